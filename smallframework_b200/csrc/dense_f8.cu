// dense_f8.cu -- dense layer on e4m3 operands with an fp32 scale for each block of 128 (one row of activations, 128 rows of weights), on the tensor
// cores (tcgen05 kind::f8f6f4).
//
// Mathematics: out[r][k] = sum_b sx[r][b] * sw[k / 128][b] * d_b, d_b the dot product of block b.  A block is 128 bytes of a row, one
// 128-byte swizzle row in shared memory and four MMAs of 32 steps; its sums go to tensor memory by themselves, and the warps behind fold them into
// fp32 registers, times the two scales.  Tensor memory holds several blocks' sums, so that the next MMAs run meanwhile.
//
// Two kernels:
//   few    weights are the 128 lanes, 16, 32 or 64 rows of activations the columns.  The weights' bytes bound it: they come once, by TMA, into all SMs,
//          the reduction cut among the CTAs of a cluster where output tiles are few; the parts go to the CTA that finishes them by asynchronous stores and are
//          added in order.  On a B200, cold: 1 row, 4096 -> 4096 6.4 us (2.6 at the copy rate; 5.0 with the weights in L2), 24 rows, 8192 -> 8192 15.1 (10.5): a
//          microsecond until the first sums, one and a half for the exchange and the end, the launch; in between the weights come at 6.0 TB/s.
//   many   256 rows of activations by 256 outputs for a pair of CTAs.  A block takes 975 cycles where its MMAs take 512: 32 KB an SM come from L2 at the device's
//          10.4 TB/s in 840, and tensor memory holds two blocks' sums, whose way to the registers and back is 1400 cycles for the two.  From 4096 rows on the
//          1 kW power cap comes first.  2048 rows, 4096 -> 8192 69 us (2.0 PFLOP/s), with bias and ReLU 71, onto old fp16 values 80; in runs of a second (1.58 GHz) 79, 82 and 90.
//          8192 rows, 8192 -> 8192 481 us, in runs of a second (1.44 GHz) 555.
#include <algorithm>
#include <type_traits>

#include "narrow_types.cuh"
#include "tc_common.cuh"

namespace
{
using namespace sb;

constexpr int KB = 128, A_BYTES = 128 * KB;

struct DenseArgs
{
    int rows, K, blocks; // blocks of 128 in the reduction
    int k_tiles, r_tiles, split;
    int first, count; // tiles that a launch does (many: of 256 x 256)
    int behind;       // few: the launch before it does the other tiles of the same call, and only the end of this one waits for it
    int accumulate;
    int act;
    float slope;
    long long out_stride;
    const float *in_scales, *filt_scales, *bias;
    void *out;
    int wide; // rows of the output begin on 16-byte boundaries
};

// ReLU and LeakyReLU of the finished sum, without branches (`below`: the slope, 1 for no activation).  Infinities get what the formula gives, unlike in the
// convolutions' form, and NaN stays NaN.
__device__ __forceinline__ float activate(float v, bool relu, float below)
{
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
    const float l = v > 0.f ? v : v * below;
    return relu ? r : l;
}

template <int TYPE>
__device__ __forceinline__ void store1(void *p, long long at, float v)
{
    if (TYPE == SMALL_B200_TYPE_F32)
        static_cast<float *>(p)[at] = v;
    else if (TYPE == SMALL_B200_TYPE_BF16)
        static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
    else
        static_cast<__half *>(p)[at] = __float2half_rn(v);
}

// Two sums times their scales onto two more, one instruction.
__device__ __forceinline__ void fold2(unsigned long long &acc, uint32_t lo, uint32_t hi, unsigned long long s2)
{
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(r), "l"(s2));
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b)
{
    unsigned long long v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// Four bytes into shared memory, past the registers; copies_done() waits for this thread's.
__device__ __forceinline__ void copy4(void *to, const float *from)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ unsigned long long activate2(unsigned long long v, bool relu, float below)
{
    float x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
    x = activate(x, relu, below);
    y = activate(y, relu, below);
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
// The two 16-bit floats of a word.
template <int TYPE>
__device__ __forceinline__ unsigned long long wide2(uint32_t w)
{
    float x, y;
    unsigned long long v;
    unpack2<TYPE>(w, x, y);
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ float2 pair_of(unsigned long long v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) { return p + ((1024u - (smem_u32(p) & 1023u)) & 1023u); }

// ------------------------------------------------------------------------------------------------ few rows
template <int BN>
struct Few
{
    // Two CTAs an SM: 113 KB of shared memory and 256 columns of tensor memory each.  Three never fit, so a launch that starts early cannot take tensor memory
    // that a CTA of the launch before it, for which it waits, has yet to allocate.
    static constexpr int STAGE = A_BYTES + BN * KB, STAGES = BN == 16 ? 5 : BN == 32 ? 4 : 3;
    static constexpr int BUFS = 4, COLS = BUFS * BN;
    static constexpr int CHUNK = 8; // blocks whose scales are brought at a time
    static constexpr int SCALES = 2 * CHUNK * BN * 4, INBOX = BN * 128 * 4;
    static constexpr int SMEM = 1024 + STAGES * STAGE + SCALES + INBOX;
    static_assert(2 * (SMEM + 2048) <= 228 * 1024 && 2 * COLS <= 512, "two CTAs an SM");
};
constexpr int FEW_THREADS = 7 * 32;

__device__ __forceinline__ float4 bias4(const DenseArgs &a, int k)
{
    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.bias)
    {
        const int last = a.K - 1;
        b = make_float4(a.bias[min(k, last)], a.bias[min(k + 1, last)], a.bias[min(k + 2, last)], a.bias[min(k + 3, last)]);
    }
    return b;
}
// Four consecutive outputs of a row as they are, and to where they are; the first `here` of them where they are not on a boundary of their own.
template <int TYPE>
__device__ __forceinline__ float4 load_few(const void *p, long long at, int here)
{
    return make_float4(load1<TYPE>(p, at), here > 1 ? load1<TYPE>(p, at + 1) : 0.f, here > 2 ? load1<TYPE>(p, at + 2) : 0.f,
                       here > 3 ? load1<TYPE>(p, at + 3) : 0.f);
}
template <int TYPE>
__device__ __forceinline__ void store_few(void *p, long long at, int here, float4 v)
{
    store1<TYPE>(p, at, v.x);
    if (here > 1)
        store1<TYPE>(p, at + 1, v.y);
    if (here > 2)
        store1<TYPE>(p, at + 2, v.z);
    if (here > 3)
        store1<TYPE>(p, at + 3, v.w);
}
template <int TYPE>
__device__ __forceinline__ float4 load4(const DenseArgs &a, int row, int k)
{
    const long long at = (long long)row * a.out_stride + k;
    if (!(a.wide && k + 4 <= a.K))
        return load_few<TYPE>(a.out, at, a.K - k);
    if (TYPE == SMALL_B200_TYPE_F32)
        return *reinterpret_cast<const float4 *>(static_cast<const float *>(a.out) + at);
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.out) + at);
    float4 v;
    unpack2<TYPE>(w.x, v.x, v.y);
    unpack2<TYPE>(w.y, v.z, v.w);
    return v;
}
template <int TYPE>
__device__ __forceinline__ void store4(const DenseArgs &a, int row, int k, float4 v)
{
    const long long at = (long long)row * a.out_stride + k;
    if (!(a.wide && k + 4 <= a.K))
        store_few<TYPE>(a.out, at, a.K - k, v);
    else if (TYPE == SMALL_B200_TYPE_F32)
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = v;
    else
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at) = make_uint2(pack2<TYPE>(v.x, v.y), pack2<TYPE>(v.z, v.w));
}
// The sum with the old value, the bias and the activation.
__device__ __forceinline__ float4 finished(const DenseArgs &a, float4 sum, float4 old, float4 bias)
{
    const bool relu = a.act == SMALL_B200_ACT_RELU;
    const float below = a.act == SMALL_B200_ACT_LEAKY ? a.slope : 1.f;
    return make_float4(activate(sum.x + old.x + bias.x, relu, below), activate(sum.y + old.y + bias.y, relu, below),
                       activate(sum.z + old.z + bias.z, relu, below), activate(sum.w + old.w + bias.w, relu, below));
}

template <int BN, int TYPE>
__global__ void __launch_bounds__(FEW_THREADS) dense_f8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                      const DenseArgs a, int *status)
{
    using G = Few<BN>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[G::STAGES], empty[G::STAGES], sum_full[G::BUFS], sum_empty[G::BUFS], sc_full[2], sc_empty[2], drained, delivered;
    __shared__ uint32_t tmem_s;
    uint8_t *ring = align1024(raw);
    float *scales = reinterpret_cast<float *>(ring + G::STAGES * G::STAGE); // [2][CHUNK][BN]
    // What the cluster's CTAs have of this CTA's share of the rows, in pairs of rows: [split][rows / split / 2][128 outputs][2]
    unsigned long long *inbox = reinterpret_cast<unsigned long long *>(ring + G::STAGES * G::STAGE + G::SCALES);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)(blockIdx.x % a.split), tile = a.first + (int)(blockIdx.x / a.split);
    const int kt = tile % a.k_tiles, r0 = tile / a.k_tiles * BN;
    const int share = (a.blocks + a.split - 1) / a.split;
    const int b0 = rank * share, n = max(0, min(a.blocks, b0 + share) - b0);
    auto load = [&](int i, int s) {
        mbar_expect_tx(&full[s], G::STAGE);
        tma_load_2d(ring + s * G::STAGE, &map_w, (b0 + i) * KB, kt * 128, &full[s]);
        tma_load_2d(ring + s * G::STAGE + A_BYTES, &map_x, (b0 + i) * KB, r0, &full[s]);
    };

    // The loading warp does not wait for the others, nor they for it: under load it takes microseconds until the last of its first copies is accepted.
    if (warp == 4)
    {
        if (elect_one())
        {
            for (int s = 0; s < G::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
            fence_barrier_init();
        }
        __syncwarp();
        asm volatile("bar.arrive 1, %0;" ::"n"(FEW_THREADS) : "memory");
        if (!a.behind) // the other launch of the call has waited for what both read, before it let this one start, and writes nothing that this one reads
            previous_kernel_done();
        next_kernel_may_start();
        if (elect_one())
            for (int i = 0; i < G::STAGES && i < n; ++i)
                load(i, i);
        __syncwarp();
    }
    else if (warp == 5)
    {
        tmem_alloc(&tmem_s, G::COLS);
        tmem_relinquish();
    }
    else if (tid == 0)
    {
        for (int s = 0; s < G::BUFS; ++s) { mbar_init(&sum_full[s], 1); mbar_init(&sum_empty[s], 4); }
        for (int s = 0; s < 2; ++s) { mbar_init(&sc_full[s], 1); mbar_init(&sc_empty[s], 4); }
        mbar_init(&drained, 1);
        mbar_init(&delivered, 1);
        fence_barrier_init();
        mbar_expect_tx(&delivered, G::INBOX);
    }
    // ---- scales: the product of a row's and the weights' scale, by block and row
    constexpr int ROWS = (BN + 31) / 32;
    float sv[ROWS][G::CHUNK], sw[G::CHUNK]; // multiplied when they are needed: until then nothing waits for them
    auto ask = [&](int c) {
#pragma unroll
        for (int j = 0; j < G::CHUNK; ++j)
            sw[j] = c * G::CHUNK + j < n ? a.filt_scales[(size_t)kt * a.blocks + b0 + c * G::CHUNK + j] : 0.f;
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
        {
            const int col = q * 32 + lane, row = r0 + col;
            const float *sx = a.in_scales + (size_t)row * a.blocks + b0;
#pragma unroll
            for (int j = 0; j < G::CHUNK; ++j)
            {
                const int b = c * G::CHUNK + j;
                sv[q][j] = col < BN && row < a.rows && b < n ? sx[b] : 0.f;
            }
        }
    };
    tc_fence_before_sync();
    if (warp != 4)
        asm volatile("bar.sync 1, %0;" ::"n"(FEW_THREADS) : "memory");
    __syncwarp();
    if (a.split > 1)
        cluster_arrive_relaxed(); // this CTA's inbox can be written to: its barrier has been made and fenced
    if (warp != 4)
    {
        if (!a.behind)
            previous_kernel_done();
        next_kernel_may_start();
    }
    tc_fence_after_sync();
    const uint32_t tmem = tmem_s;
    unsigned long long acc[BN / 2]; // of the folding warps

    if (warp < 4)
    {
        // ---- thread = one output channel: folds every block's sums into registers
#pragma unroll
        for (int c = 0; c < BN / 2; ++c)
            acc[c] = 0ull;
        bool ok = true;
        for (int i = 0; i < n; ++i)
        {
            const int buf = i % G::BUFS, chunk = i / G::CHUNK;
            if (i % G::CHUNK == 0)
                ok = mbar_wait(&sc_full[chunk & 1], (chunk >> 1) & 1, status, 101);
            ok = ok && mbar_wait(&sum_full[buf], (i / G::BUFS) & 1, status, 102);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            tc_fence_after_sync();
            const uint32_t from = tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(buf * BN);
            const ulonglong2 *s4 = reinterpret_cast<const ulonglong2 *>(scales + ((chunk & 1) * G::CHUNK + i % G::CHUNK) * BN);
            constexpr int STEP = BN < 32 ? 16 : 32;
#pragma unroll
            for (int c0 = 0; c0 < BN; c0 += STEP)
            {
                uint32_t r[STEP];
                if (STEP == 32)
                    tmem_ld32(from + c0, r);
                else
                    tmem_ld16(from + c0, r);
                tmem_ld_wait();
                if (c0 + STEP == BN)
                {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&sum_empty[buf]);
                }
#pragma unroll
                for (int c = 0; c < STEP; c += 4)
                {
                    const ulonglong2 s = s4[(c0 + c) / 4];
                    fold2(acc[(c0 + c) / 2], r[c], r[c + 1], s.x);
                    fold2(acc[(c0 + c) / 2 + 1], r[c + 2], r[c + 3], s.y);
                }
            }
            if (i % G::CHUNK == G::CHUNK - 1)
            {
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&sc_empty[chunk & 1]);
            }
        }
    }
    else if (warp == 4)
    {
        bool ok = true;
        int i = min(n, G::STAGES), s = i % G::STAGES;
        uint32_t turn = 0;
        for (; i < n; ++i)
        {
            ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], turn, status, 103));
            if (!ok)
                break;
            if (elect_one())
                load(i, s);
            __syncwarp();
            if (++s == G::STAGES)
            {
                s = 0;
                turn ^= 1;
            }
        }
        for (int j = max(0, i - G::STAGES); j < i && !ok; ++j) // its own copies in flight
            mbar_wait(&full[j % G::STAGES], (j / G::STAGES) & 1, status, 104);
    }
    else if (warp == 5)
    {
        const uint32_t idesc = make_idesc(1 /*f32*/, 0, 0, 0, 0, 128, BN);
        const uint64_t first_a = make_smem_desc(smem_u32(ring), 16, 1024, 2), first_b = make_smem_desc(smem_u32(ring) + A_BYTES, 16, 1024, 2);
        bool ok = true;
        int s = 0;
        uint32_t turn = 0;
        for (int i = 0; i < n; ++i)
        {
            const int buf = i % G::BUFS;
            const uint32_t use = ((i / G::BUFS) & 1) ^ 1; // before a buffer's first use the phase before the first counts as complete
            if (!mbar_test_both(&full[s], turn, &sum_empty[buf], use))
                ok = mbar_wait(&full[s], turn, status, 105) && mbar_wait(&sum_empty[buf], use, status, 106);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            tc_fence_after_sync();
            if (elect_one())
            {
                const uint32_t d = tmem + (uint32_t)(buf * BN);
                const uint64_t da = first_a + s * (G::STAGE / 16), db = first_b + s * (G::STAGE / 16);
                tc_mma_f8(d, da, db, idesc, 0u);
                tc_mma_f8(d, da + 2, db + 2, idesc, 1u);
                tc_mma_f8(d, da + 4, db + 4, idesc, 1u);
                tc_mma_f8(d, da + 6, db + 6, idesc, 1u);
                tc_commit(&sum_full[buf]);
                tc_commit(&empty[s]);
            }
            __syncwarp();
            if (++s == G::STAGES)
            {
                s = 0;
                turn ^= 1;
            }
        }
        if (!ok)
        {
            if (elect_one())
                tc_commit(&drained);
            __syncwarp();
            mbar_wait(&drained, 0, status, 107);
        }
    }
    else
    {
        const int chunks = (n + G::CHUNK - 1) / G::CHUNK;
        for (int c = 0; c < chunks; ++c)
        {
            ask(c);
            const bool ok = c < 2 || mbar_wait(&sc_empty[c & 1], ((c >> 1) - 1) & 1, status, 108);
            if (!__all_sync(0xffffffffu, ok))
                break;
#pragma unroll
            for (int q = 0; q < ROWS; ++q)
#pragma unroll
                for (int j = 0; j < G::CHUNK; ++j)
                    if (q * 32 + lane < BN)
                        scales[((c & 1) * G::CHUNK + j) * BN + q * 32 + lane] = sv[q][j] * sw[j];
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&sc_full[c & 1]);
        }
    }
    __syncwarp();

    // tensor memory has been read
    tc_fence_before_sync();
    if (warp < 4)
        asm volatile("bar.arrive 2, 160;" ::: "memory");
    else if (warp == 5)
    {
        asm volatile("bar.sync 2, 160;" ::: "memory");
        tmem_dealloc(tmem, G::COLS);
    }
    __syncwarp();
    // ---- every CTA of the cluster has a share of the rows: the others send it what they have of them (a wait that gave up leaves rubbish, which
    // the status word tells)
    const int per = BN / a.split;
    bool all = true;
    if (a.split == 1)
    {
        if (warp < 4)
        {
#pragma unroll
            for (int c = 0; c < BN; c += 2)
                inbox[c / 2 * 128 + tid] = acc[c / 2];
        }
        __syncthreads();
    }
    else
    {
        cluster_wait(); // all inboxes can be written to
        if (warp < 4)
        {
            const unsigned long long *mine = inbox + rank * (per / 2) * 128 + tid;
            int to = 0, left = per; // of the share that is being sent
            uint32_t at = map_to_cta(mine, 0), bar = map_to_cta(&delivered, 0);
#pragma unroll
            for (int c = 0; c < BN; c += 2)
            {
                st_async_b64(at, acc[c / 2], bar);
                at += 128 * 8;
                left -= 2;
                if (left == 0 && c + 2 < BN)
                {
                    left = per;
                    ++to;
                    at = map_to_cta(mine, to);
                    bar = map_to_cta(&delivered, to);
                }
            }
        }
        __syncwarp();
        cluster_arrive_relaxed(); // nothing more is sent
        all = mbar_wait_cluster(&delivered, 0, status, 109);
    }
    // the parts in the order of the reduction, then bias, activation and the one rounding: a warp takes two rows, a lane four outputs
    const int k = kt * 128 + 4 * lane;
    const float4 bias = bias4(a, k);
    for (int p = warp; 2 * p < per; p += FEW_THREADS / 32)
    {
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
        for (int q = 0; q < a.split; ++q)
        {
            const float4 *in = reinterpret_cast<const float4 *>(inbox + (q * (per / 2) + p) * 128 + 4 * lane);
            const float4 x = in[0], y = in[1];
            u.x += x.x; v.x += x.y; u.y += x.z; v.y += x.w;
            u.z += y.x; v.z += y.y; u.w += y.z; v.w += y.w;
        }
        const int row = r0 + rank * per + 2 * p;
        const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < a.K && row < a.rows)
            store4<TYPE>(a, row, k, finished(a, u, a.accumulate ? load4<TYPE>(a, row, k) : none, bias));
        if (k < a.K && row + 1 < a.rows)
            store4<TYPE>(a, row + 1, k, finished(a, v, a.accumulate ? load4<TYPE>(a, row + 1, k) : none, bias));
    }
    if (a.split > 1)
    {
        __syncwarp();
        cluster_wait(); // this CTA's shared memory stays while anybody may send to it
        if (!all)
            for (int i = 0; i < 1000; ++i)
                __nanosleep(1000); // and what was sent last is on its way for less than that
    }
    if (a.behind)
        previous_kernel_done(); // who waits for this launch waits for both
}

// ------------------------------------------------------------------------------------------------ many rows
// A pair of CTAs (cta_group::2) owns 256 rows by N = 256 outputs: each brings its 128 rows and half of the weights, 32 KB a block where a CTA by itself
// would bring 48 KB for the same products; traffic between L2 and the SMs is what bounded that (10.4 TB/s over the device).
//
// Tiles that leave half of the pairs idle are cut to N = 128.  That brings 24 KB for half of the products, but tensor memory then holds four blocks'
// sums, and the way from an MMA to the warps that fold and back, 900 cycles, is hidden behind three others: 0.4 of a whole tile's time.
constexpr int MANY_STAGE = 2 * A_BYTES, MANY_STAGES = 6, MANY_EPI = 8, MANY_THREADS = 384;
static_assert(MANY_STAGES % 2 == 0, "a buffer's blocks keep to every other stage");
constexpr int STAGE_OUT = 32 * 128; // a warp's way out
constexpr int MANY_SMEM = 1024 + MANY_STAGES * MANY_STAGE + MANY_EPI * STAGE_OUT;
// Registers: 384 threads start with 168 each (64512 in all); the four warps that feed keep 40, the eight that fold take 232, which adds up to the same.
// (ptxas sees 168 for all of them: with a bias, an activation or old values 20 to 28 bytes a thread are spilled; so are 24 in the kernel for few rows with 32 and 64 columns.)
constexpr int REGS_FEED = 40, REGS_FOLD = 232;
constexpr int GROUP = 8; // tiles of rows that are walked together: their activations and the weights beside them stay in L2

struct TileAt
{
    int r0, k0;
};
// Tile t of 256 x 256, or the half t & 1 of tile t / 2 (which may begin behind the last output).
template <int N>
__device__ __forceinline__ TileAt tile_at(const DenseArgs &a, int t)
{
    const int half = N == 128 ? t & 1 : 0;
    t = a.first + (N == 128 ? t >> 1 : t);
    const int per_group = GROUP * a.k_tiles, g = t / per_group, in = t - g * per_group;
    const int size = min(GROUP, a.r_tiles - g * GROUP);
    const int kt = in / size;
    return {(g * GROUP + in - kt * size) * 256, kt * 256 + half * 128};
}

__device__ __forceinline__ void fold32(unsigned long long *acc, const uint32_t *r, unsigned long long s2)
{
#pragma unroll
    for (int c = 0; c < 16; ++c)
        fold2(acc[c], r[2 * c], r[2 * c + 1], s2);
}

// A warp's copy of the bias of its COLS outputs.
template <int COLS>
__device__ __forceinline__ void copy_bias(const DenseArgs &a, uint8_t *to, int k0)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < COLS; c += 32)
        copy4(to + (c + lane) * 4, a.bias + min(k0 + c + lane, a.K - 1));
}
// 128 bytes of each of a warp's 32 rows, from output k on, between the output and the warp's shared memory (OUT: to the output): element by element, several rows
// together, which hides that a load takes its time.
template <int TYPE, bool OUT>
__device__ __forceinline__ void by_element(const DenseArgs &a, uint8_t *stage, int first, int k)
{
    using Word = typename std::conditional<TYPE == SMALL_B200_TYPE_F32, uint32_t, uint16_t>::type;
    constexpr int VE = 16 / sizeof(Word), EACH = 8 * VE / 32, TOGETHER = OUT ? 4 : 8;
    const int lane = threadIdx.x & 31, rows = min(32, a.rows - first);
    Word *out = static_cast<Word *>(a.out) + (long long)first * a.out_stride + k;
#pragma unroll 1
    for (int q0 = 0; q0 < rows; q0 += TOGETHER)
    {
        Word v[TOGETHER][EACH];
        auto all = [&](auto each) {
#pragma unroll
            for (int n = 0; n < TOGETHER; ++n)
#pragma unroll
                for (int e = 0; e < EACH; ++e)
                {
                    const int q = q0 + n, c = lane + 32 * e;
                    each(v[n][e], reinterpret_cast<Word *>(stage + q * 128 + ((c / VE ^ (q & 7)) << 4)) + c % VE, out + q * a.out_stride + c, q < rows && k + c < a.K);
                }
        };
        if (OUT)
        {
            all([](Word &v, Word *in, Word *, bool) { v = *in; });
            all([](Word &v, Word *, Word *out, bool has) { if (has) *out = v; });
        }
        else
        {
            all([](Word &v, Word *, Word *out, bool has) { v = has ? *out : (Word)0; });
            all([](Word &v, Word *in, Word *, bool) { *in = v; });
        }
    }
}

// FINISH: with a bias, an activation or old values; code that a tile jumps over costs it 0.3 us.
template <int TYPE, int N, bool FINISH>
__global__ void __launch_bounds__(MANY_THREADS, 1) dense_f8_many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                          const DenseArgs a, int *status)
{
    constexpr int BUFS = 512 / N, COLS = N / 2, BYTES = A_BYTES + N / 2 * KB; // of sums; a folding thread's outputs; of a block and CTA
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[MANY_STAGES], empty[MANY_STAGES], sum_full[BUFS], sum_empty[BUFS], drained[2];
    __shared__ uint32_t tmem_s;
    uint8_t *ring = align1024(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)cluster_ctarank(), pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const int tiles = a.count * (256 / N);
    if (tid == 0)
    {
        for (int s = 0; s < MANY_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < BUFS; ++s) { mbar_init(&sum_full[s], 1); mbar_init(&sum_empty[s], 2 * MANY_EPI); }
        for (int s = 0; s < 2; ++s) mbar_init(&drained[s], 1);
        fence_barrier_init();
    }
    if (warp == 3)
        tmem_alloc_pair(&tmem_s, 512);
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive_relaxed(); // the barriers have been made and fenced
    cluster_wait();
    tc_fence_after_sync();
    previous_kernel_done(); // tensor memory is this CTA's before the next launch may ask for it
    next_kernel_may_start();
    const uint32_t tmem = tmem_s;

    if (warp >= 4)
    {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_FOLD));
        // ---- thread = one row of activations and COLS outputs of one block of weights
        const int half = (warp - 4) >> 2, lane_row = (warp & 3) * 32 + lane;
        const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * COLS);
        const uint32_t give_back = map_to_cta(sum_empty, 0);
        bool ok = true;
        unsigned i = 0;
        for (int t = pair; t < tiles && ok; t += pairs)
        {
            const TileAt at = tile_at<N>(a, t);
            if (at.k0 >= a.K)
                continue;
            const int row = at.r0 + rank * 128 + lane_row, k0 = at.k0 + half * COLS;
            const float *sx = a.in_scales + (size_t)min(row, a.rows - 1) * a.blocks;
            const float *sw = a.filt_scales + (size_t)min(k0 / 128, (a.K - 1) / 128) * a.blocks;
            unsigned long long acc[COLS / 2];
#pragma unroll
            for (int c = 0; c < COLS / 2; ++c)
                acc[c] = 0ull;
            // Software pipeline over the blocks: while 32 columns are folded the next 32 are on their way, across blocks too, and the next block's
            // barrier is asked one step before its answer is needed.
            if (FINISH && a.bias && !a.accumulate) // asked for now, needed at the end, and until then not in registers
                copy_bias<COLS>(a, ring + MANY_STAGES * MANY_STAGE + (warp - 4) * STAGE_OUT, k0);
            float next_x = sx[0], next_w = sw[0]; // multiplied when they are needed: until then nothing waits for them
            uint32_t r[2][32];
            ok = __all_sync(0xffffffffu, mbar_wait(&sum_full[i % BUFS], (i / BUFS) & 1, status, 111));
            if (!ok)
                break;
            tc_fence_after_sync();
            tmem_ld32(from + (i % BUFS) * N, r[0]);
            for (int b = 0; b < a.blocks; ++b, ++i)
            {
                const unsigned buf = i % BUFS, then = (i + 1) % BUFS, then_phase = ((i + 1) / BUFS) & 1;
                const float s = next_x * next_w;
                const unsigned long long s2 = (unsigned long long)__float_as_uint(s) << 32 | __float_as_uint(s);
                const bool more = b + 1 < a.blocks;
                if (more)
                {
                    next_x = sx[b + 1];
                    next_w = sw[b + 1];
                }
                bool ready = false;
#pragma unroll
                for (int c = 0; c < COLS / 32; ++c)
                {
                    tmem_ld_wait();
                    if (c + 1 < COLS / 32)
                        tmem_ld32(from + buf * N + 32 * (c + 1), r[(c + 1) & 1]);
                    else
                    {
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0)
                            mbar_arrive_remote_relaxed(give_back + buf * 8);
                        if (more)
                        {
                            if (!__all_sync(0xffffffffu, ready))
                            {
                                ok = __all_sync(0xffffffffu, mbar_wait(&sum_full[then], then_phase, status, 111));
                                if (!ok)
                                    break;
                            }
                            tc_fence_after_sync();
                            tmem_ld32(from + then * N, r[0]);
                        }
                    }
                    if (c == COLS / 32 - 2)
                        ready = more && mbar_test(&sum_full[then], then_phase);
                    fold32(acc + 16 * c, r[c & 1], s2);
                }
                if (!ok)
                    break;
            }
            if (!ok)
                break;
            // Out through shared memory: a thread's 128 bytes of a row go in, whole lines of four rows come out.  Straight from the registers every
            // 16-byte store of a warp touches 32 lines, and a tile took 5000 cycles.
            constexpr int VE = TYPE == SMALL_B200_TYPE_F32 ? 4 : 8, SIZE = 16 / VE, WIDE = 8 * VE;
            uint8_t *stage = ring + MANY_STAGES * MANY_STAGE + (warp - 4) * STAGE_OUT;
            const int first = at.r0 + rank * 128 + (warp & 3) * 32; // row of the warp
            char *out = static_cast<char *>(a.out);
            auto by_vector = [&](int c0) { return a.wide && (a.K % VE == 0 || k0 + c0 + WIDE <= a.K); }; // 16 bytes are this row's or behind its end
            if (FINISH && a.accumulate)
            {
                // The old values, the same way in: whole lines of four rows, then every thread its row's.
#pragma unroll
                for (int c0 = 0; c0 < COLS; c0 += WIDE)
                {
                    if (k0 + c0 >= a.K)
                        break;
                    if (by_vector(c0))
                    {
                        uint4 old[8];
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                        {
                            const int q = n * 4 + (lane >> 3);
                            if (first + q < a.rows && k0 + c0 + (lane & 7) * VE < a.K)
                                old[n] = *reinterpret_cast<const uint4 *>(out + ((long long)(first + q) * a.out_stride + k0 + c0 + (lane & 7) * VE) * SIZE);
                            else
                                old[n] = make_uint4(0u, 0u, 0u, 0u);
                        }
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            *reinterpret_cast<uint4 *>(stage + (n * 4 + (lane >> 3)) * 128 + (((lane & 7) ^ (n * 4 + (lane >> 3) & 7)) << 4)) = old[n];
                    }
                    else
                        by_element<TYPE, false>(a, stage, first, k0 + c0);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) // what lies behind the last row or output is added to sums that go nowhere
                    {
                        const uint4 w = *reinterpret_cast<const uint4 *>(stage + lane * 128 + ((j ^ (lane & 7)) << 4));
                        unsigned long long *to = acc + (c0 + j * VE) / 2;
                        if (TYPE == SMALL_B200_TYPE_F32)
                        {
                            to[0] = add2(to[0], (unsigned long long)w.y << 32 | w.x);
                            to[1] = add2(to[1], (unsigned long long)w.w << 32 | w.z);
                        }
                        else
                        {
                            to[0] = add2(to[0], wide2<TYPE>(w.x));
                            to[1] = add2(to[1], wide2<TYPE>(w.y));
                            to[VE / 2 - 2] = add2(to[VE / 2 - 2], wide2<TYPE>(w.z));
                            to[VE / 2 - 1] = add2(to[VE / 2 - 1], wide2<TYPE>(w.w));
                        }
                    }
                    __syncwarp();
                }
                if (a.bias)
                    copy_bias<COLS>(a, stage, k0);
            }
            if (FINISH && a.bias)
            {
                // Every thread needs the same numbers: a copy in the warp's way out serves a whole warp a load.  (Loads from global memory were 5 us a tile.)
                copies_done();
                __syncwarp();
#pragma unroll
                for (int c = 0; c < COLS; c += 4)
                {
                    const ulonglong2 b = reinterpret_cast<const ulonglong2 *>(stage)[c / 4];
                    acc[c / 2] = add2(acc[c / 2], b.x);
                    acc[c / 2 + 1] = add2(acc[c / 2 + 1], b.y);
                }
                __syncwarp();
            }
            if (FINISH && a.act == SMALL_B200_ACT_RELU)
            {
#pragma unroll
                for (int c = 0; c < COLS / 2; ++c)
                    acc[c] = activate2(acc[c], true, 1.f);
            }
            else if (FINISH && a.act == SMALL_B200_ACT_LEAKY)
            {
#pragma unroll
                for (int c = 0; c < COLS / 2; ++c)
                    acc[c] = activate2(acc[c], false, a.slope);
            }
#pragma unroll
            for (int c0 = 0; c0 < COLS; c0 += WIDE)
            {
                if (k0 + c0 >= a.K)
                    break;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                {
                    float v[VE];
#pragma unroll
                    for (int c = 0; c < VE; c += 2)
                    {
                        const float2 f = pair_of(acc[(c0 + j * VE + c) / 2]);
                        v[c] = f.x;
                        v[c + 1] = f.y;
                    }
                    uint4 w;
                    if (TYPE == SMALL_B200_TYPE_F32)
                        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                    else
                        w = make_uint4(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]), pack2<TYPE>(v[VE - 4], v[VE - 3]),
                                       pack2<TYPE>(v[VE - 2], v[VE - 1]));
                    *reinterpret_cast<uint4 *>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = w; // no two lanes of eight share banks
                }
                __syncwarp();
                if (by_vector(c0))
                {
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                    {
                        const int q = n * 4 + (lane >> 3), j = lane & 7;
                        if (first + q < a.rows && k0 + c0 + j * VE < a.K)
                            *reinterpret_cast<uint4 *>(out + ((long long)(first + q) * a.out_stride + k0 + c0 + j * VE) * SIZE) =
                                *reinterpret_cast<const uint4 *>(stage + q * 128 + ((j ^ (q & 7)) << 4));
                    }
                }
                else
                    by_element<TYPE, true>(a, stage, first, k0 + c0);
                __syncwarp();
            }
        }
        if (FINISH)
            copies_done(); // also where a wait gave up
    }
    else
    {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEED));
        if (warp == 0)
        {
            // ---- this CTA's rows and its half of the weights; the first CTA's barrier counts both CTAs' bytes
            bool ok = true;
            unsigned i = 0, s = 0, turn = 0;
            const uint32_t bars = map_to_cta(full, 0);
            for (int t = pair; t < tiles && ok; t += pairs)
            {
                const TileAt at = tile_at<N>(a, t);
                if (at.k0 >= a.K)
                    continue;
                const int rx = at.r0 + rank * 128, rw = at.k0 + rank * (N / 2);
                for (int b = 0; b < a.blocks; ++b, ++i)
                {
                    if (turn > 0)
                        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (turn - 1) & 1, status, 112));
                    if (!ok)
                        break;
                    if (elect_one())
                    {
                        if (rank == 0)
                            mbar_expect_tx(&full[s], 2 * BYTES);
                        uint8_t *dst = ring + s * MANY_STAGE;
                        tma_load_2d_pair(dst, &map_x, b * KB, rx, bars + s * 8);
                        tma_load_2d_pair(dst + A_BYTES, &map_w, b * KB, rw, bars + s * 8);
                    }
                    __syncwarp();
                    if (++s == MANY_STAGES)
                    {
                        s = 0;
                        ++turn;
                    }
                }
            }
            if (!ok) // copies in flight: the first CTA sees both CTAs' arrive; a millisecond is far longer than any takes
            {
                for (unsigned j = i > MANY_STAGES ? i - MANY_STAGES : 0; j < i && rank == 0; ++j)
                    mbar_wait(&full[j % MANY_STAGES], (j / MANY_STAGES) & 1, status, 113);
                for (int n = 0; n < 1000; ++n)
                    __nanosleep(1000);
            }
        }
        else if ((warp == 1 || warp == 2) && rank == 0)
        {
            // Two warps, every other block its own: what a warp does around its MMAs (500 cycles a block, most of it waiting for answers) then passes
            // behind the other's.  The whole warp walks the loop, so that descriptors stay in uniform registers; one lane issues.
            const uint32_t idesc = make_idesc(1 /*f32*/, 0, 0, 0, 0, 256, N);
            const uint64_t first_a = make_smem_desc(smem_u32(ring), 16, 1024, 2), first_b = make_smem_desc(smem_u32(ring) + A_BYTES, 16, 1024, 2);
            unsigned total = 0;
            for (int t = pair; t < tiles; t += pairs)
                total += tile_at<N>(a, t).k0 < a.K ? (unsigned)a.blocks : 0u;
            const unsigned mine = warp - 1;
            unsigned s = mine, turn = 0, buf = mine, use = 1; // stage, parity of its phase; buffer, parity of the phase before its next use
            bool ok = true;
            for (unsigned i = mine; i < total; i += 2)
            {
                for (uint32_t n = 0; !mbar_test_both(&full[s], turn, &sum_empty[buf], use); ++n)
                    if (n >= 256) // long enough for every turn but the first ones: now the wait that gives up
                    {
                        ok = mbar_wait(&full[s], turn, status, 114) && mbar_wait(&sum_empty[buf], use, status, 115);
                        break;
                    }
                if (!__all_sync(0xffffffffu, ok))
                    break;
                tc_fence_after_sync();
                if (elect_one())
                {
                    const uint64_t da = first_a + s * (MANY_STAGE / 16), db = first_b + s * (MANY_STAGE / 16);
                    const uint32_t d = tmem + buf * N;
                    tc_mma_f8_pair(d, da, db, idesc, 0u);
                    tc_mma_f8_pair(d, da + 2, db + 2, idesc, 1u);
                    tc_mma_f8_pair(d, da + 4, db + 4, idesc, 1u);
                    tc_mma_f8_pair(d, da + 6, db + 6, idesc, 1u);
                    tc_commit_pair(&sum_full[buf]);
                    tc_commit_pair(&empty[s]);
                }
                __syncwarp();
                buf += 2;
                if (buf >= BUFS)
                {
                    buf -= BUFS;
                    use ^= 1;
                }
                s += 2;
                if (s >= MANY_STAGES)
                {
                    s -= MANY_STAGES;
                    turn ^= 1;
                }
            }
            if (!__all_sync(0xffffffffu, ok))
            {
                if (elect_one())
                    tc_commit_pair(&drained[mine]);
                __syncwarp();
                mbar_wait(&drained[mine], 0, status, 116);
            }
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all(); // neither CTA goes while the other may still write to it
    if (warp == 3)
        tmem_dealloc_pair(tmem, 512);
}

// ------------------------------------------------------------------------------------------------ host
int map_rows(CUtensorMap *map, const void *p, int rows, int C, long long stride, int box_rows)
{
    const uint64_t dims[2] = {(uint64_t)C, (uint64_t)rows}, strides[1] = {(uint64_t)stride};
    const uint32_t box[2] = {KB, (uint32_t)box_rows};
    return make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int BN, int TYPE>
int launch_few(const DenseArgs &a, const CUtensorMap &map_w, const CUtensorMap &map_x, int *status, cudaStream_t st)
{
    using G = Few<BN>;
    auto kern = dense_f8_few_kernel<BN, TYPE>;
    static PerDeviceOnce configured;
    int dev;
    if (configured.needed(&dev))
    {
        SB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
        configured.mark(dev);
    }
    // early for any number of waves: its CTAs are few and long
    const Launch l((unsigned)(a.count * a.split), FEW_THREADS, G::SMEM, st, a.split > 1 ? (unsigned)a.split : 0u);
    SB_CUDA(cudaLaunchKernelEx(&l.cfg, kern, map_w, map_x, a, status));
    return launched("dense_f8_few_kernel");
}

template <int TYPE, int N, bool FINISH>
int launch_many(const DenseArgs &a, const CUtensorMap &map_x, const CUtensorMap &map_w, int *status, cudaStream_t st)
{
    auto kern = dense_f8_many_kernel<TYPE, N, FINISH>;
    static PerDeviceOnce configured;
    int dev;
    if (configured.needed(&dev))
    {
        SB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MANY_SMEM));
        cudaFuncAttributes fa;
        SB_CUDA(cudaFuncGetAttributes(&fa, kern));
        if (fa.numRegs * MANY_THREADS < 128 * REGS_FEED + 256 * REGS_FOLD) // the split would wait for registers that the launch does not have
            return fail(SMALL_B200_CUDA_ERROR, "dense_f8_many_kernel was built with too few registers");
        configured.mark(dev);
    }
    const int pairs = std::min(a.count * (256 / N), num_sms() / 2);
    const Launch l((unsigned)(2 * pairs), MANY_THREADS, MANY_SMEM, st, 2);
    SB_CUDA(cudaLaunchKernelEx(&l.cfg, kern, map_x, map_w, a, status));
    return launched(N == 256 ? "dense_f8_many_kernel<256>" : "dense_f8_many_kernel<128>");
}

// CTAs (a cluster) that share a reduction in the kernel for few rows.  Two CTAs an SM fit; a reduction is cut while that adds CTAs to a first wave and there are
// two blocks to a CTA.  The first CTAs take the rounded-up share and the last ones what is left, which may be nothing: 17 blocks in eight parts are 3, 3, 3, 3, 3, 2, 0 and 0.  Clusters of four and eight do not fill every group of SMs (148 SMs hold 70 and 33): 1 row, 4096 inputs, 70 tiles of outputs 9.0 us in fours and 9.9 in twos, but 72 tiles 13.4 and 10.0; 8192 inputs,
// 33 tiles 8.0 in eights and 8.8 in fours, but 34 tiles 12.2 and 10.1.  Clusters of eight come up slowly (the last of 32 after 1.8 us, of 64 clusters of four
// after 0.9), so short reductions are cut in eight only where four leave SMs without a CTA: 64 rows, 2048 inputs, 20 tiles 7.2 and 6.8, 15 tiles 5.5 and 6.5.
int parts_of(long long tiles, int blocks)
{
    const long long sms = num_sms();
    int parts = 1;
    while (parts < 8 && blocks >= 4 * parts && tiles * 2 * parts <= (parts == 1 ? 2 * sms : parts == 2 ? 2 * sms - 16 : blocks >= 32 ? 2 * sms - 32 : sms))
        parts *= 2;
    return parts;
}

template <int TYPE>
int dispatch(const small_b200_dense *D, DenseArgs a, const void *in, long long in_stride, const void *filt, long long filt_stride, cudaStream_t st)
{
    int *status = device_status_ptr();
    if (!status)
        return fail(SMALL_B200_CUDA_ERROR, "device status word not available");
    CUtensorMap map_w, map_x;
    // Microseconds that either kernel takes, fitted to 136 sizes of 64 to 512 rows, 64 to 8192 outputs and 512 to 8192 inputs (none of which loses 1 % against the
    // faster one): a start and an end, a tile of 128 outputs by 64 rows and its blocks, a second CTA an SM in the one, a wave of 256 x 256 tiles, or of halves of
    // such tiles, in the other.  64 rows, 512 -> 4096: 5.6 us and 4.7; 128 rows, 4096 -> 4096: 10.9 and 12.9; 256 rows: 15.5 and 13.2; 512 rows, 8192 -> 1024: 15.1 and 21.9.
    const double b = a.blocks;
    const long long tiles_of_few = ((D->K + 127LL) / 128) * ((D->rows + 63LL) / 64);
    const long long pairs_of_tiles = ((D->K + 255LL) / 256) * ((D->rows + 255LL) / 256), at_once = std::max(1, num_sms() / 2);
    // Tiles for which there are twice as many pairs of CTAs are done in halves, a launch of its own behind whole waves.
    const long long whole = pairs_of_tiles / at_once * at_once, rest = pairs_of_tiles - whole;
    const bool halves = rest > 0 && 2 * rest <= at_once;
    const double few_us = 5.06 + 0.022 * b + (double)tiles_of_few * (0.0062 + 0.0023 * b) + (tiles_of_few * parts_of(tiles_of_few, a.blocks) > num_sms() ? 0.37 : 0.);
    const double wave = 0.47 * b + 1.9;
    // (its way out takes longer in fp32 and behind a bias or an activation, once a launch; the other's hardly does)
    const double many_us = 3.2 + (double)(whole / at_once) * wave + (rest == 0 ? 0. : halves ? 0.285 * b + (whole > 0 ? 3.2 : 0.) : wave) +
                           (TYPE == SMALL_B200_TYPE_F32 ? 0.7 : 0.) + (D->act != SMALL_B200_ACT_NONE || a.bias ? 0.5 : 0.);
    if (D->rows <= 32 || few_us < many_us)
    {
        const int bn = D->rows <= 16 ? 16 : D->rows <= 32 ? 32 : 64;
        a.k_tiles = (D->K + 127) / 128;
        a.r_tiles = (D->rows + bn - 1) / bn;
        if (int rc = map_rows(&map_w, filt, D->K, D->C, filt_stride, 128))
            return rc;
        if (int rc = map_rows(&map_x, in, D->rows, D->C, in_stride, bn))
            return rc;
        auto launch = [&](int first, int count) {
            a.first = first;
            a.count = count;
            a.behind = first > 0;
            a.split = parts_of(count, a.blocks);
            return bn == 16 ? launch_few<16, TYPE>(a, map_w, map_x, status, st) : bn == 32 ? launch_few<32, TYPE>(a, map_w, map_x, status, st)
                                                                                        : launch_few<64, TYPE>(a, map_w, map_x, status, st);
        };
        // A last wave that is not full is a launch of its own with the reductions cut, beside the end of the one before.  One launch and two: 1 row, 4096 -> 50257
        // 39.5 us and 36.8, 64 rows 53.0 and 46.1; 24 rows, 2048 -> 39680 24.7 and 21.5; but (in an earlier build) 1024 -> 50257 17.2 and 17.6, 512 -> 50257 10.6 and 11.5.
        const int tiles = a.k_tiles * a.r_tiles, resident = 2 * num_sms(), full = tiles / resident * resident;
        if (full > 0 && tiles > full && a.blocks >= 16 && parts_of(tiles - full, a.blocks) > 1)
        {
            if (int rc = launch(0, full))
                return rc;
            return launch(full, tiles - full);
        }
        return launch(0, tiles);
    }
    const bool finish = a.bias || a.accumulate || a.act != SMALL_B200_ACT_NONE;
    a.k_tiles = (D->K + 255) / 256;
    a.r_tiles = (D->rows + 255) / 256;
    a.split = 1;
    if (int rc = map_rows(&map_x, in, D->rows, D->C, in_stride, 128))
        return rc;
    if (whole > 0 || !halves)
    {
        if (int rc = map_rows(&map_w, filt, D->K, D->C, filt_stride, 128))
            return rc;
        a.first = 0;
        a.count = (int)(halves ? whole : pairs_of_tiles);
        if (int rc = finish ? launch_many<TYPE, 256, true>(a, map_x, map_w, status, st) : launch_many<TYPE, 256, false>(a, map_x, map_w, status, st))
            return rc;
    }
    if (!halves)
        return SMALL_B200_OK;
    if (int rc = map_rows(&map_w, filt, D->K, D->C, filt_stride, 64))
        return rc;
    a.first = (int)whole;
    a.count = (int)rest;
    return finish ? launch_many<TYPE, 128, true>(a, map_x, map_w, status, st) : launch_many<TYPE, 128, false>(a, map_x, map_w, status, st);
}
} // namespace

extern "C" int small_b200_dense_f8(const small_b200_dense *D, const void *in, const float *in_scales, const void *filt, const float *filt_scales,
                                   const float *bias, void *out, void *stream)
{
    const std::string name = "Dense<float8>";
    if (!D)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: null layer.");
    if (D->C <= 0 || D->C % CB != 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: in_channels unsupported.");
    if (D->K <= 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: out_channels unsupported.");
    const int size = type_size(D->out_type);
    if (size == 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: output type unsupported.");
    if (D->act != SMALL_B200_ACT_NONE && D->act != SMALL_B200_ACT_RELU && D->act != SMALL_B200_ACT_LEAKY)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: activation unsupported.");
    const long long in_stride = D->in_stride ? D->in_stride : D->C, filt_stride = D->filt_stride ? D->filt_stride : D->C,
                    out_stride = D->out_stride ? D->out_stride : D->K;
    if (D->rows < 0 || in_stride < D->C || filt_stride < D->C || out_stride < D->K || in_stride % 16 != 0 || filt_stride % 16 != 0 ||
        in_stride >= 1LL << 40 || filt_stride >= 1LL << 40) // what a tensor map holds
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: bad shape.");
    if (D->rows == 0)
        return SMALL_B200_OK;
    if (!in || !in_scales || !filt || !filt_scales || !out)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: null buffer.");
    auto off = [](const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    if (off(in, 16) || off(filt, 16) || off(in_scales, 4) || off(filt_scales, 4) || off(bias, 4) || off(out, size))
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: misaligned buffer (operands begin on 16-byte boundaries).");
    constexpr int MOST = 0x7fffffff - 512; // a tile behind the last row or output is still an int
    if (D->rows > MOST || D->K > MOST || D->C > MOST || ((D->K + 127LL) / 128) * ((D->rows + 15LL) / 16) * 8 > 0x7fffffffLL)
        return fail(SMALL_B200_INVALID_ARGUMENT, name + " ERROR: too many tiles.");
    DenseArgs a = {};
    a.rows = D->rows; a.K = D->K; a.blocks = (D->C + KB - 1) / KB;
    a.accumulate = D->accumulate; a.act = D->act; a.slope = D->slope;
    a.out_stride = out_stride; a.in_scales = in_scales; a.filt_scales = filt_scales; a.bias = bias; a.out = out;
    a.wide = !off(out, 16) && out_stride * size % 16 == 0;
    cudaStream_t st = as_stream(stream);
    switch (D->out_type)
    {
    case SMALL_B200_TYPE_F32: return dispatch<SMALL_B200_TYPE_F32>(D, a, in, in_stride, filt, filt_stride, st);
    case SMALL_B200_TYPE_BF16: return dispatch<SMALL_B200_TYPE_BF16>(D, a, in, in_stride, filt, filt_stride, st);
    default: return dispatch<SMALL_B200_TYPE_F16>(D, a, in, in_stride, filt, filt_stride, st);
    }
}
