// logprobs.cu -- log-probabilities of given classes, entropy and the best alternatives of rows of logits, in one pass over them.
//
// Mathematics, for a row x: m = max x, t_i = x_i - m, S = sum e^t_i, T = sum t_i e^t_i;
//   log p_i = t_i - log S,   H = -sum p_i log p_i = log S - T / S  (both terms non-negative: no cancellation).
// Every thread keeps (m, S, T) of the vectors it has read and rescales when its maximum has moved far; pairs merge as S = sum S_j e^(m_j - m),
// T = sum (T_j + S_j (m_j - m)) e^(m_j - m).  A masked class (minus infinity, or a value so low that its exponential is 0) adds 0 to both.
//
// Best alternatives: for each quarter of its vectors a thread also remembers the maximum and which of them first held it.  These (value, vector) keys are all
// different, and the `top` best elements lie in the `top` parts with the best keys: an element elsewhere has those parts' maxima before it.
// Only these parts' vectors are read again, and only elements not below the last of the keys are ranked.  (Rows are read by so many CTAs at once that L2
// does not hold them: with whole threads in place of quarters the second reading of 8 of 256 threads took 14 us of 107 at 2048 rows of 131072 classes.)
//
// Bound: memory, every logit read once, then the special-function pipe (62 % of its slots: an exponential a logit).  A row is cut among the CTAs of a cluster where
// rows are few, and what they found is merged over distributed shared memory (asynchronous stores to the first CTA): no workspace, and sums are always added in
// the same order.  Short rows, and longer ones where there are many, go to a warp each, which needs no barrier.
// Measured on a B200, cold: 2048x131072 bf16 with 8 alternatives 101 us (5.3 TB/s; 92 without alternatives; 83 at the copy rate; in runs of a second, at 1.73 GHz, 109 and
// 102), 6x131072 fp32 with 20 alternatives 9.6 us (10.3 where rows are masked), 160x50257 fp16 with 10 14.1 (14.6; in L2 11.2 and 12.3), 4096x1000 fp32 with 8 15.3 us (in L2
// 12.7), 1x1000 with 5 4.8 us.
#include <algorithm>

#include "narrow_types.cuh"
#include "tc_common.cuh"

namespace
{
using namespace sb;

constexpr int TOP_MOST = 32, MAX_SPLIT = 8;
constexpr int CANDIDATES = 1024, PARTS = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, SLACK = 4.f;

struct LogpArgs
{
    long long rows, stride;
    int classes, top, split, token_bytes;
};

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// Whole numbers in the order of the floats, all of them above 0; both zeros alike, NaN (which no maximum sees) as minus infinity.
__device__ __forceinline__ uint32_t order_of(float x)
{
    x = x != x ? -INFINITY : x + 0.f;
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order)
{
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ unsigned long long make_key(uint32_t order, uint32_t index) { return (unsigned long long)order << 32 | (0xffffffffu - index); }

// Pairs of floats, one instruction for both.
__device__ __forceinline__ unsigned long long pair(float x, float y)
{
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void halves(unsigned long long v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b)
{
    unsigned long long v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b)
{
    unsigned long long v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c)
{
    unsigned long long v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

struct Stats
{
    float m, S, T;
};
// Both relative to the larger maximum.
__device__ __forceinline__ Stats merge(const Stats &a, const Stats &b)
{
    Stats r;
    r.m = fmaxf(a.m, b.m);
    r.S = r.T = 0.f;
    if (a.m != -INFINITY || a.S != 0.f) // nothing seen there: S = T = 0
    {
        const float d = a.m == r.m ? 0.f : a.m - r.m, c = exp2_approx(d * LOG2E);
        r.S += a.S * c;
        r.T += c == 0.f ? 0.f : (a.T + a.S * d) * c;
    }
    if (b.m != -INFINITY || b.S != 0.f)
    {
        const float d = b.m == r.m ? 0.f : b.m - r.m, c = exp2_approx(d * LOG2E);
        r.S += b.S * c;
        r.T += c == 0.f ? 0.f : (b.T + b.S * d) * c;
    }
    return r;
}

// The 16 bytes of vector v of a row whose first element is element `skew` of vector 0; elements outside the row are minus infinity.
template <int TYPE>
__device__ __forceinline__ uint4 load_vector(const void *row, int v, int skew, int classes)
{
    constexpr int VE = TYPE == SMALL_B200_TYPE_F32 ? 4 : 8;
    const long long first = (long long)v * VE - skew;
    if (first >= 0 && first + VE <= classes)
        return *reinterpret_cast<const uint4 *>(static_cast<const char *>(row) + first * (16 / VE));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (TYPE == SMALL_B200_TYPE_F32)
            w[i] = first + i >= 0 && first + i < classes ? static_cast<const uint32_t *>(row)[first + i] : 0xff800000u;
        else
        {
            const uint32_t none = TYPE == SMALL_B200_TYPE_BF16 ? 0xff80u : 0xfc00u;
            const long long e = first + 2 * i;
            const uint32_t lo = e >= 0 && e < classes ? static_cast<const uint16_t *>(row)[e] : none;
            const uint32_t hi = e + 1 >= 0 && e + 1 < classes ? static_cast<const uint16_t *>(row)[e + 1] : none;
            w[i] = lo | hi << 16;
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int TYPE>
__device__ __forceinline__ void unpack_vector(const uint4 &w, float *x)
{
    if (TYPE == SMALL_B200_TYPE_F32)
    {
        x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
    }
    else
    {
        unpack2<TYPE>(w.x, x[0], x[1]); unpack2<TYPE>(w.y, x[2], x[3]); unpack2<TYPE>(w.z, x[4], x[5]); unpack2<TYPE>(w.w, x[6], x[7]);
    }
}

// The largest of a vector's elements; a NaN is not seen (NaN where there is nothing else).
template <int TYPE>
__device__ __forceinline__ float vector_max(const uint4 &w)
{
    if (TYPE == SMALL_B200_TYPE_F32)
        return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    auto max2 = [](uint32_t a, uint32_t b) {
        uint32_t c;
        if (TYPE == SMALL_B200_TYPE_BF16)
            asm("max.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
        else
            asm("max.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
        return c;
    };
    float lo, hi;
    unpack2<TYPE>(max2(max2(w.x, w.y), max2(w.z, w.w)), lo, hi);
    return fmaxf(lo, hi);
}

// Masked classes in a row whose maximum is ordinary: within 1e6, so that its product with log2 e is rounded by less than 0.1, and in half precision
// above -6e4, far enough from the type's lowest value.
template <int TYPE>
struct Masked
{
    static constexpr float ORDINARY = TYPE == SMALL_B200_TYPE_F16 ? -6e4f : -1e6f;
    // Minus infinity and what is as low become -1e38 (-65504 in half precision): finite, times log2 e too, and still with an exponential of 0.
    __device__ __forceinline__ static void finite(uint4 &w, float *x)
    {
        if (TYPE == SMALL_B200_TYPE_F32)
        {
            unpack_vector<TYPE>(w, x);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = max_nan(x[i], -1e38f);
            return;
        }
        constexpr uint32_t LOWEST = TYPE == SMALL_B200_TYPE_BF16 ? 0xfe96fe96u : 0xfbfffbffu;
        auto max2 = [](uint32_t a) {
            uint32_t c;
            if (TYPE == SMALL_B200_TYPE_BF16)
                asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(LOWEST));
            else
                asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(LOWEST));
            return c;
        };
        w = make_uint4(max2(w.x), max2(w.y), max2(w.z), max2(w.w));
        unpack_vector<TYPE>(w, x);
    }
};

// The barrier of a row's threads.
template <int WARPS>
__device__ __forceinline__ void sync_row()
{
    if (WARPS == 1)
        __syncwarp();
    else
        __syncthreads();
}
template <int WARPS>
__device__ __forceinline__ unsigned long long block_max(unsigned long long key, unsigned long long *part)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1)
    {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, d);
        key = key > other ? key : other;
    }
    sync_row<WARPS>();
    if ((threadIdx.x & 31) == 0)
        part[WARPS == 1 ? 0 : threadIdx.x >> 5] = key;
    sync_row<WARPS>();
    key = part[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w)
        key = part[w] > key ? part[w] : key;
    return key;
}

// How many of a list's keys are above `k`.
__device__ __forceinline__ int rank_in(const unsigned long long *list, int n, unsigned long long k)
{
    int before = 0;
#pragma unroll 4
    for (int q = 0; q + 1 < n; q += 2)
    {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(list + q);
        before += (two.x > k) + (two.y > k);
    }
    return before + ((n & 1) && list[n - 1] > k);
}
constexpr int SHORT = 96; // lists that are ranked as they are: 160 rows of 50257 fp16, some masked whole, 20 alternatives 13.3 us for 64 and 96, 13.8 for 32, 16.9 for all lists
// Leaves in a long list (at most CANDIDATES keys, none 0) those that reach a bound which `top` of them reach, and returns how many: ranking takes the square of a
// list's length.  As for the parts' bound each warp's ceil(top / 8) th best is asked for; neighbours in the list, which came from one warp, go to different ones.
// By all threads; `count` is 0 and used for nothing else.  One copy of the code for all lists.
__device__ __noinline__ int keep_best(unsigned long long *list, int n, int top, unsigned long long *bounds, int *count)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long key[CANDIDATES / 256], mine = 0ull, nth = 0ull;
#pragma unroll
    for (int j = 0; j < CANDIDATES / 256; ++j)
    {
        const int i = j * 256 + lane * 8 + warp;
        key[j] = i < n ? list[i] : 0ull;
        mine = key[j] > mine ? key[j] : mine;
    }
    for (int i = 0; i < (top + 7) / 8; ++i)
    {
        const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
        const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32) == high ? (uint32_t)mine : 0u);
        nth = (unsigned long long)high << 32 | low;
        mine = mine == nth ? 0ull : mine;
    }
    if (lane == 0)
        bounds[warp] = nth;
    __syncthreads(); // the list has been read
    unsigned long long bound = bounds[0];
#pragma unroll
    for (int w = 1; w < 8; ++w)
        bound = bounds[w] < bound ? bounds[w] : bound;
#pragma unroll
    for (int j = 0; j < CANDIDATES / 256; ++j)
        if (key[j] != 0ull && key[j] >= bound)
            list[atomicAdd(count, 1)] = key[j];
    __syncthreads();
    return *count;
}

template <int WARPS>
struct Shared
{
    Stats part[WARPS], all;
    unsigned long long bound[WARPS], last;
    unsigned long long best[TOP_MOST]; // this CTA's best elements, in order
    alignas(16) unsigned long long found[WARPS == 1 ? 256 : CANDIDATES];
    unsigned long long keys[PARTS * 32 * WARPS];
    alignas(16) unsigned long long merged[WARPS == 1 ? 2 : MAX_SPLIT * TOP_MOST];
    float4 of_cta[MAX_SPLIT]; // every CTA's maximum and sums, in the first
    int first[TOP_MOST];      // the best parts' first vectors
    int parts, parts_kept, candidates, candidates_kept; // how many are in the lists
    uint64_t delivered;
};

template <int TYPE, int WARPS>
__global__ void __launch_bounds__(256, WARPS == 1 ? 3 : TYPE == SMALL_B200_TYPE_F32 ? 4 : 5)
    logprobs_kernel(const LogpArgs a, const void *logits, const void *tokens, float *logprobs, float *entropy, float *top_logprobs, int *top_tokens, int *status)
{
    constexpr int VE = TYPE == SMALL_B200_TYPE_F32 ? 4 : 8, SIZE = 16 / VE, BATCH = 4, THREADS = 32 * WARPS;
    constexpr int ROOM = sizeof(Shared<WARPS>::found) / 8;
    constexpr int ROWS = 8 / WARPS; // of a CTA
    __shared__ Shared<WARPS> of_row[ROWS];
    Shared<WARPS> &sh = of_row[WARPS == 1 ? threadIdx.x >> 5 : 0];
    const int tid = threadIdx.x & (THREADS - 1), lane = tid & 31, warp = tid >> 5;
    const long long r = WARPS == 1 ? (long long)blockIdx.x * ROWS + (threadIdx.x >> 5) : blockIdx.x / a.split;
    if (r >= a.rows)
        return;
    const int rank = (int)(blockIdx.x % a.split);
    const char *row = static_cast<const char *>(logits) + r * a.stride * SIZE;
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / SIZE);
    const int vectors = (int)(((long long)skew + a.classes + VE - 1) / VE);
    const int share = (vectors + a.split - 1) / a.split;
    const int v0 = rank * share, v1 = min(vectors, v0 + share);
    if (WARPS > 1 && a.split > 1)
    {
        if (tid == 0)
        {
            mbar_init(&sh.delivered, 1);
            fence_barrier_init();
            mbar_expect_tx(&sh.delivered, (uint32_t)(a.split * (8 * a.top + 16)));
        }
        __syncwarp();
        cluster_arrive_relaxed();
    }
    previous_kernel_done();
    next_kernel_may_start();
    // the given class's logit, asked for before everything else
    long long token = -1;
    float given = 0.f;
    if (tid == 0 && rank == 0 && logprobs)
    {
        token = a.token_bytes == 8 ? static_cast<const long long *>(tokens)[r] : static_cast<const int *>(tokens)[r];
        if (token >= 0 && token < a.classes)
            given = load1<TYPE>(row, token);
    }

    // ---- one pass: maximum and sums of this thread's vectors, in powers of two: S = sum 2^(L x - R), T = sum (L x - R) 2^(L x - R), L = log2 e.  The
    // reference R is L mu, rounded, and mu follows the maximum only when that is SLACK above it: at every step some lane of a warp has a new maximum, but
    // one that matters is rare.  Where mu is beyond ORDINARY, L mu is not rounded but subtracted first (R = L mu, exactly).
    float m = -INFINITY, mu = 0.f, R = 0.f, limit = -INFINITY; // limit: mu + SLACK, or minus infinity while there is no mu
    bool ordinary = true;
    unsigned long long S2 = 0ull, T2 = 0ull, minus_R = 0ull;
    const unsigned long long log2e2 = pair(LOG2E, LOG2E);
    // The best elements are looked for in the parts whose maxima are the largest: a thread's vectors in PARTS parts, `part` steps each.  key[q]: the part's
    // maximum and the vector that held it first, 0 without any.
    const int part = max(1, ((v1 - v0 + THREADS - 1) / THREADS + PARTS * BATCH - 1) / (PARTS * BATCH));
    unsigned long long *keys = sh.keys + tid;
    auto reference = [&](float vm) {
        const bool now = vm > Masked<TYPE>::ORDINARY && vm < 1e6f;
        const float to = vm * LOG2E;
        if (limit != -INFINITY)
        {
            const float d = ordinary ? (now ? R - to : -fmaf(vm, LOG2E, -R)) : (now ? fmaf(mu, LOG2E, -to) : (mu - vm) * LOG2E), c = exp2_approx(d);
            const unsigned long long c2 = pair(c, c);
            T2 = c == 0.f ? 0ull : mul2(fma2(S2, pair(d, d), T2), c2);
            S2 = mul2(S2, c2);
        }
        mu = vm; R = to; limit = vm + SLACK; ordinary = now;
        minus_R = pair(-to, -to);
    };
    // One vector's terms; what masked classes become there has an exponential of 0 but is finite: 0 times minus infinity would be NaN.
    auto add = [&](uint4 w) {
        float x[VE];
        Masked<TYPE>::finite(w, x);
#pragma unroll
        for (int i = 0; i < VE; i += 2)
        {
            const unsigned long long t = fma2(pair(x[i], x[i + 1]), log2e2, minus_R);
            float p, q;
            halves(t, p, q);
            const unsigned long long e = pair(exp2_approx(p), exp2_approx(q));
            S2 = add2(S2, e);
            T2 = fma2(e, t, T2);
        }
    };
    auto add_exactly = [&](const uint4 &w) {
        float x[VE];
        unpack_vector<TYPE>(w, x);
#pragma unroll
        for (int i = 0; i < VE; i += 2)
        {
            const float p = max_nan((x[i] - mu) * LOG2E, -1e30f), q = max_nan((x[i + 1] - mu) * LOG2E, -1e30f);
            const unsigned long long e = pair(exp2_approx(p), exp2_approx(q));
            S2 = add2(S2, e);
            T2 = fma2(e, pair(p, q), T2);
        }
    };
    const uint4 *aligned = reinterpret_cast<const uint4 *>(row - skew * SIZE);
    const int whole0 = skew > 0 ? 1 : 0, whole1 = min(v1, (int)(((long long)skew + a.classes) / VE)); // vectors with elements of this row only
    int v = v0 + tid;
#pragma unroll 1
    for (int q = 0; q < PARTS; ++q)
    {
        const int end = (int)min((long long)v1, v0 + (q + 1LL) * part * BATCH * THREADS), whole = min(end, whole1), begin = v;
        float pm = -INFINITY;
        int at = v;
        for (; v + (BATCH - 1) * THREADS < whole; v += BATCH * THREADS)
        {
            uint4 w[BATCH];
            float vm[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                w[j] = j == 0 && v < whole0 ? load_vector<TYPE>(row, v, skew, a.classes) : aligned[v + j * THREADS];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                vm[j] = vector_max<TYPE>(w[j]);
            float most = fmaxf(vm[0], vm[1]);
#pragma unroll
            for (int j = 2; j < BATCH; ++j)
                most = fmaxf(most, vm[j]);
            if (most > pm)
            {
                pm = most;
                at = v + (BATCH - 1) * THREADS;
#pragma unroll
                for (int j = BATCH - 2; j >= 0; --j)
                    at = vm[j] == most ? v + j * THREADS : at;
            }
            if (most > limit)
                reference(most);
            if (ordinary)
            {
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    add(w[j]);
            }
            else
            {
#pragma unroll 1
                for (int j = 0; j < BATCH; ++j)
                    add_exactly(j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3]);
            }
        }
#pragma unroll 1
        for (; v < end; v += THREADS)
        {
            const uint4 w = load_vector<TYPE>(row, v, skew, a.classes);
            const float vm = vector_max<TYPE>(w);
            if (vm > pm)
            {
                pm = vm;
                at = v;
            }
            if (vm > limit)
                reference(vm);
            if (ordinary)
                add(w);
            else
                add_exactly(w);
        }
        keys[q * THREADS] = begin < end ? make_key(order_of(pm), (uint32_t)at) : 0ull;
        m = fmaxf(m, pm);
    }
    // relative to the maximum itself, T in natural units
    float S, T;
    {
        float p, q;
        halves(S2, p, q);
        S = p + q;
        halves(T2, p, q);
        T = p + q;
        if (m != -INFINITY)
        {
            const float d = ordinary ? -fmaf(m, LOG2E, -R) : (mu - m) * LOG2E, c = exp2_approx(d);
            T = (T + S * d) * (c * LN2);
            S *= c;
        }
    }

    // ---- the CTA's maximum and sums
    Stats st;
    {
        const float wm = value_of(__reduce_max_sync(0xffffffffu, order_of(m)));
        st = merge({wm, 0.f, 0.f}, {m, S, T}); // its own sums relative to the warp's maximum
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
        {
            st.S += __shfl_xor_sync(0xffffffffu, st.S, d);
            st.T += __shfl_xor_sync(0xffffffffu, st.T, d);
        }
    }
    if (lane == 0)
        sh.part[warp] = st;
    if (tid == 0)
        sh.parts = sh.parts_kept = sh.candidates = sh.candidates_kept = 0;

    if (a.top > 0)
    {
        // ---- a bound that at least `top` parts reach: the least of the warps' ceil(top / WARPS) th best keys of their threads
        unsigned long long key[PARTS], most = 0ull;
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
        {
            key[q] = keys[q * THREADS];
            most = key[q] > most ? key[q] : most;
        }
        unsigned long long nth = 0ull;
        {
            unsigned long long mine = most;
            for (int n = 0; n < (a.top + WARPS - 1) / WARPS; ++n)
            {
                const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
                const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32) == high ? (uint32_t)mine : 0u);
                nth = (unsigned long long)high << 32 | low;
                mine = mine == nth ? 0ull : mine;
            }
        }
        if (lane == 0)
            sh.bound[warp] = nth;
        if (tid < a.top)
            sh.best[tid] = 0ull;
        if (tid == 0)
            sh.last = 0ull;
        sync_row<WARPS>();
        unsigned long long bound = sh.bound[0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w)
            bound = sh.bound[w] < bound ? sh.bound[w] : bound;
        // ---- the parts that reach it, and of them the `top` best
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
            if (key[q] != 0ull && key[q] >= bound)
                sh.found[atomicAdd(&sh.parts, 1)] = key[q];
        sync_row<WARPS>();
        int reach = sh.parts;
        if (WARPS > 1 && reach > SHORT) // equal logits: the first warp's parts are all before the next one's
            reach = keep_best(sh.found, reach, a.top, sh.bound, &sh.parts_kept);
        for (int i = tid; i < reach; i += THREADS)
        {
            const unsigned long long k = sh.found[i];
            const int before = rank_in(sh.found, reach, k);
            if (before < a.top)
            {
                const int steps_in = (int)(0xffffffffu - (uint32_t)k - (uint32_t)v0) / THREADS, thread = (int)(0xffffffffu - (uint32_t)k - (uint32_t)v0) % THREADS;
                sh.first[before] = v0 + thread + steps_in / (part * BATCH) * (part * BATCH) * THREADS;
            }
            if (before == a.top - 1)
                sh.last = k;
        }
        sync_row<WARPS>();
        // ---- their elements that are not below the last of them
        const int best_parts = min(reach, a.top);
        const unsigned long long last = sh.last;
        const uint32_t last_order = (uint32_t)(last >> 32), last_vector = 0xffffffffu - (uint32_t)last;
        const bool all = last == 0ull; // fewer threads than that have any
        const float last_value = value_of(last_order); // (not used where `all`)
        const int in_part = part * BATCH, shift = 32 - __clz(in_part - 1); // (four vectors at least)
        auto each = [&](auto take) { // all threads over the best threads' vectors, four at a time under way together
            constexpr int HELD = WARPS == 1 ? 4 : 2;
            for (int i = tid; i < best_parts << shift; i += HELD * THREADS)
            {
                uint4 w[HELD];
                int at[HELD];
#pragma unroll
                for (int h = 0; h < HELD; ++h)
                {
                    const int n = i + h * THREADS;
                    const int i_in = n & ((1 << shift) - 1);
                    at[h] = (n >> shift) < best_parts && i_in < in_part ? sh.first[n >> shift] + i_in * THREADS : v1;
                    if (at[h] < v1)
                        w[h] = load_vector<TYPE>(row, at[h], skew, a.classes);
                }
#pragma unroll
                for (int h = 0; h < HELD; ++h)
                {
                    if (at[h] >= v1 || (!all && vector_max<TYPE>(w[h]) < last_value)) // most of them
                        continue;
                    float x[VE];
                    unpack_vector<TYPE>(w[h], x);
#pragma unroll
                    for (int e = 0; e < VE; ++e)
                    {
                        const long long index = (long long)at[h] * VE - skew + e;
                        const uint32_t o = order_of(x[e]);
                        if (index >= 0 && index < a.classes && (all || o > last_order || (o == last_order && (uint32_t)at[h] <= last_vector)))
                            take(make_key(o, (uint32_t)index));
                    }
                }
            }
        };
        each([&](unsigned long long k) {
            const int n = atomicAdd(&sh.candidates, 1);
            if (n < ROOM)
                sh.found[n] = k;
        });
        sync_row<WARPS>();
        int n = sh.candidates;
        if (n <= ROOM)
        {
            if (WARPS > 1 && n > SHORT)
                n = keep_best(sh.found, n, a.top, sh.bound, &sh.candidates_kept);
            for (int i = tid; i < n; i += THREADS)
            {
                const unsigned long long k = sh.found[i];
                const int before = rank_in(sh.found, n, k);
                if (before < a.top)
                    sh.best[before] = k;
            }
        }
        else // rows in ascending order and the like: one after the other
        {
            unsigned long long limit = ~0ull;
            for (int j = 0; j < a.top; ++j)
            {
                unsigned long long k = 0ull;
                each([&](unsigned long long c) { k = c < limit && c > k ? c : k; });
                limit = block_max<WARPS>(k, sh.found);
                if (tid == 0)
                    sh.best[j] = limit;
                if (limit == 0ull)
                    break;
            }
        }
    }
    sync_row<WARPS>();
    if (tid == 0)
    {
        Stats s = sh.part[0];
        if (WARPS > 1)
        {
            float most = s.m;
#pragma unroll
            for (int w = 1; w < WARPS; ++w)
                most = fmaxf(most, sh.part[w].m);
            s = {most, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WARPS; ++w) // the same maximum for all, so that no sum waits for the one before it
            {
                const Stats o = merge({most, 0.f, 0.f}, sh.part[w]);
                s.S += o.S;
                s.T += o.T;
            }
        }
        sh.all = s;
    }

    // ---- the cluster's, in the first CTA: the others send it what they have
    const unsigned long long *best = sh.best;
    sync_row<WARPS>();
    if (WARPS > 1 && a.split > 1)
    {
        cluster_wait(); // the first CTA's barrier is there
        const uint32_t bar = map_to_cta(&sh.delivered, 0);
        if (tid < a.top)
            st_async_b64(map_to_cta(&sh.merged[rank * a.top + tid], 0), sh.best[tid], bar);
        if (tid == 32)
        {
            const uint32_t to = map_to_cta(&sh.of_cta[rank], 0);
            st_async_b64(to, pair(sh.all.m, sh.all.S), bar);
            st_async_b64(to + 8, pair(sh.all.T, 0.f), bar);
        }
        __syncwarp();
        cluster_arrive_relaxed(); // nothing more is sent
        bool delivered = true;
        if (rank == 0)
        {
            delivered = mbar_wait_cluster(&sh.delivered, 0, status, 121);
            if (tid == 0)
            {
                float most = sh.of_cta[0].x;
                for (int q = 1; q < a.split; ++q)
                    most = fmaxf(most, sh.of_cta[q].x);
                Stats s = {most, 0.f, 0.f};
                for (int q = 0; q < a.split; ++q)
                {
                    const Stats o = merge({most, 0.f, 0.f}, {sh.of_cta[q].x, sh.of_cta[q].y, sh.of_cta[q].z});
                    s.S += o.S;
                    s.T += o.T;
                }
                sh.all = s;
            }
            const int n = a.split * a.top;
            for (int i = tid; i < n; i += THREADS)
            {
                const unsigned long long k = sh.merged[i];
                const int before = rank_in(sh.merged, n, k);
                if (k != 0ull && before < a.top)
                    sh.found[before] = k;
            }
            best = sh.found;
        }
        cluster_wait(); // the first CTA's shared memory stays while anybody may send to it
        if (!delivered)
            for (int i = 0; i < 1000; ++i)
                __nanosleep(1000); // and what was sent last is on its way for less than that
        if (rank != 0)
            return;
        sync_row<WARPS>();
    }

    // ---- outputs
    Stats s = sh.all;
    s.S = max_nan(s.S, 1.f); // the largest class alone gives 1, and what T adds is not positive: roundings apart
    s.T = s.T > 0.f ? 0.f : s.T;
    const bool nothing = s.m == -INFINITY && !(s.S != s.S); // every class is masked: no probability, no entropy
    const float log_s = nothing ? 0.f : logf(s.S);
    auto logp = [&](float x) { return nothing ? (x != x ? x : -INFINITY) : (x - s.m) - log_s; };
    if (tid == 0)
    {
        if (logprobs)
            logprobs[r] = token < 0 ? 0.f : token >= a.classes ? NAN : logp(given);
        if (entropy)
            entropy[r] = nothing ? 0.f : log_s - s.T / s.S;
    }
    if (tid < a.top)
    {
        const unsigned long long k = best[tid];
        if (top_logprobs)
            top_logprobs[r * a.top + tid] = logp(value_of((uint32_t)(k >> 32)));
        if (top_tokens)
            top_tokens[r * a.top + tid] = (int)(0xffffffffu - (uint32_t)k);
    }
}

template <int TYPE, int WARPS>
int launch_logprobs(const LogpArgs &a, const void *logits, const void *tokens, float *logprobs, float *entropy, float *top_logprobs,
                    int32_t *top_tokens, cudaStream_t st)
{
    int *status = device_status_ptr();
    if (!status)
        return fail(SMALL_B200_CUDA_ERROR, "device status word not available");
    const long long grid = WARPS == 1 ? (a.rows + 7) / 8 : a.rows * a.split;
    // early where all CTAs are resident at once, three an SM or four (fp32; 3500 rows of 2000 a call of its own each 10.0 us, 12.3 otherwise)
    const Launch l((unsigned)grid, 256, 0, st, a.split > 1 ? (unsigned)a.split : 0u, grid <= (WARPS == 1 ? 3LL : 4LL) * num_sms());
    SB_CUDA(cudaLaunchKernelEx(&l.cfg, logprobs_kernel<TYPE, WARPS>, a, logits, tokens, logprobs, entropy, top_logprobs, (int *)top_tokens, status));
    return launched("logprobs_kernel");
}
} // namespace

extern "C" int small_b200_logprobs(int32_t rows, int32_t classes, int32_t in_type, const void *logits, int64_t stride, int32_t token_bytes,
                                   const void *tokens, float *logprobs, float *entropy, int32_t top, float *top_logprobs, int32_t *top_tokens,
                                   void *stream)
{
    const char *name = "LogProbabilities";
    if (rows < 0 || classes <= 0 || (stride != 0 && stride < classes))
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: bad shape.");
    const int size = type_size(in_type);
    if (size == 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: input type unsupported.");
    if (token_bytes != 4 && token_bytes != 8)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: tokens are of 4 or 8 bytes.");
    if (top < 0 || top > TOP_MOST || top > classes)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: top unsupported (at most 32, and at most the number of classes).");
    if (rows == 0)
        return SMALL_B200_OK;
    if (!logits || (logprobs && !tokens))
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: null buffer.");
    if (!top_logprobs && !top_tokens)
        top = 0;
    if (!logprobs && !entropy && top == 0)
        return SMALL_B200_OK;
    auto off = [](const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    if (off(logits, size) || (logprobs && off(tokens, token_bytes)) || off(logprobs, 4) || off(entropy, 4) || off(top_logprobs, 4) || off(top_tokens, 4))
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: misaligned buffer.");
    LogpArgs a;
    a.rows = rows; a.stride = stride ? stride : classes; a.classes = classes; a.top = top; a.token_bytes = token_bytes;
    // CTAs to a row, while each of their threads has a vector of its own.  What a CTA does besides reading (the best alternatives, the cluster) is 4 to 5 us, so more
    // of them than two an SM pay only for rows of 256 KB on, and eight a row only for few of such rows.  With 8 alternatives, cold, one, two and four CTAs a row:
    // 160 rows of 131073 fp32 classes 33.7, 25.0 and 30.7 us, of 50259 fp16 13.9, 12.9 and 14.0 (50257 in L2 11.1, 11.2, 13.7); 148 rows of 50259 13.3, 12.2 and 13.6; 592 of
    // 131073 fp32 53.4, 61.1 and 78.9.  Four and eight: 6 rows of 131073 fp32 10.3 and 9.1, of 50259 fp16 8.0 and 8.7.
    const bool longer = (long long)classes * size >= 256 << 10;
    a.split = 1;
    while (a.split < (longer ? MAX_SPLIT : MAX_SPLIT / 2) && rows * 2LL * a.split <= (a.split == 1 && longer ? 4LL : a.split < 4 ? 2LL : 1LL) * num_sms() &&
           classes / (16 / size) >= 2 * a.split * 256)
        a.split *= 2;
    if ((long long)rows * a.split > 0x7fffffffLL)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: too many rows.");
    cudaStream_t st = as_stream(stream);
    // A warp to a row or a CTA to a row, without and with 8 alternatives, cold: 1 row of 500 fp32 classes 3.2/5.0 us and 2.8/5.3, of 1001 3.9/5.8 and 2.9/4.9; 300 rows of
    // 700 3.3/5.2 and 3.6/7.1, of 2000 5.0/6.9 and 4.3/6.8; where the warps of all rows fill the SMs 1000 rows of 4000 11.4/13.7 and 12.6/16.7, of 8000 16.6/19.6 and
    // 14.5/18.8 (called one by one 16.6/19.5 and 16.4/20.5), of 16000 27.2/31.4 and 18.2/22.7; 4096 rows of 4000 24/29 and 40/54; in bf16 1000 rows of 16001 19.4/23.2 and 16.4/21.4 (in L2
    // 12.7/16.7 and 12.7/18.2), of 32000 31.0/37.2 and 20.1/25.4.
    const bool narrow = a.split == 1 && (classes <= 768 || (rows > 4 * num_sms() && (long long)classes * size <= 32768));
#define SB_LOGP(T, W) launch_logprobs<T, W>(a, logits, tokens, logprobs, entropy, top_logprobs, top_tokens, st)
    switch (in_type)
    {
    case SMALL_B200_TYPE_F32: return narrow ? SB_LOGP(SMALL_B200_TYPE_F32, 1) : SB_LOGP(SMALL_B200_TYPE_F32, 8);
    case SMALL_B200_TYPE_BF16: return narrow ? SB_LOGP(SMALL_B200_TYPE_BF16, 1) : SB_LOGP(SMALL_B200_TYPE_BF16, 8);
    default: return narrow ? SB_LOGP(SMALL_B200_TYPE_F16, 1) : SB_LOGP(SMALL_B200_TYPE_F16, 8);
    }
#undef SB_LOGP
}
