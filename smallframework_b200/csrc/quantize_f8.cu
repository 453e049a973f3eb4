// quantize_f8.cu -- block-scaled quantisation of a matrix to e4m3: one fp32 scale for each block of 128 columns by one row (activations) or by
// 128 rows (weights), the operands of small_b200_dense_f8.
//
// Mathematics: scale = max|x| / 448 (448 is e4m3's largest value), code = x / scale to the nearest e4m3 value, ties to even, of the exact
// quotient.  A product with the rounded inverse is up to 2^-22 off, which matters only next to the middle between two codes (bf16 data meets
// middles): both ends of that interval are converted, and only where the codes differ is x compared with middle * scale, exactly.
//
// Bound: memory (2 or 4 bytes read and one written an element), and close behind it the integer ALU (70 % of its slots at 8192x8192 bf16: unpacking, conversions,
// packing).  16 lanes own 8 columns each of a block, so the largest magnitude of a row block is four shuffles away and nothing is read twice; four blocks a
// lane are under way, and 16-bit values are compared two at a time as they are.
// Measured on a B200, cold: 8192x8192 bf16 40.7 us (5.0 TB/s, 31.4 at the copy rate; in runs of a second 41.6), 5000x4112 fp32 in square blocks 19.3 us (5.3 TB/s, 15.9), 1x4096
// 2.0 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "narrow_types.cuh"
#include "tc_common.cuh"

namespace
{
using namespace sb;

constexpr float F8_MAX = 448.f;
constexpr float SCALE_MIN = 1.17549435e-38f; // 2^-126: the scale stays a normal number

// Two values to two e4m3 codes (the first in the low byte): nearest, ties to even, magnitudes beyond 448 to 448, NaN to NaN.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float from_e4m3(uint32_t code)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
// The code of x / scale where `near` and `far` (same sign, |near| < |far|) are the two candidates: |x| against middle * scale, which is the float
// `at` and what its rounding left.  Powers of two keep that remainder a normal number.
__device__ __noinline__ uint32_t exact_code(float x, float scale, uint32_t near, uint32_t far)
{
    const float up = scale < 1.f ? 1.8446744e19f : 1.f; // 2^64
    const float middle = 0.5f * (fabsf(from_e4m3(near)) + fabsf(from_e4m3(far))), s = scale * up, ax = fabsf(x) * up;
    const float at = middle * s, rest = fmaf(middle, s, -at); // middle has five significant bits
    if (ax != at)
        return ax < at ? near : far;
    if (rest != 0.f)
        return rest > 0.f ? near : far;
    return (near & 1u) ? far : near;
}
// Two products with one factor, one instruction.
__device__ __forceinline__ void mul2(float x, float y, unsigned long long f2, float &a, float &b)
{
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(f2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long twice(float f) { return (unsigned long long)__float_as_uint(f) << 32 | __float_as_uint(f); }
// Eight values to eight codes; inv is 1 / scale to within 2^-23 of it.
__device__ __forceinline__ uint2 quantize8(const float *x, float scale, float inv)
{
    constexpr float EPS = 4.76837158e-7f; // 2^-21: more than the product's and the inverse's errors together
    const unsigned long long below = twice(inv * (1.f - EPS)), above = twice(inv * (1.f + EPS));
    uint32_t n[4], f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        float a, b;
        mul2(x[2 * i], x[2 * i + 1], below, a, b);
        n[i] = to_e4m3x2(a, b);
        mul2(x[2 * i], x[2 * i + 1], above, a, b);
        f[i] = to_e4m3x2(a, b);
    }
    uint32_t lo = n[0] | n[1] << 16, hi = n[2] | n[3] << 16;
    const uint32_t flo = f[0] | f[1] << 16, fhi = f[2] | f[3] << 16;
    uint32_t dlo = lo ^ flo, dhi = hi ^ fhi;
    while (dlo | dhi) // one in 250 bf16 values: fractions of small numbers lie next to middles
    {
        const bool second = dlo == 0u;
        const int at = (__ffs((int)(second ? dhi : dlo)) - 1) & 24;
        const float p = second ? (at & 16 ? (at & 8 ? x[7] : x[6]) : (at & 8 ? x[5] : x[4]))
                               : (at & 16 ? (at & 8 ? x[3] : x[2]) : (at & 8 ? x[1] : x[0]));
        const uint32_t code = exact_code(p, scale, (second ? hi : lo) >> at & 0xffu, (second ? fhi : flo) >> at & 0xffu) << at, byte = 0xffu << at;
        if (second)
        {
            hi = (hi & ~byte) | code;
            dhi &= ~byte;
        }
        else
        {
            lo = (lo & ~byte) | code;
            dlo &= ~byte;
        }
    }
    return make_uint2(lo, hi);
}
__device__ __forceinline__ float abs_max8(const float *x)
{
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        m = fmaxf(m, fabsf(x[i])); // a NaN is not seen
    return m;
}
// Infinities take no part in the scale and become NaN, as NaN does.
__device__ __forceinline__ void infinities_to_nan(float *x)
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = fabsf(x[i]) == INFINITY ? NAN : x[i];
}
// amax / 448, rounded to nearest: the product with the rounded inverse and one correction by its exact remainder (P. Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990) give every quotient from 2^-126 on, in a sixth of a division's instructions; a test compares all significands of exponents
// over the whole range.
__device__ __forceinline__ float scale_of(float amax)
{
    constexpr float INV = 1.f / F8_MAX;
    const float s = amax * INV, rest = fmaf(-s, F8_MAX, amax);
    return amax > 0.f ? fmaxf(fmaf(rest, INV, s), SCALE_MIN) : 1.f;
}
// 1 / scale to within 2^-23 of it; scale is at least 2^-126 and below 2^120.
__device__ __forceinline__ float inverse_of(float scale)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
    return r;
}

// 16 bytes, asked for where this stands: a block's loads all go out before its first value is used.  (In the compiler's own order square blocks of 5000x4112 fp32
// take 19.7 to 20.2 us, in this one 19.2.)
__device__ __forceinline__ uint4 load16(const uint4 *p)
{
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

struct QuantArgs
{
    int rows, columns, blocks; // blocks of 128 columns in a row
    long long stride;
    long long units;
    FastDiv by_blocks;
};

// Eight elements as they are in memory; zeros where there are none.
template <int TYPE>
struct Raw8
{
    uint4 w[TYPE == SMALL_B200_TYPE_F32 ? 2 : 1];
    template <bool VEC>
    __device__ __forceinline__ void load(const void *p, long long at, bool has)
    {
        constexpr int N = TYPE == SMALL_B200_TYPE_F32 ? 2 : 1, SIZE = TYPE == SMALL_B200_TYPE_F32 ? 4 : 2;
        if (VEC)
        {
            const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) + at * SIZE);
#pragma unroll
            for (int i = 0; i < N; ++i)
                w[i] = has ? load16(q + i) : make_uint4(0u, 0u, 0u, 0u);
        }
        else
        {
            uint32_t v[4 * N];
#pragma unroll
            for (int i = 0; i < 4 * N; ++i)
                if (SIZE == 4)
                    v[i] = has ? static_cast<const uint32_t *>(p)[at + i] : 0u;
                else
                    v[i] = has ? static_cast<const uint16_t *>(p)[at + 2 * i] | (uint32_t)static_cast<const uint16_t *>(p)[at + 2 * i + 1] << 16 : 0u;
#pragma unroll
            for (int i = 0; i < N; ++i)
                w[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
    }
    // Infinities take no part in a scale and become NaN, as NaN does.
    __device__ __forceinline__ void infinities_to_nan()
    {
        constexpr int N = TYPE == SMALL_B200_TYPE_F32 ? 2 : 1;
        constexpr uint32_t INF = TYPE == SMALL_B200_TYPE_F32 ? 0x7f800000u : TYPE == SMALL_B200_TYPE_BF16 ? 0x7f80u : 0x7c00u;
        constexpr uint32_t QUIET = TYPE == SMALL_B200_TYPE_F32 ? 0x400000u : TYPE == SMALL_B200_TYPE_BF16 ? 0x40u : 0x200u;
        auto word = [](uint32_t &v) {
            if (TYPE == SMALL_B200_TYPE_F32)
                v |= (v & 0x7fffffffu) == INF ? QUIET : 0u;
            else
                v |= ((v & 0x7fffu) == INF ? QUIET : 0u) | ((v >> 16 & 0x7fffu) == INF ? QUIET << 16 : 0u);
        };
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            word(w[i].x);
            word(w[i].y);
            word(w[i].z);
            word(w[i].w);
        }
    }
    __device__ __forceinline__ void unpack(float *x) const
    {
        if (TYPE == SMALL_B200_TYPE_F32)
        {
            const uint4 &a = w[0], &b = w[TYPE == SMALL_B200_TYPE_F32 ? 1 : 0];
            x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
            x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
        }
        else
        {
            unpack2<TYPE>(w[0].x, x[0], x[1]); unpack2<TYPE>(w[0].y, x[2], x[3]); unpack2<TYPE>(w[0].z, x[4], x[5]); unpack2<TYPE>(w[0].w, x[6], x[7]);
        }
    }
};
// Of 16-bit values, two at a time, as they are: the larger ones, and the largest magnitudes of eight.
template <int TYPE>
__device__ __forceinline__ uint32_t max_of_pairs(uint32_t a, uint32_t b)
{
    uint32_t c;
    if (TYPE == SMALL_B200_TYPE_BF16)
        asm("max.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    else
        asm("max.f16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
}
template <int TYPE>
__device__ __forceinline__ uint32_t magnitudes(const Raw8<TYPE> &r)
{
    constexpr uint32_t MAG = 0x7fff7fffu;
    return max_of_pairs<TYPE>(max_of_pairs<TYPE>(r.w[0].x & MAG, r.w[0].y & MAG), max_of_pairs<TYPE>(r.w[0].z & MAG, r.w[0].w & MAG));
}
// The largest magnitude of the 16 lanes' values; a NaN is not seen.
template <int TYPE>
__device__ __forceinline__ float block_max(const Raw8<TYPE> &r, const float *x)
{
    if (TYPE == SMALL_B200_TYPE_F32)
    {
        float m = abs_max8(x);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        return m;
    }
    uint32_t m = magnitudes<TYPE>(r);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1)
        m = max_of_pairs<TYPE>(m, __shfl_xor_sync(0xffffffffu, m, d));
    float lo, hi;
    unpack2<TYPE>(m, lo, hi);
    return fmaxf(fmaxf(lo, hi), 0.f); // 0 where all are NaN
}
// A row block's codes and scale.
template <int TYPE>
__device__ __forceinline__ void finish_block(const Raw8<TYPE> &r, bool has, uint8_t *codes, float *scale_at, int lane)
{
    float x[8];
    r.unpack(x);
    float m = block_max<TYPE>(r, x);
    if (__any_sync(0xffffffffu, m == INFINITY)) // rare
    {
        infinities_to_nan(x);
        m = abs_max8(x);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    }
    const float scale = scale_of(m);
    if (has)
    {
        *reinterpret_cast<uint2 *>(codes) = quantize8(x, scale, inverse_of(scale));
        if (lane == 0)
            *scale_at = scale;
    }
}

constexpr int ROW_THREADS = 256, GROUPS = ROW_THREADS / 16, UNITS = 4; // row blocks at a time, and how many of them 16 lanes have in flight

// FLAT: packed rows of whole blocks, so that block u is elements 128 u to 128 u + 127 and scale u.
template <int TYPE, bool VEC, bool FLAT>
__global__ void __launch_bounds__(ROW_THREADS, TYPE == SMALL_B200_TYPE_F32 ? 4 : 5)
    quantize_rows_f8_kernel(const QuantArgs a, const void *in, uint8_t *out, float *scales)
{
    constexpr int SIZE = TYPE == SMALL_B200_TYPE_F32 ? 4 : 2;
    const int lane = threadIdx.x & 15;
    const long long u0 = (long long)blockIdx.x * (GROUPS * UNITS) + (threadIdx.x >> 4);
    Raw8<TYPE> r[UNITS];
    previous_kernel_done();
    next_kernel_may_start();
    if (FLAT && ((long long)blockIdx.x + 1) * (GROUPS * UNITS) <= a.units)
    {
        const char *p = static_cast<const char *>(in) + (u0 * 128 + lane * 8) * SIZE;
        uint8_t *q = out + u0 * 128 + lane * 8;
#pragma unroll
        for (int j = 0; j < UNITS; ++j)
            r[j].template load<VEC>(p + j * GROUPS * 128 * SIZE, 0, true);
#pragma unroll
        for (int j = 0; j < UNITS; ++j)
            finish_block<TYPE>(r[j], true, q + j * GROUPS * 128, scales + u0 + j * GROUPS, lane);
        return;
    }
    long long to[UNITS]; // where a lane's eight codes are
    bool has[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; ++j)
    {
        const long long u = u0 + j * GROUPS;
        has[j] = u < a.units;
        const int row = has[j] ? a.by_blocks.div((int)u) : 0, c = has[j] ? ((int)u - row * a.blocks) * 128 + lane * 8 : 0;
        has[j] = has[j] && c < a.columns;
        to[j] = (long long)row * a.columns + c;
        r[j].template load<VEC>(in, (long long)row * a.stride + c, has[j]);
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j) // all lanes of a warp together: the shuffles need them
        finish_block<TYPE>(r[j], has[j], out + to[j], scales + u0 + j * GROUPS, lane);
}

// A CTA owns a square block: 16 lanes by 16 rows at a time, eight times, all of it in registers, 16-bit values as they are.  A block's loads and stores take turns,
// so it is CTAs that hide them: 5000x4112 fp32 20.9 us with two an SM, 19.2 with three; 8192x8192 bf16 56 with two (values kept as floats), 45 with three, 41.2 with four.
// The bounds cost a few registers in local memory (80 a thread and 28 bytes stored in fp32, 64 and 4 in 16 bits; rows that are read element by element 48 and 12).
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256, TYPE == SMALL_B200_TYPE_F32 ? 3 : 4)
    quantize_square_f8_kernel(const QuantArgs a, const void *in, uint8_t *out, float *scales)
{
    __shared__ float part[8];
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int br = a.by_blocks.div((int)blockIdx.x), bc = (int)blockIdx.x - br * a.blocks;
    const int c = bc * 128 + lane * 8;
    Raw8<TYPE> r[8];
    previous_kernel_done();
    next_kernel_may_start();
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const int row = br * 128 + j * 16 + group;
        r[j].template load<VEC>(in, (long long)row * a.stride + c, row < a.rows && c < a.columns);
    }
    for (int pass = 0;; ++pass)
    {
        float m = 0.f;
        if (TYPE == SMALL_B200_TYPE_F32)
        {
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                float x[8];
                r[j].unpack(x);
                m = fmaxf(m, abs_max8(x));
            }
        }
        else
        {
            uint32_t most = magnitudes<TYPE>(r[0]);
#pragma unroll
            for (int j = 1; j < 8; ++j)
                most = max_of_pairs<TYPE>(most, magnitudes<TYPE>(r[j]));
            float lo, hi;
            unpack2<TYPE>(most, lo, hi);
            m = fmaxf(fmaxf(lo, hi), 0.f); // 0 where all are NaN
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        if ((threadIdx.x & 31) == 0)
            part[threadIdx.x >> 5] = m;
        __syncthreads();
        m = part[0];
#pragma unroll
        for (int w = 1; w < 8; ++w)
            m = fmaxf(m, part[w]);
        if (m == INFINITY && pass == 0) // the same for all threads
        {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                r[j].infinities_to_nan();
            __syncthreads();
            continue;
        }
        const float scale = scale_of(m), inv = inverse_of(scale);
#pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            const int row = br * 128 + j * 16 + group;
            if (row < a.rows && c < a.columns)
            {
                float x[8];
                r[j].unpack(x);
                *reinterpret_cast<uint2 *>(out + (long long)row * a.columns + c) = quantize8(x, scale, inv);
            }
        }
        if (threadIdx.x == 0)
            scales[blockIdx.x] = scale;
        return;
    }
}

template <int TYPE, bool VEC>
int launch_quantize(const QuantArgs &a, int block_rows, const void *in, uint8_t *out, float *scales, cudaStream_t st)
{
    if (block_rows == 128)
    {
        const Launch l((unsigned)a.units, 256, 0, st, 0, a.units <= 3LL * num_sms());
        SB_CUDA(cudaLaunchKernelEx(&l.cfg, quantize_square_f8_kernel<TYPE, VEC>, a, in, out, scales));
        return launched("quantize_square_f8_kernel");
    }
    const Launch l((unsigned)((a.units + GROUPS * UNITS - 1) / (GROUPS * UNITS)), ROW_THREADS, 0, st, 0, a.units <= 4LL * num_sms() * GROUPS * UNITS);
    if (VEC && a.stride == a.columns && a.columns % 128 == 0)
        SB_CUDA(cudaLaunchKernelEx(&l.cfg, quantize_rows_f8_kernel<TYPE, VEC, VEC>, a, in, out, scales));
    else
        SB_CUDA(cudaLaunchKernelEx(&l.cfg, quantize_rows_f8_kernel<TYPE, VEC, false>, a, in, out, scales));
    return launched("quantize_rows_f8_kernel");
}
} // namespace

extern "C" int small_b200_quantize_blocks_f8(int32_t rows, int32_t columns, int32_t block_rows, int32_t in_type, const void *in, int64_t in_stride,
                                             void *out, float *scales, void *stream)
{
    const char *name = "QuantizeBlocks<float8>";
    if (columns <= 0 || columns % CB != 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: in_channels unsupported.");
    if (rows < 0 || (block_rows != 1 && block_rows != 128) || (in_stride != 0 && in_stride < columns))
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: bad shape.");
    const int size = type_size(in_type);
    if (size == 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: input type unsupported.");
    if (rows == 0)
        return SMALL_B200_OK;
    if (!in || !out || !scales)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: null buffer.");
    if (reinterpret_cast<uintptr_t>(in) % size != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 4 != 0)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: misaligned buffer (the codes begin on a 16-byte boundary).");
    QuantArgs a;
    a.rows = rows; a.columns = columns; a.blocks = (int)((columns + 127LL) / 128);
    a.stride = in_stride ? in_stride : columns;
    a.units = (long long)(block_rows == 1 ? rows : (rows + 127LL) / 128) * a.blocks;
    if (a.units > 0x7fffffffLL)
        return fail(SMALL_B200_INVALID_ARGUMENT, std::string(name) + " ERROR: too many blocks.");
    a.by_blocks.set(a.blocks);
    const bool vec = reinterpret_cast<uintptr_t>(in) % 16 == 0 && a.stride * size % 16 == 0;
    uint8_t *o = static_cast<uint8_t *>(out);
    cudaStream_t st = as_stream(stream);
#define SB_QUANT(T) (vec ? launch_quantize<T, true>(a, block_rows, in, o, scales, st) : launch_quantize<T, false>(a, block_rows, in, o, scales, st))
    switch (in_type)
    {
    case SMALL_B200_TYPE_F32: return SB_QUANT(SMALL_B200_TYPE_F32);
    case SMALL_B200_TYPE_BF16: return SB_QUANT(SMALL_B200_TYPE_BF16);
    default: return SB_QUANT(SMALL_B200_TYPE_F16);
    }
#undef SB_QUANT
}
