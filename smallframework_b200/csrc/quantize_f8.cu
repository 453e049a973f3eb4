// quantize_f8.cu -- block-scaled quantisation of a matrix to e4m3: one fp32 scale for each block of 128 columns by one row (activations) or by
// 128 rows (weights), the operands of small_b200_dense_f8.
//
// Mathematics: scale = max|x| / 448 (448 is e4m3's largest value), code = x / scale to the nearest e4m3 value, ties to even, of the exact
// quotient.  A product with the rounded inverse is up to 2^-22 off, which matters only next to the middle between two codes (bf16 data meets
// middles exactly): both ends of that interval are converted, and only where the codes differ is x compared with middle * scale, exactly, in 64
// bits.
//
// Bound: memory (2 or 4 bytes read and one written an element).  16 lanes own 8 columns each of a block, so the largest magnitude of a row block is
// four shuffles away and nothing is read twice.
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
// The code of x / scale where `near` and `far` (same sign, |near| <= |far|) are the two candidates.
__device__ __noinline__ uint32_t exact_code(float x, float scale, uint32_t near, uint32_t far)
{
    if (near == far)
        return near;
    const double middle = 0.5 * ((double)fabsf(from_e4m3(near)) + (double)fabsf(from_e4m3(far))); // five significant bits
    const double ax = fabs((double)x), at = middle * (double)scale;                               // exact: 5 + 24 bits
    if (ax != at)
        return ax < at ? near : far;
    return (near & 1u) ? far : near;
}
// Eight values to eight codes; inv is 1 / scale to within one rounding.
__device__ __forceinline__ uint2 quantize8(const float *x, float scale, float inv)
{
    constexpr float EPS = 4.76837158e-7f; // 2^-21: more than the product's and the inverse's roundings together
    uint32_t n[4], f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float a = x[2 * i] * inv, b = x[2 * i + 1] * inv;
        n[i] = to_e4m3x2(a * (1.f - EPS), b * (1.f - EPS));
        f[i] = to_e4m3x2(a * (1.f + EPS), b * (1.f + EPS));
    }
    uint32_t lo = n[0] | n[1] << 16, hi = n[2] | n[3] << 16;
    const uint32_t flo = f[0] | f[1] << 16, fhi = f[2] | f[3] << 16;
    if (lo != flo || hi != fhi)
    {
        uint32_t l = 0, h = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            l |= exact_code(x[i], scale, lo >> (8 * i) & 0xffu, flo >> (8 * i) & 0xffu) << (8 * i);
            h |= exact_code(x[4 + i], scale, hi >> (8 * i) & 0xffu, fhi >> (8 * i) & 0xffu) << (8 * i);
        }
        lo = l; hi = h;
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
__device__ __forceinline__ float scale_of(float amax) { return amax > 0.f ? fmaxf(__fdiv_rn(amax, F8_MAX), SCALE_MIN) : 1.f; }

struct QuantArgs
{
    int rows, columns, blocks; // blocks of 128 columns in a row
    long long stride;
    long long units;
    FastDiv by_blocks;
};

constexpr int ROW_THREADS = 256, UNITS = 2; // row blocks that 16 lanes have in flight

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(ROW_THREADS) quantize_rows_f8_kernel(const QuantArgs a, const void *__restrict__ in, uint8_t *__restrict__ out,
                                                                         float *__restrict__ scales)
{
    constexpr int GROUPS = ROW_THREADS / 16;
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    // all lanes of a warp stay in the loop together: the shuffles need them
    for (long long u0 = (long long)blockIdx.x * (GROUPS * UNITS); u0 < a.units; u0 += (long long)gridDim.x * (GROUPS * UNITS))
    {
        float x[UNITS][8];
        int row[UNITS], block[UNITS];
        bool has[UNITS];
#pragma unroll
        for (int j = 0; j < UNITS; ++j)
        {
            const long long u = u0 + j * GROUPS + group;
            row[j] = u < a.units ? a.by_blocks.div((int)u) : 0;
            block[j] = u < a.units ? (int)u - row[j] * a.blocks : 0;
            const int c = block[j] * 128 + lane * 8;
            has[j] = u < a.units && c < a.columns;
            load8<TYPE, VEC>(in, (long long)row[j] * a.stride + c, has[j], x[j]);
        }
#pragma unroll
        for (int j = 0; j < UNITS; ++j)
        {
            float m = abs_max8(x[j]);
#pragma unroll
            for (int d = 8; d > 0; d >>= 1)
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            if (__any_sync(0xffffffffu, m == INFINITY)) // rare
            {
                infinities_to_nan(x[j]);
                m = abs_max8(x[j]);
#pragma unroll
                for (int d = 8; d > 0; d >>= 1)
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            }
            const float scale = scale_of(m);
            if (has[j])
            {
                *reinterpret_cast<uint2 *>(out + (long long)row[j] * a.columns + block[j] * 128 + lane * 8) = quantize8(x[j], scale, __frcp_rn(scale));
                if (lane == 0)
                    scales[(long long)row[j] * a.blocks + block[j]] = scale;
            }
        }
    }
}

// A CTA owns a square block: 16 lanes by 16 rows at a time, eight times, all of it in registers.
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) quantize_square_f8_kernel(const QuantArgs a, const void *__restrict__ in, uint8_t *__restrict__ out,
                                                                   float *__restrict__ scales)
{
    __shared__ float part[8];
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const int br = a.by_blocks.div((int)blockIdx.x), bc = (int)blockIdx.x - br * a.blocks;
    const int c = bc * 128 + lane * 8;
    float x[8][8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const int row = br * 128 + j * 16 + group;
        const bool has = row < a.rows && c < a.columns;
        load8<TYPE, VEC>(in, (long long)row * a.stride + c, has, x[j]);
    }
    for (int pass = 0;; ++pass)
    {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            m = fmaxf(m, abs_max8(x[j]));
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
                infinities_to_nan(x[j]);
            __syncthreads();
            continue;
        }
        const float scale = scale_of(m), inv = __frcp_rn(scale);
#pragma unroll
        for (int j = 0; j < 8; ++j)
        {
            const int row = br * 128 + j * 16 + group;
            if (row < a.rows && c < a.columns)
                *reinterpret_cast<uint2 *>(out + (long long)row * a.columns + c) = quantize8(x[j], scale, inv);
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
        quantize_square_f8_kernel<TYPE, VEC><<<(unsigned)a.units, 256, 0, st>>>(a, in, out, scales);
        return launched("quantize_square_f8_kernel");
    }
    long long blocks = (a.units + ROW_THREADS / 16 * UNITS - 1) / (ROW_THREADS / 16 * UNITS);
    const long long most = (long long)num_sms() * 16;
    quantize_rows_f8_kernel<TYPE, VEC><<<(unsigned)(blocks < most ? blocks : most), ROW_THREADS, 0, st>>>(a, in, out, scales);
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
    a.rows = rows; a.columns = columns; a.blocks = (columns + 127) / 128;
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
