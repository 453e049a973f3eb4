// narrow_types.cuh -- element types of the layers that take or give 16-bit floats beside fp32.
//
// Times in the comments of these layers' kernels, unless they say otherwise: a B200, calls in a row in a captured graph that runs for some milliseconds.  "Cold":
// with inputs in turn that are larger than L2 (126 MB) together.  In runs of a second the card's 1 kW power cap lowers the clock to 1.4 to 1.7 GHz; those times are named so.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace sb
{
// Bytes of an element, 0 for a type that does not exist.
inline int type_size(int type)
{
    return type == SMALL_B200_TYPE_F32 ? 4 : (type == SMALL_B200_TYPE_BF16 || type == SMALL_B200_TYPE_F16) ? 2 : 0;
}

// A launch of clusters of `cluster` CTAs along x, 0 for none (the kernels then use no cluster instructions: stores to shared::cluster and cluster barriers raised
// illegal instructions in a launch without clusters).  With `early` it may come up while the kernel before it in its stream ends: its kernel sets itself up,
// calls previous_kernel_done() before it touches global memory, and next_kernel_may_start() once; what comes behind it waits for the whole of it all the same.
// (One launch reads without that wait: the second of a dense layer on few rows that is two launches, whose first one has waited.)
// Calls in a row on a B200: dense 1 row, 2048 -> 512, 4.3 us and 3.2, 4096 -> 4096 5.8 and 5.4; but the quantisation of 8192x8192, whose 8192 CTAs come and
// go, 40.5 and 46.2: early only where the grid is resident at once, or is a few waves of long CTAs (dense on few rows, up to four waves: 1 row, 512 -> 40000, 12.2 us
// and 9.9, 1024 -> 131072 32.6 and 30.0; 64 rows, 1920 -> 60000, 33.9 and 31.7).
struct Launch
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    Launch(unsigned grid, unsigned threads, size_t smem, cudaStream_t st, unsigned cluster = 0, bool early = true)
    {
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = cluster > 0 ? 2 : 1;
    }
};

#ifdef __CUDACC__
// What the kernel before wrote is read by plain loads behind the wait: __ldg and const __restrict__ are for data that nobody writes while a kernel exists, and
// the compiler may move such loads over the wait.
__device__ __forceinline__ void previous_kernel_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_kernel_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// The two 16-bit floats of a word.
template <int TYPE>
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi)
{
    if (TYPE == SMALL_B200_TYPE_BF16)
    {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    }
    else
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x;
        hi = f.y;
    }
}
template <int TYPE>
__device__ __forceinline__ float load1(const void *p, long long at)
{
    if (TYPE == SMALL_B200_TYPE_F32)
        return static_cast<const float *>(p)[at];
    if (TYPE == SMALL_B200_TYPE_BF16)
        return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
    return __half2float(static_cast<const __half *>(p)[at]);
}
// Two floats rounded to nearest into a word.
template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if (TYPE == SMALL_B200_TYPE_BF16)
    {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
#endif
} // namespace sb
