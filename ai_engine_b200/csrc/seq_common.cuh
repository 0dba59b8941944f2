// Types and small device helpers of the sequence operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/aie_seq.h"
#include "common.cuh"

namespace aie {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x)
{
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
    else return x;
}

// Two values rounded to a pair of 16-bit ones.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t y;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}

// [tokens][heads][dim] of type T (aie_heads)
template <typename T>
struct HeadsOf {
    T *p;
    long long ts, hs;
    __device__ __forceinline__ T *at(long long t, int h) const { return p + t * ts + h * hs; }
};

template <typename T>
static inline HeadsOf<T> heads_of(const aie_heads &h)
{
    return HeadsOf<T>{(T *)h.data, (long long)h.token_stride, (long long)h.head_stride};
}

// One page's places of one head (aie_kv_pages)
struct PagesGeom {
    long long ps, ts, hs;
    int pages, size;
};

static inline PagesGeom pages_geom(const aie_kv_pages &p)
{
    return PagesGeom{(long long)p.page_stride, (long long)p.token_stride, (long long)p.head_stride, (int)p.pages,
                     (int)p.page_size};
}

// Every launch of these kernels may be set up while the one before it in the
// stream still runs (programmatic stream serialization): nothing in memory is
// touched before this, which waits for that one's end, and only then lets the
// launch behind this one be set up.  Back to back, a frame's prompt took 10.25
// us a call without, of which the kernel is 8.7 us.
//
// One exception: with a shared part, prefix_step_kernel reads a call's inputs
// (lengths, table, queries, the cache's pages) before its wait, and only the
// shared part's results and its own output after it.  That is right because it
// stands directly behind attn_tc_kernel in the stream, all of whose blocks have
// waited for whatever wrote those inputs before they let it start.  Neither may
// change: no launch between the two, and attn_tc_kernel's wait ahead of its
// launch_dependents.
__device__ __forceinline__ void behind_last_launch()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... P, typename... A>
static cudaError_t launch_behind(void (*fn)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, const A &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

}  // namespace aie
