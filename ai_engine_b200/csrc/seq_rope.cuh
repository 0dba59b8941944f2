// Norm of queries and keys and the position rotation, with keys and values
// filed into a paged cache.
//
//   r = rsqrt(sum_d x_d^2 / D + eps),  y_d = x_d r w_d
//   (y_i, y_j) -> (y_i cos a - y_j sin a, y_j cos a + y_i sin a)
//
// in f32, rounded once.  A head is read once and written once (keys twice
// when they also go to the cache): memory-bound.
#pragma once
#include "seq_common.cuh"

namespace aie {

template <typename T>
struct RopeArgs {
    HeadsOf<T> q, k, v, qo, ko;
    T *kp, *vp;
    PagesGeom pg;
    const float *wq, *wk, *cs;
    const int32_t *pos;
    const int64_t *slots;
    int tokens, hq, hk, d, rot, max_pos, interleaved;
    float eps;
};

// Where a token's head stands in the cache, or nullptr.
template <typename T>
__device__ __forceinline__ T *rope_slot(T *pages, const PagesGeom &g, const int64_t *slots, int t, int h)
{
    if (!pages) return nullptr;
    const long long s = slots[t];
    if (s < 0 || s >= (long long)g.pages * g.size) return nullptr;
    return pages + (s / g.size) * g.ps + (s % g.size) * g.ts + h * g.hs;
}

constexpr int kRopeMaxDim = 512;

// Any head size, stride and alignment: one warp per head of a token (query
// heads, then key heads, then value heads, which are only filed), the normed
// head in shared memory while it is rotated.
template <typename T>
__global__ void __launch_bounds__(128) rope_row_kernel(RopeArgs<T> a)
{
    __shared__ float buf[4][kRopeMaxDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = a.hq + a.hk + (a.vp ? a.hk : 0);
    const long long unit = (long long)blockIdx.x * 4 + warp;
    if (unit >= (long long)a.tokens * rows) return;
    const int t = (int)(unit / rows);
    int h = (int)(unit % rows);
    if (h >= a.hq + a.hk) {
        h -= a.hq + a.hk;
        T *dst = rope_slot(a.vp, a.pg, a.slots, t, h);
        if (!dst) return;
        const T *src = a.v.at(t, h);
        for (int i = lane; i < a.d; i += 32) dst[i] = src[i];
        return;
    }
    const bool key = h >= a.hq;
    if (key) h -= a.hq;
    const T *src = key ? a.k.at(t, h) : a.q.at(t, h);
    const float *w = key ? a.wk : a.wq;
    float *y = buf[warp];
    float sum = 0.f;
    for (int i = lane; i < a.d; i += 32) {
        const float x = to_f32(src[i]);
        y[i] = x;
        sum = fmaf(x, x, sum);
    }
    __syncwarp();
    if (w) {
        const float r = 1.0f / sqrtf(warp_sum(sum) / (float)a.d + a.eps);
        for (int i = lane; i < a.d; i += 32) y[i] = y[i] * r * w[i];
        __syncwarp();
    }
    T *o1 = key ? (a.ko.p ? a.ko.at(t, h) : nullptr) : a.qo.at(t, h);
    T *o2 = key ? rope_slot(a.kp, a.pg, a.slots, t, h) : nullptr;
    const int half = a.rot >> 1;
    const int pos = a.rot ? a.pos[t] : 0;
    const bool ok = pos >= 0 && pos < a.max_pos;
    const float *cs = a.cs + (long long)(ok ? pos : 0) * a.rot;
    for (int i = lane; i < a.d; i += 32) {
        float v = y[i];
        if (i < a.rot) {
            const int f = a.interleaved ? i >> 1 : (i < half ? i : i - half);
            const bool first = a.interleaved ? !(i & 1) : i < half;
            const float other = y[a.interleaved ? i ^ 1 : (first ? i + half : i - half)];
            const float c = cs[f], s = cs[half + f];
            v = first ? v * c - other * s : v * c + other * s;
            if (!ok) v = __int_as_float(0x7fffffff);
        }
        const T r = from_f32<T>(v);
        if (o1) o1[i] = r;
        if (o2) o2[i] = r;
    }
}

template <typename T>
static cudaError_t rope_launch(const RopeArgs<T> &a, cudaStream_t s)
{
    const long long units = (long long)a.tokens * (a.hq + a.hk + (a.vp ? a.hk : 0));
    rope_row_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace aie
