// Attention by rows: one warp per query row, keys in the lanes.  Any head
// size up to 256, any stride and alignment, f32 too.
//
//   s_j = scale q . k_j,  m = max s,  l = sum e^(s_j - m),
//   out = sum e^(s_j - m) v_j / l
//
// with m, l and the sum carried along 32 keys at a time.  For the calls that the
// tensor cores do not take (seq_attn.cuh); bound by the dot products, a key a
// lane, at a few TFLOP/s: 826 ms for two prompts of 8192 and 6001 tokens, 32
// heads of 128, that take 0.8 ms there.
#pragma once
#include "seq_common.cuh"

namespace aie {

constexpr int kRowsMaxDim = 256;

// Keys of packed prompts: token j of the sequence that starts at `first`.
template <typename T>
struct PackedKeys {
    HeadsOf<T> k, v;
    long long first;
    int head;
    __device__ __forceinline__ bool find(int j, const T *&kj, const T *&vj) const
    {
        kj = k.at(first + j, head);
        vj = v.at(first + j, head);
        return true;
    }
};

// Keys of a paged cache: places below `shared` through the prefix's pages.
template <typename T>
struct PagedKeys {
    const T *k, *v;
    PagesGeom g;
    const int32_t *prefix, *row;
    int shared, head;
    __device__ __forceinline__ bool find(int j, const T *&kj, const T *&vj) const
    {
        const int i = j / g.size;
        const int page = j < shared ? prefix[i] : row[i];
        if (page < 0 || page >= g.pages) return false;
        const long long at = page * g.ps + (j - i * g.size) * g.ts + head * g.hs;
        kj = k + at;
        vj = v + at;
        return true;
    }
};

// One row over its first n keys.  qs: this warp's scaled query in shared memory.
template <typename T, typename Keys>
__device__ __forceinline__ void attend_row(const float *qs, const Keys &keys, int n, int d, T *out, int lane)
{
    float acc[kRowsMaxDim / 32];
#pragma unroll
    for (int i = 0; i < kRowsMaxDim / 32; i++) acc[i] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        const T *kj = nullptr, *vj = nullptr;
        const bool real = j < n && keys.find(j, kj, vj);
        float s = -INFINITY;
        if (real) {
            s = 0.f;
            for (int i = 0; i < d; i++) s = fmaf(qs[i], to_f32(kj[i]), s);
        }
        const float top = fmaxf(m, warp_max(s));
        // no score above -inf yet: e^(-inf - -inf) is 1 for the sums so far
        // (all 0) and 0 for these keys; a NaN score stays NaN
        const float old = m == top ? 1.f : expf(m - top);
        const float p = !real || (top == -INFINITY && s == -INFINITY) ? 0.f : expf(s - top);
        l = fmaf(l, old, warp_sum(p));
        m = top;
#pragma unroll
        for (int i = 0; i < kRowsMaxDim / 32; i++) acc[i] *= old;
        unsigned todo = __ballot_sync(0xffffffffu, real);
        while (todo) {
            const int src = __ffs(todo) - 1;
            todo &= todo - 1;
            const float pj = __shfl_sync(0xffffffffu, p, src);
            const T *vrow = (const T *)__shfl_sync(0xffffffffu, (unsigned long long)vj, src);
#pragma unroll
            for (int i = 0; i < kRowsMaxDim / 32; i++)
                if (lane + 32 * i < d) acc[i] = fmaf(pj, to_f32(vrow[lane + 32 * i]), acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kRowsMaxDim / 32; i++)
        if (lane + 32 * i < d) out[lane + 32 * i] = from_f32<T>(n > 0 ? acc[i] / l : 0.f);
}

template <typename T>
struct PromptRows {
    HeadsOf<T> q, k, v, o;
    const int32_t *cu;
    int tokens, seqs, hq, group, d, causal;
    float scale;
};

// The sequence that holds token t: the first s with cu[s + 1] > t.
__device__ __forceinline__ int find_seq(const int32_t *cu, int seqs, int t)
{
    int lo = 0, hi = seqs;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(PromptRows<T> a)
{
    __shared__ float qs[4][kRowsMaxDim];
    behind_last_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= (long long)a.tokens * a.hq) return;
    const int t = (int)(row / a.hq), h = (int)(row % a.hq);
    const int s = find_seq(a.cu, a.seqs, t);
    if (s >= a.seqs) return;
    const int first = max(a.cu[s], 0), end = min(a.cu[s + 1], a.tokens);
    if (t < first) return;
    const T *q = a.q.at(t, h);
    for (int i = lane; i < a.d; i += 32) qs[warp][i] = to_f32(q[i]) * a.scale;
    __syncwarp();
    const PackedKeys<T> keys{a.k, a.v, first, h / a.group};
    attend_row<T>(qs[warp], keys, (a.causal ? t + 1 : end) - first, a.d, a.o.at(t, h), lane);
}

// Packed tokens and the states that their sequences see.
template <typename T>
struct CrossRows {
    HeadsOf<T> q, k, v, o;
    const int32_t *cu_q, *cu_k;
    int tokens, keys, seqs, hq, group, d;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(128) cross_rows_kernel(CrossRows<T> a)
{
    __shared__ float qs[4][kRowsMaxDim];
    behind_last_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= (long long)a.tokens * a.hq) return;
    const int t = (int)(row / a.hq), h = (int)(row % a.hq);
    const int s = a.cu_q ? find_seq(a.cu_q, a.seqs, t) : t;
    if (s >= a.seqs || (a.cu_q && t < a.cu_q[s])) return;
    const int first = min(max(a.cu_k[s], 0), a.keys), end = min(a.cu_k[s + 1], a.keys);
    const T *q = a.q.at(t, h);
    for (int i = lane; i < a.d; i += 32) qs[warp][i] = to_f32(q[i]) * a.scale;
    __syncwarp();
    const PackedKeys<T> keys{a.k, a.v, first, h / a.group};
    attend_row<T>(qs[warp], keys, end - first, a.d, a.o.at(t, h), lane);
}

template <typename T>
struct PrefixRows {
    HeadsOf<T> q, o;
    const T *k, *v;
    PagesGeom g;
    const int32_t *prefix, *table, *lens;
    int batch, hq, group, d, shared, max_len, table_stride;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(128) prefix_rows_kernel(PrefixRows<T> a)
{
    __shared__ float qs[4][kRowsMaxDim];
    behind_last_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= (long long)a.batch * a.hq) return;
    const int b = (int)(row / a.hq), h = (int)(row % a.hq);
    const T *q = a.q.at(b, h);
    for (int i = lane; i < a.d; i += 32) qs[warp][i] = to_f32(q[i]) * a.scale;
    __syncwarp();
    const PagedKeys<T> keys{a.k, a.v, a.g, a.prefix, a.table + (long long)b * a.table_stride, a.shared, h / a.group};
    attend_row<T>(qs[warp], keys, min(a.lens[b], a.max_len), a.d, a.o.at(b, h), lane);
}

}  // namespace aie
