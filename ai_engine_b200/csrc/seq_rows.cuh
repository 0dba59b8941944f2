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

// Packed tokens over states where the tensor cores cannot take them (f32, heads of
// more than 128, strides that TMA does not address): 64 rows, tokens times the
// query heads of a group, by 32 states at a time in shared memory, all in f32.
//
//   S = Q K^T, P = e^(S - m), O = O e^(m' - m) + P V
//
// A thread has 4 rows by 2 states of S and 4 rows by 4 J columns of O: about as
// many cycles of shared memory as of multiply-adds, and few warps to hide what is
// late in either.  2048 tokens over 2048 states, f32: 8 heads of 64 357 us, 24
// TFLOP/s (533 without the next states' loads ahead, a warp per row 9072); 8/2
// heads of 128 676 us (781 with them); bf16, 8/2 heads of 256 1.69 ms, 20 TFLOP/s (a
// warp per row 32.3).
constexpr int kTileRows = 64, kTileKeys = 32, kTileThreads = 256;

constexpr uint32_t cross_tile_smem(int d)
{
    const uint32_t dp = (d + 3) / 4 * 4;
    return 4 * ((kTileRows + kTileKeys) * (dp + 4) + kTileKeys * dp + kTileRows * (kTileKeys + 4));
}

template <typename T, int J>
__global__ void __launch_bounds__(kTileThreads, J == 4 ? 1 : 2) cross_tile_kernel(const CrossRows<T> a, int heads)
{
    extern __shared__ __align__(16) float tile_smem[];
    __shared__ int work[5];  // found; the sequence's tokens and states; the tile's first row
    behind_last_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.x % heads;
    const long long unit = blockIdx.x / heads;

    // ---- whose rows these are
    if (!a.cu_q) {
        // a token each: as many tiles for every sequence
        if (tid == 0) {
            const int tiles = (a.group + kTileRows - 1) / kTileRows;
            const long long s = unit / tiles;
            work[0] = s < a.seqs ? (int)s + 1 : 0;
            if (s < a.seqs) {
                work[1] = (int)s; work[2] = 1;
                work[3] = min(max(a.cu_k[s], 0), a.keys);
                work[4] = max(min(a.cu_k[s + 1], a.keys) - work[3], 0);
                *(long long *)tile_smem = (unit - s * tiles) * kTileRows;
            }
        }
    } else if (warp == 0) {
        if (lane == 0) work[0] = 0;
        __syncwarp();
        long long before = 0;
        for (int s0 = 0; s0 < a.seqs; s0 += 32) {
            const int s = min(s0 + lane, a.seqs), next = min(s + 1, a.seqs);
            const int from = min(max(a.cu_q[s], 0), a.tokens), n = max(min(a.cu_q[next], a.tokens) - from, 0);
            const long long mine = ((long long)n * a.group + kTileRows - 1) / kTileRows;
            long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            upto += before;
            if (unit < upto && unit >= upto - mine) {
                work[0] = s + 1;
                work[1] = from; work[2] = n;
                work[3] = min(max(a.cu_k[s], 0), a.keys);
                work[4] = max(min(a.cu_k[next], a.keys) - work[3], 0);
                before = upto - mine;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, unit < upto);
            if (hit) {
                before = __shfl_sync(0xffffffffu, before, __ffs(hit) - 1);
                break;
            }
            before = __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) *(long long *)tile_smem = (unit - before) * kTileRows;
    }
    __syncthreads();
    if (!work[0]) return;
    const int first = work[1], key0 = work[3], n = work[4];
    const long long row0 = *(const long long *)tile_smem, rows = (long long)work[2] * a.group;
    __syncthreads();

    const int dp = (a.d + 3) / 4 * 4, ld = dp + 4;
    float *const qs = tile_smem, *const ks = qs + kTileRows * ld, *const vs = ks + kTileKeys * ld, *const ps = vs + kTileKeys * dp;
    auto row_of = [&](const HeadsOf<T> &x, long long r) {
        const int tok = (int)(r / a.group), g = (int)(r - (long long)tok * a.group);
        return x.at(first + tok, kvh * a.group + g);
    };
    // a warp a row, a lane every 32nd element
    constexpr int kWarps = kTileThreads / 32, kRows = kTileKeys / kWarps;
    auto load = [&](const T *p, bool real, T (&x)[2 * J]) {
#pragma unroll
        for (int i = 0; i < 2 * J; i++) x[i] = real && lane + 32 * i < a.d ? p[lane + 32 * i] : from_f32<T>(0.f);
    };
    auto keep = [&](const T (&x)[2 * J], float f, float *to) {
#pragma unroll
        for (int i = 0; i < 2 * J; i++)
            if (lane + 32 * i < dp) to[lane + 32 * i] = to_f32(x[i]) * f;
    };
    for (int r = warp; r < kTileRows; r += kWarps) {
        const bool real = row0 + r < rows;
        T x[2 * J];
        load(real ? row_of(a.q, row0 + r) : nullptr, real, x);
        keep(x, a.scale, qs + r * ld);
    }
    // the next states are on their way while these are worked on, but for J = 2, where that
    // takes more registers than two blocks an SM have
    constexpr bool kAhead = J != 2;
    T kx[kRows][2 * J], vx[kRows][2 * J];
    auto ahead = [&](int k0) {
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const int r = k0 + warp + i * kWarps;
            load(r < n ? a.k.at(key0 + r, kvh) : nullptr, r < n, kx[i]);
            load(r < n ? a.v.at(key0 + r, kvh) : nullptr, r < n, vx[i]);
        }
    };
    if constexpr (kAhead) ahead(0);

    const int ty = tid >> 4, tx = tid & 15;
    float m[4], l[4] = {}, o[4][J][4] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = -INFINITY;
    for (int k0 = 0; k0 < n; k0 += kTileKeys) {
        if constexpr (!kAhead) ahead(k0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const int r = warp + i * kWarps;
            keep(kx[i], 1.f, ks + r * ld);
            keep(vx[i], 1.f, vs + r * dp);
        }
        __syncthreads();
        if constexpr (kAhead) ahead(k0 + kTileKeys);
        float s[4][2] = {};
        for (int c = 0; c < dp; c += 4) {
            float4 q[4], k[2];
#pragma unroll
            for (int i = 0; i < 4; i++) q[i] = *(const float4 *)(qs + (ty * 4 + i) * ld + c);
#pragma unroll
            for (int j = 0; j < 2; j++) k[j] = *(const float4 *)(ks + (tx + 16 * j) * ld + c);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    s[i][j] = fmaf(q[i].w, k[j].w, fmaf(q[i].z, k[j].z, fmaf(q[i].y, k[j].y, fmaf(q[i].x, k[j].x, s[i][j]))));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (k0 + tx + 16 * j >= n) s[i][j] = -INFINITY;
            float top = fmaxf(m[i], fmaxf(s[i][0], s[i][1]));
#pragma unroll
            for (int e = 1; e < 16; e <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
            // nothing but scores of -inf so far: no weight, and no 0 / 0 either
            const float ref = top == -INFINITY ? 0.f : top, f = ex2((m[i] - ref) * 1.4426950408889634f);
            m[i] = top;
            l[i] *= f;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float p = ex2((s[i][j] - ref) * 1.4426950408889634f);
                l[i] += p;
                ps[(ty * 4 + i) * (kTileKeys + 4) + tx + 16 * j] = p;
            }
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][j][e] *= f;
        }
        __syncwarp();  // a row's weights are its half warp's own
        for (int k = 0; k < kTileKeys; k += 4) {
            float4 p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = *(const float4 *)(ps + (ty * 4 + i) * (kTileKeys + 4) + k);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int j = 0; j < J; j++) {
                    if (tx * 4 + 64 * j >= dp) continue;
                    const float4 v = *(const float4 *)(vs + (k + e) * dp + tx * 4 + 64 * j);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float w = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
                        o[i][j][0] = fmaf(w, v.x, o[i][j][0]); o[i][j][1] = fmaf(w, v.y, o[i][j][1]);
                        o[i][j][2] = fmaf(w, v.z, o[i][j][2]); o[i][j][3] = fmaf(w, v.w, o[i][j][3]);
                    }
                }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float sum = l[i];
#pragma unroll
        for (int e = 1; e < 16; e <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, e);
        const long long r = row0 + ty * 4 + i;
        if (r >= rows) continue;
        const float f = n ? 1.f / sum : 0.f;
        T *out = row_of(a.o, r);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (tx * 4 + 64 * j + e < a.d) out[tx * 4 + 64 * j + e] = from_f32<T>(o[i][j][e] * f);
    }
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
