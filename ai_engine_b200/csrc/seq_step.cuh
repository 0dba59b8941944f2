// One query token for each of a batch of streams over the places of its own
// (16-bit operands), joined with the shared prefix's partial results.
//
//   S = Q K^T for the query heads that read one key/value head,
//   m, l, O carried along; at the end every partial result (m_i, l_i, O_i)
//   has weight 2^(m_i - m):  out = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i
//
// Each place is read once and used for a group of query heads: memory-bound.
// A block takes a piece of one stream's places for one key/value head, 64 at
// a time through a ring of shared memory filled by asynchronous copies; each
// of its four warps multiplies 16 of the 64 (m16n8k16, the group padded to
// 16 rows) and carries its own m, l and O.  Where streams are few, the pieces
// of one stream are a cluster of up to 8 blocks, whose results meet in
// distributed shared memory.  Fixed order throughout: results repeat bit for
// bit.
//
// Rounding to fewer bits: the weights to the operands' type for the product
// with V (l sums them unrounded), and the result.
#pragma once
#include <cooperative_groups.h>

#include "seq_attn.cuh"

namespace aie {

constexpr int kStKeys = 64;      // places of one ring stage
constexpr int kStStages = 3;
constexpr int kStThreads = 128;
constexpr int kStList = 1024;    // page numbers held at a time

template <typename T>
struct StepArgs {
    HeadsOf<T> q, o;
    const T *k, *v;
    PagesGeom g;
    FastDiv size;
    const int32_t *prefix, *table, *lens;
    const float *part_o, *part_lse;  // the shared part's results, `splits` of them
    int batch, hq, hk, group, d, from, shared, max_len, table_stride, splits;
    int q_pairs;  // two elements of q are 4-byte aligned
    float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool real)
{
    const int n = real ? 16 : 0;  // 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void add_scaled(float4 &x, float f, const float4 &y)
{
    x.x = fmaf(f, y.x, x.x);
    x.y = fmaf(f, y.y, x.y);
    x.z = fmaf(f, y.z, x.z);
    x.w = fmaf(f, y.w, x.w);
}

template <int DK>
struct StepSmem {
    static constexpr uint32_t kTile = kStKeys * DK * 2;          // K or V of a stage
    static constexpr uint32_t kRing = kStStages * 2 * kTile;     // reused for the warps' O at the end
    static constexpr uint32_t kO = 16 * DK * 4;                  // one result of 16 rows
    static constexpr uint32_t kBytes = kRing + kO;               // ring, the block's result
    static_assert(4 * kO <= kRing, "the warps' results fit the ring");
};

template <typename T, int DK>
__global__ void __launch_bounds__(kStThreads)
prefix_step_kernel(const StepArgs<T> a)
{
    namespace cg = cooperative_groups;
    using Sm = StepSmem<DK>;
    constexpr int kChunks = DK / 8;  // 16-byte pieces of a head
    extern __shared__ __align__(128) char smem[];
    __shared__ int32_t list[kStList];
    __shared__ float warp_m[4][16], warp_l[4][16], block_m[16], block_l[16];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.y, row0 = blockIdx.z * 16;
    const int b = blockIdx.x / ranks;
    const int heads = min(a.group - row0, 16);
    float *const block_o = (float *)(smem + Sm::kRing);

    // this block's places [lo, hi): whole tiles of 64
    const int len = min(max(a.lens[b], 0), a.max_len);
    const int tiles = (max(len - a.from, 0) + kStKeys - 1) / kStKeys, per = (tiles + ranks - 1) / ranks;
    const int lo = a.from + min(rank * per, tiles) * kStKeys, hi = min(a.from + min((rank + 1) * per, tiles) * kStKeys, len);

    // the group's queries, padded to 16 rows, as the A operand
    uint32_t qa[DK / 16][4];
    {
        const int r = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < DK / 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = r + (i & 1) * 8, col = k * 16 + c + (i >> 1) * 8;
                uint32_t x = 0;
                if (row < heads && col < a.d) {  // d is even
                    const T *p = a.q.at(b, kvh * a.group + row0 + row) + col;
                    x = a.q_pairs ? *(const uint32_t *)p
                                  : (uint32_t)*(const unsigned short *)p | (uint32_t)*(const unsigned short *)(p + 1) << 16;
                }
                qa[k][i] = x;
            }
    }
    float o[DK / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DK / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    const int32_t *row = a.table + (long long)b * a.table_stride;
    const int edge = fdiv(a.shared, a.size);  // the page in which the shared part ends, if inside
    const int edge_page = a.shared > edge * a.g.size && a.from < a.shared ? a.prefix[edge] : -1;
    const float sl = a.scale_log2;
    // as many places at a time as the list of page numbers covers
    const int most = (kStList - 1) * a.g.size / kStKeys * kStKeys;
    for (int s0 = lo; s0 < hi; s0 += most) {
        const int s1 = min(hi, s0 + most), page0 = fdiv(s0, a.size), pages = fdiv(s1 - 1, a.size) + 1 - page0;
        __syncthreads();
        // pages of shared places alone come from the prefix; a table row is
        // only there if places behind the shared ones are wanted
        for (int i = tid; i < pages; i += kStThreads)
            list[i] = page0 + i < edge && a.from < a.shared ? a.prefix[page0 + i] : s1 > a.shared ? row[page0 + i] : -1;
        __syncthreads();
        const int n = (s1 - s0 + kStKeys - 1) / kStKeys;
        auto load = [&](int tile) {
            char *dst = smem + (tile % kStStages) * 2 * Sm::kTile;
            const int c = tid % kChunks;
#pragma unroll
            for (int r = tid / kChunks; r < kStKeys; r += kStThreads / kChunks) {
                const int place = s0 + tile * kStKeys + r;
                bool real = place < s1 && c * 8 < a.d;
                long long at = 0;
                if (real) {
                    const int i = fdiv(place, a.size);
                    const int page = i == edge && place < a.shared && a.from < a.shared ? edge_page : list[i - page0];
                    real = page >= 0 && page < a.g.pages;
                    if (real) at = page * a.g.ps + (place - i * a.g.size) * a.g.ts + kvh * a.g.hs + c * 8;
                }
                const uint32_t to = smem_u32(dst) + r * DK * 2 + ((c ^ (r & 7)) << 4);
                cp_async16(to, a.k + at, real);
                cp_async16(to + Sm::kTile, a.v + at, real);
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < kStStages - 1; i++) {
            if (i < n) load(i);
            else cp_async_commit();
        }
        for (int tile = 0; tile < n; tile++) {
            cp_async_wait<kStStages - 2>();
            __syncthreads();
            if (tile + kStStages - 1 < n) load(tile + kStStages - 1);
            else cp_async_commit();
            const uint32_t kt = smem_u32(smem + (tile % kStStages) * 2 * Sm::kTile), vt = kt + Sm::kTile;
            const int key0 = warp * 16;
            float s[2][4] = {};
#pragma unroll
            for (int k = 0; k < DK / 16; k++) {
                uint32_t kb[4];
                const int r = key0 + (lane & 7) + (lane >> 4) * 8, c = k * 2 + (lane >> 3 & 1);
                ldmatrix4(kt + r * DK * 2 + ((c ^ (r & 7)) << 4), kb);
                mma16816<T>(s[0], qa[k], kb[0], kb[1]);
                mma16816<T>(s[1], qa[k], kb[2], kb[3]);
            }
            // places behind the last one carry no weight
            const int here = s1 - (s0 + tile * kStKeys + key0);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i * 8 + (lane & 3) * 2 + (j & 1) >= here) s[i][j] = -INFINITY;
            uint32_t p[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {  // rows lane / 4 and lane / 4 + 8
                float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, m[h]);
                const float f = top == m[h] ? 1.f : ex2((m[h] - top) * sl);
                m[h] = top;
                const float off = top == -INFINITY ? 0.f : -top * sl;
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) e[i] = ex2(fmaf(s[i >> 1][2 * h + (i & 1)], sl, off));
                l[h] = fmaf(l[h], f, (e[0] + e[1]) + (e[2] + e[3]));
                p[h] = pack2<T>(e[0], e[1]);
                p[h + 2] = pack2<T>(e[2], e[3]);
#pragma unroll
                for (int i = 0; i < DK / 8; i++) {
                    o[i][2 * h] *= f;
                    o[i][2 * h + 1] *= f;
                }
            }
#pragma unroll
            for (int i = 0; i < DK / 16; i++) {
                uint32_t vb[4];
                const int r = key0 + (lane & 7) + (lane >> 3 & 1) * 8, c = i * 2 + (lane >> 4);
                ldmatrix4_t(vt + r * DK * 2 + ((c ^ (r & 7)) << 4), vb);
                mma16816<T>(o[2 * i], p, vb[0], vb[1]);
                mma16816<T>(o[2 * i + 1], p, vb[2], vb[3]);
            }
        }
        cp_async_wait<0>();
    }

    // ---- the four warps' results become the block's, in log2 units
    __syncthreads();
    {
        float *wo = (float *)(smem + warp * Sm::kO);
        const int r = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3) == 0) {
                warp_m[warp][r + 8 * h] = m[h] * sl;
                warp_l[warp][r + 8 * h] = l[h];
            }
#pragma unroll
            for (int i = 0; i < DK / 8; i++)
                *(float2 *)(wo + (r + 8 * h) * DK + i * 8 + c) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        }
    }
    __syncthreads();
    for (int e = tid; e < heads * (DK / 4); e += kStThreads) {
        const int r = e / (DK / 4), c = e % (DK / 4);
        const float top = fmaxf(fmaxf(warp_m[0][r], warp_m[1][r]), fmaxf(warp_m[2][r], warp_m[3][r]));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = warp_m[w][r] == -INFINITY && warp_l[w][r] == 0.f ? 0.f : ex2(warp_m[w][r] - top);
            add_scaled(x, f, ((const float4 *)(smem + w * Sm::kO))[r * (DK / 4) + c]);
            sum = fmaf(f, warp_l[w][r], sum);
        }
        ((float4 *)block_o)[r * (DK / 4) + c] = x;
        if (c == 0) {
            block_m[r] = top;
            block_l[r] = sum;
        }
    }
    // the shared part's launch may still run: its results from here on
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    // ---- a row's partial results: the cluster's blocks, then the shared
    // part's pieces.  Their weights first, a warp per row.
    const long long rows = (long long)a.batch * a.hq, prow0 = (long long)b * a.hq + kvh * a.group + row0;
    const int parts = ranks + a.splits;
    float *const weight = (float *)smem;  // [row][part], over the ring
    for (int r = warp; r < heads; r += 4) {
        float top = -INFINITY;
        for (int i = lane; i < parts; i += 32) {
            float w;
            if (i < ranks) {
                w = *cluster.map_shared_rank(&block_m[r], i);
                if (w == -INFINITY && *cluster.map_shared_rank(&block_l[r], i) != 0.f) w = __int_as_float(0x7fffffff);
            } else w = a.part_lse[(i - ranks) * rows + prow0 + r];
            weight[r * parts + i] = w;
            top = fmaxf(top, w);
        }
        top = warp_max(top);
        float sum = 0.f;
        for (int i = lane; i < parts; i += 32) {
            // nothing seen: no weight
            const float w = weight[r * parts + i], f = w == -INFINITY ? 0.f : ex2(w - top);
            weight[r * parts + i] = f;
            sum += i < ranks ? f * *cluster.map_shared_rank(&block_l[r], i) : f;
        }
        sum = warp_sum(sum);
        if (lane == 0) warp_l[0][r] = len > 0 ? 1.f / sum : 0.f;
    }
    __syncthreads();
    // the cluster's blocks take turns at the elements
    const int quads = a.d / 4;
    for (int e = rank * kStThreads + tid; e < heads * quads; e += ranks * kStThreads) {
        const int r = e / quads, c = e % quads;
        const float *w = weight + r * parts;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < ranks; i++) add_scaled(x, w[i], ((const float4 *)cluster.map_shared_rank(block_o, i))[r * (DK / 4) + c]);
        const float4 *o = (const float4 *)(a.part_o + (prow0 + r) * a.d) + c;
#pragma unroll 8
        for (int i = 0; i < a.splits; i++) add_scaled(x, w[ranks + i], o[i * rows * quads]);
        const float f = warp_l[0][r];
        T *dst = a.o.at(b, kvh * a.group + row0 + r) + 4 * c;
        dst[0] = from_f32<T>(len > 0 ? x.x * f : 0.f);
        dst[1] = from_f32<T>(len > 0 ? x.y * f : 0.f);
        dst[2] = from_f32<T>(len > 0 ? x.z * f : 0.f);
        dst[3] = from_f32<T>(len > 0 ? x.w * f : 0.f);
    }
    if (ranks > 1) cluster.sync();  // a block's results stay until the others have read them
}

// Largest number of blocks that share one stream's places.
constexpr int kStMostPieces = 8;

template <typename T, int DK>
static cudaError_t step_launch(const StepArgs<T> &a, int pieces, bool behind_shared, cudaStream_t s)
{
    auto *fn = &prefix_step_kernel<T, DK>;
    cudaError_t e = ensure_smem_attr((const void *)fn, StepSmem<DK>::kBytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.batch * pieces), (unsigned)a.hk, (unsigned)((a.group + 15) / 16));
    cfg.blockDim = dim3(kStThreads);
    cfg.dynamicSmemBytes = StepSmem<DK>::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)pieces;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    // may begin while the shared part's last blocks run (griddepcontrol.wait)
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = behind_shared ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fn, a);
}

}  // namespace aie
