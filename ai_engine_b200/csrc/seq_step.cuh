// One query token for each of a batch of streams over the places of its own
// (16-bit operands), joined with the shared prefix's partial results.
//
//   S = Q K^T for the query heads that read one key/value head,
//   m, l, O carried along; at the end every partial result (m_i, l_i, O_i)
//   has weight 2^(m_i - m):  out = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i
//
// Each place is read once and used for a group of query heads: memory-bound.
// A block goes through (stream, key/value head) pairs.  One warp copies tiles
// of 64 places into a ring of shared memory (TMA, a box per page or part of
// one) and runs ahead into the next pair; four warps multiply 16 of the 64
// places each (m16n8k16, the group padded to 16 rows) and carry their own m, l
// and O.  Where streams are few, the places of one stream are split over a
// cluster of up to 8 blocks, whose results meet in distributed shared memory.
// Fixed order throughout: results repeat bit for bit.
//
// A stream that ends inside the shared part has no places of its own.  The
// shared part multiplies its weights of 0 with values that it does not see, and
// 0 times a value that is not finite is NaN.  Only then its places are gone
// through here too, and the shared part's results left out.
//
// Rounding to fewer bits: the weights to the operands' type for the product
// with V (l sums them unrounded; f16 weights 2^7 times as large, as in
// attn_tc_kernel), and the result.
#pragma once
#include <cooperative_groups.h>

#include "seq_attn.cuh"

namespace aie {

constexpr int kStKeys = 64;        // places of one ring stage
constexpr int kStThreads = 160;    // four warps that multiply, one that copies
constexpr int kStMostPieces = 8;   // largest number of blocks that share one stream's places
constexpr int kStMostStages = 3;
constexpr uint32_t kStErr = 0x42000000u;

template <typename T>
struct StepArgs {
    HeadsOf<T> q, o;
    FastDiv size;
    const int32_t *prefix, *table, *lens;
    const float *part_o, *part_lse;  // the shared part's results, `splits` of them
    int batch, hq, hk, group, d, from, max_len, table_stride, splits;
    int pages, page_size, box_rows;  // places of one box: the greatest common divisor of a page's and a tile's
    int units, zs, rows;             // (stream, key head, 16 heads of the group) triples; rows kept: min(group, 16)
    int ends_in, split_places;       // streams shorter than this end in the shared part; places of one of its pieces
    int stages;
    int q_pairs;                     // two elements of q are 4-byte aligned
    float scale_log2;
};

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
    static constexpr uint32_t kBlock = kStKeys * 128;             // 64 places of 64 elements
    static constexpr uint32_t kTile = DK / 64 * kBlock;           // K or V of a stage
    static constexpr uint32_t kStage = 2 * kTile;
    // the warps' results, then the weights of `parts` partial results per row
    static uint32_t bytes(int stages, int rows, int parts) { return stages * kStage + 4 * rows * DK * 4 + rows * parts * 4 + 1024; }
};

struct StepShared {
    uint64_t full[kStMostStages], empty[kStMostStages];
    float warp_m[4][16], warp_l[4][16], block_m[16], block_l[16], inv[16];
    uint32_t abort;
};

__device__ __forceinline__ void step_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the four multiplying warps

template <typename T, int DK>
__global__ void __launch_bounds__(kStThreads)
prefix_step_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const StepArgs<T> a)
{
    namespace cg = cooperative_groups;
    using Sm = StepSmem<DK>;
    extern __shared__ char smem_raw[];
    __shared__ StepShared sh;
    char *const smem = (char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float *const result = (float *)(smem + a.stages * Sm::kStage);  // [warp][row][DK]; the first becomes the block's
    float *const weight = result + 4 * a.rows * DK;                 // [row][part]
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // behind the shared part's launch, which has waited for the inputs, only its
    // results have to be waited for, below
    if (!a.splits) behind_last_launch();
    if (tid == 0) {
        for (int i = 0; i < a.stages; i++) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 4);
        }
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    volatile uint32_t *abort = &sh.abort;
    auto wait = [&](uint64_t *bar, uint32_t parity, uint32_t site) {
        if (mbar_wait(bar, parity)) return true;
        report_error(kStErr | site);
        *abort = 1;
        return false;
    };
    // a unit's tiles of 64 places, this block's part of them, and the first place:
    // a.from, or 0 for a stream whose shared part is worked out anew
    auto tiles_of = [&](int b, int head0, int heads, int &len, int &from, int &lo, int &hi) {
        len = min(max(a.lens[b], 0), a.max_len);
        from = a.from;
        if (__builtin_expect(len > 0 && len < a.ends_in, 0)) {
            // the shared part's word on the piece that the stream ends in
            asm volatile("griddepcontrol.wait;" ::: "memory");
            const long long row = ((long long)((len - 1) / a.split_places) * a.batch + b) * a.hq + head0 + lane;
            if (__any_sync(0xffffffffu, lane < heads && isnan(a.part_lse[row]))) from = 0;
        }
        const int first = from / kStKeys, end = len > from ? (len - 1) / kStKeys + 1 : first;
        const int per = (end - first + ranks - 1) / ranks;
        lo = min(first + rank * per, end);
        hi = min(lo + per, end);
    };
    int ring = 0;  // tiles so far, over all units
    bool ok = true;

    if (warp == 4) {
        // ---- copies; each lane one box of a tile
        const int boxes = kStKeys / a.box_rows;
        for (int u = blockIdx.x / ranks; u < a.units; u += gridDim.x / ranks) {
            // the multiplying warps hold the first pair's result back until the shared
            // part is done, however long that takes: no bounded wait runs meanwhile
            if (u != blockIdx.x / ranks && a.splits) asm volatile("griddepcontrol.wait;" ::: "memory");
            const int b = u / (a.hk * a.zs), kvh = u / a.zs % a.hk, row0 = u % a.zs * 16;
            int len, from, lo, hi;
            tiles_of(b, kvh * a.group + row0, min(a.group - row0, 16), len, from, lo, hi);
            const int32_t *row = from < a.from ? a.prefix : a.table + (long long)b * a.table_stride;
            auto page_of = [&](int tile) {
                const int place = tile * kStKeys + lane * a.box_rows;
                // outside the stream's places, or no page of the cache: one that does not exist, read as zeros
                const int page = lane < boxes && place < len && place + a.box_rows > from ? row[fdiv(place, a.size)] : a.pages;
                return page < 0 || page > a.pages ? a.pages : page;
            };
            int next = lo < hi ? page_of(lo) : 0;
            for (int tile = lo; tile < hi && ok; tile++, ring++) {
                const int page = next, st = ring % a.stages, round = ring / a.stages;
                if (tile + 1 < hi) next = page_of(tile + 1);
                int go = 1;
                if (lane == 0) {
                    go = !*abort && (!round || wait(&sh.empty[st], (round - 1) & 1, 1));
                    if (go) mbar_expect_tx(&sh.full[st], Sm::kStage);
                }
                ok = __shfl_sync(0xffffffffu, go, 0);
                if (ok && lane < boxes) {
                    const int place = tile * kStKeys + lane * a.box_rows, at = place - fdiv(place, a.size) * a.page_size;
                    char *dst = smem + st * Sm::kStage + lane * a.box_rows * 128;
#pragma unroll
                    for (int i = 0; i < DK / 64; i++) {
                        tma_load_4d(dst + i * Sm::kBlock, &tm_k, &sh.full[st], i * 64, kvh, at, page);
                        tma_load_4d(dst + Sm::kTile + i * Sm::kBlock, &tm_v, &sh.full[st], i * 64, kvh, at, page);
                    }
                }
            }
            if (ranks > 1) {
                cluster.sync();
                cluster.sync();
            }
        }
        // nothing may still be written to this block's memory when it ends
        if (!ok && lane == 0)
            for (int i = max(ring - a.stages, 0); i < ring; i++) mbar_wait(&sh.full[i % a.stages], (i / a.stages) & 1);
        __syncwarp();
        return;
    }

    // ---- products
    const float sl = a.scale_log2;
    bool first_unit = true;
    for (int u = blockIdx.x / ranks; u < a.units; u += gridDim.x / ranks) {
        const int b = u / (a.hk * a.zs), kvh = u / a.zs % a.hk, row0 = u % a.zs * 16, heads = min(a.group - row0, 16);
        int len, from, lo, hi;
        tiles_of(b, kvh * a.group + row0, heads, len, from, lo, hi);
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

        for (int tile = lo; tile < hi; tile++, ring++) {
            const int st = ring % a.stages;
            ok = ok && __all_sync(0xffffffffu, wait(&sh.full[st], (ring / a.stages) & 1, 2));
            if (!ok) continue;
            const uint32_t kt = smem_u32(smem + st * Sm::kStage), vt = kt + Sm::kTile;
            const int key0 = warp * 16, place0 = tile * kStKeys + key0;
            const int skip = from - place0, here = len - place0;  // of this warp's 16 places: skip .. here - 1 count
            if (skip < 16 && here > 0) {
                const bool edge = skip > 0 || here < 16;
                if (edge) {
                    // values of other places may be anything, and 0 times them NaN: zeros
                    for (int i = lane; i < 16 * 8; i += 32)
                        if (i / 8 < skip || i / 8 >= here)
#pragma unroll
                            for (int k = 0; k < DK / 64; k++)
                                *(uint4 *)(smem + st * Sm::kStage + Sm::kTile + k * Sm::kBlock + (key0 * 8 + i) * 16) =
                                    make_uint4(0, 0, 0, 0);
                    __syncwarp();
                }
                float s[2][4] = {};
#pragma unroll
                for (int k = 0; k < DK / 16; k++) {
                    uint32_t kb[4];
                    const int r = key0 + (lane & 7) + (lane >> 4) * 8, c = (k & 3) * 2 + (lane >> 3 & 1);
                    ldmatrix4(kt + (k >> 2) * Sm::kBlock + r * 128 + ((c ^ (r & 7)) << 4), kb);
                    mma16816<T>(s[0], qa[k], kb[0], kb[1]);
                    mma16816<T>(s[1], qa[k], kb[2], kb[3]);
                }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int key = i * 8 + (lane & 3) * 2 + (j & 1);
                            if (key < skip || key >= here) s[i][j] = -INFINITY;
                        }
                }
                uint32_t p[4];
                float top[2];
                bool grow = false;
#pragma unroll
                for (int h = 0; h < 2; h++) {  // rows lane / 4 and lane / 4 + 8
                    float x = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    top[h] = fmaxf(x, m[h]);
                    grow |= (top[h] - m[h]) * sl > 8.f;  // as in attn_tc_kernel: smaller steps leave m
                }
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float f = top[h] == m[h] ? 1.f : ex2((m[h] - top[h]) * sl);
                        m[h] = top[h];
                        l[h] *= f;
#pragma unroll
                        for (int i = 0; i < DK / 8; i++) {
                            o[i][2 * h] *= f;
                            o[i][2 * h + 1] *= f;
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float off = m[h] == -INFINITY ? 0.f : fmaf(-m[h], sl, kWeightShift<T>);
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) e[i] = ex2(fmaf(s[i >> 1][2 * h + (i & 1)], sl, off));
                    l[h] += (e[0] + e[1]) + (e[2] + e[3]);
                    p[h] = pack2<T>(e[0], e[1]);
                    p[h + 2] = pack2<T>(e[2], e[3]);
                }
#pragma unroll
                for (int i = 0; i < DK / 16; i++) {
                    uint32_t vb[4];
                    const int r = key0 + (lane & 7) + (lane >> 3 & 1) * 8, c = (i & 3) * 2 + (lane >> 4);
                    ldmatrix4_t(vt + (i >> 2) * Sm::kBlock + r * 128 + ((c ^ (r & 7)) << 4), vb);
                    mma16816<T>(o[2 * i], p, vb[0], vb[1]);
                    mma16816<T>(o[2 * i + 1], p, vb[2], vb[3]);
                }
                if (edge) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the zeros before the next copy
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[st]);
        }

        // ---- the four warps' results become the block's, in log2 units: m less
        // the weights' shift, so that 2^m l is the sum
        step_sync();  // the last unit's are read
        {
            float *wo = result + warp * a.rows * DK;
            const int r = lane >> 2, c = (lane & 3) * 2;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                if (r + 8 * h < heads) {
                    if ((lane & 3) == 0) {
                        sh.warp_m[warp][r + 8 * h] = fmaf(m[h], sl, -kWeightShift<T>);
                        sh.warp_l[warp][r + 8 * h] = l[h];
                    }
#pragma unroll
                    for (int i = 0; i < DK / 8; i++)
                        *(float2 *)(wo + (r + 8 * h) * DK + i * 8 + c) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
                }
            }
        }
        step_sync();
        for (int e = tid; e < heads * (DK / 4); e += 128) {
            const int r = e / (DK / 4);
            const float top = fmaxf(fmaxf(sh.warp_m[0][r], sh.warp_m[1][r]), fmaxf(sh.warp_m[2][r], sh.warp_m[3][r]));
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = sh.warp_m[w][r] == -INFINITY && sh.warp_l[w][r] == 0.f ? 0.f : ex2(sh.warp_m[w][r] - top);
                add_scaled(x, f, ((const float4 *)(result + w * a.rows * DK))[e]);
                sum = fmaf(f, sh.warp_l[w][r], sum);
            }
            ((float4 *)result)[e] = x;
            if (e % (DK / 4) == 0) {
                sh.block_m[r] = top;
                sh.block_l[r] = sum;
            }
        }
        // the shared part's launch may still run: its results from here on
        if (first_unit && a.splits) behind_last_launch();
        first_unit = false;
        if (ranks > 1) cluster.sync();
        else step_sync();
        // ---- a row's partial results: the cluster's blocks, then the shared
        // part's pieces.  Their weights first, a warp per row.
        const long long rows = (long long)a.batch * a.hq, prow0 = (long long)b * a.hq + kvh * a.group + row0;
        const int splits = from < a.from ? 0 : a.splits, parts = ranks + splits;
        for (int r = warp; r < heads; r += 4) {
            float top = -INFINITY;
            for (int i = lane; i < parts; i += 32) {
                float w;
                if (i < ranks) {
                    w = *cluster.map_shared_rank(&sh.block_m[r], i);
                    if (w == -INFINITY && *cluster.map_shared_rank(&sh.block_l[r], i) != 0.f) w = __int_as_float(0x7fffffff);
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
                sum += i < ranks ? f * *cluster.map_shared_rank(&sh.block_l[r], i) : f;
            }
            sum = warp_sum(sum);
            if (lane == 0) sh.inv[r] = 1.f / sum;
        }
        step_sync();
        // the cluster's blocks take turns at the elements
        const int quads = a.d / 4;
        for (int e = rank * 128 + tid; e < heads * quads; e += ranks * 128) {
            const int r = e / quads, c = e % quads;
            const float *w = weight + r * parts;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < ranks; i++) add_scaled(x, w[i], ((const float4 *)cluster.map_shared_rank(result, i))[r * (DK / 4) + c]);
            const float4 *po = (const float4 *)(a.part_o + (prow0 + r) * a.d) + c;
#pragma unroll 8
            for (int i = 0; i < splits; i++) add_scaled(x, w[ranks + i], po[i * rows * quads]);
            const float f = sh.inv[r];
            T *dst = a.o.at(b, kvh * a.group + row0 + r) + 4 * c;
            dst[0] = from_f32<T>(len > 0 ? x.x * f : 0.f);
            dst[1] = from_f32<T>(len > 0 ? x.y * f : 0.f);
            dst[2] = from_f32<T>(len > 0 ? x.z * f : 0.f);
            dst[3] = from_f32<T>(len > 0 ? x.w * f : 0.f);
        }
        if (ranks > 1) cluster.sync();  // a block's results stay until the others have read them
    }
}

template <typename T, int DK>
static cudaError_t step_launch(const CUtensorMap &k, const CUtensorMap &v, StepArgs<T> a, int pieces, cudaStream_t s)
{
    auto *fn = &prefix_step_kernel<T, DK>;
    // the deepest ring with which two blocks fit an SM
    const int parts = pieces + a.splits;
    a.stages = kStMostStages;
    while (a.stages > 2 && StepSmem<DK>::bytes(a.stages, a.rows, parts) + sizeof(StepShared) + 1024 > 228 * 1024 / 2) a.stages--;
    cudaError_t e = ensure_smem_attr((const void *)fn, StepSmem<DK>::bytes(kStMostStages, 16, kStMostPieces + kAtMostSplits));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min(a.units, std::max(1, 2 * tc_sm_count() / pieces)) * pieces));
    cfg.blockDim = dim3(kStThreads);
    cfg.dynamicSmemBytes = StepSmem<DK>::bytes(a.stages, a.rows, parts);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)pieces;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    // may begin while the last launch's blocks run (behind_last_launch)
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, fn, k, v, a);
}

}  // namespace aie
