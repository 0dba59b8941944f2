// C ABI of the sequence operators (declared in include/aie_seq.h): argument
// checks and launches.  The kernels are in the seq_*.cuh files.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <numeric>
#include <utility>
#include <vector>

#include "host.cuh"
#include "tc_ptx.cuh"
#include "seq_common.cuh"
#include "seq_attn.cuh"
#include "seq_kv4.cuh"
#include "seq_pages.cuh"
#include "seq_read.cuh"
#include "seq_rope.cuh"
#include "seq_rows.cuh"
#include "seq_step.cuh"

using namespace aie;

// the sizes that C callers and _lib.py's packed layouts go by
static_assert(sizeof(aie_qk_rope) == 248 && sizeof(aie_prompt) == 136 && sizeof(aie_prefix) == 176 &&
                  sizeof(aie_pages) == 80 && sizeof(aie_cross) == 160 && sizeof(aie_kv4_rows) == 104 && sizeof(aie_kv4_step) == 144,
              "argument layouts");

cudaError_t aie::seq_take_device_error(uint32_t *code)
{
    uint32_t zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(code, g_aie_error, sizeof *code);
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_aie_error, &zero, sizeof zero);
    return e;
}

extern "C" int aie_seq_selftest_wait_timeout(uint32_t timeout_us, void *stream)
{
    if (timeout_us == 0 || timeout_us > 2000000) return fail(AIE_E_INVALID, "timeout must be 1..2000000 us");
    selftest_wait_kernel<<<1, 32, 0, (cudaStream_t)stream>>>((unsigned long long)timeout_us * 1000ull, kSeqSelftestCode);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AIE_OK : cuda_fail(e, "selftest launch");
}

// ------------------------------------------------------------- checks ---

static int launched(cudaError_t e, const char *what)
{
    return e == cudaSuccess ? AIE_OK : cuda_fail(e, what);
}

static int check_dtype(int32_t dt)
{
    if (dt < AIE_DT_F32 || dt > AIE_DT_BF16) return fail(AIE_E_INVALID, "unknown dtype %d", dt);
    return AIE_OK;
}

static int check_group(uint32_t hq, uint32_t hk, uint32_t d, uint32_t most)
{
    if (!hk || !hq || hq % hk) return fail(AIE_E_INVALID, "%u query heads over %u key heads", hq, hk);
    if (hq > 4096) return fail(AIE_E_UNSUPPORTED, "%u query heads: at most 4096", hq);
    if (!d) return fail(AIE_E_INVALID, "head_dim is 0");
    if (d > most) return fail(AIE_E_UNSUPPORTED, "head_dim %u: at most %u", d, most);
    return AIE_OK;
}

static uint32_t dtype_size(int32_t dt) { return dt == AIE_DT_F32 ? 4 : 2; }

static int check_heads(const aie_heads &h, int32_t dt, const char *what)
{
    if (!h.data) return fail(AIE_E_INVALID, "%s is NULL", what);
    if ((uintptr_t)h.data % dtype_size(dt)) return fail(AIE_E_ALIGN, "%s is not aligned to its elements", what);
    if (h.token_stride < 0 || h.head_stride < 0) return fail(AIE_E_INVALID, "%s has a negative stride", what);
    return AIE_OK;
}

static int check_pages(const aie_kv_pages &p, int32_t dt)
{
    if (!p.k || !p.v) return fail(AIE_E_INVALID, "the cache's k or v is NULL");
    if ((uintptr_t)p.k % dtype_size(dt) || (uintptr_t)p.v % dtype_size(dt))
        return fail(AIE_E_ALIGN, "the cache is not aligned to its elements");
    if (!p.pages || !p.page_size || p.pages > 0x7fffffffu || p.page_size > 65536)
        return fail(AIE_E_INVALID, "a cache of %u pages of %u places", p.pages, p.page_size);
    if (p.page_stride < 0 || p.token_stride < 0 || p.head_stride < 0)
        return fail(AIE_E_INVALID, "the cache has a negative stride");
    return AIE_OK;
}

#define TRY(call)             \
    do {                      \
        int st_ = (call);     \
        if (st_) return st_;  \
    } while (0)

// ------------------------------------------------------ norm, rotation ---

template <typename T>
static int qk_norm_rope(const aie_qk_rope &p, const uint8_t *pair_axis, uint32_t axes, cudaStream_t s)
{
    RopeArgs<T> a;
    a.q = heads_of<T>(p.q); a.k = heads_of<T>(p.k); a.v = heads_of<T>(p.v);
    a.qo = heads_of<T>(p.q_out); a.ko = heads_of<T>(p.k_out);
    a.kp = (T *)p.pages.k; a.vp = (T *)p.pages.v;
    a.pg = pages_geom(p.pages);
    a.wq = p.q_weight; a.wk = p.k_weight; a.cs = p.cos_sin;
    a.pos = p.positions; a.slots = p.slots;
    a.tokens = (int)p.tokens; a.hq = p.q.data ? (int)p.q_heads : 0; a.hk = (int)p.kv_heads;
    a.d = (int)p.head_dim; a.rot = (int)p.rot_dim; a.max_pos = (int)p.max_pos; a.interleaved = p.interleaved != 0;
    a.eps = p.eps;
    a.axis = p.rot_dim ? pair_axis : nullptr; a.axes = (int)axes;
    return launched(rope_launch(a, s), "norm and rotation");
}

// pair_axis NULL: one position a token
static int qk_norm_rope(const aie_qk_rope *p, const uint8_t *pair_axis, uint32_t axes, void *stream)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    TRY(check_dtype(p->dtype));
    TRY(check_group(p->q_heads, p->kv_heads, p->head_dim, kRopeMaxDim));
    if (p->rot_dim > p->head_dim || p->rot_dim % 2)
        return fail(AIE_E_INVALID, "rot_dim %u of a head of %u", p->rot_dim, p->head_dim);
    if (p->tokens > 0x7fffffffu || p->max_pos > 0x7fffffffu) return fail(AIE_E_INVALID, "too many tokens or positions");
    if (!p->tokens) return AIE_OK;
    if (p->q.data || p->q_out.data) {
        TRY(check_heads(p->q, p->dtype, "q"));
        TRY(check_heads(p->q_out, p->dtype, "q_out"));
    }
    TRY(check_heads(p->k, p->dtype, "k"));
    if (p->k_out.data) TRY(check_heads(p->k_out, p->dtype, "k_out"));
    if (p->rot_dim && (!p->positions || !p->cos_sin)) return fail(AIE_E_INVALID, "a rotation needs positions and cos_sin");
    if (p->pages.k || p->pages.v) {
        TRY(check_pages(p->pages, p->dtype));
        TRY(check_heads(p->v, p->dtype, "v"));
        if (!p->slots) return fail(AIE_E_INVALID, "slots is NULL");
    } else if (!p->k_out.data) return fail(AIE_E_INVALID, "the keys have neither an output nor a cache");
    if ((uint64_t)p->tokens * (p->q_heads + 2 * p->kv_heads) > 0x1ffffffffull)
        return fail(AIE_E_UNSUPPORTED, "more than 2^33 heads in one call");
    cudaStream_t s = (cudaStream_t)stream;
    if (p->dtype == AIE_DT_F32) return qk_norm_rope<float>(*p, pair_axis, axes, s);
    return p->dtype == AIE_DT_F16 ? qk_norm_rope<__half>(*p, pair_axis, axes, s) : qk_norm_rope<__nv_bfloat16>(*p, pair_axis, axes, s);
}

extern "C" int aie_qk_norm_rope(const aie_qk_rope *p, void *stream) { return qk_norm_rope(p, nullptr, 1, stream); }

extern "C" int aie_qk_norm_rope_axes(const aie_qk_rope *p, const uint8_t *pair_axis, uint32_t axes, void *stream)
{
    if (!axes || axes > 255) return fail(AIE_E_INVALID, "%u axes: 1 to 255", axes);
    if (!pair_axis && p && p->rot_dim) return fail(AIE_E_INVALID, "pair_axis is NULL");
    return qk_norm_rope(p, pair_axis, axes, stream);
}

// ---------------------------------------------------- prompt attention ---

template <typename T>
static int prompt_rows(const aie_prompt &p, cudaStream_t s)
{
    PromptRows<T> a;
    a.q = heads_of<T>(p.q); a.k = heads_of<T>(p.k); a.v = heads_of<T>(p.v); a.o = heads_of<T>(p.out);
    a.cu = p.cu;
    a.tokens = (int)p.tokens; a.seqs = (int)p.seqs; a.hq = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads);
    a.d = (int)p.head_dim; a.causal = p.causal != 0;
    a.scale = p.scale;
    const long long rows = (long long)p.tokens * p.q_heads;
    return launched(launch_behind(prompt_rows_kernel<T>, (unsigned)((rows + 3) / 4), 128, 0, s, a), "prompt attention");
}

// Whether the tensor cores take these heads: 16-bit operands, a head of at
// most 128 elements in whole 16-byte pieces, a group of query heads that fits
// a tile, and a scale under which the largest product has the largest weight.
static bool attn_heads_ok(int32_t dtype, uint32_t hq, uint32_t hk, uint32_t d, float scale)
{
    return dtype != AIE_DT_F32 && d % 8 == 0 && d <= 128 && hq / hk <= kAtTile && scale >= 1e-30f && scale <= 1e30f;
}

template <typename T>
static cudaError_t attn_prompt_launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const AttnArgs &a,
                                      unsigned grid, cudaStream_t s)
{
    return a.d <= 64 ? attn_launch<T, 1, kAtPrompt>(q, k, v, a, grid, s) : attn_launch<T, 2, kAtPrompt>(q, k, v, a, grid, s);
}

// What 16-bit results are aligned to in every row.
static int out_bytes(const aie_heads &out, uint32_t head_dim)
{
    const uint64_t bits = (uintptr_t)out.data | 2 * out.token_stride | 2 * out.head_stride;
    return bits % 32 == 0 && head_dim % 16 == 0 ? 32 : bits % 16 == 0 ? 16 : 2;
}

static int prompt_tc(const aie_prompt &p, cudaStream_t s)
{
    AttnArgs a = {};
    a.cu = p.cu;
    a.out = p.out.data;
    a.out_ts = p.out.token_stride; a.out_hs = p.out.head_stride;
    a.tokens = (int)p.tokens; a.seqs = (int)p.seqs;
    a.kv_heads = (int)p.kv_heads; a.q_heads = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads);
    a.d = (int)p.head_dim; a.tokens_per_tile = kAtTile / a.group;
    a.causal = p.causal != 0;
    a.out_bytes = out_bytes(p.out, p.head_dim);
    a.scale_log2 = p.scale * 1.4426950408889634f;
    const bool bf16 = p.dtype == AIE_DT_BF16;
    CUtensorMap q, k, v;
    if (!attn_map(&q, bf16, p.q.data, p.head_dim, p.q_heads, p.q.head_stride, p.tokens, p.q.token_stride, 0, 0, a.group,
                  a.tokens_per_tile) ||
        !attn_map(&k, bf16, p.k.data, p.head_dim, p.kv_heads, p.k.head_stride, p.tokens, p.k.token_stride, 0, 0, 1, kAtTile) ||
        !attn_map(&v, bf16, p.v.data, p.head_dim, p.kv_heads, p.v.head_stride, p.tokens, p.v.token_stride, 0, 0, 1, kAtTile))
        return fail(AIE_E_CUDA, "cuTensorMapEncodeTiled failed");
    // no more pairs of tiles than whole ones, and one that is not whole per sequence
    const uint64_t pairs = p.tokens / (2 * a.tokens_per_tile) + std::min(p.seqs, p.tokens);
    const uint64_t grid = pairs * p.kv_heads;
    if (grid > 0x7fffffffull) return fail(AIE_E_UNSUPPORTED, "too many tiles");
    return launched(bf16 ? attn_prompt_launch<__nv_bfloat16>(q, k, v, a, (unsigned)grid, s)
                         : attn_prompt_launch<__half>(q, k, v, a, (unsigned)grid, s),
                    "prompt attention");
}

extern "C" int aie_prompt_attn(const aie_prompt *p, void *stream)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    TRY(check_dtype(p->dtype));
    TRY(check_group(p->q_heads, p->kv_heads, p->head_dim, kRowsMaxDim));
    if (p->tokens > 0x3fffffffu || p->seqs > 0x3fffffffu) return fail(AIE_E_INVALID, "too many tokens or sequences");
    if (!(p->scale == p->scale)) return fail(AIE_E_INVALID, "scale is NaN");
    if (!p->tokens || !p->seqs) return AIE_OK;
    if (!p->cu) return fail(AIE_E_INVALID, "cu is NULL");
    TRY(check_heads(p->q, p->dtype, "q"));
    TRY(check_heads(p->k, p->dtype, "k"));
    TRY(check_heads(p->v, p->dtype, "v"));
    TRY(check_heads(p->out, p->dtype, "out"));
    if ((uint64_t)p->tokens * p->q_heads > 0x1ffffffffull) return fail(AIE_E_UNSUPPORTED, "more than 2^33 query rows");
    cudaStream_t s = (cudaStream_t)stream;
    if (attn_heads_ok(p->dtype, p->q_heads, p->kv_heads, p->head_dim, p->scale) &&
        attn_addressable(p->q.data, p->q.token_stride, p->q.head_stride, p->tokens, p->q_heads) &&
        attn_addressable(p->k.data, p->k.token_stride, p->k.head_stride, p->tokens, p->kv_heads) &&
        attn_addressable(p->v.data, p->v.token_stride, p->v.head_stride, p->tokens, p->kv_heads))
        return prompt_tc(*p, s);
    if (p->dtype == AIE_DT_F32) return prompt_rows<float>(*p, s);
    return p->dtype == AIE_DT_F16 ? prompt_rows<__half>(*p, s) : prompt_rows<__nv_bfloat16>(*p, s);
}

// ---------------------------------------------------- prefix attention ---

static int check_prefix(const aie_prefix *p)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    TRY(check_dtype(p->dtype));
    TRY(check_group(p->q_heads, p->kv_heads, p->head_dim, kRowsMaxDim));
    if (p->batch > 65535) return fail(AIE_E_UNSUPPORTED, "%u streams: at most 65535", p->batch);
    if (p->max_len > 0x3fffffffu || p->prefix_len > 0x3fffffffu) return fail(AIE_E_INVALID, "too many places");
    if (!p->pages.page_size) return fail(AIE_E_INVALID, "page_size is 0");
    return AIE_OK;
}

// How a call is computed.  The shared part: over key tiles in `splits` pieces
// on the tensor cores, or (0) with the streams' own part.  That: `pieces`
// blocks per stream and key head, or (0) row by row.
struct PrefixPlan {
    int splits, tiles_per_split, row_pairs, pieces;
    uint64_t bytes;  // of the workspace
};

static PrefixPlan prefix_plan(const aie_prefix &p)
{
    PrefixPlan w = {};
    const uint32_t keys = std::min(p.prefix_len, p.max_len), size = p.pages.page_size;
    const uint64_t units = (uint64_t)p.batch * p.kv_heads * ((p.q_heads / p.kv_heads + 15) / 16);
    // pages of whole swizzle atoms: 8 places
    const bool heads_ok = units <= 0x3fffffffu && attn_heads_ok(p.dtype, p.q_heads, p.kv_heads, p.head_dim, p.scale) && size % 8 == 0 &&
                          attn_addressable(p.pages.k, p.pages.token_stride, p.pages.head_stride, size, p.kv_heads) &&
                          attn_addressable(p.pages.v, p.pages.page_stride, 8, p.pages.pages, 1);
    if (keys && p.batch && heads_ok &&
        attn_addressable(p.q.data, p.q.token_stride, p.q.head_stride, p.batch, p.q_heads)) {
        const int tiles = (int)((keys + kAtTile - 1) / kAtTile);
        const int tpt = kAtTile / (int)(p.q_heads / p.kv_heads);
        w.row_pairs = ((int)p.batch + 2 * tpt - 1) / (2 * tpt);
        // one block per SM at a time: the pieces (of whole tiles) that give the
        // shortest run, a block costing about three tiles besides its own
        const long long blocks = (long long)w.row_pairs * p.kv_heads, sms = tc_sm_count();
        long long best = 0;
        for (int want = 1; want <= std::min(tiles, kAtMostSplits); want++) {
            const int per = (tiles + want - 1) / want, splits = (tiles + per - 1) / per;
            const long long cost = (blocks * splits + sms - 1) / sms * (per + 3);
            if (!best || cost < best) {
                best = cost;
                w.splits = splits;
                w.tiles_per_split = per;
            }
        }
    }
    if (heads_ok && (w.splits || !keys)) {
        // up to two blocks per SM, each with four tiles of places or more
        const int places = (int)(p.max_len - keys);
        w.pieces = 1;
        while (w.pieces < kStMostPieces && 2 * w.pieces * units <= 2ull * tc_sm_count() && w.pieces * 4 * kStKeys < places) w.pieces *= 2;
    }
    const uint64_t rows = (uint64_t)p.batch * p.q_heads;
    w.bytes = w.splits * rows * (4 + 4 * (uint64_t)p.head_dim) + 64;
    return w;
}

// The partial results: their weights' sums at the front, then whole sectors.
static float *part_o(const aie_prefix &p, const PrefixPlan &w)
{
    const uintptr_t at = (uintptr_t)p.workspace + (uint64_t)w.splits * p.batch * p.q_heads * 4;
    return (float *)((at + 31) / 32 * 32);
}

extern "C" uint64_t aie_prefix_attn_workspace(const aie_prefix *p)
{
    return check_prefix(p) ? 0 : prefix_plan(*p).bytes;
}

template <typename T>
static cudaError_t attn_prefix_launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const AttnArgs &a,
                                      unsigned grid, cudaStream_t s)
{
    return a.d <= 64 ? attn_launch<T, 1, kAtPaged>(q, k, v, a, grid, s) : attn_launch<T, 2, kAtPaged>(q, k, v, a, grid, s);
}

// The cache's maps, for both parts: boxes inside one page, whole boxes to both
// kernels' tiles.
struct PageMaps {
    CUtensorMap k, v;
    int box_rows;
};

static int page_maps(const aie_prefix &p, PageMaps *m)
{
    const aie_kv_pages &g = p.pages;
    const bool bf16 = p.dtype == AIE_DT_BF16;
    static_assert(kAtTile % kStKeys == 0, "whole boxes to either tile");
    m->box_rows = std::gcd((int)g.page_size, kStKeys);
    if (!attn_map(&m->k, bf16, g.k, p.head_dim, p.kv_heads, g.head_stride, g.page_size, g.token_stride, g.pages, g.page_stride, 1,
                  m->box_rows) ||
        !attn_map(&m->v, bf16, g.v, p.head_dim, p.kv_heads, g.head_stride, g.page_size, g.token_stride, g.pages, g.page_stride, 1,
                  m->box_rows))
        return fail(AIE_E_CUDA, "cuTensorMapEncodeTiled failed");
    return AIE_OK;
}

static int prefix_tc(const aie_prefix &p, const PrefixPlan &w, const PageMaps &m, cudaStream_t s)
{
    AttnArgs a = {};
    a.prefix = p.prefix; a.lens = p.lens;
    a.part_lse = (float *)p.workspace;
    a.part_o = part_o(p, w);
    a.tokens = (int)p.batch;
    a.kv_heads = (int)p.kv_heads; a.q_heads = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads);
    a.d = (int)p.head_dim; a.tokens_per_tile = kAtTile / a.group;
    a.shared = (int)p.prefix_len; a.max_len = (int)p.max_len;
    a.page_size = (int)p.pages.page_size; a.pages = (int)p.pages.pages;
    a.splits = w.splits; a.tiles_per_split = w.tiles_per_split;
    a.scale_log2 = p.scale * 1.4426950408889634f;
    a.box_rows = m.box_rows;
    const bool bf16 = p.dtype == AIE_DT_BF16;
    CUtensorMap q;
    if (!attn_map(&q, bf16, p.q.data, p.head_dim, p.q_heads, p.q.head_stride, p.batch, p.q.token_stride, 0, 0, a.group,
                  a.tokens_per_tile))
        return fail(AIE_E_CUDA, "cuTensorMapEncodeTiled failed");
    const uint64_t grid = (uint64_t)w.row_pairs * p.kv_heads * w.splits;
    if (grid > 0x7fffffffull) return fail(AIE_E_UNSUPPORTED, "too many tiles");
    return launched(bf16 ? attn_prefix_launch<__nv_bfloat16>(q, m.k, m.v, a, (unsigned)grid, s)
                         : attn_prefix_launch<__half>(q, m.k, m.v, a, (unsigned)grid, s),
                    "prefix attention");
}

template <typename T>
static int prefix_rows(const aie_prefix &p, cudaStream_t s)
{
    PrefixRows<T> a;
    a.q = heads_of<T>(p.q); a.o = heads_of<T>(p.out);
    a.k = (const T *)p.pages.k; a.v = (const T *)p.pages.v;
    a.g = pages_geom(p.pages);
    a.prefix = p.prefix; a.table = p.table; a.lens = p.lens;
    a.batch = (int)p.batch; a.hq = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads); a.d = (int)p.head_dim;
    a.shared = (int)p.prefix_len; a.max_len = (int)p.max_len; a.table_stride = (int)p.table_stride;
    a.scale = p.scale;
    const long long rows = (long long)p.batch * p.q_heads;
    return launched(launch_behind(prefix_rows_kernel<T>, (unsigned)((rows + 3) / 4), 128, 0, s, a), "prefix attention");
}

template <typename T>
static int prefix_step(const aie_prefix &p, const PrefixPlan &w, const PageMaps &m, cudaStream_t s)
{
    const aie_kv_pages &g = p.pages;
    StepArgs<T> a = {};
    a.q = heads_of<T>(p.q); a.o = heads_of<T>(p.out);
    a.size = make_fastdiv((int)g.page_size);
    a.prefix = p.prefix; a.table = p.table; a.lens = p.lens;
    a.part_lse = (const float *)p.workspace;
    a.part_o = part_o(p, w);
    a.batch = (int)p.batch; a.hq = (int)p.q_heads; a.hk = (int)p.kv_heads; a.group = (int)(p.q_heads / p.kv_heads);
    a.d = (int)p.head_dim;
    a.from = (int)p.prefix_len;
    a.max_len = (int)p.max_len; a.table_stride = (int)p.table_stride; a.splits = w.splits;
    a.ends_in = w.splits ? std::min(a.from, a.max_len) : 0; a.split_places = w.tiles_per_split * kAtTile;
    a.pages = (int)g.pages; a.page_size = (int)g.page_size; a.box_rows = m.box_rows;
    a.zs = (a.group + 15) / 16; a.units = a.batch * a.hk * a.zs; a.rows = std::min(a.group, 16);
    a.q_pairs = (uintptr_t)p.q.data % 4 == 0 && p.q.token_stride % 2 == 0 && p.q.head_stride % 2 == 0;
    a.scale_log2 = p.scale * 1.4426950408889634f;
    return launched(a.d <= 64 ? step_launch<T, 64>(m.k, m.v, a, w.pieces, s) : step_launch<T, 128>(m.k, m.v, a, w.pieces, s),
                    "prefix attention");
}

extern "C" int aie_prefix_attn(const aie_prefix *p, void *stream)
{
    TRY(check_prefix(p));
    if (!(p->scale == p->scale)) return fail(AIE_E_INVALID, "scale is NaN");
    if (!p->batch) return AIE_OK;
    TRY(check_heads(p->q, p->dtype, "q"));
    TRY(check_heads(p->out, p->dtype, "out"));
    TRY(check_pages(p->pages, p->dtype));
    if (!p->lens) return fail(AIE_E_INVALID, "lens is NULL");
    if (p->prefix_len && !p->prefix) return fail(AIE_E_INVALID, "prefix is NULL");
    if (p->max_len > p->prefix_len) {
        if (!p->table) return fail(AIE_E_INVALID, "table is NULL");
        if ((uint64_t)p->table_stride * p->pages.page_size < p->max_len)
            return fail(AIE_E_INVALID, "rows of %u pages of %u do not hold max_len %u", p->table_stride,
                        p->pages.page_size, p->max_len);
    }
    const PrefixPlan w = prefix_plan(*p);
    if (p->workspace_bytes < w.bytes || !p->workspace || (uintptr_t)p->workspace % 16)
        return fail(AIE_E_INVALID, "workspace: %llu bytes, 16-byte aligned, are needed", (unsigned long long)w.bytes);
    cudaStream_t s = (cudaStream_t)stream;
    if (w.pieces) {
        PageMaps m;
        TRY(page_maps(*p, &m));
        if (w.splits) TRY(prefix_tc(*p, w, m, s));
        return p->dtype == AIE_DT_F16 ? prefix_step<__half>(*p, w, m, s) : prefix_step<__nv_bfloat16>(*p, w, m, s);
    }
    if (p->dtype == AIE_DT_F32) return prefix_rows<float>(*p, s);
    return p->dtype == AIE_DT_F16 ? prefix_rows<__half>(*p, s) : prefix_rows<__nv_bfloat16>(*p, s);
}

// ----------------------------------------------------- cross attention ---

static int check_cross(const aie_cross *p)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    TRY(check_dtype(p->dtype));
    TRY(check_group(p->q_heads, p->kv_heads, p->head_dim, kRowsMaxDim));
    if (p->tokens > 0x3fffffffu || p->keys > 0x3fffffffu || p->seqs > 0x3fffffffu)
        return fail(AIE_E_INVALID, "too many tokens, states or sequences");
    if (!p->cu_q && p->tokens != p->seqs) return fail(AIE_E_INVALID, "%u tokens of %u sequences without cu_q", p->tokens, p->seqs);
    if ((uint64_t)p->tokens * p->q_heads > 0x1ffffffffull) return fail(AIE_E_UNSUPPORTED, "more than 2^33 query rows");
    return AIE_OK;
}

// Whether one token of each sequence goes over the states in equal parts:
// 16-bit heads in whole 16-byte pieces.
static bool cross_read_ok(const aie_cross &p)
{
    auto ok = [](const aie_heads &h) { return (uintptr_t)h.data % 16 == 0 && h.token_stride % 8 == 0 && h.head_stride % 8 == 0; };
    return !p.cu_q && p.dtype != AIE_DT_F32 && p.head_dim % 8 == 0 && ok(p.k) && ok(p.v) &&
           (uint64_t)p.seqs * p.q_heads <= 0x7fffffffull;
}

// Whether packed tokens go over the states on the tensor cores.
static bool cross_tc_ok(const aie_cross &p)
{
    return p.keys && attn_heads_ok(p.dtype, p.q_heads, p.kv_heads, p.head_dim, p.scale) && p.cu_q &&
           attn_addressable(p.q.data, p.q.token_stride, p.q.head_stride, p.tokens, p.q_heads) &&
           attn_addressable(p.k.data, p.k.token_stride, p.k.head_stride, p.keys, p.kv_heads) &&
           attn_addressable(p.v.data, p.v.token_stride, p.v.head_stride, p.keys, p.kv_heads);
}

// No more pairs of tiles than whole ones, and one that is not whole per
// sequence.  Where they fill the SMs less than twice, their steps are cut.
struct CrossPlan {
    bool few;
    int capacity;
    uint64_t pairs, grid, rows, bytes;  // rows of a partial result
};

static CrossPlan cross_plan(const aie_cross &p)
{
    CrossPlan w = {};
    const uint32_t tpt = kAtTile / (p.q_heads / p.kv_heads), sms = (uint32_t)tc_sm_count();
    auto pairs = [&](uint32_t tokens) { return p.tokens / tokens + (uint64_t)std::min(p.seqs, p.tokens); };
    // no more tokens a sequence than a tile holds: pairs of the same rows
    w.few = p.tokens <= (uint64_t)tpt * p.seqs && pairs(tpt) * p.kv_heads < 2 * sms;
    w.pairs = pairs(w.few ? tpt : 2 * tpt);
    if (w.pairs * p.kv_heads < 2 * sms) w.capacity = (int)std::max(1u, sms / p.kv_heads);
    w.grid = (w.pairs + w.capacity) * p.kv_heads;
    w.rows = (w.few ? 1 : 2) * kAtTile;
    w.bytes = 64 + (w.capacity ? w.grid * w.rows * (p.head_dim + 1) * 4 : 0);
    return w;
}

extern "C" uint64_t aie_cross_attn_workspace(const aie_cross *p)
{
    if (check_cross(p)) return 0;
    if (cross_read_ok(*p)) return read_plan(false, p->seqs, p->keys, p->kv_heads, p->q_heads / p->kv_heads, p->head_dim).bytes;
    return cross_tc_ok(*p) ? cross_plan(*p).bytes : 64;
}

template <typename T>
static cudaError_t attn_cross_launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const AttnArgs &a,
                                     const CrossPlan &w, cudaStream_t s)
{
    const unsigned grid = (unsigned)w.grid, rows = (unsigned)(w.pairs * a.kv_heads * w.rows / kJoinRows);
    cudaError_t e;
    if (w.few) {
        e = a.d <= 64 ? attn_launch<T, 1, kAtFew>(q, k, v, a, grid, s) : attn_launch<T, 2, kAtFew>(q, k, v, a, grid, s);
        return e != cudaSuccess ? e : launch_behind(cross_join_kernel<T, true>, rows, 32 * kJoinRows, 0, s, a);
    }
    e = a.d <= 64 ? attn_launch<T, 1, kAtCross>(q, k, v, a, grid, s) : attn_launch<T, 2, kAtCross>(q, k, v, a, grid, s);
    return e != cudaSuccess || !a.capacity ? e : launch_behind(cross_join_kernel<T, false>, rows, 32 * kJoinRows, 0, s, a);
}

static int cross_tc(const aie_cross &p, cudaStream_t s)
{
    const CrossPlan w = cross_plan(p);
    if (w.grid > 0x7fffffffull) return fail(AIE_E_UNSUPPORTED, "too many tiles");
    AttnArgs a = {};
    a.cu = p.cu_q; a.cu_k = p.cu_k;
    a.out = p.out.data;
    a.out_ts = p.out.token_stride; a.out_hs = p.out.head_stride;
    char *ws = (char *)(((uintptr_t)p.workspace + 31) / 32 * 32);
    a.part_o = (float *)ws;
    a.part_lse = (float *)(ws + (w.capacity ? w.grid * w.rows * p.head_dim * 4 : 0));
    a.tokens = (int)p.tokens; a.seqs = (int)p.seqs; a.keys = (int)p.keys; a.capacity = w.capacity;
    a.splits = (int)(w.grid / p.kv_heads);
    a.kv_heads = (int)p.kv_heads; a.q_heads = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads);
    a.d = (int)p.head_dim; a.tokens_per_tile = kAtTile / a.group;
    a.pair_tokens = (w.few ? 1 : 2) * a.tokens_per_tile;
    a.out_bytes = out_bytes(p.out, p.head_dim);
    a.scale_log2 = p.scale * 1.4426950408889634f;
    const bool bf16 = p.dtype == AIE_DT_BF16;
    CUtensorMap q, k, v;
    if (!attn_map(&q, bf16, p.q.data, p.head_dim, p.q_heads, p.q.head_stride, p.tokens, p.q.token_stride, 0, 0, a.group,
                  a.tokens_per_tile) ||
        !attn_map(&k, bf16, p.k.data, p.head_dim, p.kv_heads, p.k.head_stride, p.keys, p.k.token_stride, 0, 0, 1, kCrossBox) ||
        !attn_map(&v, bf16, p.v.data, p.head_dim, p.kv_heads, p.v.head_stride, p.keys, p.v.token_stride, 0, 0, 1, kCrossBox))
        return fail(AIE_E_CUDA, "cuTensorMapEncodeTiled failed");
    return launched(bf16 ? attn_cross_launch<__nv_bfloat16>(q, k, v, a, w, s) : attn_cross_launch<__half>(q, k, v, a, w, s),
                    "cross attention");
}

static int cross_read(const aie_cross &p, cudaStream_t s)
{
    ReadArgs a = {};
    const ReadPlan w = read_plan(false, p.seqs, p.keys, p.kv_heads, p.q_heads / p.kv_heads, p.head_dim);
    if (w.tiles > 0x7fffffffull) return fail(AIE_E_UNSUPPORTED, "more than 2^35 (state, key head) pairs in one call");
    a.seqs = (int)p.seqs;
    read_args(a, w, p.q, p.out, p.workspace);
    a.k = p.k.data; a.k_ts = p.k.token_stride; a.k_hs = p.k.head_stride;
    a.v = p.v.data; a.v_ts = p.v.token_stride; a.v_hs = p.v.head_stride;
    a.cu = p.cu_k; a.keys = (int)p.keys;
    a.hq = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads); a.d = (int)p.head_dim;
    a.bf16 = p.dtype == AIE_DT_BF16; a.scale = p.scale;
    return launched(read16_run(a, w.nt, s), "cross attention");
}

// Rows a sequence from which tiles are worth it with heads of more than 128, where
// few blocks fit an SM (64 sequences over 2000 states, 8 heads of 256: a warp per row
// 2.1, 2.9 and 4.5 ms with 1, 2 and 4 rows, tiles 3.3); others always are (8 heads
// of 128, 1 row: 1.65 ms and 1.33; one sequence over 20000: 16.4 and 4.5).
constexpr int kTileLeast = 3;

template <typename T>
static int cross_rows(const aie_cross &p, cudaStream_t s)
{
    CrossRows<T> a;
    a.q = heads_of<T>(p.q); a.k = heads_of<T>(p.k); a.v = heads_of<T>(p.v); a.o = heads_of<T>(p.out);
    a.cu_q = p.cu_q; a.cu_k = p.cu_k;
    a.tokens = (int)p.tokens; a.keys = (int)p.keys; a.seqs = (int)p.seqs;
    a.hq = (int)p.q_heads; a.group = (int)(p.q_heads / p.kv_heads); a.d = (int)p.head_dim;
    a.scale = p.scale;
    const long long rows = (long long)p.tokens * p.q_heads;
    // tiles of rows, no more than whole ones and one that is not per sequence
    const uint64_t units = ((uint64_t)p.tokens * a.group / kTileRows + std::min(p.seqs, p.tokens)) * p.kv_heads;
    if ((p.head_dim <= 128 || (uint64_t)p.tokens * a.group >= (uint64_t)kTileLeast * p.seqs) && units <= 0x7fffffffull) {
        auto *fn = a.d <= 64 ? &cross_tile_kernel<T, 1> : a.d <= 128 ? &cross_tile_kernel<T, 2> : &cross_tile_kernel<T, 4>;
        const uint32_t smem = cross_tile_smem(a.d);
        cudaError_t e = ensure_smem_attr((const void *)fn, cross_tile_smem(a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256));
        if (e == cudaSuccess) e = launch_behind(fn, (unsigned)units, kTileThreads, smem, s, a, (int)p.kv_heads);
        return launched(e, "cross attention");
    }
    return launched(launch_behind(cross_rows_kernel<T>, (unsigned)((rows + 3) / 4), 128, 0, s, a), "cross attention");
}

extern "C" int aie_cross_attn(const aie_cross *p, void *stream)
{
    TRY(check_cross(p));
    if (!(p->scale == p->scale)) return fail(AIE_E_INVALID, "scale is NaN");
    if (!p->tokens || !p->seqs) return AIE_OK;
    if (!p->cu_k) return fail(AIE_E_INVALID, "cu_k is NULL");
    TRY(check_heads(p->q, p->dtype, "q"));
    TRY(check_heads(p->out, p->dtype, "out"));
    if (p->keys) {
        TRY(check_heads(p->k, p->dtype, "k"));
        TRY(check_heads(p->v, p->dtype, "v"));
    }
    const uint64_t need = aie_cross_attn_workspace(p);
    if (p->workspace_bytes < need || !p->workspace || (uintptr_t)p->workspace % 16)
        return fail(AIE_E_INVALID, "workspace: %llu bytes, 16-byte aligned, are needed", (unsigned long long)need);
    cudaStream_t s = (cudaStream_t)stream;
    if (cross_read_ok(*p)) return cross_read(*p, s);
    if (cross_tc_ok(*p)) return cross_tc(*p, s);
    if (p->dtype == AIE_DT_F32) return cross_rows<float>(*p, s);
    return p->dtype == AIE_DT_F16 ? cross_rows<__half>(*p, s) : cross_rows<__nv_bfloat16>(*p, s);
}

// ---------------------------------------------------------- 4-bit cache ---

static int check_kv4(const aie_kv4 &c)
{
    if (!c.k || !c.v) return fail(AIE_E_INVALID, "the cache's k or v is NULL");
    if (!c.head_dim || c.head_dim % 32) return fail(AIE_E_INVALID, "head_dim %u: a multiple of 32", c.head_dim);
    if (c.head_dim > 256) return fail(AIE_E_UNSUPPORTED, "head_dim %u: at most 256", c.head_dim);
    if (!c.kv_heads) return fail(AIE_E_INVALID, "no key heads");
    if (c.kv_heads > 4096) return fail(AIE_E_UNSUPPORTED, "%u key heads: at most 4096", c.kv_heads);
    if (!c.pages || !c.page_size || c.page_size % 8 || c.pages > 0x3fffffffu || c.page_size > 65536)
        return fail(AIE_E_INVALID, "a cache of %u pages of %u places (a multiple of 8)", c.pages, c.page_size);
    const int64_t page = (int64_t)c.kv_heads * c.page_size * c.head_dim * 5 / 8;
    if (c.page_stride < 0 || (c.pages > 1 && c.page_stride < page))
        return fail(AIE_E_INVALID, "page_stride %lld for pages of %lld bytes", (long long)c.page_stride, (long long)page);
    if ((uintptr_t)c.k % 16 || (uintptr_t)c.v % 16 || c.page_stride % 16)
        return fail(AIE_E_ALIGN, "the cache and its pages must be 16-byte aligned");
    return AIE_OK;
}

static int kv4_rows(const aie_kv4_rows *p, bool file, void *stream)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    TRY(check_dtype(p->dtype));
    TRY(check_kv4(p->cache));
    if (!p->tokens) return AIE_OK;
    TRY(check_heads(p->k, p->dtype, "k"));
    TRY(check_heads(p->v, p->dtype, "v"));
    if (!p->slots) return fail(AIE_E_INVALID, "slots is NULL");
    if ((uint64_t)p->tokens * p->cache.kv_heads * (p->cache.head_dim / 8) > 0x7fffff00ull)
        return fail(AIE_E_UNSUPPORTED, "more than 2^34 elements in one call");
    cudaStream_t s = (cudaStream_t)stream;
    const char *what = file ? "filing in 4 bits" : "reading 4 bits";
    if (p->dtype == AIE_DT_F32) return launched(kv4_rows_launch<float>(*p, file, s), what);
    return launched(p->dtype == AIE_DT_F16 ? kv4_rows_launch<__half>(*p, file, s) : kv4_rows_launch<__nv_bfloat16>(*p, file, s), what);
}

extern "C" int aie_kv4_file(const aie_kv4_rows *p, void *stream) { return kv4_rows(p, true, stream); }
extern "C" int aie_kv4_load(const aie_kv4_rows *p, void *stream) { return kv4_rows(p, false, stream); }

static int check_kv4_step(const aie_kv4_step *p)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    if (p->dtype != AIE_DT_F16 && p->dtype != AIE_DT_BF16) return fail(AIE_E_UNSUPPORTED, "dtype %d: f16 or bf16", p->dtype);
    TRY(check_kv4(p->cache));
    TRY(check_group(p->q_heads, p->cache.kv_heads, p->cache.head_dim, 256));
    if (p->batch > 65535) return fail(AIE_E_UNSUPPORTED, "%u streams: at most 65535", p->batch);
    if (p->max_len > 0x3fffffffu) return fail(AIE_E_INVALID, "too many places");
    return AIE_OK;
}

static ReadPlan kv4_plan(const aie_kv4_step &p)
{
    return read_plan(true, p.batch, (uint64_t)p.batch * p.max_len, p.cache.kv_heads, p.q_heads / p.cache.kv_heads, p.cache.head_dim);
}

extern "C" uint64_t aie_kv4_attn_workspace(const aie_kv4_step *p) { return check_kv4_step(p) ? 0 : kv4_plan(*p).bytes; }

static int kv4_step(const aie_kv4_step &p, cudaStream_t s)
{
    ReadArgs a = {};
    const ReadPlan w = kv4_plan(p);
    if (w.tiles > 0x7fffffffull) return fail(AIE_E_UNSUPPORTED, "more than 2^36 (place, key head) pairs in one call");
    a.seqs = (int)p.batch;
    read_args(a, w, p.q, p.out, p.workspace);
    a.g = kv4_geom(p.cache); a.size = make_fastdiv(a.g.size);
    a.table = p.table; a.lens = p.lens; a.max_len = (int)p.max_len; a.table_stride = (int)p.table_stride;
    a.hq = (int)p.q_heads; a.group = (int)(p.q_heads / p.cache.kv_heads); a.d = a.g.d;
    a.bf16 = p.dtype == AIE_DT_BF16; a.scale = p.scale;
    const cudaError_t e = a.bf16 ? read4_run_bf16(a, w.nt, s) : read4_run_f16(a, w.nt, s);
    return launched(e, "attention over 4 bits");
}

extern "C" int aie_kv4_attn(const aie_kv4_step *p, void *stream)
{
    TRY(check_kv4_step(p));
    if (!(p->scale == p->scale)) return fail(AIE_E_INVALID, "scale is NaN");
    if (!p->batch) return AIE_OK;
    TRY(check_heads(p->q, p->dtype, "q"));
    TRY(check_heads(p->out, p->dtype, "out"));
    if (!p->lens) return fail(AIE_E_INVALID, "lens is NULL");
    if (p->max_len) {
        if (!p->table) return fail(AIE_E_INVALID, "table is NULL");
        if ((uint64_t)p->table_stride * p->cache.page_size < p->max_len)
            return fail(AIE_E_INVALID, "rows of %u pages of %u do not hold max_len %u", p->table_stride, p->cache.page_size, p->max_len);
    }
    const uint64_t need = aie_kv4_attn_workspace(p);
    if (p->workspace_bytes < need || !p->workspace || (uintptr_t)p->workspace % 16)
        return fail(AIE_E_INVALID, "workspace: %llu bytes, 16-byte aligned, are needed", (unsigned long long)need);
    return kv4_step(*p, (cudaStream_t)stream);
}

// --------------------------------------------------------------- pages ---

constexpr uint32_t kPagesMaxRows = 1u << 18;  // the row bitmap: 32 KB of shared memory

static int pages_args(const aie_pages *p, bool rows, bool places, bool kv, PagesArgs *a)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    if (!p->pages || p->pages >= (uint32_t)kSumCap) return fail(AIE_E_INVALID, "a cache of %u pages", p->pages);
    if (kv) {
        if (!p->kv || !p->layers || !p->page_bytes) return fail(AIE_E_INVALID, "the cache is NULL or empty");
        if ((uintptr_t)p->kv % 16 || p->page_bytes % 16)
            return fail(AIE_E_ALIGN, "the cache and its pages must be 16-byte aligned (pages of %llu bytes)",
                        (unsigned long long)p->page_bytes);
    }
    if (rows) {
        if (!p->refs || !p->lens || !p->table || !p->status) return fail(AIE_E_INVALID, "a part of the state is NULL");
        if (!p->rows || !p->width) return fail(AIE_E_INVALID, "%u rows of %u pages", p->rows, p->width);
        if (p->rows > kPagesMaxRows) return fail(AIE_E_UNSUPPORTED, "%u rows: at most %u", p->rows, kPagesMaxRows);
        if (places && (!p->page_size || p->page_size > 65536)) return fail(AIE_E_INVALID, "pages of %u places", p->page_size);
        if (p->width > 0x3fffffffu || (uint64_t)p->width * p->page_size > 0x3fffffffu)
            return fail(AIE_E_UNSUPPORTED, "rows of more than 2^30 places");
    }
    a->kv = (char *)p->kv;
    a->refs = p->refs; a->lens = p->lens; a->table = p->table; a->status = p->status; a->ws = p->workspace;
    a->page_bytes = (long long)p->page_bytes;
    a->layers = (int)p->layers; a->pages = (int)p->pages; a->page_size = (int)p->page_size;
    a->rows = (int)p->rows; a->width = (int)p->width;
    return AIE_OK;
}

extern "C" uint64_t aie_pages_workspace(uint32_t pages, uint32_t n)
{
    return 4ull * (2 + 2 * (uint64_t)pages + 3 * (uint64_t)n);
}

static int check_list(const void *l, const char *what, uint32_t n)
{
    if (!l) return fail(AIE_E_INVALID, "%s is NULL", what);
    if (n > 1u << 20) return fail(AIE_E_UNSUPPORTED, "%u entries: at most 2^20", n);
    return AIE_OK;
}

static int check_ws(const aie_pages *p)
{
    if (!p->workspace || (uintptr_t)p->workspace % 8) return fail(AIE_E_INVALID, "workspace is NULL or not 8-byte aligned");
    return AIE_OK;
}

// Blocks for a copy of `chunks` pieces of page_bytes.
static unsigned copy_grid(long long chunks) { return (unsigned)std::min<long long>(chunks, 8ll * tc_sm_count()); }

extern "C" int aie_pages_grow(const aie_pages *p, const int32_t *rows, const int32_t *counts, uint32_t n,
                              int64_t *slots, uint32_t tokens, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, true, true, false, &a));
    if (tokens > 0x3fffffffu || (tokens && !slots)) return fail(AIE_E_INVALID, "slots is NULL or too long");
    if (!n && !tokens) return AIE_OK;
    TRY(check_ws(p));
    if (n) {
        TRY(check_list(rows, "rows", n));
        TRY(check_list(counts, "counts", n));
    }
    return launched(launch_behind(pages_grow_kernel, 1, kPagesThreads, (p->rows + 31) / 32 * 4, (cudaStream_t)stream, a, rows, counts,
                                  (int)n, slots, (int)tokens),
                    "grow");
}

extern "C" int aie_pages_fork(const aie_pages *p, const int32_t *src, const int32_t *dst, uint32_t n, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, true, true, true, &a));
    if (!n) return AIE_OK;
    TRY(check_ws(p));
    TRY(check_list(src, "src", n));
    TRY(check_list(dst, "dst", n));
    cudaStream_t s = (cudaStream_t)stream;
    TRY(launched(launch_behind(pages_fork_plan_kernel, 1, kPagesThreads, (p->rows + 31) / 32 * 4, s, a, src, dst, (int)n), "fork"));
    return launched(launch_behind(pages_fork_kernel, copy_grid(2ll * p->layers * n), 256, 0, s, a, src, dst, (int)n), "fork");
}

extern "C" int aie_pages_copy(const aie_pages *p, const int32_t *src, const int32_t *dst, uint32_t n, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, false, false, true, &a));
    if (!n) return AIE_OK;
    TRY(check_list(src, "src", n));
    TRY(check_list(dst, "dst", n));
    return launched(launch_behind(pages_copy_kernel, copy_grid(2ll * p->layers * n), 256, 0, (cudaStream_t)stream, a, src, dst, (int)n),
                    "copy");
}

extern "C" int aie_pages_free(const aie_pages *p, const int32_t *rows, uint32_t n, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, true, false, false, &a));
    if (!n) return AIE_OK;
    TRY(check_list(rows, "rows", n));
    return launched(launch_behind(pages_free_kernel, n, 256, 0, (cudaStream_t)stream, a, rows), "free");
}

extern "C" int aie_pages_compact(const aie_pages *p, int32_t *remap, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, true, false, true, &a));
    TRY(check_ws(p));
    if (!remap) return fail(AIE_E_INVALID, "remap is NULL");
    cudaStream_t s = (cudaStream_t)stream;
    TRY(launched(launch_behind(pages_compact_plan_kernel, 1, kPagesThreads, 0, s, a, remap), "compact"));
    return launched(launch_behind(pages_compact_kernel, copy_grid(2ll * p->layers * p->pages), 256, 0, s, a, (const int32_t *)remap),
                    "compact");
}
