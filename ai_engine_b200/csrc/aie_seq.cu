// C ABI of the sequence operators (declared in include/aie_seq.h): argument
// checks and launches.  The kernels are in the seq_*.cuh files.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <utility>
#include <vector>

#include "host.cuh"
#include "tc_ptx.cuh"
#include "seq_common.cuh"
#include "seq_pages.cuh"
#include "seq_rope.cuh"
#include "seq_rows.cuh"

using namespace aie;

// the sizes that the Python layer packs (ai_engine_b200/_lib.py)
static_assert(sizeof(aie_qk_rope) == 248 && sizeof(aie_prompt) == 136 && sizeof(aie_prefix) == 176 &&
                  sizeof(aie_pages) == 80,
              "argument layouts");

cudaError_t aie::seq_take_device_error(uint32_t *code)
{
    uint32_t zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(code, g_aie_error, sizeof *code);
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_aie_error, &zero, sizeof zero);
    return e;
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
static int qk_norm_rope(const aie_qk_rope &p, cudaStream_t s)
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
    return launched(rope_launch(a, s), "norm and rotation");
}

extern "C" int aie_qk_norm_rope(const aie_qk_rope *p, void *stream)
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
    if (p->dtype == AIE_DT_F32) return qk_norm_rope<float>(*p, s);
    return p->dtype == AIE_DT_F16 ? qk_norm_rope<__half>(*p, s) : qk_norm_rope<__nv_bfloat16>(*p, s);
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
    prompt_rows_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(a);
    return launched(cudaGetLastError(), "prompt attention");
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

extern "C" uint64_t aie_prefix_attn_workspace(const aie_prefix *p)
{
    return check_prefix(p) ? 0 : 16;
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
    prefix_rows_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(a);
    return launched(cudaGetLastError(), "prefix attention");
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
    if (p->workspace_bytes < aie_prefix_attn_workspace(p) || !p->workspace || (uintptr_t)p->workspace % 16)
        return fail(AIE_E_INVALID, "workspace: %llu bytes, 16-byte aligned, are needed",
                    (unsigned long long)aie_prefix_attn_workspace(p));
    cudaStream_t s = (cudaStream_t)stream;
    if (p->dtype == AIE_DT_F32) return prefix_rows<float>(*p, s);
    return p->dtype == AIE_DT_F16 ? prefix_rows<__half>(*p, s) : prefix_rows<__nv_bfloat16>(*p, s);
}

// --------------------------------------------------------------- pages ---

constexpr uint32_t kPagesMaxRows = 1u << 18;  // the row bitmap: 32 KB of shared memory

static int pages_args(const aie_pages *p, bool rows, bool places, bool kv, PagesArgs *a)
{
    if (!p) return fail(AIE_E_INVALID, "null arguments");
    if (!p->pages || p->pages > 0x3fffffffu) return fail(AIE_E_INVALID, "a cache of %u pages", p->pages);
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
    pages_grow_kernel<<<1, kPagesThreads, (p->rows + 31) / 32 * 4, (cudaStream_t)stream>>>(a, rows, counts, (int)n, slots,
                                                                                           (int)tokens);
    return launched(cudaGetLastError(), "grow");
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
    pages_fork_plan_kernel<<<1, kPagesThreads, (p->rows + 31) / 32 * 4, s>>>(a, src, dst, (int)n);
    TRY(launched(cudaGetLastError(), "fork"));
    pages_fork_kernel<<<copy_grid(2ll * p->layers * n), 256, 0, s>>>(a, src, dst, (int)n);
    return launched(cudaGetLastError(), "fork");
}

extern "C" int aie_pages_copy(const aie_pages *p, const int32_t *src, const int32_t *dst, uint32_t n, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, false, false, true, &a));
    if (!n) return AIE_OK;
    TRY(check_list(src, "src", n));
    TRY(check_list(dst, "dst", n));
    pages_copy_kernel<<<copy_grid(2ll * p->layers * n), 256, 0, (cudaStream_t)stream>>>(a, src, dst, (int)n);
    return launched(cudaGetLastError(), "copy");
}

extern "C" int aie_pages_free(const aie_pages *p, const int32_t *rows, uint32_t n, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, true, false, false, &a));
    if (!n) return AIE_OK;
    TRY(check_list(rows, "rows", n));
    pages_free_kernel<<<n, 256, 0, (cudaStream_t)stream>>>(a, rows);
    return launched(cudaGetLastError(), "free");
}

extern "C" int aie_pages_compact(const aie_pages *p, int32_t *remap, void *stream)
{
    PagesArgs a;
    TRY(pages_args(p, true, false, true, &a));
    TRY(check_ws(p));
    if (!remap) return fail(AIE_E_INVALID, "remap is NULL");
    cudaStream_t s = (cudaStream_t)stream;
    pages_compact_plan_kernel<<<1, kPagesThreads, 0, s>>>(a, remap);
    TRY(launched(cudaGetLastError(), "compact"));
    pages_compact_kernel<<<copy_grid(2ll * p->layers * p->pages), 256, 0, s>>>(a, remap);
    return launched(cudaGetLastError(), "compact");
}
