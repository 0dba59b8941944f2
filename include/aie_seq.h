/*
 * aie_seq.h -- C ABI of the sequence operators (sm_100a): what a serving loop
 * needs when the frames' features of many streams feed a sequence model.
 *
 *   aie_qk_norm_rope       RMS norm of every query and key head and the
 *                          position rotation in one pass; keys and values
 *                          can go straight into the pages of a cache
 *   aie_prompt_attn        attention over whole packed prompts, causal or not
 *   aie_prefix_attn        one-token attention of a batch of streams over a
 *                          paged cache, the part they share computed once
 *   aie_pages_*            upkeep of the cache's pages: grow, fork, copy,
 *                          free, compact
 *
 * ai_engine has no counterpart of these.  The conventions are aie_conv.h's:
 * caller-owned device buffers, calls that are asynchronous on the caller's
 * cudaStream_t, allocate nothing and never abort, an aie_status in return
 * and the detail in aie_last_error.  Arguments come in one struct, all of
 * whose unused bytes are zero.  Strides are in elements.  Query head h reads
 * key/value head h / (q_heads / kv_heads).
 */
#ifndef AIE_SEQ_H
#define AIE_SEQ_H

#include "aie_conv.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum aie_dtype { AIE_DT_F32 = 0, AIE_DT_F16 = 1, AIE_DT_BF16 = 2 } aie_dtype;

/* [tokens][heads][head_dim]: element (t, h, d) at data[t * token_stride +
 * h * head_stride + d]. */
typedef struct aie_heads {
    void *data;
    int64_t token_stride, head_stride;
} aie_heads;

/* A paged cache of keys and values: token t of page p, head h, element d at
 * k[p * page_stride + t * token_stride + h * head_stride + d] (v alike). */
typedef struct aie_kv_pages {
    void *k, *v;
    int64_t page_stride, token_stride, head_stride;
    uint32_t pages, page_size;
} aie_kv_pages;

/* y = x * rsqrt(mean(x^2) + eps) * weight over each query and key head, then
 * a rotation of its first rot_dim elements by the angles of the token's
 * position; one rounding, at the end.  cos_sin is [max_pos][rot_dim] f32,
 * each row the rot_dim / 2 cosines, then the sines.  Pair i is elements
 * (i, i + rot_dim / 2), or (2i, 2i + 1) when interleaved:
 * (a, b) -> (a cos - b sin, b cos + a sin).
 * A weight of NULL leaves that tensor's heads unnormed.  A position outside
 * [0, max_pos) gives NaN in the token's rotated elements.
 * k_out.data NULL: the new keys go to the pages only.  q.data NULL (then
 * q_out.data too) leaves the queries out.  q_out may be q, k_out may be k.
 * pages.k NULL: nothing is filed.  Else the new keys, and v as it is, go to
 * slot slots[t] = page * page_size + place of the cache; a slot outside the
 * cache (-1) files nothing.  Two tokens with one slot leave either's values.
 * positions and slots are read on the device. */
typedef struct aie_qk_rope {
    aie_heads q, k, v, q_out, k_out;
    aie_kv_pages pages;
    const float *q_weight, *k_weight, *cos_sin;
    const int32_t *positions;
    const int64_t *slots;
    uint32_t tokens, q_heads, kv_heads, head_dim, rot_dim, max_pos;
    int32_t dtype, interleaved;
    float eps;
    uint32_t reserved;
} aie_qk_rope;
AIE_API int aie_qk_norm_rope(const aie_qk_rope *p, void *stream);

/* out[t] = sum_j softmax_j(scale q[t] . k[j]) v[j] over the tokens j of t's
 * own sequence (causal: j <= t).  Sequence s is tokens cu[s] .. cu[s + 1];
 * cu (device, [seqs + 1], not decreasing, within 0 .. tokens) is read on the
 * device.  A sequence may be empty; tokens of no sequence are left unwritten.
 * Values of other sequences, infinities and NaN among them, never reach a
 * result; a NaN or infinity in v within a sequence may also reach earlier
 * tokens of that sequence (0 times infinity is NaN). */
typedef struct aie_prompt {
    aie_heads q, k, v, out;
    const int32_t *cu;
    uint32_t tokens, seqs, q_heads, kv_heads, head_dim;
    int32_t dtype, causal;
    float scale;
} aie_prompt;
AIE_API int aie_prompt_attn(const aie_prompt *p, void *stream);

/* One query token for each of `batch` streams: out[b] = sum_j softmax_j(scale
 * q[b] . k[j]) v[j] over the first lens[b] places of stream b.  Places below
 * prefix_len are shared: place j stands in page prefix[j / page_size].  The
 * others are the stream's own: place j stands in page table[b * table_stride
 * + j / page_size] (entries of whole shared pages are not read).  A stream
 * with lens[b] <= 0 gives zeros; lens above max_len count as max_len.
 * prefix, table and lens are read on the device.  Page numbers outside the
 * cache are never read from; the stream's result is then unspecified.
 * Places from lens[b] on, infinities and NaN among them, never reach stream
 * b's result.
 * workspace: aie_prefix_attn_workspace(p) bytes, 16-byte aligned, its
 * contents unspecified before and after; calls that may overlap need one
 * each. */
typedef struct aie_prefix {
    aie_heads q, out;
    aie_kv_pages pages;
    const int32_t *prefix, *table, *lens;
    void *workspace;
    uint64_t workspace_bytes;
    uint32_t batch, q_heads, kv_heads, head_dim, prefix_len, max_len, table_stride;
    int32_t dtype;
    float scale;
    uint32_t reserved;
} aie_prefix;
AIE_API uint64_t aie_prefix_attn_workspace(const aie_prefix *p);
AIE_API int aie_prefix_attn(const aie_prefix *p, void *stream);

/* The cache's bookkeeping, all on the device: how many rows (streams) hold
 * each page, how many tokens each row has, and its pages in order
 * (table[r * width + i], -1 behind the last).  status collects what the
 * calls below could not do (aie_pages_status bits, OR'ed, never cleared). */
typedef struct aie_pages {
    void *kv;                    /* [layers][2][pages][page_bytes], K and V */
    int32_t *refs, *lens, *table, *status;
    int32_t *workspace;          /* aie_pages_workspace(pages, n) bytes */
    uint64_t page_bytes;         /* of one page of one layer's K */
    uint32_t layers, pages, page_size, rows, width, reserved;
} aie_pages;

typedef enum aie_pages_status {
    AIE_PAGES_FULL = 1,    /* too few free pages, or table rows too short: the call changed nothing */
    AIE_PAGES_BAD_ROW = 2  /* a row out of range or listed twice; a fork's destination that is a source or not
                              empty: the call changed nothing */
} aie_pages_status;

/* Bytes of scratch for a call with n list entries. */
AIE_API uint64_t aie_pages_workspace(uint32_t pages, uint32_t n);

/* Row rows[i] gets counts[i] (0 if negative) more tokens, and pages for them: the lowest
 * free pages, in the order of the list.  slots (tokens of them, the list's
 * order, nullable when tokens is 0) receives where each new token stands:
 * page * page_size + place; entries past the counts' sum become -1. */
AIE_API int aie_pages_grow(const aie_pages *p, const int32_t *rows, const int32_t *counts, uint32_t n,
                           int64_t *slots, uint32_t tokens, void *stream);

/* Row dst[i] (empty, and no entry of src) becomes a copy of row src[i]: it shares src's whole
 * pages, and a page that src fills in part is copied to the lowest free one
 * (in the order of the list). */
AIE_API int aie_pages_fork(const aie_pages *p, const int32_t *src, const int32_t *dst, uint32_t n, void *stream);

/* Page dst[i] becomes a copy of page src[i] in every layer.  Pairs with a
 * page out of range are left out.  No page is a destination twice, nor both
 * a source and a destination. */
AIE_API int aie_pages_copy(const aie_pages *p, const int32_t *src, const int32_t *dst, uint32_t n, void *stream);

/* Rows rows[i] become empty; pages that no row holds any more are free.
 * Rows out of range are left out, a row listed twice is freed once. */
AIE_API int aie_pages_free(const aie_pages *p, const int32_t *rows, uint32_t n, void *stream);

/* The pages in use move to the front of the cache: with n of them, those at
 * n and above go, in ascending order, to the free ones below n.  remap
 * ([pages]) receives each page's new number, -1 for a free one. */
AIE_API int aie_pages_compact(const aie_pages *p, int32_t *remap, void *stream);

/* aie_selftest_wait_timeout for these operators: a wait that gives up after
 * timeout_us (1..2e6) and records its code, which aie_device_status reports. */
AIE_API int aie_seq_selftest_wait_timeout(uint32_t timeout_us, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* AIE_SEQ_H */
