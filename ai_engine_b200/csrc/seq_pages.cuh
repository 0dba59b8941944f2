// Upkeep of a paged cache's pages: who holds which page, and moving them.
//
// Every call is one block that decides (prefix sums over the list, a scan of
// the reference counts for the lowest free pages) and, where contents move, a
// second launch over all SMs that copies what the first one listed.  All
// decisions depend on the lists' order alone, never on the order of atomics.
#pragma once
#include "seq_common.cuh"

namespace aie {

constexpr int kPagesThreads = 1024;

struct PagesArgs {
    char *kv;
    int32_t *refs, *lens, *table, *status;
    int32_t *ws;  // [0] pages to copy, [1] whether the call goes ahead, [2..] (source, destination) pairs
    long long page_bytes;
    int layers, pages, page_size, rows, width;
};

// Sums stop here: more pages than a cache may have, as many tokens as slots can
// list.  Two of them still fit 32 bits.
constexpr int kSumCap = 0x3fffffff;

__device__ __forceinline__ int cap_add(int a, int b) { return min(a + b, kSumCap); }

// Exclusive prefix sum over the block's threads; *total for all of them.  Values
// from 0 to kSumCap; sums stop at kSumCap, so they ascend whatever a list asks for.
__device__ __forceinline__ int block_scan(int v, int *total, int *smem)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = cap_add(x, y);
    }
    if (lane == 31) smem[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = lane < warps ? smem[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w = cap_add(w, y);
        }
        smem[lane] = w;
    }
    __syncthreads();
    const int before = warp ? smem[warp - 1] : 0;
    *total = smem[warps - 1];
    __syncthreads();
    const int y = __shfl_up_sync(0xffffffffu, x, 1);
    return lane ? cap_add(before, y) : before;
}

// The lowest `need` free pages, in ascending order, to list[0..]; how many there were.
__device__ __forceinline__ int lowest_free(const int32_t *refs, int pages, int need, int32_t *list, int *smem)
{
    int have = 0;
    for (int p0 = 0; p0 < pages && have < need; p0 += blockDim.x) {
        const int p = p0 + threadIdx.x;
        const int is_free = p < pages && refs[p] == 0;
        int total;
        const int at = have + block_scan(is_free, &total, smem);
        if (is_free && at < need) list[at] = p;
        have += total;
    }
    return min(have, need);
}

// A row's tokens, never more than its table row holds.
__device__ __forceinline__ int row_len(const PagesArgs &a, int r) { return min(max(a.lens[r], 0), a.width * a.page_size); }

// The last of n ascending values that is at most x (at[0] <= x).
__device__ __forceinline__ int last_at_most(const int32_t *at, int n, int x)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Marks the list's rows in a bitmap: false (for all threads) when one is out
// of range, listed twice or, if asked, not empty.
__device__ __forceinline__ bool rows_ok(const int32_t *list, int n, const PagesArgs &a, bool empty, unsigned *map)
{
    for (int i = threadIdx.x; i < (a.rows + 31) / 32; i += blockDim.x) map[i] = 0u;
    __syncthreads();
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int r = list[i];
        if (r < 0 || r >= a.rows) bad = 1;
        else if (atomicOr(&map[r >> 5], 1u << (r & 31)) & (1u << (r & 31))) bad = 1;
        else if (empty && a.lens[r] != 0) bad = 1;
    }
    return !__syncthreads_or(bad);
}

__global__ void __launch_bounds__(kPagesThreads)
pages_grow_kernel(PagesArgs a, const int32_t *rows, const int32_t *counts, int n, int64_t *slots, int tokens)
{
    extern __shared__ unsigned map[];
    __shared__ int smem[32];
    int32_t *list = a.ws + 2;           // the pages handed out
    int32_t *need_at = list + a.pages;  // each entry's first page in it, then its first slot
    int32_t *slot_at = need_at + n;
    behind_last_launch();
    const bool ok = rows_ok(rows, n, a, false, map);
    int need = 0, sum = 0, bad = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        int pages = 0, count = 0;
        if (ok && i < n) {
            const int len = row_len(a, rows[i]);
            count = max(counts[i], 0);
            const long long after = ((long long)len + count + a.page_size - 1) / a.page_size;
            if (after > a.width) {
                bad = 1;
                count = 0;
            } else pages = (int)after - (len + a.page_size - 1) / a.page_size;
        }
        int total;
        const int p = cap_add(need, block_scan(pages, &total, smem));
        need = cap_add(need, total);
        const int c = cap_add(sum, block_scan(count, &total, smem));
        sum = cap_add(sum, total);
        if (i < n) {
            need_at[i] = p;
            slot_at[i] = c;
        }
    }
    bad = __syncthreads_or(bad);
    const int have = ok && !bad ? lowest_free(a.refs, a.pages, need, list, smem) : 0;
    __syncthreads();
    const bool go = ok && !bad && have == need;
    if (!go && threadIdx.x == 0) atomicOr(a.status, ok ? AIE_PAGES_FULL : AIE_PAGES_BAD_ROW);
    if (go) {
        for (int i = threadIdx.x; i < need; i += blockDim.x) a.refs[list[i]] = 1;
        // every new page, then every new token, looks its entry up
        for (int k = threadIdx.x; k < need; k += blockDim.x) {
            const int i = last_at_most(need_at, n, k), r = rows[i];
            const int first = (row_len(a, r) + a.page_size - 1) / a.page_size;
            a.table[(long long)r * a.width + first + k - need_at[i]] = list[k];
        }
        __syncthreads();
        for (int k = threadIdx.x; k < min(sum, tokens); k += blockDim.x) {
            const int i = last_at_most(slot_at, n, k), r = rows[i];
            const int place = row_len(a, r) + k - slot_at[i];
            const int page = a.table[(long long)r * a.width + place / a.page_size];
            slots[k] = (long long)page * a.page_size + place % a.page_size;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += blockDim.x) a.lens[rows[i]] = row_len(a, rows[i]) + max(counts[i], 0);
    }
    for (int s = (go ? sum : 0) + threadIdx.x; s < tokens; s += blockDim.x) slots[s] = -1;
}

// Fork, first part: which page each partly filled last page is copied to.
__global__ void __launch_bounds__(kPagesThreads)
pages_fork_plan_kernel(PagesArgs a, const int32_t *src, const int32_t *dst, int n)
{
    behind_last_launch();
    extern __shared__ unsigned map[];
    __shared__ int smem[32];
    bool ok = rows_ok(dst, n, a, true, map);
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int r = src[i];
        bad |= r < 0 || r >= a.rows || (map[r >> 5] >> (r & 31) & 1);  // a source is no destination
    }
    ok = !__syncthreads_or(bad) && ok;
    int2 *pairs = (int2 *)(a.ws + 2);
    int32_t *list = a.ws + 2 + 2 * n;
    int need = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const int len = ok && i < n ? row_len(a, src[i]) : 0;
        int total;
        const int at = need + block_scan(len % a.page_size > 0, &total, smem);
        need += total;
        // .y: the entry's place in the list of free pages, replaced below
        if (i < n) pairs[i] = make_int2(len % a.page_size ? a.table[(long long)src[i] * a.width + len / a.page_size]
                                                              : -1, at);
    }
    const int have = ok ? lowest_free(a.refs, a.pages, need, list, smem) : 0;
    __syncthreads();
    const bool go = ok && have == need;
    if (go)
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const int2 p = pairs[i];
            const int page = p.x >= 0 ? list[p.y] : -1;
            pairs[i].y = page;
            if (page >= 0) a.refs[page] = 1;
        }
    if (threadIdx.x == 0) {
        a.ws[0] = go ? n : 0;
        a.ws[1] = go;
        if (!go) atomicOr(a.status, ok ? AIE_PAGES_FULL : AIE_PAGES_BAD_ROW);
    }
}

// One block copies 16-byte pieces, 4 a thread in flight at a time.  Memory-bound:
// 790 MB of moving pages of 32 KB take 131 us, 6.0 TB/s (one at a time 157 us; 8
// at a time 130 us, but 22 us against 18 for 96 forks' pages of 16 KB).
__device__ __forceinline__ void copy_chunk(const char *src, char *dst, long long vecs)
{
    constexpr int kAhead = 4;
    const uint4 *from = (const uint4 *)src;
    uint4 *to = (uint4 *)dst;
    for (long long i0 = threadIdx.x; i0 < vecs; i0 += kAhead * blockDim.x) {
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (i0 + k * blockDim.x < vecs)
                v[k] = from[i0 + k * blockDim.x];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (i0 + k * blockDim.x < vecs) to[i0 + k * blockDim.x] = v[k];
    }
}

// Copies the listed pages in every layer, K and V: one block per chunk at a time.
__device__ __forceinline__ void copy_pages(const PagesArgs &a, const int2 *pairs, int n, int block, int blocks)
{
    const long long vecs = a.page_bytes / 16;
    const int chunks = 2 * a.layers;
    for (long long u = block; u < (long long)n * chunks; u += blocks) {
        const int2 p = pairs[u / chunks];
        if (p.x < 0 || p.y < 0 || p.x >= a.pages || p.y >= a.pages) continue;
        const long long c = u % chunks * a.pages;
        copy_chunk(a.kv + (c + p.x) * a.page_bytes, a.kv + (c + p.y) * a.page_bytes, vecs);
    }
}

// Fork, second part: the new rows, the counts of the shared pages, the copies.
__global__ void __launch_bounds__(256)
pages_fork_kernel(PagesArgs a, const int32_t *src, const int32_t *dst, int n)
{
    behind_last_launch();  // the first part's decisions
    if (!a.ws[1]) return;
    const int2 *pairs = (const int2 *)(a.ws + 2);
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int len = row_len(a, src[i]), whole = len / a.page_size;
        const int32_t *from = a.table + (long long)src[i] * a.width;
        int32_t *to = a.table + (long long)dst[i] * a.width;
        for (int k = threadIdx.x; k < a.width; k += blockDim.x) {
            int page = -1;
            if (k < whole) {
                page = from[k];
                if (page >= 0 && page < a.pages) atomicAdd(&a.refs[page], 1);
            } else if (k == whole) page = pairs[i].y;
            to[k] = page;
        }
        if (threadIdx.x == 0) a.lens[dst[i]] = len;
    }
    copy_pages(a, pairs, a.ws[0], blockIdx.x, gridDim.x);
}

// A copy's pairs as copy_pages wants them.
__global__ void __launch_bounds__(256)
pages_copy_kernel(PagesArgs a, const int32_t *src, const int32_t *dst, int n)
{
    behind_last_launch();
    const long long vecs = a.page_bytes / 16;
    const int chunks = 2 * a.layers;
    for (long long u = blockIdx.x; u < (long long)n * chunks; u += gridDim.x) {
        const int x = src[u / chunks], y = dst[u / chunks];
        if (x < 0 || y < 0 || x >= a.pages || y >= a.pages) continue;
        const long long c = u % chunks * a.pages;
        copy_chunk(a.kv + (c + x) * a.page_bytes, a.kv + (c + y) * a.page_bytes, vecs);
    }
}

// One block per row of the list.  A row listed twice: each entry of its table
// row is taken by one of the blocks.
__global__ void __launch_bounds__(256) pages_free_kernel(PagesArgs a, const int32_t *rows)
{
    behind_last_launch();
    const int r = rows[blockIdx.x];
    if (r < 0 || r >= a.rows) return;
    int32_t *row = a.table + (long long)r * a.width;
    for (int k = threadIdx.x; k < a.width; k += blockDim.x) {
        const int page = atomicExch(&row[k], -1);
        if (page >= 0 && page < a.pages) atomicSub(&a.refs[page], 1);
    }
    if (threadIdx.x == 0) a.lens[r] = 0;
}

// Compact, first part: new numbers, the pages to move, the counts in their new places.
__global__ void __launch_bounds__(kPagesThreads) pages_compact_plan_kernel(PagesArgs a, int32_t *remap)
{
    behind_last_launch();
    __shared__ int smem[32];
    int live = 0;
    for (int p = threadIdx.x; p < a.pages; p += blockDim.x) live += a.refs[p] > 0;
    int used;
    block_scan(live, &used, smem);
    int2 *pairs = (int2 *)(a.ws + 2);
    int holes = 0, late = 0;
    for (int p0 = 0; p0 < a.pages; p0 += blockDim.x) {
        const int p = p0 + threadIdx.x;
        const bool on = p < a.pages && a.refs[p] > 0;
        const bool hole = p < used && !on, move = p >= used && on;
        int total;
        int at = holes + block_scan(hole, &total, smem);
        holes += total;
        if (hole) pairs[at].y = p;
        at = late + block_scan(move, &total, smem);
        late += total;
        if (move) pairs[at].x = p;
        if (p < a.pages && !move) remap[p] = on ? p : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < late; i += blockDim.x) {
        const int2 p = pairs[i];
        remap[p.x] = p.y;
        a.refs[p.y] = a.refs[p.x];
        a.refs[p.x] = 0;
    }
    if (threadIdx.x == 0) a.ws[0] = late;
}

// Compact, second part: the moves, and the rows' new page numbers.
__global__ void __launch_bounds__(256) pages_compact_kernel(PagesArgs a, const int32_t *remap)
{
    behind_last_launch();  // the first part's decisions
    const long long all = (long long)a.rows * a.width;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long long)gridDim.x * blockDim.x) {
        const int page = a.table[i];
        if (page >= 0) a.table[i] = page < a.pages ? remap[page] : -1;
    }
    copy_pages(a, (const int2 *)(a.ws + 2), a.ws[0], blockIdx.x, gridDim.x);
}

}  // namespace aie
