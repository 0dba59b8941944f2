// One query token for each of many sequences over the sequence's own keys: the
// frames' states (packed, 16 bits) or the places of the 4-bit cache.
//
//   S^T = K Q^T,  P = 2^(S - m),  O^T = V^T P^T,  out = O / l
//
// with m, l and O carried along.  Each key is read once for the group of query
// heads that share it: memory-bound, so everything goes by keeping copies in
// flight.  K and V are the M side of the products (m16n8k16): 16 keys or 16
// elements of V by 8 query heads, so that a group of up to 8 heads wastes no
// more than the rest of 8 columns, and 4-bit codes become operands in the
// registers that they are loaded to.
//
// The sequences' tiles of keys, for every key head one after the other, are one
// long list, and each warp takes an equal part of it, whatever the lengths are:
// no sequence is too long for a warp, nor many short ones too uneven.  A warp
// copies its own tiles ahead (cp.async, a ring of its own; nothing is waited for
// but its own copies) and shares nothing with the others.  Where a sequence's
// tiles end up in several warps, each leaves a partial result (O / l and log2 of
// the weights' sum), and a second launch joins them:
//   out = sum 2^(lse_i - lse) O_i.
// A warp leaves two at most: number `warp` of the sequence that its part begins
// within, `warps + warp` of the one that it ends within.  Fixed order throughout: results
// repeat bit for bit.
//
// Rounding to fewer bits: the weights to 16 bits for the product with V (l sums
// them unrounded; f16 weights 2^7 times as large, as in attn_tc_kernel), the
// result, and over the 4-bit cache the weights times the scales to f16 for the
// product with the codes.  What that last rounding loses is put back, times the
// middle code, where results are f16 (1.75 times a 32-bit computation's error
// without, 1.3 with); a bf16 result's own rounding is 8 times as large, and in
// the second case below the kernel takes 139 us without it, 151 with it.
//
// Over the 4-bit cache the work is on the codes: 32 elements of a place and head
// are 20 bytes, which come in 0.9 cycles of an SM at the memory's rate; one
// instruction a pair of codes takes the logic pipe 0.25 of them.  So codes are not
// made into numbers at all: masked in place they are subnormal f16 (n 2^-24; the
// odd ones 16 times as large), which the products multiply exactly and at full
// rate; scales go into the weights, lowest values into a product of their own.
//
// Measured (states larger than L2): 96 streams of up to 2855 states of 8 heads of
// 128, bf16: 109 us a call, 561 MB at 5.1 TB/s; its issue slots are used 25%.  4
// bits, 64 streams of up to 16384 places of 8 heads of 128, 4 query heads each:
// 137 us a call (666 MB at 4.9 TB/s) in runs of some milliseconds, 155 in long
// ones, where the power limit takes the clock from 1.95 to 1.72 GHz (f16 results
// 149 and 166); issue slots 52%, logic pipe about 50%; 5.6 TB/s once all warps
// run, after 9 us to a warp's first tile, and blocks of an SM end unevenly (with
// the f16 results' correction between 102 and 153 us).  Parts taken from a counter end together but
// cost 165-178 us (each part begins with its own queries); 4 blocks an SM of 128
// registers 146-148; 16 places a tile 154.
#pragma once
#include "seq_kv4.cuh"
#include "seq_step.cuh"

namespace aie {

constexpr int kRdWarps = 4, kRdThreads = 32 * kRdWarps;

struct ReadArgs {
    const void *q;
    void *out;
    long long q_ts, q_hs, o_ts, o_hs;
    // the sequences' keys: packed states ...
    const void *k, *v;
    long long k_ts, k_hs, v_ts, v_hs;
    const int32_t *cu;
    int keys;
    // ... or places of pages
    Kv4Geom g;
    FastDiv size;
    const int32_t *table, *lens;
    int max_len, table_stride;
    int seqs, hq, group, d;
    unsigned most;           // tiles of all sequences, at most
    int zs, heads;           // blocks of a group's query heads; key heads times those
    int rows;                // query heads of a block that are kept
    int bf16;
    int q_vec, o_vec;        // bytes that q and out are aligned to, in every row
    float scale;
    // workspace
    unsigned *before;        // [seqs + 1]: tiles of the sequences before
    float *part_lse, *part_o;
    int workers;
    unsigned parts_each;     // host: of a sequence and head, where its share is like the others'
};

__device__ __forceinline__ int read_len(const ReadArgs &a, int s)
{
    if (a.lens) return min(max(a.lens[s], 0), a.max_len);
    const int from = min(max(a.cu[s], 0), a.keys), to = min(max(a.cu[s + 1], 0), a.keys);
    return max(to - from, 0);
}

// Tiles a warp takes of `total`.
__device__ __forceinline__ unsigned read_share(unsigned total, unsigned workers) { return max((total + workers - 1) / workers, 1u); }

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix2(uint32_t addr, uint32_t (&r)[2])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix2_t(uint32_t addr, uint32_t (&r)[2])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The four codes of each half of a word as f16 pairs, code i of the lower half and
// of the upper.  A code in the lowest bits of an f16 is that many times 2^-24, a
// subnormal, which the products take as it is: exact, at one instruction a pair.
// The odd ones stand four bits higher, 16 times as large.
struct Codes {
    uint32_t p[4];
    __device__ __forceinline__ Codes(uint32_t w)
    {
        const uint32_t high = __byte_perm(w, 0, 0x4341);  // codes 2 and 3, in each half's lower byte
        p[0] = w & 0x000F000Fu;
        p[1] = w & 0x00F000F0u;
        p[2] = high & 0x000F000Fu;
        p[3] = high & 0x00F000F0u;
    }
};

// The same with the odd ones still on top of the even: p[1] is code 0 + 16 code 1.
// For a sum over them from which that over the even ones can be taken away.
struct StackedCodes {
    uint32_t p[4];
    __device__ __forceinline__ StackedCodes(uint32_t w)
    {
        p[1] = w & 0x00FF00FFu;
        p[3] = __byte_perm(w, 0, 0x4341);
        p[0] = w & 0x000F000Fu;
        p[2] = p[3] & 0x000F000Fu;
    }
};

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b)
{
    const __half2 y = __hmul2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&y;
}

// a b - y
__device__ __forceinline__ uint32_t lost2(uint32_t a, uint32_t b, uint32_t y)
{
    const __half2 z = __hfma2(*(const __half2 *)&a, *(const __half2 *)&b, __hneg2(*(const __half2 *)&y));
    return *(const uint32_t *)&z;
}

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b)
{
    const __half2 y = __hmax2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&y;
}

// c = a b
template <typename T>
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%10, %10, %10, %10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%10, %10, %10, %10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// N 32-bit words of shared memory from an address aligned to the whole of them.
template <int N>
__device__ __forceinline__ void shared_words(const uint32_t *p, uint32_t (&w)[N])
{
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *(const uint4 *)(p + i);
            w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 x = *(const uint2 *)(p + i);
            w[i] = x.x; w[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = p[i];
    }
}

// DC: groups of 32 elements (4 bits) or steps of 16 (16 bits).  A stage of a
// warp's ring holds one tile: K rows, then V rows, a row padded to an odd number
// of 16-byte pieces so that eight rows' pieces are in different banks; then, in
// 4 bits, the groups' pairs of K and of V.
template <bool KV4, int DC>
struct ReadTile {
    static constexpr int kKeys = KV4 ? 32 : 16;
    static constexpr int kPieces = KV4 ? DC : 2 * DC;       // of a row
    static constexpr uint32_t kRow = (kPieces | 1) * 16;
    static constexpr uint32_t kSide = kKeys * kRow;         // K or V
    static constexpr uint32_t kPairs = KV4 ? kKeys * DC * 4 : 0;
    static constexpr uint32_t kStage = 2 * kSide + 2 * kPairs;
};

// Four neighbouring elements of a result.
template <typename T>
__device__ __forceinline__ void read_store4(const ReadArgs &a, long long at, const float (&x)[4])
{
    unsigned short *out = (unsigned short *)a.out + at;
    const uint2 y = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    if (a.o_vec >= 8) *(uint2 *)out = y;
    else {
        out[0] = (unsigned short)y.x; out[1] = (unsigned short)(y.x >> 16);
        out[2] = (unsigned short)y.y; out[3] = (unsigned short)(y.y >> 16);
    }
}

// Blocks of an SM.  With 16-bit heads of more than 128 the rings of two would hold one
// tile a warp.  (One block of three stages, all at once: 64 sequences of 2000 states, 8/2
// heads of 256, 57 us, one after the other of two stages 64.5; 500 of 1-999, 8/4 heads of
// 160, 152 and 158; 300 of 500, 8 heads of 200, 214 and 199.)
constexpr int read_blocks(bool kv4, int dc, int nt) { return nt == 1 && dc <= 4 ? 3 : !kv4 && dc > 8 ? 1 : 2; }

// A ring's stages: as many, up to six, as let all blocks of an SM fit it with their
// static shared memory and what the system keeps (1 KB a block).
constexpr uint32_t kReadOther = 1024 + 1280;
template <bool KV4, int DC, int NT>
struct ReadRing {
    static constexpr uint32_t kOne = kRdWarps * ReadTile<KV4, DC>::kStage;
    static constexpr uint32_t kRoom = 228 * 1024 / read_blocks(KV4, DC, NT) - kReadOther;
    static constexpr int kStages = kRoom / kOne > 6 ? 6 : kRoom / kOne;
    static_assert(kStages >= 2 && kStages * kOne <= 227 * 1024, "two tiles a warp, all blocks of an SM at once");
};

// T: the type of queries and results; that of the products is f16 in 4 bits.
template <typename T, bool KV4, int DC, int NT, int STAGES>
__global__ void __launch_bounds__(kRdThreads, read_blocks(KV4, DC, NT)) read_kernel(const ReadArgs a)
{
    using Tile = ReadTile<KV4, DC>;
    using M = std::conditional_t<KV4, __half, T>;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    // Binary orders by which m may lag behind the scores.  In 4 bits weights are also
    // multiplied with the groups' scales: weights of 2^7 2^4 times scales below 2^4 are
    // what f16 holds.  In a tile with a larger scale, or with none of 2^-8, each group's
    // are multiplied by a power of two before they are used, and its sums follow (both
    // exactly, but for scales that become subnormal beside a larger one in their tile);
    // weights stay as they are, so that no group or place coarsens what others add.  (64
    // streams of up to 16384 places, bf16, 600 calls: 141 us each, 164 where every tile has
    // scales above 2^4, that is values that span 240; 152 where none has 2^-8.  Lifted
    // before the scores instead of behind the weights, ordinary values took 1.5% longer.)
    constexpr float kLag = KV4 ? 4.f : 8.f;
    constexpr uint32_t kLeastScale = 0x1C00u << 16, kMostScale = 0x4C00u << 16;  // 2^-8, 2^4
    constexpr int MT = Tile::kKeys / 16, OT = KV4 ? 2 * DC : DC;  // tiles of 16 keys; of 16 elements of V
    extern __shared__ __align__(16) char smem[];
    __shared__ unsigned scan[kRdThreads], warp_sums[kRdWarps];
    behind_last_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- tiles before each thread's sequences, and in all
    const int per = (a.seqs + kRdThreads - 1) / kRdThreads, s_from = tid * per, s_to = min(s_from + per, a.seqs);
    // (sums stop at 2^31 - 1 instead of wrapping: a cu that decreases can have any number)
    auto sum = [](unsigned x, unsigned y) { return min(x + y, 0x7fffffffu); };
    unsigned mine = 0;
    for (int s = s_from; s < s_to; s++) mine = sum(mine, (read_len(a, s) + Tile::kKeys - 1) / Tile::kKeys);
    unsigned upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto = sum(upto, y);
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    unsigned tiles = 0, base = upto - mine;
#pragma unroll
    for (int i = 0; i < kRdWarps; i++) {
        if (i < warp) base = sum(base, warp_sums[i]);
        tiles = sum(tiles, warp_sums[i]);
    }
    if (tiles > a.most) tiles = 0;  // no list of starts: zeros
    scan[tid] = base;
    if (blockIdx.x == 0) {  // for the joining launch
        for (int s = s_from; s < s_to; s++) {
            a.before[s] = tiles ? base : 0u;
            base += (read_len(a, s) + Tile::kKeys - 1) / Tile::kKeys;
        }
        if (tid == 0) a.before[a.seqs] = tiles;
    }
    __syncthreads();
    const unsigned total = tiles * a.heads, share = read_share(total, a.workers);
    const int worker = blockIdx.x * kRdWarps + warp;
    const unsigned long long first_of = (unsigned long long)worker * share;
    if (first_of >= total) return;
    const unsigned begin = (unsigned)first_of;
    const int count = (int)min(share, total - begin);

    // ---- where the warp's part begins
    struct Place {
        int s, head, tile, len;  // sequence; key head and block of query heads; tile of the sequence
        long long head_at;       // 4 bits: the key head's blocks in a page; 16 bits: the key head
    } at;
    auto head_at = [&](int head) { return (long long)(head / a.zs) * (KV4 ? a.g.block() : 1); };
    {
        at.head = (int)(begin / tiles);
        unsigned left = begin - at.head * tiles;
        // the last thread whose sequences begin at or before it
        int t = 0;
#pragma unroll
        for (int i = 0; i < kRdWarps; i++) t += __popc(__ballot_sync(0xffffffffu, scan[i * 32 + lane] <= left));
        t--;
        left -= scan[t];
        for (at.s = t * per;; at.s++) {
            at.len = read_len(a, at.s);
            const unsigned n = (at.len + Tile::kKeys - 1) / Tile::kKeys;
            if (left < n) break;
            left -= n;
        }
        at.tile = (int)left;
        at.head_at = head_at(at.head);
    }
    auto advance = [&](Place &p) {
        if (++p.tile * Tile::kKeys < p.len) return;
        p.tile = 0;
        do {
            if (++p.s == a.seqs) {
                p.s = 0;
                p.head_at = head_at(++p.head);
            }
            p.len = read_len(a, p.s);
        } while (!p.len);
    };

    const int r = lane >> 2, c2 = (lane & 3) * 2;  // a lane's rows r, r + 8 and columns c2, c2 + 1 of a product
    char *const ring = smem + warp * (STAGES * Tile::kStage);
    const uint32_t ring_at = smem_u32(ring);

    // ---- the queries of a sequence, as they come: of head r the elements 32 g + 8 (lane & 3)
    // .. + 7 of each group, or 16 k + c2, + 1 and + 8, + 9 of each step
    uint32_t raw[NT][KV4 ? 4 * DC : 2 * DC];
    auto load_q = [&] {
        const int row0 = at.head % a.zs * (8 * NT), heads = min(a.group - row0, 8 * NT);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const bool real = nt * 8 + r < heads;
            const unsigned short *q = (const unsigned short *)a.q + (long long)at.s * a.q_ts +
                                      (long long)(at.head / a.zs * a.group + row0 + (real ? nt * 8 + r : 0)) * a.q_hs;
            auto two = [&](int d) { return a.q_vec >= 4 ? *(const uint32_t *)(q + d) : (uint32_t)q[d] | (uint32_t)q[d + 1] << 16; };
            if constexpr (KV4) {
#pragma unroll
                for (int g = 0; g < DC; g++) {
                    const int d = g * 32 + (lane & 3) * 8;
                    uint4 x;
                    if (a.q_vec >= 16) x = *(const uint4 *)(q + d);
                    else x = make_uint4(two(d), two(d + 2), two(d + 4), two(d + 6));
                    raw[nt][g * 4] = real ? x.x : 0u;
                    raw[nt][g * 4 + 1] = real ? x.y : 0u;
                    raw[nt][g * 4 + 2] = real ? x.z : 0u;
                    raw[nt][g * 4 + 3] = real ? x.w : 0u;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2 * DC; k++) raw[nt][k] = real && k * 8 + c2 < a.d ? two(k * 8 + c2) : 0u;  // head_dim is even
            }
        }
    };
    load_q();

    // ---- copies
    Place ahead = at;
    // 4 bits: four lanes to 8 places of the tile (the lane's are those of lane & 3), eight
    // lanes to a piece of every one of them: how many exist, and where their codes
    // and pairs are
    const int in8 = lane >> 2;
    const uint8_t *codes_at = nullptr, *pairs_at = nullptr;
    const long long v_from_k = a.g.v - a.g.k;
    int real = 0;
    auto look_up = [&] {
        if constexpr (KV4) {
            const int place = ahead.tile * Tile::kKeys + (lane & 3) * 8, i = fdiv(place, a.size), in = place - i * a.g.size;
            const int page = place < ahead.len ? a.table[(long long)ahead.s * a.table_stride + i] : -1;
            const bool exists = page >= 0 && page < a.g.pages;
            real = exists ? min(ahead.len - place, 8) : 0;
            const uint8_t *block = a.g.k + ahead.head_at + (exists ? page * a.g.page_stride : 0);
            codes_at = block + in * (16 * DC) + in8 * 16;
            pairs_at = block + a.g.size * (16 * DC) + in * (4 * DC) + in8 * 16;
        }
    };
    auto copy_tile = [&](int stage) {
        const uint32_t dst = ring_at + stage * Tile::kStage;
        // keys that do not exist: zeros
        if constexpr (KV4) {
            // 8 places' codes are 8 DC pieces of 16 bytes side by side, their pairs 2 DC
            const uint32_t codes_to = dst + (lane & 3) * 8 * Tile::kRow, pairs_to = dst + 2 * Tile::kSide + ((lane & 3) * 2 * DC + in8) * 16;
#pragma unroll
            for (int i = 0; i < DC; i++) {
                const int c = i * 8 + in8, row = c / DC, n = row < real ? 16 : 0;
                const uint32_t to = codes_to + row * Tile::kRow + (c - row * DC) * 16;
                copy16(to, codes_at + i * 128, n);
                copy16(to + Tile::kSide, codes_at + v_from_k + i * 128, n);
            }
#pragma unroll
            for (int i = 0; i < (DC + 3) / 4; i++) {
                const int n = min(max(real * (4 * DC) - (i * 8 + in8) * 16, 0), 16);
                if (i * 8 + in8 < 2 * DC) {
                    copy16(pairs_to + i * 128, pairs_at + i * 128, n);
                    copy16(pairs_to + Tile::kPairs + i * 128, pairs_at + v_from_k + i * 128, n);
                }
            }
        } else {
            const int rows = ahead.len - ahead.tile * Tile::kKeys;
            const long long key = min(max(a.cu[ahead.s], 0), a.keys) + (long long)ahead.tile * Tile::kKeys;
            const int kvh = (int)ahead.head_at;
            const T *k = (const T *)a.k + key * a.k_ts + kvh * a.k_hs, *v = (const T *)a.v + key * a.v_ts + kvh * a.v_hs;
#pragma unroll
            for (int i = 0; i < DC; i++) {
                const int c = i * 32 + lane, row = c / (2 * DC), piece = c % (2 * DC);
                const bool real = row < rows && piece * 8 < a.d;
                copy16(dst + row * Tile::kRow + piece * 16, real ? k + row * a.k_ts + piece * 8 : k, real ? 16 : 0);
                copy16(dst + Tile::kSide + row * Tile::kRow + piece * 16, real ? v + row * a.v_ts + piece * 8 : v, real ? 16 : 0);
            }
        }
    };
    int copied = 0;
    look_up();
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) {
        if (copied < count) {
            copy_tile(i);
            if (++copied < count) {
                advance(ahead);
                look_up();
            }
        }
        copies_commit();
    }

    // ---- products
    const float sl = fabsf(a.scale) * 1.4426950408889634f, sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
    uint32_t qb[NT][KV4 ? 2 * DC : DC][2], qs[NT][2];  // queries; 4 bits: each group's sum of them, in two f16
    float slq[NT][2];                                  // scale of a column's scores, in binary orders
    float ref[NT][2], most_s[NT][2];                   // weights are 2^(slq (s - ref) + shift), ref = m; scores above most_s move m
    float o[OT][NT][4], m[NT][2], l[NT][2];
    float o_lo[KV4 ? NT : 1][4];  // 4 bits: the weighted sums of the groups' lo
    int lift = 0;                 // the lane's group's (lane / 4) scales, and its sums in o, are 2^-lift of what they stand for
    bool fresh = true;
    int first_tile = 0, stage = 0;  // of the sequence's tiles; of the ring
    for (int i = 0; i < count; i++) {
        if (fresh) {
            fresh = false;
            first_tile = at.tile;
            if (i) load_q();
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if constexpr (KV4) {
                    float f[DC][8], top = 0.f;
#pragma unroll
                    for (int g = 0; g < DC; g++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t x = raw[nt][g * 4 + e];
                            const float2 y = kBf16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u))
                                                    : __half22float2(*(const __half2 *)&x);
                            f[g][2 * e] = y.x * sign;
                            f[g][2 * e + 1] = y.y * sign;
                            top = fmaxf(top, fmaxf(fabsf(f[g][2 * e]), fabsf(f[g][2 * e + 1])));
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // a power of two that brings the largest to 2^8 .. 2^9: exact, and in f16
                    // nothing that counts is subnormal
                    const int ex = (int)(__float_as_uint(top) >> 23);
                    const int k = top > 0.f ? min(max(8 + 127 - ex, -120), 120) : 0;
                    const float up = __uint_as_float((uint32_t)(127 + k) << 23), down = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
                    for (int g = 0; g < DC; g++) {
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            f[g][e] = __half2float(__float2half_rn(f[g][e] * up));
                            sum += f[g][e];
                        }
                        // element e + 4 is the same code of a word's upper half; odd codes are 16 times as large
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float x = e & 1 ? 0.0625f : 1.f;
                            qb[nt][2 * g + (e >> 1)][e & 1] = pack2<__half>(f[g][e] * x, f[g][e + 4] * x);
                        }
                        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                        if (!(g & 3)) qs[nt][g >> 2] = 0u;
                        if ((lane & 3) == (g & 3)) {
                            const float hi = __half2float(__float2half_rn(sum));
                            qs[nt][g >> 2] = pack2<__half>(hi, sum - hi);
                        }
                    }
                    if (DC <= 4) qs[nt][1] = 0u;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        // 2^127 at most: larger (queries beyond 2^115), and scores that differ at all
                        // have weights 1 and 0 either way
                        slq[nt][j] = fminf(fmaxf(sl * 0x1p24f * __shfl_sync(0xffffffffu, down, (c2 + j) * 4), 1e-37f), 0x1p127f);
                    }
                    o_lo[nt][0] = o_lo[nt][1] = o_lo[nt][2] = o_lo[nt][3] = 0.f;
                    lift = 0;
                } else {
#pragma unroll
                    for (int k = 0; k < 2 * DC; k++) {
                        const T *x = (const T *)&raw[nt][k];
                        qb[nt][k >> 1][k & 1] = pack2<T>(sign * to_f32(x[0]), sign * to_f32(x[1]));
                    }
                    slq[nt][0] = slq[nt][1] = fmaxf(sl, 1e-37f);
                }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    m[nt][j] = most_s[nt][j] = -INFINITY;
                    l[nt][j] = ref[nt][j] = 0.f;
                }
#pragma unroll
                for (int x = 0; x < OT; x++) o[x][nt][0] = o[x][nt][1] = o[x][nt][2] = o[x][nt][3] = 0.f;
            }
        }

        // the next copy goes where the last tile was
        if (copied < count) {
            copy_tile(stage ? stage - 1 : STAGES - 1);
            if (++copied < count) {
                advance(ahead);
                look_up();
            }
        }
        copies_commit();
        copies_wait<STAGES - 1>();
        __syncwarp();

        const char *const st = ring + stage * Tile::kStage;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        const uint32_t kt = smem_u32(st), vt = kt + Tile::kSide;
        bool tiny = false, odd = false;  // no scale of 2^-8; one of 2^4, or some that are lifted
        if constexpr (KV4) {
            uint32_t pv[DC], most = 0;
            shared_words<DC>((const uint32_t *)(st + 2 * Tile::kSide + Tile::kPairs) + lane * DC, pv);
#pragma unroll
            for (int g = 0; g < DC; g++) most = max2(most, pv[g]);  // of the lower halves
            most <<= 16;
            tiny = !__any_sync(0xffffffffu, most >= kLeastScale);
            odd = __any_sync(0xffffffffu, most >= kMostScale || lift);
        }
        {
            const int here = at.len - at.tile * Tile::kKeys;
            // ---- scores: keys r and r + 8 of each 16, query heads c2 and c2 + 1
            float s[MT][NT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if constexpr (KV4) {
                    // S 2^-24 = sum over the groups of s (codes 2^-24) q, and of lo sum(q) 2^-24
                    const uint32_t *pk = (const uint32_t *)(st + 2 * Tile::kSide) + (mt * 16 + r) * DC;
                    uint32_t p0[DC], p1[DC];
                    shared_words<DC>(pk, p0);
                    shared_words<DC>(pk + 8 * DC, p1);
                    uint32_t low[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // row r or r + 8, group lane & 3 or 4 further on
                        const int g = (lane & 3) + (i >> 1) * 4;
                        low[i] = g < DC ? __byte_perm(pk[(i & 1) * 8 * DC + g], 0, 0x3232) : 0u;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        mma16816_first<M>(s[mt][nt], low, qs[nt][0], qs[nt][1]);
#pragma unroll
                        for (int j = 0; j < 4; j++) s[mt][nt][j] *= 0x1p-24f;
                    }
                    uint32_t w[4];
#pragma unroll
                    for (int g = 0; g < DC; g++) {
                        // of 16 keys, two groups at a time
                        if (g + 1 < DC && !(g & 1)) ldmatrix4(kt + (mt * 16 + (lane & 15)) * Tile::kRow + (g + (lane >> 4)) * 16, w);
                        else if (!(g & 1)) ldmatrix2(kt + (mt * 16 + (lane & 15)) * Tile::kRow + g * 16, *(uint32_t(*)[2])w);
                        const Codes x0(w[(g & 1) * 2]), x1(w[(g & 1) * 2 + 1]);
                        const float f0 = __half2float(__ushort_as_half((unsigned short)p0[g])), f1 = __half2float(__ushort_as_half((unsigned short)p1[g]));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            float acc[4];
                            mma16816_first<M>(acc, {x0.p[0], x1.p[0], x0.p[1], x1.p[1]}, qb[nt][2 * g][0], qb[nt][2 * g][1]);
                            mma16816<M>(acc, {x0.p[2], x1.p[2], x0.p[3], x1.p[3]}, qb[nt][2 * g + 1][0], qb[nt][2 * g + 1][1]);
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                s[mt][nt][j] = fmaf(f0, acc[j], s[mt][nt][j]);
                                s[mt][nt][2 + j] = fmaf(f1, acc[2 + j], s[mt][nt][2 + j]);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < DC; k++) {
                        uint32_t w[4];
                        ldmatrix4(kt + (mt * 16 + (lane & 15)) * Tile::kRow + (2 * k + (lane >> 4)) * 16, w);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if (k) mma16816<M>(s[mt][nt], w, qb[nt][k][0], qb[nt][k][1]);
                            else mma16816_first<M>(s[mt][nt], w, qb[nt][k][0], qb[nt][k][1]);
                        }
                    }
                }
            }
            if (here < Tile::kKeys) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (mt * 16 + r + (j >> 1) * 8 >= here) s[mt][nt][j] = -INFINITY;
            }
            // ---- weights
            float top[NT][2];
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float x = m[nt][j];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) x = max3(x, s[mt][nt][j], s[mt][nt][2 + j]);
                    top[nt][j] = x;
                    grow |= x > most_s[nt][j];
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float x = top[nt][j];
#pragma unroll
                        for (int e = 4; e < 32; e <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, e));
                        const float f = x == m[nt][j] ? 1.f : ex2((m[nt][j] - x) * slq[nt][j]);
                        if (x != -INFINITY) {
                            m[nt][j] = ref[nt][j] = x;
                            // as in attn_tc_kernel: steps of a few binary orders leave m (rounded down:
                            // what f16 holds allows no more, however large the scores are)
                            most_s[nt][j] = __fadd_rd(x, __fdividef(kLag, slq[nt][j]));
                        }
                        l[nt][j] *= f;
                        if constexpr (KV4) o_lo[nt][j] *= f;
#pragma unroll
                        for (int t = 0; t < OT; t++) {
                            o[t][nt][j] *= f;
                            o[t][nt][2 + j] *= f;
                        }
                    }
            }
            // (the difference first: slq s - slq ref would be as far off as slq ref is rounded,
            // more than f16 holds from scores of 2^27 on)
            const float shift = kWeightShift<M>;
            uint32_t pb[NT][MT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    float e[4];
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const float2 x = __ffma2_rn(__fadd2_rn(make_float2(s[mt][nt][j], s[mt][nt][j + 1]), make_float2(-ref[nt][0], -ref[nt][1])),
                                                    make_float2(slq[nt][0], slq[nt][1]), make_float2(shift, shift));
                        e[j] = ex2(x.x);
                        e[j + 1] = ex2(x.y);
                    }
                    l[nt][0] += e[0] + e[2];
                    l[nt][1] += e[1] + e[3];
                    pb[nt][mt][0] = transpose8x8(pack2<M>(e[0], e[1]));
                    pb[nt][mt][1] = transpose8x8(pack2<M>(e[2], e[3]));
                }
            if constexpr (KV4) {
                if (tiny | odd) {
                    // a lane has a place's (s, lo) of V
                    uint32_t *const pairs = (uint32_t *)(st + 2 * Tile::kSide + Tile::kPairs) + lane * DC;
                    int next = tiny && r < DC ? -8 : 0;
                    if (!tiny) {
#pragma unroll
                        for (int g = 0; g < DC; g++) {
                            // s < 2^(need + 4); lift is left alone where it is one too many
                            const int need = (int)(__reduce_max_sync(0xffffffffu, pairs[g] & 0xffffu) >> 10) - 18;
                            if (r == g) next = lift > 0 && lift == need + 1 ? lift : min(max(need, 0), 12);
                        }
                    }
                    if (__any_sync(0xffffffffu, next != lift)) {
                        const float f = __uint_as_float((uint32_t)(127 + lift - next) << 23);
                        lift = next;
#pragma unroll
                        for (int t = 0; t < OT; t++) {
                            const float x = __shfl_sync(0xffffffffu, f, (t >> 1) * 4);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int j = 0; j < 4; j++) o[t][nt][j] *= x;
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int g = 0; g < DC; g++) {
                        const int k = __shfl_sync(0xffffffffu, lift, g * 4);
                        const __half y = __hmul(__ushort_as_half((unsigned short)pairs[g]), __ushort_as_half((unsigned short)(15 - k << 10)));
                        pairs[g] = __byte_perm(pairs[g], __half_as_ushort(y), 0x3254);
                    }
                    __syncwarp();
                }
            }
            // ---- values
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if constexpr (KV4) {
                    // O = sum over the keys of (p s) codes, and of p lo.  (s, lo) of keys c2, c2 + 1
                    // and of 8 further on, two keys to a register
                    const uint32_t *pv = (const uint32_t *)(st + 2 * Tile::kSide + Tile::kPairs) + (mt * 16 + c2) * DC;
                    uint32_t p0[DC], p1[DC], p2[DC], p3[DC], low[4] = {0u, 0u, 0u, 0u};
                    shared_words<DC>(pv, p0);
                    shared_words<DC>(pv + DC, p1);
                    shared_words<DC>(pv + 8 * DC, p2);
                    shared_words<DC>(pv + 9 * DC, p3);
                    if (r < DC) {  // row r: group r
                        low[0] = __byte_perm(pv[r], pv[DC + r], 0x7632);
                        low[2] = __byte_perm(pv[8 * DC + r], pv[9 * DC + r], 0x7632);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma16816<M>(o_lo[nt], low, pb[nt][mt][0], pb[nt][mt][1]);
                    uint32_t w[4];
#pragma unroll
                    for (int g = 0; g < DC; g++) {
                        // of 16 keys, two groups at a time
                        if (g + 1 < DC && !(g & 1)) ldmatrix4_t(vt + (mt * 16 + (lane & 15)) * Tile::kRow + (g + (lane >> 4)) * 16, w);
                        else if (!(g & 1)) ldmatrix2_t(vt + (mt * 16 + (lane & 15)) * Tile::kRow + g * 16, *(uint32_t(*)[2])w);
                        const StackedCodes x0(w[(g & 1) * 2]), x1(w[(g & 1) * 2 + 1]);
                        const uint32_t s0 = __byte_perm(p0[g], p1[g], 0x5410), s1 = __byte_perm(p2[g], p3[g], 0x5410);
                        // rows r: elements 4 r + 0 (+ 2), rows r + 8: these and 16 times 4 r + 1 (+ 3)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint32_t b0 = mul2(pb[nt][mt][0], s0), b1 = mul2(pb[nt][mt][1], s1);
                            mma16816<M>(o[2 * g][nt], {x0.p[0], x0.p[1], x1.p[0], x1.p[1]}, b0, b1);
                            mma16816<M>(o[2 * g + 1][nt], {x0.p[2], x0.p[3], x1.p[2], x1.p[3]}, b0, b1);
                            // what p s lost in f16 (exactly f16 again), times the middle code, to the lo of
                            // row g: else lo + code s, which cancel, would not lose the same (f16 results
                            // 1.7 times as far off as a 16-bit cache's; 1.3 with it).  bf16 cannot tell.
                            if constexpr (!kBf16) {
                                const uint32_t middle = r == g ? (uint32_t)(0x4780 + lift * 1024) * 0x10001u : 0u;  // 7.5 2^lift
                                mma16816<M>(o_lo[nt], {middle, 0u, middle, 0u}, lost2(pb[nt][mt][0], s0, b0), lost2(pb[nt][mt][1], s1, b1));
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < DC; t++) {
                        // as stored: keys 0-7 and 8-15 by elements 0-7, then 8-15
                        uint32_t w[4];
                        ldmatrix4_t(vt + (mt * 16 + (lane & 7) + (lane >> 4) * 8) * Tile::kRow + (2 * t + (lane >> 3 & 1)) * 16, w);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma16816<M>(o[t][nt], w, pb[nt][mt][0], pb[nt][mt][1]);
                    }
                }
            }
        }
        __syncwarp();  // the tile is read before the copy that replaces it

        // ---- end of the sequence, or of the warp's part
        const bool ends = (at.tile + 1) * Tile::kKeys >= at.len;
        if (ends || i + 1 == count) {
            const bool whole = ends && first_tile == 0;
            const int kvh = at.head / a.zs, row0 = at.head % a.zs * (8 * NT), heads = min(a.group - row0, 8 * NT);
            const long long part = worker + (first_tile ? 0 : a.workers);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float sum = l[nt][j];
#pragma unroll
                    for (int e = 4; e < 32; e <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, e);
                    float low[KV4 ? DC : 1], code[KV4 ? DC : 1];
                    if constexpr (KV4) {
#pragma unroll
                        for (int g = 0; g < DC; g++) {
                            low[g] = __shfl_sync(0xffffffffu, o_lo[nt][j], g * 4 + (lane & 3));
                            code[g] = __uint_as_float((uint32_t)(127 + 24 + __shfl_sync(0xffffffffu, lift, g * 4)) << 23);
                        }
                    }
                    const int n = nt * 8 + c2 + j;
                    if (n >= heads) continue;
                    // of several parts, one with scores of -inf alone (the sum is 0) has no weight
                    const float f = sum == 0.f && !whole ? 0.f : 1.f / sum;
                    const long long oat = (long long)at.s * a.o_ts + (long long)(kvh * a.group + row0 + n) * a.o_hs;
                    const long long pat = (part * a.rows + n) * a.d;
                    if (!whole && r == 0)
                        a.part_lse[part * a.rows + n] = sum == 0.f ? -INFINITY : fmaf(ref[nt][j], slq[nt][j], log2f(sum) - kWeightShift<M>);
                    if constexpr (KV4) {
                        // four neighbouring elements of each group
#pragma unroll
                        for (int g = 0; g < DC; g++) {
                            float x[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const float *t = o[2 * g + (e >> 1)][nt];
                                x[e] = f * fmaf(e & 1 ? t[2 + j] - t[j] : t[j], e & 1 ? code[g] * 0.0625f : code[g], low[g]);
                            }
                            const int d = g * 32 + r * 4;
                            if (!whole) *(float4 *)(a.part_o + pat + d) = make_float4(x[0], x[1], x[2], x[3]);
                            else read_store4<T>(a, oat + d, x);
                        }
                    } else {
#pragma unroll
                        for (int t = 0; t < OT; t++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const int d = t * 16 + e * 8 + r;
                                if (d >= a.d) continue;
                                const float x = o[t][nt][2 * e + j] * f;
                                if (!whole) a.part_o[pat + d] = x;
                                else ((T *)a.out)[oat + d] = from_f32<T>(x);
                            }
                    }
                }
            fresh = true;
        }
        if (i + 1 < count) advance(at);
    }
}

// Sequences whose tiles more than one warp took, and those without any: a block
// per sequence and query head, of more warps where there are more parts.
struct JoinArgs {
    void *out;
    long long o_ts, o_hs;
    const unsigned *before;
    const float *part_lse, *part_o;
    int seqs, hq, group, d, zs, heads, rows, bf16, workers;
};

template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) read_join_kernel(const JoinArgs a)
{
    constexpr bool MANY = WARPS > 4;
    extern __shared__ float weight[];  // MANY: of each part
    __shared__ float sums[WARPS][256], tops[WARPS], totals[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int s = blockIdx.x / a.hq, h = blockIdx.x % a.hq, kvh = h / a.group, in = h % a.group;
    const int head = kvh * a.zs + in / a.rows, row = in % a.rows;
    const long long oat = (long long)s * a.o_ts + (long long)h * a.o_hs;
    behind_last_launch();
    const unsigned tiles = a.before[a.seqs], from = a.before[s], n = a.before[s + 1] - from;
    auto store = [&](int d, float x) {
        if (a.bf16) ((__nv_bfloat16 *)a.out)[oat + d] = __float2bfloat16_rn(x);
        else ((__half *)a.out)[oat + d] = __float2half_rn(x);
    };
    if (n == 0) {
        for (int d = threadIdx.x; d < a.d; d += 32 * WARPS) store(d, 0.f);
        return;
    }
    const unsigned share = read_share(tiles * a.heads, a.workers), at = head * tiles + from, first = at / share;
    const int parts = (int)((at + n - 1) / share - first + 1);
    if (parts == 1) return;
    // of the first warp the part that it ends within, of the others those that they begin within
    auto part = [&](int i) { return (long long)(i ? i : a.workers); };
    const long long id = first, next = (long long)a.rows * a.d;
    const float *lse = a.part_lse + id * a.rows + row, *po = a.part_o + (id * a.rows + row) * a.d + lane * 4;
    // a warp every WARPS-th part, a lane four neighbouring elements (of 128 at a time);
    // the first on their way before the weights are known
    constexpr int kFirst = 2;
    float4 y[kFirst][2];
#pragma unroll
    for (int i = 0; i < kFirst; i++)
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (warp + i * WARPS < parts && k * 128 + lane * 4 < a.d)
                y[i][k] = *(const float4 *)(po + part(warp + i * WARPS) * next + k * 128);
    float top = -INFINITY, sum = 0.f;
    float4 x[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    auto weigh = [&](float w) { return w == -INFINITY ? 0.f : ex2(w - top); };
    auto add = [&](float f, const float4 (&z)[2]) {
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k * 128 + lane * 4 < a.d) add_scaled(x[k], f, z[k]);
    };
    auto load = [&](int i, float4 (&z)[2]) {
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k * 128 + lane * 4 < a.d) z[k] = *(const float4 *)(po + part(i) * next + k * 128);
    };
    if constexpr (MANY) {
        // the weights first, by all threads
        for (int i = threadIdx.x; i < parts; i += 32 * WARPS) {
            const float w = lse[part(i) * a.rows];
            weight[i] = w;
            top = fmaxf(top, w);
        }
        top = warp_max(top);
        if (lane == 0) tops[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WARPS; i++) top = fmaxf(top, tops[i]);
        for (int i = threadIdx.x; i < parts; i += 32 * WARPS) {
            weight[i] = weigh(weight[i]);
            sum += weight[i];
        }
        sum = warp_sum(sum);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kFirst; i++)
            if (warp + i * WARPS < parts) add(weight[warp + i * WARPS], y[i]);
#pragma unroll 8
        for (int i = warp + kFirst * WARPS; i < parts; i += WARPS) {
            float4 z[2];
            load(i, z);
            add(weight[i], z);
        }
    } else {
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, lse[part(i) * a.rows]);
        top = warp_max(top);
#pragma unroll
        for (int i = 0; i < kFirst; i++)
            if (warp + i * WARPS < parts) {
                const float f = weigh(lse[part(warp + i * WARPS) * a.rows]);
                sum += f;
                add(f, y[i]);
            }
#pragma unroll 4
        for (int i = warp + kFirst * WARPS; i < parts; i += WARPS) {
            float4 z[2];
            load(i, z);
            const float f = weigh(lse[part(i) * a.rows]);
            sum += f;
            add(f, z);
        }
    }
    if (lane == 0) totals[warp] = sum;
#pragma unroll
    for (int k = 0; k < 2; k++) *(float4 *)&sums[warp][k * 128 + lane * 4] = x[k];
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; i++) all += totals[i];
    for (int d = threadIdx.x; d < a.d; d += 32 * WARPS) {
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; i++) z += sums[i][d];
        store(d, z / all);
    }
}

// --------------------------------------------------------------- host ---

// How a call is computed: query heads of a block of a group, how many blocks, and
// the workspace.
struct ReadPlan {
    int nt, zs, heads, rows, workers;
    uint64_t tiles, lse_at, o_at, bytes;  // tiles: of all key heads, at most
};

// DC as the kernels are instantiated for it
static int read_dc(bool kv4, uint32_t d) { return kv4 ? (int)d / 32 : d <= 64 ? 4 : d <= 128 ? 8 : 16; }

// most: as many keys as all sequences have together, or more.
static ReadPlan read_plan(bool kv4, uint32_t seqs, uint64_t most, uint32_t kv_heads, uint32_t group, uint32_t d)
{
    ReadPlan w;
    w.nt = group > 8 && d <= 128 ? 2 : 1;  // with heads of 256 the results of 16 would not fit the registers
    w.zs = (int)(group + 8 * w.nt - 1) / (8 * w.nt);
    w.heads = (int)kv_heads * w.zs;
    w.rows = (int)std::min<uint32_t>(group, 8 * w.nt);
    w.workers = read_blocks(kv4, read_dc(kv4, d), w.nt) * tc_sm_count() * kRdWarps;
    w.tiles = (most / (kv4 ? 32 : 16) + seqs) * w.heads;
    const uint64_t parts = 2ull * w.workers;
    auto up = [](uint64_t x) { return (x + 31) / 32 * 32; };
    w.lse_at = up((seqs + 1ull) * 4);
    w.o_at = up(w.lse_at + parts * w.rows * 4);
    w.bytes = w.o_at + parts * w.rows * d * 4 + 32;
    return w;
}

// The kernels' launches, each compiled apart (aie_read16.cu, aie_read4_f16.cu, aie_read4_bf16.cu).
cudaError_t read16_run(const ReadArgs &a, int nt, cudaStream_t s);
cudaError_t read4_run_f16(const ReadArgs &a, int nt, cudaStream_t s);
cudaError_t read4_run_bf16(const ReadArgs &a, int nt, cudaStream_t s);

template <typename T, bool KV4, int DC, int NT>
static cudaError_t read_launch(const ReadArgs &a, cudaStream_t s)
{
    constexpr int stages = ReadRing<KV4, DC, NT>::kStages;
    constexpr uint32_t one = ReadRing<KV4, DC, NT>::kOne;
    auto *fn = &read_kernel<T, KV4, DC, NT, stages>;
    cudaError_t e = ensure_smem_attr((const void *)fn, stages * one);
    if (e != cudaSuccess) return e;
    e = launch_behind(fn, (unsigned)(a.workers / kRdWarps), kRdThreads, stages * one, s, a);
    if (e != cudaSuccess) return e;
    const JoinArgs j{a.out, a.o_ts, a.o_hs, a.before, a.part_lse, a.part_o, a.seqs, a.hq, a.group, a.d, a.zs, a.heads, a.rows, a.bf16,
                     a.workers};
    // warps a row, by its parts, as many as there were if all sequences had the same length
    // (the host does not know them; a long one among many short ones is joined by few warps
    // for its parts: 50000 states among 95 sequences of 100, 73 us a call): with two each (256 streams of up to 1900 places in 4 bits)
    // 87.4 us a call of two warps, 91.3 of four; with three (96 of 5000) 83.4 and 81.5; with
    // 600 (one of 9682 states) 14.8 of sixteen, 21 of eight, 31 of four; with 15, 14.4 of
    // four and 15.5 of sixteen
    const unsigned rows = (unsigned)((long long)a.seqs * a.hq);
    if (a.parts_each <= 2) return launch_behind(read_join_kernel<2>, rows, 64, 0, s, j);
    if (a.parts_each <= 24) return launch_behind(read_join_kernel<4>, rows, 128, 0, s, j);
    return launch_behind(read_join_kernel<16>, rows, 512, (a.workers + 2) * 4, s, j);
}

static void read_args(ReadArgs &a, const ReadPlan &w, const aie_heads &q, const aie_heads &out, void *workspace)
{
    a.q = q.data; a.q_ts = q.token_stride; a.q_hs = q.head_stride;
    a.out = out.data; a.o_ts = out.token_stride; a.o_hs = out.head_stride;
    a.most = (unsigned)(w.tiles / w.heads);
    a.zs = w.zs; a.heads = w.heads; a.rows = w.rows; a.workers = w.workers;
    a.parts_each = (unsigned)(std::min<uint64_t>(w.workers, w.tiles) / ((uint64_t)w.heads * a.seqs)) + 1;
    char *ws = (char *)(((uintptr_t)workspace + 31) / 32 * 32);
    a.before = (unsigned *)ws;
    auto vec = [](const aie_heads &h) {
        const uint64_t bits = (uintptr_t)h.data | 2 * h.token_stride | 2 * h.head_stride;
        return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
    };
    a.q_vec = vec(q); a.o_vec = vec(out);
    a.part_lse = (float *)(ws + w.lse_at);
    a.part_o = (float *)(ws + w.o_at);
}

template <typename T>
static cudaError_t read4_launch(const ReadArgs &a, int nt, cudaStream_t s)
{
    switch (a.d / 32) {
    case 1: return nt == 2 ? read_launch<T, true, 1, 2>(a, s) : read_launch<T, true, 1, 1>(a, s);
    case 2: return nt == 2 ? read_launch<T, true, 2, 2>(a, s) : read_launch<T, true, 2, 1>(a, s);
    case 3: return nt == 2 ? read_launch<T, true, 3, 2>(a, s) : read_launch<T, true, 3, 1>(a, s);
    case 4: return nt == 2 ? read_launch<T, true, 4, 2>(a, s) : read_launch<T, true, 4, 1>(a, s);
    case 5: return read_launch<T, true, 5, 1>(a, s);
    case 6: return read_launch<T, true, 6, 1>(a, s);
    case 7: return read_launch<T, true, 7, 1>(a, s);
    default: return read_launch<T, true, 8, 1>(a, s);
    }
}

template <typename T>
static cudaError_t read16_launch(const ReadArgs &a, int nt, cudaStream_t s)
{
    if (a.d > 128) return read_launch<T, false, 16, 1>(a, s);
    if (a.d > 64) return nt == 2 ? read_launch<T, false, 8, 2>(a, s) : read_launch<T, false, 8, 1>(a, s);
    return nt == 2 ? read_launch<T, false, 4, 2>(a, s) : read_launch<T, false, 4, 1>(a, s);
}

}  // namespace aie
