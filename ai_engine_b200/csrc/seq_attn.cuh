// Attention on the tensor cores (tcgen05, f16 / bf16 operands, f32 sums):
// whole packed prompts, the shared prefix of a batch of streams, and packed
// tokens over states of another length.
//
//   S = Q K^T,  P = e^(scale (S - m)),  l = sum P,  O = P V,  out = O / l
//
// over 128 keys at a time with the maximum m, the sum l and O carried along.
// A tile is 128 query rows of one key/value head: `tokens_per_tile` tokens
// times the group of query heads that read that head, so that grouped heads
// share each key tile.  A block works on two tiles in turn: while the tensor
// core multiplies for one, the other's rows are exponentiated.
//
//   warps 0-3, 4-7   rows of tile 0 and 1, one thread per row: S from tensor
//                    memory, running maximum and sum, P back to tensor memory
//   warp 8           TMA: Q once, then K and V tiles through a ring
//   warp 9           MMA issue, the two tiles in turn: S_w(j+1) follows
//                    O_w += P_w(j) V(j), so a finished S tells the rows that O
//                    may be touched too.  (An issuer for each tile lets their
//                    products interleave and both tiles' rows wait at the same
//                    time: 962 us for two prompts of 8192 and 6001 tokens, 32
//                    heads, against 771 us.)
//   warp 10          tells it when K and V tiles have arrived
//   warp 11          nothing (it fills the issuing warpgroup)
//
// The carried m is only moved when a row's maximum has grown by more than 8
// binary orders: until then P <= 2^8, and out = O / l is the same ratio for
// any m.  Moving it rescales O in tensor memory, which few tiles need.
//
// Rounding to fewer bits: P to the operands' type (as the tensor core wants
// it; l sums the unrounded P in f32), and the result.  f16 weights are held
// 2^7 times as large (kWeightShift), up to 2^15: at 1 for the largest, those
// below 2^-14 would lose bits and those below 2^-25 vanish, which adds up over
// a long context (one key 22.6 binary orders above 32768 equal ones: 0.0058
// for 0.0051).  Exponents only: no instruction more.
//
// Tokens over states (CROSS): where there are fewer pairs of tiles than SMs, a
// pair's steps are cut into parts of about as many as make one wave of blocks;
// each part leaves (O / l, log2 of the weights' sum), which cross_join_kernel
// joins as the shared prefix's pieces are.  Every block works the cut out from
// the sequences' lengths, which the host does not know.
//
// Where sequences have no more tokens than fill one tile (FEW), both tiles are the
// same rows, and take the steps in turn: a step's chain of scores, exponentials
// and products is 1.7 us long, and nothing else would hide it.  (Short questions
// about long clips, 12 steps a block: 15.6 us for the steps, which is 5.7 TB/s,
// against 24 with one tile, or with half of every step's keys for each.)  Such a
// question takes 35.5 us a call for 89 MB, of them 34 here: cutting the work, the
// first copies and the exchange are the rest.  Long texts over states (5095 tokens,
// 32/8 heads of 128) run at the prompts' rate, 1.02 PFLOP/s.
//
// At 168 registers a thread the prompts' form spills 8 bytes, the paged one 12,
// that of states 8, FEW 72 (32 with heads of up to 64).
//
// Every wait is bounded (1 s); on expiry the block records an error code,
// waits for its copies in flight, frees its tensor memory and returns.
#pragma once
#include "seq_common.cuh"
#include "tc_ptx.cuh"

namespace aie {

constexpr int kAtThreads = 384;
// Registers a thread: 384 x 168 at launch; a row's 128 scores stay in
// registers, so the two row warpgroups take 216 each (2 x 128 x 216 + 128 x 72
// = 384 x 168) and the third, which only issues, keeps 72.
constexpr int kAtRowRegs = 216, kAtIssueRegs = 72;
constexpr int kAtTile = 128;      // query rows of a tile, keys of a step
constexpr uint32_t kAtBlockBytes = kAtTile * 128;  // 128 rows of 64 16-bit elements
constexpr int kAtMostSplits = 64; // pieces of the shared prefix
constexpr uint32_t kAtErr = 0x41000000u;

// Binary orders by which a row's weights (and with them l and O) are larger
// than 2^(s - m), which is at most 2^8: as much as f16 holds.  bf16 has the
// range of f32.
template <typename T>
constexpr float kWeightShift = std::is_same<T, __half>::value ? 7.f : 0.f;

// --------------------------------------------------------------- PTX ---

// Instruction descriptor, kind::f16: D f32, A and B of one type, A K-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t n, bool b_mn_major)
{
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) |
           ((uint32_t)(kAtTile >> 4) << 24);
}

// V as B operand: its rows (keys) are the K side, 64 elements of a head wide
// per 128-byte swizzled row; the next 64 elements one block further on.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr)
{
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)(kAtBlockBytes >> 4) << 16;  // leading: to the next 64 elements
    d |= (uint64_t)(1024 >> 4) << 32;           // stride: to the next 8 keys
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v)
{
    uint32_t *r = (uint32_t *)v;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// Completes the loads; the destinations go through it so that no use moves above.
__device__ __forceinline__ void tmem_wait_ld32(float *v)
{
    uint32_t *r = (uint32_t *)v;
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void store32(void *p, const uint32_t *v)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------- kernel ---

struct AttnArgs {
    const int32_t *cu;        // prompts: the sequences' starts
    const int32_t *prefix;    // shared prefix: its pages
    const int32_t *lens;      // shared prefix: the streams' lengths
    void *out;                // prompts: the result
    long long out_ts, out_hs;
    float *part_o, *part_lse; // shared prefix: [split][row][d] and [split][row], row = stream * q_heads + head
    int tokens, seqs;         // prompts: packed tokens; shared prefix: streams
    int kv_heads, q_heads, group, d, tokens_per_tile;
    int pair_tokens;          // states: tokens of a pair of tiles, that of one where both are the same rows
    int causal;
    int out_bytes;            // what `out` is aligned to, in every row: 32, 16 or less
    int shared, max_len, page_size, pages, box_rows, splits, tiles_per_split;
    float scale_log2;
    const int32_t *cu_k;      // states: the sequences' starts
    int keys;                 // packed states
    // splits: parts that there is room for
    int capacity;             // blocks of a key head that run at once; 0: steps are not cut
};

constexpr int kAtPrompt = 0, kAtPaged = 1, kAtCross = 2, kAtFew = 3;  // what attn_tc_kernel attends to
constexpr int kCrossBox = 32;  // states of a copy
constexpr int kAtLeast = 4;  // steps that a block is worth starting for: its start and end take about 3

template <int DB, bool FEW>
struct AttnSmem {
    static constexpr int kStages = DB == 2 ? (FEW ? 6 : 5) : 8;
    static constexpr uint32_t kQ = (FEW ? 1 : 2) * DB * kAtBlockBytes;
    static constexpr uint32_t kStage = DB * kAtBlockBytes;
    static constexpr uint32_t kBytes = kQ + kStages * kStage + 1024 /* alignment */;
};

struct AttnShared {
    uint64_t q_full, kv_full[8], kv_empty[8], s_full[2], p_full[2][2], o_full[2], drain;
    uint32_t tmem, abort;
    int seq_first, seq_len, pair, key_first, key_len, part, parts, per;
};

// What one block does: tile pair `pair` of tokens first .. first + len.
struct AttnWork {
    int first, len, pair, kvh, split;
};

// A pair of tiles of tokens over states, and its share of their steps: part
// `part` of `parts`, `per` steps each; base is the number of its first part.
struct CrossWork {
    int first, len, pair, key_first, key_len, part, parts, per;
    long long base;
};

// By one warp: the pair with number `pair` among all, or the part with number
// `unit` among all pairs' parts (the other is -1).  128 sequences at a time, 4 a
// lane.  Only the lane that returns true has it.
__device__ __forceinline__ bool cross_find(const AttnArgs &a, int unit, int pair, int lane, CrossWork &w)
{
    const int two = a.pair_tokens;
    int start[4], len[4], key[4], key_len[4], pairs[4], steps[4];
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = min(s0 + 4 * lane + i, a.seqs), next = min(s + 1, a.seqs);
            start[i] = min(max(a.cu[s], 0), a.tokens);
            len[i] = max(min(max(a.cu[next], 0), a.tokens) - start[i], 0);
            key[i] = min(max(a.cu_k[s], 0), a.keys);
            key_len[i] = max(min(max(a.cu_k[next], 0), a.keys) - key[i], 0);
            pairs[i] = (len[i] + two - 1) / two;
            steps[i] = (key_len[i] + kAtTile - 1) / kAtTile;
        }
    };
    int per = 0x7fffffff;  // steps of a part
    if (a.capacity) {
        long long work = 0, n = 0;
        for (int s0 = 0; s0 < a.seqs; s0 += 128) {
            load(s0);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                work += (long long)pairs[i] * steps[i];
                n += pairs[i];
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            work += __shfl_xor_sync(0xffffffffu, work, o);
            n += __shfl_xor_sync(0xffffffffu, n, o);
        }
        // a pair's last part is not full: room for one more each, where there is any
        const long long room = a.capacity > 2 * n ? a.capacity - n : a.capacity;
        per = (int)min(max((work + room - 1) / room, (long long)kAtLeast), 0x7fffffffll);
    }
    long long units_before = 0;
    int pairs_before = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += 128) {
        if (s0 || a.seqs > 128 || !a.capacity) load(s0);
        int sum = 0, sum_units = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sum += pairs[i];
            sum_units += pairs[i] * max((steps[i] + per - 1ll) / per, 1ll);
        }
        int upto = sum, upto_units = sum_units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o), z = __shfl_up_sync(0xffffffffu, upto_units, o);
            if (lane >= o) {
                upto += y;
                upto_units += z;
            }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, unit >= 0 ? unit < units_before + upto_units : pair < pairs_before + upto);
        if (hit) {
            if (lane != __ffs(hit) - 1) return false;
            long long u = units_before + upto_units - sum_units;
            int n = pairs_before + upto - sum;
            bool found = false;  // always, unless a list that decreases overflowed the sums
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int parts = (int)max((steps[i] + per - 1ll) / per, 1ll);
                if (unit >= 0 ? unit >= u && unit < u + pairs[i] * parts : pair >= n && pair < n + pairs[i]) {
                    const int in = unit >= 0 ? (int)(unit - u) : (pair - n) * parts;
                    w = CrossWork{start[i], len[i], in / parts, key[i], key_len[i], in % parts, parts, per, u + in / parts * parts};
                    found = true;
                }
                u += pairs[i] * parts;
                n += pairs[i];
            }
            return found;
        }
        units_before += __shfl_sync(0xffffffffu, upto_units, 31);
        pairs_before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <typename T, int DB, int MODE>
__global__ void __launch_bounds__(kAtThreads, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const AttnArgs a)
{
    constexpr bool PAGED = MODE == kAtPaged, FEW = MODE == kAtFew, CROSS = MODE == kAtCross || FEW;
    constexpr int kTurns = FEW ? 2 : 1;  // tiles that take the steps in turn
    using Sm = AttnSmem<DB, FEW>;
    extern __shared__ char smem_raw[];
    __shared__ AttnShared sh;
    char *smem = (char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    char *const sq = smem, *const skv = smem + Sm::kQ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tpt = a.tokens_per_tile;

    // tensor memory, barriers, the maps' descriptors: each by a warp of its own
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 32 * 8) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_q)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
    }
    if (threadIdx.x == 32 * 10) {
        mbar_init(&sh.q_full, 1);
        for (int i = 0; i < Sm::kStages; i++) {
            mbar_init(&sh.kv_full[i], 1);
            mbar_init(&sh.kv_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i][0], 5);
            mbar_init(&sh.p_full[i][1], 4);
            mbar_init(&sh.o_full[i], 1);
        }
        mbar_init(&sh.drain, 1);
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // also for the streams' own part (prefix_step_kernel), which may then start
    // beside this one
    behind_last_launch();

    // ---- which tokens, which keys
    AttnWork w;
    w.kvh = blockIdx.x % a.kv_heads;
    int unit = blockIdx.x / a.kv_heads;
    if constexpr (PAGED) {
        w.split = unit % a.splits;
        w.pair = unit / a.splits;
        w.first = 0;
        w.len = a.tokens;
    } else if constexpr (CROSS) {
        if (warp == 0) {
            if (lane == 0) sh.seq_len = 0;
            __syncwarp();
            CrossWork c;
            if (cross_find(a, unit, -1, lane, c)) {
                sh.seq_first = c.first;
                sh.seq_len = c.len;
                sh.pair = c.pair;
                sh.key_first = c.key_first;
                sh.key_len = c.key_len;
                sh.part = c.part;
                sh.parts = c.parts;
                sh.per = c.per;
            }
        }
    } else {
        w.split = 0;
        if (warp == 0) {
            // unit -> (sequence, pair of tiles): 128 sequences at a time, 4 a lane
            int at = 0;
            bool found = false;
            for (int s0 = 0; s0 < a.seqs && !found; s0 += 128) {
                int start[5], pairs[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 5; i++) start[i] = min(max(a.cu[min(s0 + 4 * lane + i, a.seqs)], 0), a.tokens);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    pairs[i] = (max(start[i + 1] - start[i], 0) + 2 * tpt - 1) / (2 * tpt);
                    sum += pairs[i];
                }
                int upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, unit < at + upto);
                if (hit) {
                    found = true;
                    if (lane == __ffs(hit) - 1) {
                        int left = unit - (at + upto - sum);  // among this lane's pairs
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (left >= 0 && left < pairs[i]) {
                                sh.seq_first = start[i];
                                sh.seq_len = start[i + 1] - start[i];
                                // a causal sequence's last tiles see the most keys: first
                                sh.pair = pairs[i] - 1 - left;
                            }
                            left -= pairs[i];
                        }
                    }
                }
                at += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (!found && lane == 0) sh.seq_len = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    if constexpr (!PAGED) {
        w.first = sh.seq_first;
        w.len = sh.seq_len;
        w.pair = sh.pair;
        if constexpr (CROSS) w.split = sh.part;
        if (w.len == 0) {  // a block past the last pair
            if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
            return;
        }
    }
    // keys seen by a tile's last token; `keys` also bounds the values that exist
    const int tok0 = w.pair * (FEW ? 1 : 2) * tpt;
    const int keys = PAGED ? min(a.shared, a.max_len) : CROSS ? sh.key_len : w.len;
    const int key_first = CROSS ? sh.key_first : w.first;
    const int per_split = PAGED ? a.tiles_per_split : CROSS ? sh.per : 0, step0 = w.split * per_split;
    const bool parts = PAGED || (CROSS && sh.parts > 1);  // a partial result, not the result
    auto steps_of = [&](int t) {
        const int first = tok0 + (FEW ? 0 : t * tpt), last = min(first + tpt, w.len);
        const int seen = first >= w.len ? 0 : (MODE == kAtPrompt && a.causal) ? last : keys;
        const int steps = (seen + kAtTile - 1) / kAtTile;
        return MODE != kAtPrompt ? max(min(steps - step0, per_split), 0) + step0 : steps;
    };
    const int n0 = steps_of(0), n1 = FEW && n0 - step0 < 2 ? step0 : steps_of(1), n = max(n0, n1);
    auto n_of = [&](int t) { return t ? n1 : n0; };
    volatile uint32_t *abort = &sh.abort;
    auto wait = [&](uint64_t *bar, uint32_t parity, uint32_t site) {
        if (mbar_wait(bar, parity)) return true;
        report_error(kAtErr | site);
        *abort = 1;
        return false;
    };

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kAtRowRegs));
        // ---- rows
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const int tok = tok0 + (FEW ? 0 : t * tpt) + row / a.group, head = w.kvh * a.group + row % a.group;
        const bool real = row < tpt * a.group && tok < w.len;
        int seen = keys;
        if constexpr (PAGED) {
            if (real) seen = min(seen, max(a.lens[tok], 0));
        } else if constexpr (!CROSS) {
            if (a.causal) seen = min(tok + 1, keys);
        }
        const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * 128, to = ts + 256;
        const float sl = a.scale_log2;
        float m = -INFINITY;           // carried reference maximum, in units of S
        float2 l2 = make_float2(0.f, 0.f);
        bool ok = true;
        const int nt = n_of(t);
        for (int j = step0 + (FEW ? t : 0); j < nt; j += kTurns) {
            ok = wait(&sh.s_full[t], ((j - step0) / kTurns) & 1, 7);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            float s[kAtTile];
#pragma unroll
            for (int i = 0; i < kAtTile / 32; i++) tmem_ld32(ts + 32 * i, s + 32 * i);
#pragma unroll
            for (int i = 0; i < kAtTile / 32; i++) tmem_wait_ld32(s + 32 * i);
            const int here = seen - j * kAtTile;
            if (__any_sync(0xffffffffu, here < kAtTile)) {
#pragma unroll
                for (int i = 0; i < kAtTile; i++) s[i] = i < here ? s[i] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < kAtTile - 4; i += 8) {
                mx[0] = max3(mx[0], s[i], s[i + 1]);
                mx[1] = max3(mx[1], s[i + 2], s[i + 3]);
                mx[2] = max3(mx[2], s[i + 4], s[i + 5]);
                mx[3] = max3(mx[3], s[i + 6], s[i + 7]);
            }
            mx[0] = max3(mx[0], s[kAtTile - 4], s[kAtTile - 3]);
            mx[1] = max3(mx[1], s[kAtTile - 2], s[kAtTile - 1]);
            const float top = fmaxf(max3(mx[0], mx[1], mx[2]), fmaxf(mx[3], m));
            // -inf - -inf is NaN: not greater, nothing to move
            const bool grow = (top - m) * sl > 8.f;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2((m - top) * sl) : 1.f;  // from -inf: 0
                if (grow) m = top;
                if (j >= step0 + kTurns) {
                    l2.x *= f;
                    l2.y *= f;
#pragma unroll
                    for (int c = 0; c < 2 * DB; c++) {
                        float o[32];
                        tmem_ld32(to + 32 * c, o);
                        tmem_wait_ld32(o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] *= f;
                        tmem_st32(to + 32 * c, (const uint32_t *)o);
                    }
                }
            }
            float off = m == -INFINITY ? 0.f : fmaf(-m, sl, kWeightShift<T>);
            if constexpr (CROSS) {
                // Scores so large that the rounding of m sl counts (beyond 2^27 it is more than
                // f16 holds): the difference first.  Too dear for every step.
                if (__any_sync(0xffffffffu, m != -INFINITY && fabsf(m) * sl >= 65536.f)) {
                    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int i = 0; i < kAtTile; i++) s[i] -= base;
                    off = m == -INFINITY ? 0.f : kWeightShift<T>;
                }
            }
            const float2 sl2 = make_float2(sl, sl), off2 = make_float2(off, off);
#pragma unroll
            for (int c = 0; c < kAtTile / 64; c++) {
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const float2 x = __ffma2_rn(make_float2(s[64 * c + 2 * i], s[64 * c + 2 * i + 1]), sl2, off2);
                    const float2 e = make_float2(ex2(x.x), ex2(x.y));
                    l2 = __fadd2_rn(l2, e);
                    p[i] = pack2<T>(e.x, e.y);
                }
                tmem_st32(ts + 32 * c, p);
                // half of the keys are enough to begin
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t][c]);
            }
        }
        // ---- result
        const float l = l2.x + l2.y;
        if (nt > step0 && ok) ok = __all_sync(0xffffffffu, wait(&sh.o_full[t], 0, 8));
        tc_fence_after();
        // of this split's keys; scores of -inf alone (l is 0) count as none here
        const bool none = nt <= step0 || seen <= (step0 + (FEW ? t : 0)) * kAtTile || ((parts || FEW) && l == 0.f);
        const float r = none ? 0.f : 1.f / l;
        const float lse = none ? -INFINITY : fmaf(m, sl, log2f(l) - kWeightShift<T>);  // log2 of the weights' sum
        const long long prow = PAGED   ? ((long long)w.split * a.tokens + tok) * a.q_heads + head
                               : FEW   ? (long long)blockIdx.x * kAtTile + row
                               : CROSS ? (long long)blockIdx.x * (2 * kAtTile) + t * kAtTile + row
                                       : 0;
        const long long at = parts ? prow * a.d : (w.first + tok) * a.out_ts + head * a.out_hs;
        // 32 columns at a time out of tensor memory: a thread holds a row and
        // writes whole 32-byte sectors of it (16-byte pieces: 2 us a tile, so: 1)
        auto fetch = [&](int c, float (&o)[32]) {
            if (nt > step0) {
                tmem_ld32(to + 32 * c, o);
                tmem_wait_ld32(o);
            }
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = none ? 0.f : o[i] * r;
        };
        auto put = [&](int c, float (&o)[32]) {
#pragma unroll
            for (int i = 0; i < 32; i += PAGED ? 8 : 16) {
                if (32 * c + i >= a.d) break;
                if constexpr (PAGED) {
                    store32(a.part_o + at + 32 * c + i, (const uint32_t *)&o[i]);
                } else if (CROSS && parts) {
                    store32(a.part_o + at + 32 * c + i, (const uint32_t *)&o[i]);
                    if (32 * c + i + 8 < a.d) store32(a.part_o + at + 32 * c + i + 8, (const uint32_t *)&o[i + 8]);
                } else {
                    T *dst = (T *)a.out + at + 32 * c + i;
                    uint32_t v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = pack2<T>(o[i + 2 * e], o[i + 2 * e + 1]);
                    if (a.out_bytes == 32) store32(dst, v);
                    else if (a.out_bytes == 16) {
                        ((uint4 *)dst)[0] = make_uint4(v[0], v[1], v[2], v[3]);
                        if (32 * c + i + 8 < a.d) ((uint4 *)dst)[1] = make_uint4(v[4], v[5], v[6], v[7]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (32 * c + i + e < a.d) dst[e] = from_f32<T>(o[i + e]);
                    }
                }
            }
        };
        if constexpr (FEW) {
            // a row's two results become one: the other tile's thread gets half of the
            // columns, by way of the ring, which is free once all products are done
            constexpr int kPad = 32 * DB + 4;
            float *const halves = (float *)skv, *const lses = halves + 2 * kAtTile * kPad;
            if (ok && n_of(1 - t) > step0) ok = __all_sync(0xffffffffu, wait(&sh.o_full[1 - t], 0, 8));
            tc_fence_after();
            if (ok) {
                lses[t * kAtTile + row] = lse;
#pragma unroll 1
                for (int c = 0; c < DB; c++) {
                    float o[32];
                    fetch((1 - t) * DB + c, o);
                    float4 *const to_ = (float4 *)(halves + (t * kAtTile + row) * kPad + 32 * c);
#pragma unroll
                    for (int i = 0; i < 8; i++) to_[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (ok) {
                const float other = lses[(1 - t) * kAtTile + row], top = fmaxf(lse, other);
                const float w0 = lse == -INFINITY ? 0.f : ex2(lse - top), w1 = other == -INFINITY ? 0.f : ex2(other - top), sum = w0 + w1;
                // no keys: zeros; keys with scores of -inf alone: NaN, or a part without weight
                const float f = sum == 0.f && (parts || !keys) ? 0.f : 1.f / sum;
                if (parts && t == 0 && real) a.part_lse[prow] = sum == 0.f ? -INFINITY : top + log2f(sum);
#pragma unroll 1
                for (int c = t * DB; c < t * DB + DB; c++) {
                    float o[32];
                    fetch(c, o);
                    const float4 *const from = (const float4 *)(halves + ((1 - t) * kAtTile + row) * kPad + 32 * (c - t * DB));
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float4 x = from[i];
                        o[4 * i] = f * fmaf(w0, o[4 * i], w1 * x.x);
                        o[4 * i + 1] = f * fmaf(w0, o[4 * i + 1], w1 * x.y);
                        o[4 * i + 2] = f * fmaf(w0, o[4 * i + 2], w1 * x.z);
                        o[4 * i + 3] = f * fmaf(w0, o[4 * i + 3], w1 * x.w);
                    }
                    if (real) put(c, o);
                    __syncwarp();
                }
            }
        } else if (ok && (nt > step0 || MODE != kAtPrompt)) {
            if (MODE != kAtPrompt && parts && real) a.part_lse[prow] = lse;
            bool nan = false;
#pragma unroll 1
            for (int c = 0; c < 2 * DB; c++) {
                float o[32];
                fetch(c, o);
                if (PAGED && seen < keys)
#pragma unroll
                    for (int i = 0; i < 32; i++) nan |= o[i] != o[i];
                if (real) put(c, o);
                __syncwarp();
            }
            // A stream that ends in the prefix, and a result of NaN: values that it does
            // not see may have made it so (0 times them).  prefix_step_kernel works
            // it out anew where this says so.
            if (nan && real) a.part_lse[prow] = __int_as_float(0x7fffffff);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAtIssueRegs));
        if (warp == 8) {
            // ---- copies.  Ring order: K(0) V(0) K(1) V(1) ...
            if (n > step0) {
                if (lane == 0) {
                    const uint32_t q_bytes = (uint32_t)tpt * a.group * 128 * DB;
                    const int tiles = !FEW && n1 > step0 ? 2 : 1;
                    mbar_expect_tx(&sh.q_full, q_bytes * tiles);
                    for (int t = 0; t < tiles; t++)
                        for (int b = 0; b < DB; b++)
                            tma_load_3d(sq + (t * DB + b) * kAtBlockBytes, &tm_q, &sh.q_full, b * 64, w.kvh * a.group,
                                        w.first + tok0 + t * tpt);
                }
                // paged: each lane copies one page's part of a tile
                const int rows = PAGED ? a.box_rows : kAtTile;
                auto page_of = [&](int step) {
                    const int place = step * kAtTile + lane * rows;
                    // past the prefix: a page that does not exist, read as zeros
                    const int page = lane * rows < kAtTile && place < a.shared ? a.prefix[place / a.page_size] : a.pages;
                    return page < 0 || page > a.pages ? a.pages : page;
                };
                int page = 0, next = 0;
                if constexpr (PAGED) next = page_of(step0);
                int issued = 0;
                for (int i = 0; i < 2 * (n - step0) + (FEW ? 1 : 0); i++) {
                    // (FEW: K of two steps, then V of both; an odd last step has no second)
                    const int st = i % Sm::kStages, round = i / Sm::kStages, step = step0 + (FEW ? i / 4 * 2 + (i & 1) : i / 2);
                    if (FEW && step >= n) continue;
                    const CUtensorMap *tm = (FEW ? i & 2 : i & 1) ? &tm_v : &tm_k;
                    char *dst = skv + st * Sm::kStage;
                    int go = 1;
                    if (lane == 0) {
                        go = !*abort && (!round || wait(&sh.kv_empty[st], (round - 1) & 1, 1));
                        if (go) mbar_expect_tx(&sh.kv_full[st], Sm::kStage);
                    }
                    go = __shfl_sync(0xffffffffu, go, 0);
                    if (!go) break;
                    if constexpr (PAGED) {
                        if (!(i & 1)) {
                            page = next;
                            if (step + 1 < n) next = page_of(step + 1);
                        }
                        if (lane * rows < kAtTile)
                            for (int b = 0; b < DB; b++)
                                tma_load_4d(dst + b * kAtBlockBytes + lane * rows * 128, tm, &sh.kv_full[st], b * 64, w.kvh,
                                            (step * kAtTile + lane * rows) % a.page_size, page);
                    } else if constexpr (CROSS) {
                        // four lanes to 64 elements of 128 states (texts over clips: 589 us, 600 with one)
                        if (lane < DB * (kAtTile / kCrossBox))
                            tma_load_3d(dst + lane % DB * kAtBlockBytes + lane / DB * (kCrossBox * 128), tm, &sh.kv_full[st], lane % DB * 64,
                                        w.kvh, key_first + step * kAtTile + lane / DB * kCrossBox);
                    } else if (lane == 0) {
                        for (int b = 0; b < DB; b++)
                            tma_load_3d(dst + b * kAtBlockBytes, tm, &sh.kv_full[st], b * 64, w.kvh, key_first + step * kAtTile);
                    }
                    issued = i + 1;
                }
                // nothing may still be written to this block's memory when it ends
                if (*abort && lane == 0) {
                    mbar_wait(&sh.q_full, 0);
                    for (int i = max(issued - Sm::kStages, 0); i < issued; i++)
                        if (!FEW || step0 + i / 4 * 2 + (i & 1) < n) mbar_wait(&sh.kv_full[i % Sm::kStages], (i / Sm::kStages) & 1);
                }
                __syncwarp();
            }
        } else if (warp == 9) {
            // ---- products, all from one thread
            constexpr uint32_t id_s = idesc_f16<T>(kAtTile, false), id_o = idesc_f16<T>(64 * DB, true);
            if (lane == 0 && n > step0) {
                const uint64_t qd0 = smem_desc_sw128(smem_u32(sq)), kd0 = smem_desc_sw128(smem_u32(skv)),
                               vd0 = smem_desc_mn_sw128(smem_u32(skv));
                auto s_mma = [&](int t, uint32_t k) {
                    const uint64_t qd = qd0 + (FEW ? 0 : t * (DB * kAtBlockBytes >> 4)), kd = kd0 + k * (Sm::kStage >> 4);
#pragma unroll
                    for (int i = 0; i < 4 * DB; i++) {
                        const uint32_t off = ((i / 4) * kAtBlockBytes + (i % 4) * 32) >> 4;
                        mma_f16_ss(tmem + t * 128, qd + off, kd + off, id_s, i > 0);
                    }
                    mma_commit(&sh.s_full[t]);
                };
                // half h of the keys: 64 of them
                auto o_mma = [&](int t, uint32_t v, int h, bool first) {
                    const uint64_t vd = vd0 + v * (Sm::kStage >> 4);
#pragma unroll
                    for (int i = 4 * h; i < 4 * h + 4; i++)
                        mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + i * 8, vd + (uint32_t)(i * 2048 >> 4), id_o,
                                   !first || i > 0);
                };
                bool ok = wait(&sh.q_full, 0, 2) && wait(&sh.kv_full[0], 0, 3);
                if constexpr (FEW) {
                    // step i by tile i % 2: its K is copy 4 (i / 2) + i % 2, its V two further on
                    const int steps = n - step0;
                    for (int i = 0; ok && i < min(steps, 2); i++) {
                        if (i && !(ok = wait(&sh.kv_full[i], 0, 3))) break;
                        tc_fence_after();
                        s_mma(i, i);
                        mma_commit(&sh.kv_empty[i]);
                    }
                    for (int i = 0; ok && i < steps; i++) {
                        const int t = i & 1, iv = 2 * (i & ~1) + 2 + t, ik = iv + 2;
                        const uint32_t par = (i >> 1) & 1;
                        if (!(ok = wait(&sh.p_full[t][0], par, 6))) break;
                        tc_fence_after();
                        o_mma(t, iv % Sm::kStages, 0, i < 2);
                        if (!(ok = wait(&sh.p_full[t][1], par, 6))) break;
                        tc_fence_after();
                        o_mma(t, iv % Sm::kStages, 1, false);
                        mma_commit(&sh.kv_empty[iv % Sm::kStages]);
                        if (i + 2 < steps) {
                            s_mma(t, ik % Sm::kStages);
                            mma_commit(&sh.kv_empty[ik % Sm::kStages]);
                        } else mma_commit(&sh.o_full[t]);
                    }
                } else if (ok) {
                    tc_fence_after();
                    if (n0 > step0) s_mma(0, 0);
                    if (n1 > step0) s_mma(1, 0);
                    mma_commit(&sh.kv_empty[0]);
                }
                uint32_t vj = 1, kj = 2 % Sm::kStages, v_old = 0, k_old = 0;  // ring places of V(j), K(j + 1)
                for (int j = step0; !FEW && ok && j < n; j++) {
                    const uint32_t par = (j - step0) & 1;
                    if (j < n0) {
                        if (!(ok = wait(&sh.p_full[0][0], par, 6))) break;
                        tc_fence_after();
                        o_mma(0, vj, 0, j == step0);
                    }
                    // the last step's places, once this step's products run
                    if (j > step0 && j + 1 < n) {
                        mma_commit(&sh.kv_empty[v_old]);
                        mma_commit(&sh.kv_empty[k_old]);
                    }
                    if (j < n0) {
                        if (!(ok = wait(&sh.p_full[0][1], par, 6))) break;
                        tc_fence_after();
                        o_mma(0, vj, 1, false);
                        if (j + 1 < n0) s_mma(0, kj);
                        else mma_commit(&sh.o_full[0]);
                    }
                    if (j < n1) {
                        if (!(ok = wait(&sh.p_full[1][0], par, 6))) break;
                        tc_fence_after();
                        o_mma(1, vj, 0, j == step0);
                        if (!(ok = wait(&sh.p_full[1][1], par, 6))) break;
                        tc_fence_after();
                        o_mma(1, vj, 1, false);
                        if (j + 1 < n1) s_mma(1, kj);
                        else mma_commit(&sh.o_full[1]);
                    }
                    v_old = vj;
                    k_old = kj;
                    vj = vj + 2 >= Sm::kStages ? vj + 2 - Sm::kStages : vj + 2;
                    kj = kj + 2 >= Sm::kStages ? kj + 2 - Sm::kStages : kj + 2;
                }
                if (!ok) {
                    mma_commit(&sh.drain);
                    mbar_wait(&sh.drain, 0);
                }
            }
            __syncwarp();
        } else if (warp == 10 && n > step0) {
            // ---- the copies' side of p_full: V(j) and K(j + 1) are there.  (A
            // wait costs the issuing thread about 200 cycles even when there
            // is nothing to wait for, so it makes as few as it can.)
            for (int j = step0; j < n; j++) {
                const int turn = (j - step0) % kTurns, iv = FEW ? 2 * (j - step0 - turn) + 2 + turn : 2 * (j - step0) + 1, ik = FEW ? iv + 2 : iv + 1;
                bool ok = wait(&sh.kv_full[iv % Sm::kStages], (iv / Sm::kStages) & 1, 4);
                // values behind the last key may be anything, and 0 times them NaN: zeros
                const int real = keys - j * kAtTile;
                if (real < kAtTile) {
                    for (int i = real * 8 + lane; ok && i < kAtTile * 8; i += 32)
#pragma unroll
                        for (int b = 0; b < DB; b++)
                            *(uint4 *)(skv + iv % Sm::kStages * Sm::kStage + b * kAtBlockBytes + i * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (ok && j + kTurns < n) ok = wait(&sh.kv_full[ik % Sm::kStages], (ik / Sm::kStages) & 1, 5);
                // one arrival per step
                if constexpr (FEW) {
                    if (ok && j >= step0 + 2) ok = wait(&sh.p_full[turn][0], ((j - step0) / 2 - 1) & 1, 11);
                } else {
                    for (int t = 0; t < 2 && ok && j > step0; t++)
                        if (j - 1 < n_of(t)) ok = wait(&sh.p_full[t][0], (j - 1 - step0) & 1, 11);
                }
                if (!__all_sync(0xffffffffu, ok)) break;
                if (FEW && lane == 0) mbar_arrive(&sh.p_full[turn][0]);
                else if (lane == 0) {
                    if (j < n0) mbar_arrive(&sh.p_full[0][0]);
                    if (j < n1) mbar_arrive(&sh.p_full[1][0]);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Pairs of tiles whose steps were cut: the parts' results joined, a warp per row.
constexpr int kJoinRows = 8;  // of a block
template <typename T, bool FEW>
__global__ void __launch_bounds__(32 * kJoinRows) cross_join_kernel(const AttnArgs a)
{
    __shared__ CrossWork shared;
    __shared__ int found;
    behind_last_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    constexpr int kRows = FEW ? kAtTile : 2 * kAtTile;
    const int i = unit % (kRows / kJoinRows) * kJoinRows + warp, pair = unit / (kRows / kJoinRows);
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    if (warp == 0) {
        CrossWork c;
        if (cross_find(a, -1, pair, lane, c)) {
            shared = c;
            found = 1;
        }
    }
    __syncthreads();
    // (the last only where cu is no list of starts, and parts are missing)
    if (!found || shared.parts == 1 || shared.base + shared.parts > a.splits) return;
    const CrossWork w = shared;
    const int t = i / kAtTile, row = i % kAtTile, tok = w.pair * a.pair_tokens + t * a.tokens_per_tile + row / a.group;
    const int head = kvh * a.group + row % a.group;
    if (row >= a.tokens_per_tile * a.group || tok >= w.len) return;
    T *dst = (T *)a.out + (w.first + tok) * a.out_ts + head * a.out_hs + lane * 4;
    const long long first = (w.base * a.kv_heads + kvh) * kRows + i, next = a.kv_heads * kRows;
    const int parts = w.parts;
    auto at = [&](int part) { return first + part * next; };
    float top = -INFINITY;
    for (int part = lane; part < parts; part += 32) top = fmaxf(top, a.part_lse[at(part)]);
    top = warp_max(top);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int part0 = 0; part0 < parts; part0 += 32) {
        const int n = min(parts - part0, 32);
        const float lse = lane < n ? a.part_lse[at(part0 + lane)] : -INFINITY, mine = lse == -INFINITY ? 0.f : ex2(lse - top);
        sum += mine;
#pragma unroll 8
        for (int k = 0; k < n; k++) {
            const float f = __shfl_sync(0xffffffffu, mine, k);
            if (lane * 4 < a.d) {
                const float4 y = *(const float4 *)(a.part_o + at(part0 + k) * a.d + lane * 4);
                x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
            }
        }
    }
    const float f = 1.f / warp_sum(sum);
    if (lane * 4 < a.d) {
        dst[0] = from_f32<T>(x.x * f); dst[1] = from_f32<T>(x.y * f); dst[2] = from_f32<T>(x.z * f); dst[3] = from_f32<T>(x.w * f);
    }
}

// --------------------------------------------------------------- host ---

// A [tokens][heads][d] tensor, or pages of it, as a tensor map with boxes of
// 64 elements of `heads_box` heads of `tokens_box` tokens.  False when TMA
// cannot address it.
static inline bool attn_addressable(const void *p, int64_t ts, int64_t hs, uint32_t tokens, uint32_t heads)
{
    auto fits = [](int64_t s, uint32_t extent) { return extent <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
    return (uintptr_t)p % 16 == 0 && fits(ts, tokens) && fits(hs, heads);
}

static inline bool attn_map(CUtensorMap *tm, bool bf16, const void *p, uint32_t d, uint32_t heads, int64_t hs, uint32_t tokens,
                            int64_t ts, uint32_t pages, int64_t ps, uint32_t heads_box, uint32_t tokens_box)
{
    PFN_encodeTiled enc = tc_encoder();
    if (!enc) return false;
    // a dimension of one needs no stride, but the encoder wants a valid one
    auto bytes = [](int64_t s, uint32_t extent) { return (cuuint64_t)(extent <= 1 ? 16 : 2 * s); };
    const cuuint64_t dims[4] = {d, heads, tokens, pages};
    const cuuint64_t strides[3] = {bytes(hs, heads), bytes(ts, tokens), bytes(ps, pages)};
    const cuuint32_t box[4] = {64, heads_box, tokens_box, 1}, ones[4] = {1, 1, 1, 1};
    return enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, pages ? 4 : 3, (void *)p, dims,
               strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DB, int MODE>
static cudaError_t attn_launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const AttnArgs &a,
                               unsigned grid, cudaStream_t s)
{
    auto *fn = &attn_tc_kernel<T, DB, MODE>;
    cudaError_t e = ensure_smem_attr((const void *)fn, AttnSmem<DB, MODE == kAtFew>::kBytes);
    if (e != cudaSuccess) return e;
    return launch_behind(fn, grid, kAtThreads, AttnSmem<DB, MODE == kAtFew>::kBytes, s, q, k, v, a);
}

}  // namespace aie
