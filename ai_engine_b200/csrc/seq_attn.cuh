// Attention on the tensor cores (tcgen05, f16 / bf16 operands, f32 sums):
// whole packed prompts, and the shared prefix of a batch of streams.
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

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
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
    int causal;
    int out_bytes;            // what `out` is aligned to, in every row: 32, 16 or less
    int shared, max_len, page_size, pages, box_rows, splits, tiles_per_split;
    float scale_log2;
};

template <int DB>
struct AttnSmem {
    static constexpr int kStages = DB == 2 ? 5 : 8;
    static constexpr uint32_t kQ = 2 * DB * kAtBlockBytes;
    static constexpr uint32_t kStage = DB * kAtBlockBytes;
    static constexpr uint32_t kBytes = kQ + kStages * kStage + 1024 /* alignment */;
};

struct AttnShared {
    uint64_t q_full, kv_full[8], kv_empty[8], s_full[2], p_full[2][2], o_full[2], drain;
    uint32_t tmem, abort;
    int seq_first, seq_len, pair;
};

// What one block does: tile pair `pair` of tokens first .. first + len.
struct AttnWork {
    int first, len, pair, kvh, split;
};

template <typename T, int DB, bool PAGED>
__global__ void __launch_bounds__(kAtThreads, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const AttnArgs a)
{
    using Sm = AttnSmem<DB>;
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
        if (w.len == 0) {  // a block past the last pair
            if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
            return;
        }
    }
    // keys seen by a tile's last token; `keys` also bounds the values that exist
    const int tok0 = w.pair * 2 * tpt;
    const int keys = PAGED ? min(a.shared, a.max_len) : w.len;
    const int step0 = PAGED ? w.split * a.tiles_per_split : 0;
    auto steps_of = [&](int t) {
        const int first = tok0 + t * tpt, last = min(first + tpt, w.len);
        const int seen = first >= w.len ? 0 : (!PAGED && a.causal) ? last : keys;
        const int steps = (seen + kAtTile - 1) / kAtTile;
        return PAGED ? max(min(steps, step0 + a.tiles_per_split), step0) : steps;
    };
    const int n0 = steps_of(0), n1 = steps_of(1), n = max(n0, n1);
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
        const int tok = tok0 + t * tpt + row / a.group, head = w.kvh * a.group + row % a.group;
        const bool real = row < tpt * a.group && tok < w.len;
        int seen = keys;
        if constexpr (PAGED) {
            if (real) seen = min(seen, max(a.lens[tok], 0));
        } else {
            if (a.causal) seen = min(tok + 1, keys);
        }
        const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * 128, to = ts + 256;
        const float sl = a.scale_log2;
        float m = -INFINITY;           // carried reference maximum, in units of S
        float2 l2 = make_float2(0.f, 0.f);
        bool ok = true;
        const int nt = n_of(t);
        for (int j = step0; j < nt; j++) {
            ok = wait(&sh.s_full[t], (j - step0) & 1, 7);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            float s[128];
#pragma unroll
            for (int i = 0; i < 4; i++) tmem_ld32(ts + 32 * i, s + 32 * i);
#pragma unroll
            for (int i = 0; i < 4; i++) tmem_wait_ld32(s + 32 * i);
            const int here = seen - j * kAtTile;
            if (__any_sync(0xffffffffu, here < kAtTile)) {
#pragma unroll
                for (int i = 0; i < 128; i++) s[i] = i < here ? s[i] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 124; i += 8) {
                mx[0] = max3(mx[0], s[i], s[i + 1]);
                mx[1] = max3(mx[1], s[i + 2], s[i + 3]);
                mx[2] = max3(mx[2], s[i + 4], s[i + 5]);
                mx[3] = max3(mx[3], s[i + 6], s[i + 7]);
            }
            mx[0] = max3(mx[0], s[124], s[125]);
            mx[1] = max3(mx[1], s[126], s[127]);
            const float top = fmaxf(max3(mx[0], mx[1], mx[2]), fmaxf(mx[3], m));
            // -inf - -inf is NaN: not greater, nothing to move
            const bool grow = (top - m) * sl > 8.f;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2((m - top) * sl) : 1.f;  // from -inf: 0
                if (grow) m = top;
                if (j > step0) {
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
            const float off = m == -INFINITY ? 0.f : fmaf(-m, sl, kWeightShift<T>);
            const float2 sl2 = make_float2(sl, sl), off2 = make_float2(off, off);
#pragma unroll
            for (int c = 0; c < 2; c++) {
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
        if (ok && (nt > step0 || PAGED)) {
            // of this split's keys; scores of -inf alone (l is 0) count as none here
            const bool none = nt <= step0 || seen <= step0 * kAtTile || (PAGED && l == 0.f);
            const float r = none ? 0.f : 1.f / l;
            const long long prow = PAGED ? ((long long)w.split * a.tokens + tok) * a.q_heads + head : 0;
            // 32 columns at a time out of tensor memory: a thread holds a row and
            // writes whole 32-byte sectors of it (16-byte pieces: 2 us a tile, so: 1)
            const long long at = PAGED ? prow * a.d : (w.first + tok) * a.out_ts + head * a.out_hs;
            if constexpr (PAGED) {
                // log2 of the weights' sum; -inf where nothing was seen
                if (real) a.part_lse[prow] = none ? -INFINITY : fmaf(m, sl, log2f(l) - kWeightShift<T>);
            }
            bool nan = false;
#pragma unroll 1
            for (int c = 0; c < 2 * DB; c++) {
                float o[32];
                if (nt > step0) {
                    tmem_ld32(to + 32 * c, o);
                    tmem_wait_ld32(o);
                }
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] = none ? 0.f : o[i] * r;
                if (PAGED && seen < keys)
#pragma unroll
                    for (int i = 0; i < 32; i++) nan |= o[i] != o[i];
                if (real) {
#pragma unroll
                    for (int i = 0; i < 32; i += PAGED ? 8 : 16) {
                        if (32 * c + i >= a.d) break;
                        if constexpr (PAGED) {
                            store32(a.part_o + at + 32 * c + i, (const uint32_t *)&o[i]);
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
                }
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
                    const int tiles = n1 > step0 ? 2 : 1;
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
                for (int i = 0; i < 2 * (n - step0); i++) {
                    const int st = i % Sm::kStages, round = i / Sm::kStages, step = step0 + i / 2;
                    const CUtensorMap *tm = i & 1 ? &tm_v : &tm_k;
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
                    } else if (lane == 0) {
                        for (int b = 0; b < DB; b++)
                            tma_load_3d(dst + b * kAtBlockBytes, tm, &sh.kv_full[st], b * 64, w.kvh, w.first + step * kAtTile);
                    }
                    issued = i + 1;
                }
                // nothing may still be written to this block's memory when it ends
                if (*abort && lane == 0) {
                    mbar_wait(&sh.q_full, 0);
                    for (int i = max(issued - Sm::kStages, 0); i < issued; i++)
                        mbar_wait(&sh.kv_full[i % Sm::kStages], (i / Sm::kStages) & 1);
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
                    const uint64_t qd = qd0 + t * (DB * kAtBlockBytes >> 4), kd = kd0 + k * (Sm::kStage >> 4);
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
                if (ok) {
                    tc_fence_after();
                    if (n0 > step0) s_mma(0, 0);
                    if (n1 > step0) s_mma(1, 0);
                    mma_commit(&sh.kv_empty[0]);
                }
                uint32_t vj = 1, kj = 2 % Sm::kStages, v_old = 0, k_old = 0;  // ring places of V(j), K(j + 1)
                for (int j = step0; ok && j < n; j++) {
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
                const int iv = 2 * (j - step0) + 1, ik = iv + 1;
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
                if (ok && j + 1 < n) ok = wait(&sh.kv_full[ik % Sm::kStages], (ik / Sm::kStages) & 1, 5);
                // one arrival per step
                for (int t = 0; t < 2 && ok && j > step0; t++)
                    if (j - 1 < n_of(t)) ok = wait(&sh.p_full[t][0], (j - 1 - step0) & 1, 11);
                if (!__all_sync(0xffffffffu, ok)) break;
                if (lane == 0) {
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

template <typename T, int DB, bool PAGED>
static cudaError_t attn_launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const AttnArgs &a,
                               unsigned grid, cudaStream_t s)
{
    auto *fn = &attn_tc_kernel<T, DB, PAGED>;
    cudaError_t e = ensure_smem_attr((const void *)fn, AttnSmem<DB>::kBytes);
    if (e != cudaSuccess) return e;
    return launch_behind(fn, grid, kAtThreads, AttnSmem<DB>::kBytes, s, q, k, v, a);
}

}  // namespace aie
