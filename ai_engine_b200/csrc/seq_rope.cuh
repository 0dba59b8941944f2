// Norm of queries and keys and the position rotation, with keys and values
// filed into a paged cache.
//
//   r = rsqrt(sum_d x_d^2 / D + eps),  y_d = x_d r w_d
//   (y_i, y_j) -> (y_i cos a - y_j sin a, y_j cos a + y_i sin a)
//
// in f32, rounded once.  A head is read once and written once (keys twice
// when they also go to the cache): memory-bound.
#pragma once
#include "seq_common.cuh"
#include "tc_ptx.cuh"

namespace aie {

template <typename T>
struct RopeArgs {
    HeadsOf<T> q, k, v, qo, ko;
    T *kp, *vp;
    PagesGeom pg;
    const float *wq, *wk, *cs;
    const int32_t *pos;
    const int64_t *slots;
    int tokens, hq, hk, d, rot, max_pos, interleaved;
    float eps;
    const uint8_t *axis;  // each pair's axis, or nullptr: one position a token
    int axes;             // positions of a token
};

// The table's row for a token's position (along an axis), nullptr outside it.
template <bool AXES, typename T>
__device__ __forceinline__ const float *rope_angles(const RopeArgs<T> &a, int t, int axis)
{
    if (AXES && axis >= a.axes) return nullptr;
    const int pos = a.pos[AXES ? (long long)t * a.axes + axis : t];
    return pos >= 0 && pos < a.max_pos ? a.cs + (long long)pos * a.rot : nullptr;
}

// Where a token's head stands in the cache, or nullptr.
template <typename T>
__device__ __forceinline__ T *rope_slot(T *pages, const PagesGeom &g, const int64_t *slots, int t, int h)
{
    if (!pages) return nullptr;
    const long long s = slots[t];
    if (s < 0 || s >= (long long)g.pages * g.size) return nullptr;
    return pages + (s / g.size) * g.ps + (s % g.size) * g.ts + h * g.hs;
}

constexpr int kRopeMaxDim = 512;

// Any head size, stride and alignment: one warp per head of a token (query
// heads, then key heads, then value heads, which are only filed), the normed
// head in shared memory while it is rotated.
template <typename T, bool AXES>
__global__ void __launch_bounds__(128) rope_row_kernel(RopeArgs<T> a)
{
    __shared__ float buf[4][kRopeMaxDim];
    behind_last_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = a.hq + a.hk + (a.vp ? a.hk : 0);
    const long long unit = (long long)blockIdx.x * 4 + warp;
    if (unit >= (long long)a.tokens * rows) return;
    const int t = (int)(unit / rows);
    int h = (int)(unit % rows);
    if (h >= a.hq + a.hk) {
        h -= a.hq + a.hk;
        T *dst = rope_slot(a.vp, a.pg, a.slots, t, h);
        if (!dst) return;
        const T *src = a.v.at(t, h);
        for (int i = lane; i < a.d; i += 32) dst[i] = src[i];
        return;
    }
    const bool key = h >= a.hq;
    if (key) h -= a.hq;
    const T *src = key ? a.k.at(t, h) : a.q.at(t, h);
    const float *w = key ? a.wk : a.wq;
    float *y = buf[warp];
    float sum = 0.f;
    for (int i = lane; i < a.d; i += 32) {
        const float x = to_f32(src[i]);
        y[i] = x;
        sum = fmaf(x, x, sum);
    }
    __syncwarp();
    if (w) {
        const float r = 1.0f / sqrtf(warp_sum(sum) / (float)a.d + a.eps);
        for (int i = lane; i < a.d; i += 32) y[i] = y[i] * r * w[i];
        __syncwarp();
    }
    T *o1 = key ? (a.ko.p ? a.ko.at(t, h) : nullptr) : a.qo.at(t, h);
    T *o2 = key ? rope_slot(a.kp, a.pg, a.slots, t, h) : nullptr;
    const int half = a.rot >> 1;
    const float *cs = !AXES && a.rot ? rope_angles<AXES>(a, t, 0) : nullptr;
    for (int i = lane; i < a.d; i += 32) {
        float v = y[i];
        if (i < a.rot) {
            const int f = a.interleaved ? i >> 1 : (i < half ? i : i - half);
            const bool first = a.interleaved ? !(i & 1) : i < half;
            const float other = y[a.interleaved ? i ^ 1 : (first ? i + half : i - half)];
            if constexpr (AXES) cs = rope_angles<AXES>(a, t, a.axis[f]);
            if (cs) {
                const float c = cs[f], s = cs[half + f];
                v = first ? v * c - other * s : v * c + other * s;
            } else v = __int_as_float(0x7fffffff);
        }
        const T r = from_f32<T>(v);
        if (o1) o1[i] = r;
        if (o2) o2[i] = r;
    }
}

// 8 neighbouring elements in registers as they come, one or two 16-byte loads.
template <typename T>
struct Vec8 {
    uint4 u[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T *p)
{
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.u[i].x), "=r"(v.u[i].y), "=r"(v.u[i].z), "=r"(v.u[i].w)
                     : "l"((const uint4 *)p + i));
    return v;
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const Vec8<T> &v)
{
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4 *)p)[i] = v.u[i];
}

template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T> &v, float *f)
{
    const uint32_t *u = (const uint32_t *)&v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // a bf16 is the upper half of an f32
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 y = __half22float2(*(const __half2 *)&u[i]);
            f[2 * i] = y.x;
            f[2 * i + 1] = y.y;
        } else {
            f[2 * i] = __uint_as_float(u[2 * i]);
            f[2 * i + 1] = __uint_as_float(u[2 * i + 1]);
        }
    }
}

template <typename T>
__device__ __forceinline__ Vec8<T> pack8(const float *f)
{
    Vec8<T> v;
    uint32_t *u = (uint32_t *)&v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 2) u[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        else {
            u[2 * i] = __float_as_uint(f[2 * i]);
            u[2 * i + 1] = __float_as_uint(f[2 * i + 1]);
        }
    }
    return v;
}

// A piece of 8 elements, or of 4 16-bit ones.
template <typename T, int N>
struct Piece : Vec8<T> {
    __device__ __forceinline__ void load(const T *p) { *(Vec8<T> *)this = load8(p); }
    __device__ __forceinline__ void store(T *p) const { store8(p, *this); }
    __device__ __forceinline__ void unpack(float *f) const { unpack8<T>(*this, f); }
    __device__ __forceinline__ void pack(const float *f) { *(Vec8<T> *)this = pack8<T>(f); }
};
template <typename T>
struct Piece<T, 4> {
    static_assert(sizeof(T) == 2, "16-bit elements");
    uint2 u;
    __device__ __forceinline__ void load(const T *p)
    {
        asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p));
    }
    __device__ __forceinline__ void store(T *p) const { *(uint2 *)p = u; }
    __device__ __forceinline__ void unpack(float *f) const
    {
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 y = std::is_same<T, __half>::value ? __half22float2(*(const __half2 *)&w[i])
                                                            : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            f[2 * i] = y.x;
            f[2 * i + 1] = y.y;
        }
    }
    __device__ __forceinline__ void pack(const float *f) { u = make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3])); }
};

template <int N>
__device__ __forceinline__ void load_floats(const float *p, float *f)
{
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 a = *(const float4 *)(p + i);
        f[i] = a.x; f[i + 1] = a.y; f[i + 2] = a.z; f[i + 3] = a.w;
    }
}

// Heads in whole 16-element pieces, everything 16-byte aligned: LPR lanes per
// head (a power of two, at least d / 2 N), each with two pieces of N = 8 elements
// (4 for heads that allow no more) that the rotation pairs with each other, so
// that it needs no exchange: with halves, elements i and i + rot / 2; interleaved
// or not rotated, neighbours.
// A lane keeps its pieces' weights and its token's angles in registers for
// HPT heads of the token, whose loads are all in flight at once.
//
// Bound by memory: 16384 tokens of 32 + 8 heads of 128 with keys and values
// filed take 87 us, 444 MB at 5.1 TB/s.  Measured there: 5 blocks an SM (96
// registers) 86 us, 4 89, 6 (80 registers) 93; 2 heads a lane 101; blocks of 256
// threads 99.  At 5 blocks the four-heads form spills 20 to 36 bytes a thread in
// 16 bits.  In f32, where the heads alone take 64 registers, it spills 108 to
// 164: the same tokens take 187 us, 881 MB at 4.7 TB/s.
//
// By several axes (AXES) a pair's angle is that of its token's position on the
// pair's axis.  A lane whose pairs all have one axis reads its angles as before,
// from that axis' row; others read theirs one by one (1297 tokens of 20 + 5 heads
// of 96, axes taking turns: 6.7 us a call).  16350 tokens of 32 + 8 heads of 128,
// three axes, filed: 87 us, 436 MB at 5.0 TB/s; with the axes taking turns 89; pairs
// of neighbours 92, and 95 with turns.
constexpr int kRopeThreads = 128, kRopeBlocks = 5;
struct RopeVec {
    unsigned q_units, k_units;  // groups of HPT heads of a token
    unsigned q_end, k_end, end; // units: all of q, then of k, then of v
    int slots32;                // the cache's places fit 32 bits
    float inv_d;
};

template <typename T, int LPR, int HPT, bool INTERLEAVED, bool AXES, int N>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) rope_vec_kernel(const RopeArgs<T> a, const RopeVec g)
{
    behind_last_launch();
    unsigned unit = (unsigned)(((unsigned long long)blockIdx.x * blockDim.x + threadIdx.x) / LPR);
    const int lane = threadIdx.x % LPR;
    if (unit >= g.end) return;  // whole groups of LPR lanes
    const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (threadIdx.x % 32 / LPR * LPR);
    // q, k and v one after the other: few warps hold more than one of them
    const bool key = unit >= g.q_end, value = unit >= g.k_end;
    unit -= value ? g.k_end : key ? g.q_end : 0;
    const unsigned per = key ? g.k_units : g.q_units;
    const int t = (int)(unit / per), h0 = (int)(unit - (unsigned)t * per) * HPT;
    const int n = min(HPT, (key ? a.hk : a.hq) - h0);
    const bool on = lane * (2 * N) < a.d;
    // the lane's pieces: elements e0 and e0 + gap on
    const int half = a.rot >> 1;
    const bool turn = !value && lane * (2 * N) < a.rot;
    const int e0 = !INTERLEAVED && turn ? lane * N : lane * (2 * N), gap = !INTERLEAVED && turn ? half : N;

    const HeadsOf<T> &src = value ? a.v : key ? a.k : a.q;
    Piece<T, N> x[HPT][2];
    if (on) {
        const T *p = src.at(t, h0) + e0;
#pragma unroll
        for (int i = 0; i < HPT; i++)
            if (i < n) {
                x[i][0].load(p);
                x[i][1].load(p + gap);
                p += src.hs;
            }
    }
    // the token's place in the cache
    T *page = !key ? nullptr : value ? a.vp : a.kp;
    if (page) {
        const long long s = a.slots[t];
        if (s < 0 || s >= (long long)a.pg.pages * a.pg.size) page = nullptr;
        else {
            if (g.slots32) {
                const unsigned number = (unsigned)s / (unsigned)a.pg.size;
                page += number * a.pg.ps + ((unsigned)s - number * (unsigned)a.pg.size) * a.pg.ts;
            } else page += s / a.pg.size * a.pg.ps + s % a.pg.size * a.pg.ts;
            page += h0 * a.pg.hs + e0;
        }
    }
    if (value) {
#pragma unroll
        for (int i = 0; i < HPT; i++)
            if (on && page && i < n) {
                x[i][0].store(page);
                x[i][1].store(page + gap);
                page += a.pg.hs;
            }
        return;
    }
    // y0 = r (x0 a0 + x1 b0), y1 = r (x1 a1 + x0 b1): weight and angle in one
    // factor, the same for all heads of the token.  Two elements to a register pair.
    const float *w = key ? a.wk : a.wq;
    float2 a0[N / 2], a1[N / 2], b0[N / 2], b1[N / 2];
    if (on) {
        float c[N], sn[N], w0[N], w1[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            c[k] = w0[k] = w1[k] = 1.f;
            sn[k] = 0.f;
        }
        if (turn) {
            // angles: e0 .. e0 + N - 1 of the halves, or of the N neighbouring pairs
            uint2 ax = make_uint2(0, 0);  // their axes
            if constexpr (AXES && N == 8) ax = *(const uint2 *)(a.axis + lane * N);
            else if constexpr (AXES) ax.x = ax.y = *(const uint32_t *)(a.axis + lane * N);
            if (!AXES || (ax.x == ax.y && ax.x == (ax.x & 255) * 0x01010101u)) {
                if (const float *cs = rope_angles<AXES>(a, t, ax.x & 255)) {
                    load_floats<N>(cs + lane * N, c);
                    load_floats<N>(cs + lane * N + half, sn);
                } else {
#pragma unroll
                    for (int k = 0; k < N; k++) c[k] = sn[k] = __int_as_float(0x7fffffff);
                }
            } else {
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const float *cs = rope_angles<AXES>(a, t, ((k < 4 ? ax.x : ax.y) >> 8 * (k & 3)) & 255);
                    c[k] = cs ? cs[lane * N + k] : __int_as_float(0x7fffffff);
                    sn[k] = cs ? cs[lane * N + k + half] : __int_as_float(0x7fffffff);
                }
            }
        }
        if (w) {
            load_floats<N>(w + e0, w0);
            load_floats<N>(w + e0 + gap, w1);
        }
#pragma unroll
        for (int k = 0; k < N / 2; k++) {
            const int i = 2 * k, j = i + 1;
            if (INTERLEAVED && turn) {  // pairs (i, j) of either piece; b goes with the pair swapped
                a0[k] = make_float2(w0[i] * c[k], w0[j] * c[k]);
                b0[k] = make_float2(-w0[j] * sn[k], w0[i] * sn[k]);
                a1[k] = make_float2(w1[i] * c[k + N / 2], w1[j] * c[k + N / 2]);
                b1[k] = make_float2(-w1[j] * sn[k + N / 2], w1[i] * sn[k + N / 2]);
            } else {
                a0[k] = make_float2(w0[i] * c[i], w0[j] * c[j]);
                b0[k] = make_float2(-w1[i] * sn[i], -w1[j] * sn[j]);
                a1[k] = make_float2(w1[i] * c[i], w1[j] * c[j]);
                b1[k] = make_float2(w0[i] * sn[i], w0[j] * sn[j]);
            }
        }
    }
    const HeadsOf<T> &dst = key ? a.ko : a.qo;
    T *out = dst.p ? dst.at(t, h0) + e0 : nullptr;
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        if (i >= n) break;
        float2 f0[N / 2], f1[N / 2];
        float r = 1.f;
        if (on) {
            x[i][0].unpack((float *)f0);
            x[i][1].unpack((float *)f1);
        }
        if (w) {
            float2 sum = make_float2(0.f, 0.f);
            if (on)
#pragma unroll
                for (int k = 0; k < N / 2; k++) sum = __ffma2_rn(f0[k], f0[k], __ffma2_rn(f1[k], f1[k], sum));
            float total = sum.x + sum.y;
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) total += __shfl_xor_sync(mask, total, o);
            r = rsqrtf(fmaf(total, g.inv_d, a.eps));
        }
        if (!on) continue;
        const float2 r2 = make_float2(r, r);
#pragma unroll
        for (int k = 0; k < N / 2; k++) {
            const float2 p = f0[k], q = f1[k];
            float2 y0 = __fmul2_rn(p, a0[k]), y1 = __fmul2_rn(q, a1[k]);
            if (turn) {
                y0 = __ffma2_rn(INTERLEAVED ? make_float2(p.y, p.x) : q, b0[k], y0);
                y1 = __ffma2_rn(INTERLEAVED ? make_float2(q.y, q.x) : p, b1[k], y1);
            }
            f0[k] = __fmul2_rn(y0, r2);
            f1[k] = __fmul2_rn(y1, r2);
        }
        Piece<T, N> y0, y1;
        y0.pack((const float *)f0);
        y1.pack((const float *)f1);
        if (out) {
            y0.store(out);
            y1.store(out + gap);
            out += dst.hs;
        }
        if (page) {
            y0.store(page);
            y1.store(page + gap);
            page += a.pg.hs;
        }
    }
}

// Pieces of n elements.
template <typename T>
static bool rope_vec_ok(const RopeArgs<T> &a, int n)
{
    const int bytes = std::min(16, n * (int)sizeof(T));
    const long long unit = bytes / (int)sizeof(T);
    auto ok = [&](const HeadsOf<T> &h) { return !h.p || ((uintptr_t)h.p % bytes == 0 && h.ts % unit == 0 && h.hs % unit == 0); };
    auto ptr = [](const void *p, int b) { return (uintptr_t)p % b == 0; };
    return a.d % (2 * n) == 0 && a.rot % (2 * n) == 0 && (unsigned long long)a.tokens * (a.hq + 2 * a.hk) < 1ull << 32 && ok(a.q) &&
           ok(a.k) && ok(a.v) && ok(a.qo) && ok(a.ko) && ptr(a.kp, bytes) && ptr(a.vp, bytes) &&
           (!a.kp || (a.pg.ps % unit == 0 && a.pg.ts % unit == 0 && a.pg.hs % unit == 0)) && ptr(a.wq, 16) && ptr(a.wk, 16) && ptr(a.cs, 16) &&
           ptr(a.axis, n);
}

template <typename T, int LPR, int HPT, int N = 8>
static cudaError_t rope_vec_launch(const RopeArgs<T> &a, cudaStream_t s)
{
    RopeVec g;
    g.q_units = (unsigned)(a.hq + HPT - 1) / HPT;
    g.k_units = (unsigned)(a.hk + HPT - 1) / HPT;
    g.q_end = a.tokens * g.q_units;  // all under 2^32: rope_vec_ok
    g.k_end = g.q_end + a.tokens * g.k_units;
    g.end = g.k_end + (a.vp ? a.tokens * g.k_units : 0);
    g.slots32 = (unsigned long long)a.pg.pages * a.pg.size <= 0xffffffffull;
    g.inv_d = 1.0f / (float)a.d;
    const unsigned grid = (unsigned)(((unsigned long long)g.end * LPR + kRopeThreads - 1) / kRopeThreads);
    auto *fn = a.axis ? (a.interleaved ? rope_vec_kernel<T, LPR, HPT, true, true, N> : rope_vec_kernel<T, LPR, HPT, false, true, N>)
                      : (a.interleaved ? rope_vec_kernel<T, LPR, HPT, true, false, N> : rope_vec_kernel<T, LPR, HPT, false, false, N>);
    return launch_behind(fn, grid, kRopeThreads, 0, s, a, g);
}

// So few heads that one at a time they are all resident at once: one at a time
// (8 tokens of 24 heads of 64: 2.6 us against 3.8 us four at a time; 1237 tokens
// of 25 heads of 96, beyond that: 5.6 us four at a time against 6.6 us).
template <typename T, int LPR>
static cudaError_t rope_vec_launch(const RopeArgs<T> &a, cudaStream_t s)
{
    const long long threads = (long long)a.tokens * (a.hq + 2 * a.hk) * LPR;
    return threads <= (long long)kRopeThreads * kRopeBlocks * tc_sm_count() ? rope_vec_launch<T, LPR, 1>(a, s)
                                                                            : rope_vec_launch<T, LPR, 4>(a, s);
}

template <typename T>
static cudaError_t rope_launch(const RopeArgs<T> &a, cudaStream_t s)
{
    if (rope_vec_ok(a, 8)) {
        if (a.d <= 64) return rope_vec_launch<T, 4>(a, s);
        if (a.d <= 128) return rope_vec_launch<T, 8>(a, s);
        return rope_vec_launch<T, 32>(a, s);
    }
    if constexpr (sizeof(T) == 2) {
        // heads or rotations in multiples of 8 only, or rows aligned to 8 bytes: pieces of 4
        // (2345 tokens of 32 + 8 heads of 80, 40 rotated, filed: 18 us; a warp a head: 51)
        if (a.d <= 128 && rope_vec_ok(a, 4)) return a.d <= 64 ? rope_vec_launch<T, 8, 2, 4>(a, s) : rope_vec_launch<T, 16, 2, 4>(a, s);
    }
    const long long units = (long long)a.tokens * (a.hq + a.hk + (a.vp ? a.hk : 0));
    return launch_behind(a.axis ? rope_row_kernel<T, true> : rope_row_kernel<T, false>, (unsigned)((units + 3) / 4), 128, 0, s, a);
}

}  // namespace aie
