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
};

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
template <typename T>
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
    const int pos = a.rot ? a.pos[t] : 0;
    const bool ok = pos >= 0 && pos < a.max_pos;
    const float *cs = a.cs + (long long)(ok ? pos : 0) * a.rot;
    for (int i = lane; i < a.d; i += 32) {
        float v = y[i];
        if (i < a.rot) {
            const int f = a.interleaved ? i >> 1 : (i < half ? i : i - half);
            const bool first = a.interleaved ? !(i & 1) : i < half;
            const float other = y[a.interleaved ? i ^ 1 : (first ? i + half : i - half)];
            const float c = cs[f], s = cs[half + f];
            v = first ? v * c - other * s : v * c + other * s;
            if (!ok) v = __int_as_float(0x7fffffff);
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

__device__ __forceinline__ void load8f(const float *p, float *f)
{
    const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// Heads in whole 16-element pieces, everything 16-byte aligned: LPR lanes per
// head (a power of two, at least d / 16), each with two pieces of 8 elements
// that the rotation pairs with each other, so that it needs no exchange: with
// halves, elements i and i + rot / 2; interleaved or not rotated, neighbours.
// A lane keeps its pieces' weights and its token's angles in registers for
// HPT heads of the token, whose loads are all in flight at once.
//
// Bound by memory: 16384 tokens of 32 + 8 heads of 128 with keys and values
// filed take 87 us, 444 MB at 5.1 TB/s.  Measured there: 5 blocks an SM (96
// registers) 86 us, 4 89, 6 (80 registers) 93; 2 heads a lane 101; blocks of 256
// threads 99.  At 5 blocks the four-heads form spills 20 to 36 bytes a thread in
// 16 bits.  In f32, where the heads alone take 64 registers, it spills 108 to
// 164: the same tokens take 187 us, 881 MB at 4.7 TB/s.
constexpr int kRopeThreads = 128, kRopeBlocks = 5;
struct RopeVec {
    unsigned q_units, k_units;  // groups of HPT heads of a token
    unsigned q_end, k_end, end; // units: all of q, then of k, then of v
    int slots32;                // the cache's places fit 32 bits
    float inv_d;
};

template <typename T, int LPR, int HPT, bool INTERLEAVED>
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
    const bool on = lane * 16 < a.d;
    // the lane's pieces: elements e0 and e0 + gap on
    const int half = a.rot >> 1;
    const bool turn = !value && lane * 16 < a.rot;
    const int e0 = !INTERLEAVED && turn ? lane * 8 : lane * 16, gap = !INTERLEAVED && turn ? half : 8;

    const HeadsOf<T> &src = value ? a.v : key ? a.k : a.q;
    Vec8<T> x[HPT][2];
    if (on) {
        const T *p = src.at(t, h0) + e0;
#pragma unroll
        for (int i = 0; i < HPT; i++)
            if (i < n) {
                x[i][0] = load8(p);
                x[i][1] = load8(p + gap);
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
                store8(page, x[i][0]);
                store8(page + gap, x[i][1]);
                page += a.pg.hs;
            }
        return;
    }
    // y0 = r (x0 a0 + x1 b0), y1 = r (x1 a1 + x0 b1): weight and angle in one
    // factor, the same for all heads of the token.  Two elements to a register pair.
    const float *w = key ? a.wk : a.wq;
    float2 a0[4], a1[4], b0[4], b1[4];
    if (on) {
        float c[8], sn[8], w0[8], w1[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            c[k] = w0[k] = w1[k] = 1.f;
            sn[k] = 0.f;
        }
        if (turn) {
            const int pos = a.pos[t];
            if (pos >= 0 && pos < a.max_pos) {
                // angles: e0 .. e0 + 7 of the halves, or of the eight neighbouring pairs
                const float *cs = a.cs + (long long)pos * a.rot + lane * 8;
                load8f(cs, c);
                load8f(cs + half, sn);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) c[k] = sn[k] = __int_as_float(0x7fffffff);
            }
        }
        if (w) {
            load8f(w + e0, w0);
            load8f(w + e0 + gap, w1);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = 2 * k, j = i + 1;
            if (INTERLEAVED && turn) {  // pairs (i, j) of either piece; b goes with the pair swapped
                a0[k] = make_float2(w0[i] * c[k], w0[j] * c[k]);
                b0[k] = make_float2(-w0[j] * sn[k], w0[i] * sn[k]);
                a1[k] = make_float2(w1[i] * c[k + 4], w1[j] * c[k + 4]);
                b1[k] = make_float2(-w1[j] * sn[k + 4], w1[i] * sn[k + 4]);
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
        float2 f0[4], f1[4];
        float r = 1.f;
        if (on) {
            unpack8(x[i][0], (float *)f0);
            unpack8(x[i][1], (float *)f1);
        }
        if (w) {
            float2 sum = make_float2(0.f, 0.f);
            if (on)
#pragma unroll
                for (int k = 0; k < 4; k++) sum = __ffma2_rn(f0[k], f0[k], __ffma2_rn(f1[k], f1[k], sum));
            float total = sum.x + sum.y;
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) total += __shfl_xor_sync(mask, total, o);
            r = rsqrtf(fmaf(total, g.inv_d, a.eps));
        }
        if (!on) continue;
        const float2 r2 = make_float2(r, r);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 p = f0[k], q = f1[k];
            float2 y0 = __fmul2_rn(p, a0[k]), y1 = __fmul2_rn(q, a1[k]);
            if (turn) {
                y0 = __ffma2_rn(INTERLEAVED ? make_float2(p.y, p.x) : q, b0[k], y0);
                y1 = __ffma2_rn(INTERLEAVED ? make_float2(q.y, q.x) : p, b1[k], y1);
            }
            f0[k] = __fmul2_rn(y0, r2);
            f1[k] = __fmul2_rn(y1, r2);
        }
        const Vec8<T> y0 = pack8<T>((const float *)f0), y1 = pack8<T>((const float *)f1);
        if (out) {
            store8(out, y0);
            store8(out + gap, y1);
            out += dst.hs;
        }
        if (page) {
            store8(page, y0);
            store8(page + gap, y1);
            page += a.pg.hs;
        }
    }
}

template <typename T>
static bool rope_vec_ok(const RopeArgs<T> &a)
{
    const long long unit = 16 / sizeof(T);
    auto ok = [&](const HeadsOf<T> &h) { return !h.p || ((uintptr_t)h.p % 16 == 0 && h.ts % unit == 0 && h.hs % unit == 0); };
    auto ptr = [](const void *p) { return (uintptr_t)p % 16 == 0; };
    return a.d % 16 == 0 && a.rot % 16 == 0 && (unsigned long long)a.tokens * (a.hq + 2 * a.hk) < 1ull << 32 && ok(a.q) && ok(a.k) && ok(a.v) && ok(a.qo) && ok(a.ko) && ptr(a.kp) && ptr(a.vp) &&
           (!a.kp || (a.pg.ps % unit == 0 && a.pg.ts % unit == 0 && a.pg.hs % unit == 0)) && ptr(a.wq) && ptr(a.wk) && ptr(a.cs);
}

template <typename T, int LPR, int HPT>
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
    return launch_behind(a.interleaved ? rope_vec_kernel<T, LPR, HPT, true> : rope_vec_kernel<T, LPR, HPT, false>, grid, kRopeThreads,
                         0, s, a, g);
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
    if (rope_vec_ok(a)) {
        if (a.d <= 64) return rope_vec_launch<T, 4>(a, s);
        if (a.d <= 128) return rope_vec_launch<T, 8>(a, s);
        return rope_vec_launch<T, 32>(a, s);
    }
    const long long units = (long long)a.tokens * (a.hq + a.hk + (a.vp ? a.hk : 0));
    return launch_behind(rope_row_kernel<T>, (unsigned)((units + 3) / 4), 128, 0, s, a);
}

}  // namespace aie
