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
    for (int i = 0; i < (int)sizeof(T) / 2; i++) v.u[i] = ((const uint4 *)p)[i];
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
    const T *e = (const T *)&v;
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = to_f32(e[i]);
}

template <typename T>
__device__ __forceinline__ Vec8<T> pack8(const float *f)
{
    Vec8<T> v;
    T *e = (T *)&v;
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = from_f32<T>(f[i]);
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
struct RopeVec {
    int units_per_token, q_units, k_units;  // groups of HPT heads of q, k, v
    unsigned units;
    int slots32;  // the cache's places fit 32 bits
};

template <typename T, int LPR, int HPT, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_vec_kernel(const RopeArgs<T> a, const RopeVec g)
{
    const unsigned unit = (unsigned)(((unsigned long long)blockIdx.x * blockDim.x + threadIdx.x) / LPR);
    const int lane = threadIdx.x % LPR;
    if (unit >= g.units) return;  // whole groups of LPR lanes
    const unsigned mask = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (threadIdx.x % 32 / LPR * LPR);
    const int t = (int)(unit / (unsigned)g.units_per_token);
    int u = (int)(unit - (unsigned)t * g.units_per_token);
    const int kind = u < g.q_units ? 0 : u < g.q_units + g.k_units ? 1 : 2;
    u -= kind == 0 ? 0 : kind == 1 ? g.q_units : g.q_units + g.k_units;
    const int heads = kind == 0 ? a.hq : a.hk, h0 = u * HPT;
    const bool on = lane * 16 < a.d;
    // the lane's pieces
    const int half = a.rot >> 1;
    const bool turn = kind < 2 && lane * 16 < a.rot;
    const int e0 = !INTERLEAVED && turn ? lane * 8 : lane * 16, e1 = !INTERLEAVED && turn ? e0 + half : e0 + 8;

    const HeadsOf<T> &src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    Vec8<T> x[HPT][2];
#pragma unroll
    for (int i = 0; i < HPT; i++)
        if (on && h0 + i < heads) {
            const T *p = src.at(t, h0 + i);
            x[i][0] = load8(p + e0);
            x[i][1] = load8(p + e1);
        }
    // the token's place in the cache
    T *pages = kind == 0 ? nullptr : kind == 1 ? a.kp : a.vp;
    if (pages) {
        const long long s = a.slots[t];
        if (s < 0 || s >= (long long)a.pg.pages * a.pg.size) pages = nullptr;
        else if (g.slots32) {
            const unsigned page = (unsigned)s / (unsigned)a.pg.size;
            pages += page * a.pg.ps + ((unsigned)s - page * (unsigned)a.pg.size) * a.pg.ts;
        } else pages += s / a.pg.size * a.pg.ps + s % a.pg.size * a.pg.ts;
    }
    if (kind == 2) {
#pragma unroll
        for (int i = 0; i < HPT; i++)
            if (on && pages && h0 + i < heads) {
                T *p = pages + (h0 + i) * a.pg.hs;
                store8(p + e0, x[i][0]);
                store8(p + e1, x[i][1]);
            }
        return;
    }
    float c[8], sn[8], w0[8], w1[8];
    if (on && turn) {
        const int pos = a.pos[t];
        if (pos >= 0 && pos < a.max_pos) {
            // angles: e0 .. e0 + 7 of the halves, or of the eight neighbouring pairs
            const float *cs = a.cs + (long long)pos * a.rot + lane * 8;
            load8f(cs, c);
            load8f(cs + half, sn);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = sn[i] = __int_as_float(0x7fffffff);
        }
    }
    const float *w = kind == 0 ? a.wq : a.wk;
    if (on && w) {
        load8f(w + e0, w0);
        load8f(w + e1, w1);
    }
    const HeadsOf<T> &dst = kind == 0 ? a.qo : a.ko;
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        if (h0 + i >= heads) break;
        float f0[8], f1[8];
        float sum = 0.f;
        if (on) {
            unpack8(x[i][0], f0);
            unpack8(x[i][1], f1);
#pragma unroll
            for (int k = 0; k < 8; k++) sum = fmaf(f0[k], f0[k], fmaf(f1[k], f1[k], sum));
        }
        if (w) {
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
            if (on) {
                const float r = 1.0f / sqrtf(sum / (float)a.d + a.eps);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    f0[k] = f0[k] * r * w0[k];
                    f1[k] = f1[k] * r * w1[k];
                }
            }
        }
        if (!on) continue;
        if (turn) {
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float p = f0[2 * k], q = f0[2 * k + 1], v = f1[2 * k], z = f1[2 * k + 1];
                    f0[2 * k] = p * c[k] - q * sn[k];
                    f0[2 * k + 1] = q * c[k] + p * sn[k];
                    f1[2 * k] = v * c[k + 4] - z * sn[k + 4];
                    f1[2 * k + 1] = z * c[k + 4] + v * sn[k + 4];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float p = f0[k], q = f1[k];
                    f0[k] = p * c[k] - q * sn[k];
                    f1[k] = q * c[k] + p * sn[k];
                }
            }
        }
        const Vec8<T> y0 = pack8<T>(f0), y1 = pack8<T>(f1);
        if (dst.p) {
            T *p = dst.at(t, h0 + i);
            store8(p + e0, y0);
            store8(p + e1, y1);
        }
        if (pages) {
            T *p = pages + (h0 + i) * a.pg.hs;
            store8(p + e0, y0);
            store8(p + e1, y1);
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
    g.q_units = (a.hq + HPT - 1) / HPT;
    g.k_units = (a.hk + HPT - 1) / HPT;
    g.units_per_token = g.q_units + g.k_units * (a.vp ? 2 : 1);
    g.units = (unsigned)a.tokens * g.units_per_token;  // under 2^32: rope_vec_ok
    g.slots32 = (unsigned long long)a.pg.pages * a.pg.size <= 0xffffffffull;
    const unsigned grid = (unsigned)(((unsigned long long)g.units * LPR + 255) / 256);
    if (a.interleaved) rope_vec_kernel<T, LPR, HPT, true><<<grid, 256, 0, s>>>(a, g);
    else rope_vec_kernel<T, LPR, HPT, false><<<grid, 256, 0, s>>>(a, g);
    return cudaGetLastError();
}

// Few heads: one at a time, over as many SMs as they reach.
template <typename T, int LPR>
static cudaError_t rope_vec_launch(const RopeArgs<T> &a, cudaStream_t s)
{
    const long long threads = (long long)a.tokens * (a.hq + 2 * a.hk) * LPR;
    return threads < 4ll * 2048 * tc_sm_count() ? rope_vec_launch<T, LPR, 1>(a, s) : rope_vec_launch<T, LPR, 4>(a, s);
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
    rope_row_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace aie
