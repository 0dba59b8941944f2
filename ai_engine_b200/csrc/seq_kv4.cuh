// A paged cache in 4 bits: filing and reading back.
//
//   lo = f16(min x),  s = f16((max x - lo) / 15),  code = rint((x - lo) / s),
//   x' = lo + code s
//
// for each group of 32 elements of a head: 5 bits an element.  All four steps are
// as in 64 bits, so that a cache can be told from its inputs to the bit; in f32
// arithmetic wherever that cannot make a difference.
//
// Two lanes hold a group, 16 elements each: the least and the largest in the
// inputs' own type (exact), one exchange, then a multiply-add and a subtraction an
// element, and the sign of what is left tells a code's side of a border; only where
// f32 cannot tell are the 64-bit forms called.  Reading back is one multiply-add.
// A group is read once and written once: memory-bound.  16384 tokens of 8 heads
// of 128 in bf16, k and v: 67 MB read, 21 MB written in 30 us (2.9 TB/s; issue slots
// 67%: the arithmetic of two roundings an element); read back in 20 us (4.4 TB/s).
// Filing with 64 registers (8 blocks an SM) spills 28 bytes a thread, 60 in f32.
#pragma once
#include "seq_rope.cuh"

namespace aie {

// The block of a page and head: codes of all places, then (s, lo) pairs.
struct Kv4Geom {
    uint8_t *k, *v;
    long long page_stride;
    int pages, size, heads, d;
    __host__ __device__ __forceinline__ long long block() const { return (long long)size * d * 5 / 8; }
    __device__ __forceinline__ uint8_t *at(uint8_t *base, long long page, int head) const
    {
        return base + page * page_stride + head * block();
    }
};

static inline Kv4Geom kv4_geom(const aie_kv4 &c)
{
    return Kv4Geom{(uint8_t *)c.k, (uint8_t *)c.v, (long long)c.page_stride, (int)c.pages, (int)c.page_size, (int)c.kv_heads,
                   (int)c.head_dim};
}

template <typename T>
struct Kv4Rows {
    Kv4Geom g;
    HeadsOf<T> k, v;
    const int64_t *slots;
    long long block;  // bytes of a page and head
    int pieces;       // of `each` elements: tokens * heads * d / each
    int each;
    FastDiv per_token, per_head, size;
    int slots32;      // the cache's places fit 31 bits
    int vec;          // 16-byte accesses
};

// 8 neighbouring elements, in one access where they are aligned.
template <typename T>
__device__ __forceinline__ Vec8<T> read8(const T *p, int vec)
{
    if (vec) return load8(p);
    Vec8<T> x;
#pragma unroll
    for (int i = 0; i < 8; i++) ((T *)&x)[i] = p[i];
    return x;
}

// Next to a border between two codes, where f32 may be on the wrong side, and
// wherever codes have to be kept within 0 .. 15.
static __device__ __noinline__ uint32_t kv4_code64(float x, float lo, float s)
{
    return s > 0.f ? (uint32_t)fmin(fmax(rint(((double)x - (double)lo) / (double)s), 0.0), 15.0) : 0u;
}
static __device__ __noinline__ float kv4_scale64(float hi, float lo) { return (float)fmax(((double)hi - (double)lo) / 15.0, 0.0); }

__device__ __forceinline__ __half lower(__half2 x) { return __low2half(x); }
__device__ __forceinline__ __half upper(__half2 x) { return __high2half(x); }
__device__ __forceinline__ __nv_bfloat16 lower(__nv_bfloat162 x) { return __low2bfloat16(x); }
__device__ __forceinline__ __nv_bfloat16 upper(__nv_bfloat162 x) { return __high2bfloat16(x); }

// A lane's 16 of a group's 32 elements (two neighbouring lanes): the group's
// smallest and largest, NaN where it holds one.
template <typename T>
__device__ __forceinline__ void kv4_range(const Vec8<T> (&x)[2], float &lo, float &hi)
{
    if constexpr (sizeof(T) == 2) {
        // pairs, in their own type: exact
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        const T2 *u = (const T2 *)x;
        T2 a = u[0], b = u[0];
#pragma unroll
        for (int i = 1; i < 8; i++) {
            a = __hmin2_nan(a, u[i]);
            b = __hmax2_nan(b, u[i]);
        }
        a = __hmin2_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
        b = __hmax2_nan(b, __shfl_xor_sync(0xffffffffu, b, 1));
        lo = to_f32(__hmin_nan(lower(a), upper(a)));
        hi = to_f32(__hmax_nan(lower(b), upper(b)));
    } else {
        const float *f = (const float *)x;
        lo = hi = f[0];
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            lo = fminf(lo, f[i]);
            hi = fmaxf(hi, f[i]);
            nan |= f[i] != f[i];
        }
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
        nan |= (bool)__shfl_xor_sync(0xffffffffu, (int)nan, 1);
        if (nan) lo = hi = __int_as_float(0x7fffffff);
    }
}

// Their codes, and the group's (s, lo).
template <typename T>
__device__ __forceinline__ uint2 kv4_quantise(const Vec8<T> (&x)[2], uint32_t &pair)
{
    float lo, hi;
    kv4_range(x, lo, hi);
    const bool bad = !(fabsf(lo) <= 3.402823466e38f && fabsf(hi) <= 3.402823466e38f);
    const float least = lo, most = hi;
    lo = fminf(fmaxf(lo, -65504.f), 65504.f);
    hi = fminf(fmaxf(hi, -65504.f), 65504.f);
    const __half low = __float2half_rn(lo);
    lo = __half2float(low);
    // the f16 next to (hi - lo) / 15: three roundings of f32 move that by less
    // than 2^-21 of it, which rarely reaches over a border of f16
    const float t = fmaxf(hi - lo, 0.f) * (1.f / 15.f);
    __half scale = __float2half_rn(t * (1.f - 0x1p-21f));
    if (__half_as_ushort(scale) != __half_as_ushort(__float2half_rn(t * (1.f + 0x1p-21f)))) scale = __float2half_rn(kv4_scale64(hi, lo));
    const float s = __half2float(scale), inv = s > 0.f ? __frcp_rn(s) : 0.f;
    pair = bad ? 0x7fff0000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(low) << 16;
    // (x - lo) / s in f32, less than 2^-18 off; its nearest integer by way of 1.5 2^23, and how far that is
    float2 f[8];
    unpack8<T>(x[0], (float *)f);
    unpack8<T>(x[1], (float *)(f + 4));
    const float2 less = make_float2(-lo, -lo), by = make_float2(inv, inv), up = make_float2(12582912.f, 12582912.f),
                 down = make_float2(-12582912.f, -12582912.f), minus = make_float2(-1.f, -1.f);
    float far = 0.f;
    float2 r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float2 q = __fmul2_rn(__fadd2_rn(f[i], less), by);
        r[i] = __fadd2_rn(__fadd2_rn(q, up), down);
        const float2 d = __ffma2_rn(r[i], minus, q);
        far = max3(far, fabsf(d.x), fabsf(d.y));
    }
    const bool inside = (most - lo) * inv < 15.25f && (least - lo) * inv > -0.25f && !bad;
    if (inside && far >= 0.5f - 0x1p-17f) {
        // Next to a border b = n + 1/2, as some of a hundred groups of bf16 are exactly: by the
        // sign of x - lo - s b, where s b is exact (16 bits) and x - lo a sum of two f32
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float y = ((const float *)f)[i], d = y - lo, n = floorf(d * inv);
            if (fabsf(d * inv - n - 0.5f) < 0x1p-16f) {
                const float e = fmaf(-s, n + 0.5f, d), z = d - y, rest = (y - (d - z)) + (-lo - z);
                if (e == 0.f && rest != 0.f) ((float *)r)[i] = (float)kv4_code64(y, lo, s);
                else ((float *)r)[i] = n + (e > 0.f || (e == 0.f && ((int)n & 1)) ? 1.f : 0.f);
            }
        }
    }
    if (!inside)
#pragma unroll
        for (int i = 0; i < 16; i++)
            ((float *)r)[i] = bad ? 0.f : (float)kv4_code64(fminf(fmaxf(((const float *)f)[i], -65504.f), 65504.f), lo, s);
    // two to a byte, two bytes to a number below 2^16, in f32: exact
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        c[i] = __float_as_uint(fmaf(r[2 * i + 1].y, 4096.f, fmaf(r[2 * i + 1].x, 256.f, fmaf(r[2 * i].y, 16.f, r[2 * i].x))) + 8388608.f);
    return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}

// Where a piece's codes and its group's pair stand in the block of its page and
// head, or false for no slot.
template <typename T>
struct Kv4Piece {
    int t, head, d0;
    long long off;  // of the block from the cache's start
    int code, pair; // bytes within it
    __device__ __forceinline__ bool find(const Kv4Rows<T> &a, int piece)
    {
        t = fdiv(piece, a.per_token);
        const int left = piece - t * a.per_token.d;
        head = fdiv(left, a.per_head);
        d0 = (left - head * a.per_head.d) * a.each;
        const long long slot = a.slots[t];
        if (slot < 0 || slot >= (long long)a.g.pages * a.g.size) return false;
        const long long page = a.slots32 ? fdiv((int)slot, a.size) : slot / a.g.size;
        const int place = (int)(slot - page * a.g.size);
        off = page * a.g.page_stride + (long long)head * a.block;
        code = (place * a.g.d + d0) >> 1;
        pair = a.g.size * (a.g.d >> 1) + ((place * a.g.d) >> 3) + (d0 >> 5) * 4;
        return true;
    }
};

// 16 elements of K and the same of V a thread.
template <typename T>
__global__ void __launch_bounds__(128, 8) kv4_file_kernel(const Kv4Rows<T> a)
{
    behind_last_launch();
    const int piece = (int)(blockIdx.x * 128 + threadIdx.x);
    Kv4Piece<T> p;
    const bool kept = piece < a.pieces && p.find(a, piece);  // both lanes of a group, or neither
    Vec8<T> k[2] = {}, v[2] = {};
    if (kept) {
        const T *kt = a.k.at(p.t, p.head) + p.d0, *vt = a.v.at(p.t, p.head) + p.d0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            k[i] = read8(kt + 8 * i, a.vec);
            v[i] = read8(vt + 8 * i, a.vec);
        }
    }
    uint32_t kp, vp;
    const uint2 kc = kv4_quantise<T>(k, kp), vc = kv4_quantise<T>(v, vp);
    if (!kept) return;
    *(uint2 *)(a.g.k + p.off + p.code) = kc;
    *(uint2 *)(a.g.v + p.off + p.code) = vc;
    if (!(p.d0 & 31)) {
        *(uint32_t *)(a.g.k + p.off + p.pair) = kp;
        *(uint32_t *)(a.g.v + p.off + p.pair) = vp;
    }
}

__device__ __forceinline__ void kv4_values(uint32_t codes, uint32_t pair, float *f)
{
    const float2 m = __half22float2(*(const __half2 *)&pair);
    const float2 s = make_float2(m.x, m.x), lo = make_float2(m.y, m.y), less = make_float2(-8388608.f, -8388608.f);
    // a code in a byte of its own, that byte the lowest of 2^23's: 2^23 + code
    const uint32_t even = codes & 0x0F0F0F0Fu, odd = codes >> 4 & 0x0F0F0F0Fu;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 c = make_float2(__uint_as_float(__byte_perm(even, 0x4B000000u, 0x7440 + i)), __uint_as_float(__byte_perm(odd, 0x4B000000u, 0x7440 + i)));
        ((float2 *)f)[i] = __ffma2_rn(__fadd2_rn(c, less), s, lo);
    }
}

template <typename T>
__device__ __forceinline__ void write8(T *p, int vec, const float *f)
{
    if (vec) store8(p, pack8<T>(f));
    else
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = from_f32<T>(f[i]);
}

template <typename T>
__global__ void __launch_bounds__(128) kv4_load_kernel(const Kv4Rows<T> a)
{
    behind_last_launch();
    const int piece = (int)(blockIdx.x * 128 + threadIdx.x);
    if (piece >= a.pieces) return;
    Kv4Piece<T> p;
    const bool kept = p.find(a, piece);
    float k[8] = {}, v[8] = {};
    if (kept) {
        kv4_values(*(const uint32_t *)(a.g.k + p.off + p.code), *(const uint32_t *)(a.g.k + p.off + p.pair), k);
        kv4_values(*(const uint32_t *)(a.g.v + p.off + p.code), *(const uint32_t *)(a.g.v + p.off + p.pair), v);
    }
    write8(a.k.at(p.t, p.head) + p.d0, a.vec, k);
    write8(a.v.at(p.t, p.head) + p.d0, a.vec, v);
}

template <typename T>
static cudaError_t kv4_rows_launch(const aie_kv4_rows &p, bool file, cudaStream_t s)
{
    Kv4Rows<T> a;
    a.g = kv4_geom(p.cache);
    a.k = heads_of<T>(p.k); a.v = heads_of<T>(p.v);
    a.slots = p.slots;
    // a lane's elements: half of a group that it has the range of; 8, whose values it writes
    // (16: 21.9 us for 16384 tokens of 8 heads of 128, against 20.1)
    a.each = file ? 16 : 8;
    const int per_head = a.g.d / a.each, per_token = a.g.heads * per_head;
    a.pieces = (int)p.tokens * per_token;
    a.per_token = make_fastdiv(per_token); a.per_head = make_fastdiv(per_head); a.size = make_fastdiv(a.g.size);
    a.slots32 = (long long)a.g.pages * a.g.size <= 0x7fffffffll;
    a.block = a.g.block();
    auto ok = [](const aie_heads &h) {
        const int64_t unit = 16 / sizeof(T);
        return (uintptr_t)h.data % 16 == 0 && h.token_stride % unit == 0 && h.head_stride % unit == 0;
    };
    a.vec = ok(p.k) && ok(p.v);
    return launch_behind(file ? kv4_file_kernel<T> : kv4_load_kernel<T>, (a.pieces + 127) / 128, 128, 0, s, a);
}

}  // namespace aie
