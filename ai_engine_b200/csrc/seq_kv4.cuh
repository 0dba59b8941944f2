// A paged cache in 4 bits: filing and reading back.
//
//   lo = f16(min x),  s = f16((max x - lo) / 15),  code = rint((x - lo) / s),
//   x' = lo + code s
//
// for each group of 32 elements of a head: 5 bits an element.  All four steps are
// as in 64 bits, so that a cache can be told from its inputs to the bit; in f32
// arithmetic wherever that cannot make a difference.
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
    int pieces;       // of 8 elements: tokens * heads * d / 8
    FastDiv per_token, per_head;
    int vec;          // 16-byte accesses
};

// 8 neighbouring elements, in one access where they are aligned.
template <typename T>
__device__ __forceinline__ void read8(const T *p, int vec, float *f)
{
    if (vec) unpack8<T>(load8(p), f);
    else
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = to_f32(p[i]);
}

// Next to a border between two codes, where f32 may be on the wrong side.
__device__ __noinline__ float kv4_code64(float x, float lo, float s) { return (float)rint(((double)x - (double)lo) / (double)s); }
__device__ __noinline__ float kv4_scale64(float hi, float lo) { return (float)(((double)hi - (double)lo) / 15.0); }

// A lane's 8 of a group's 32 elements (four neighbouring lanes): their codes,
// and the group's (s, lo).
__device__ __forceinline__ uint32_t kv4_quantise(float *f, uint32_t &pair)
{
    bool bad = false;
    float lo = 65504.f, hi = -65504.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        bad |= !(fabsf(f[i]) <= 3.402823466e38f);
        f[i] = fminf(fmaxf(f[i], -65504.f), 65504.f);
        lo = fminf(lo, f[i]);
        hi = fmaxf(hi, f[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
    }
    const __half low = __float2half_rn(lo);
    lo = __half2float(low);
    // the f16 next to (hi - lo) / 15: three roundings of f32 move that by less
    // than 2^-21 of it, which rarely reaches over a border of f16
    const float t = fmaxf(hi - lo, 0.f) * (1.f / 15.f);
    __half scale = __float2half_rn(t * (1.f - 0x1p-21f));
    if (__half_as_ushort(scale) != __half_as_ushort(__float2half_rn(t * (1.f + 0x1p-21f)))) scale = __float2half_rn(kv4_scale64(hi, lo));
    const float s = __half2float(scale), inv = s > 0.f ? 1.f / s : 0.f;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float q = (f[i] - lo) * inv;  // less than 2^-18 off
        float r = rintf(q);
        if (fabsf(fabsf(q - r) - 0.5f) < 0x1p-15f) r = kv4_code64(f[i], lo, s);
        codes |= (uint32_t)fminf(fmaxf(r, 0.f), 15.f) << 4 * i;
    }
    pair = bad ? 0x7fff0000u : (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(low) << 16;
    return bad ? 0 : codes;
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
        d0 = (left - head * (a.g.d >> 3)) * 8;
        const long long slot = a.slots[t];
        if (slot < 0 || slot >= (long long)a.g.pages * a.g.size) return false;
        const long long page = slot / a.g.size;
        const int place = (int)(slot - page * a.g.size);
        off = page * a.g.page_stride + head * a.g.block();
        code = (place * a.g.d + d0) >> 1;
        pair = a.g.size * (a.g.d >> 1) + ((place * a.g.d) >> 3) + (d0 >> 5) * 4;
        return true;
    }
};

// A piece of K and the same of V a thread.
template <typename T>
__global__ void __launch_bounds__(128) kv4_file_kernel(const Kv4Rows<T> a)
{
    behind_last_launch();
    const int piece = (int)(blockIdx.x * 128 + threadIdx.x);
    Kv4Piece<T> p;
    const bool real = piece < a.pieces;  // whole groups of four lanes
    const bool kept = real && p.find(a, piece);
    float k[8] = {}, v[8] = {};
    if (kept) {
        read8(a.k.at(p.t, p.head) + p.d0, a.vec, k);
        read8(a.v.at(p.t, p.head) + p.d0, a.vec, v);
    }
    uint32_t kp, vp;
    const uint32_t kc = kv4_quantise(k, kp), vc = kv4_quantise(v, vp);
    if (!kept) return;
    *(uint32_t *)(a.g.k + p.off + p.code) = kc;
    *(uint32_t *)(a.g.v + p.off + p.code) = vc;
    if (!(p.d0 & 31)) {
        *(uint32_t *)(a.g.k + p.off + p.pair) = kp;
        *(uint32_t *)(a.g.v + p.off + p.pair) = vp;
    }
}

__device__ __forceinline__ void kv4_values(uint32_t codes, uint32_t pair, float *f)
{
    const float2 m = __half22float2(*(const __half2 *)&pair);
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = fmaf((float)(codes >> 4 * i & 15u), m.x, m.y);
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
    const int per_head = a.g.d / 8, per_token = a.g.heads * per_head;
    a.pieces = (int)p.tokens * per_token;
    a.per_token = make_fastdiv(per_token); a.per_head = make_fastdiv(per_head);
    auto ok = [](const aie_heads &h) {
        const int64_t unit = 16 / sizeof(T);
        return (uintptr_t)h.data % 16 == 0 && h.token_stride % unit == 0 && h.head_stride % unit == 0;
    };
    a.vec = ok(p.k) && ok(p.v);
    return launch_behind(file ? kv4_file_kernel<T> : kv4_load_kernel<T>, (a.pieces + 127) / 128, 128, 0, s, a);
}

}  // namespace aie
