// Device helpers of the paged cache's kernels: element types, their conversions, and the matrix-instruction operands
// built from what the cache holds.
#pragma once
#include "paged.h"

namespace bg {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// two values rounded to nearest, the first in the low half
__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a, b}, v2b));
}

// eight consecutive elements (16-byte aligned) <-> fp32
template <int T>
__device__ __forceinline__ void load8(const void *p, size_t at, float *x)
{
    if (T == PT_F32) {
        const v4f a = ((const v4f *)((const float *)p + at))[0], b = ((const v4f *)((const float *)p + at))[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    } else if (T == PT_F16) {
        const v8h a = *(const v8h *)((const uint16_t *)p + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = (float)a[i];
        }
    } else {
        const v4u a = *(const v4u *)((const uint16_t *)p + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
}

template <int T>
__device__ __forceinline__ void store8(void *p, size_t at, const float *x)
{
    if (T == PT_F32) {
        v4f a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = x[i];
            b[i] = x[4 + i];
        }
        ((v4f *)((float *)p + at))[0] = a;
        ((v4f *)((float *)p + at))[1] = b;
    } else if (T == PT_F16) {
        v8h a;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = (_Float16)x[i];
        }
        *(v8h *)((uint16_t *)p + at) = a;
    } else {
        v4u a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
        }
        *(v4u *)((uint16_t *)p + at) = a;
    }
}

// a list that no kernel running now writes, for reads at the wave's own index: they go through the scalar unit, so that no
// vector load behind them has to be waited for
typedef const __attribute__((address_space(4))) int32_t *uniform_list;

// ---- sums over a wave ---------------------------------------------------------------------------------
// Inclusive sums over the 64 lanes, on the vector unit alone (rows of 16, then 15 -> 16.., 31 -> 32..)
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v)
{
#define BG_SCAN_STEP(ctrl, rows) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false)
    BG_SCAN_STEP(0x111, 0xf);  // row_shr:1
    BG_SCAN_STEP(0x112, 0xf);
    BG_SCAN_STEP(0x114, 0xf);
    BG_SCAN_STEP(0x118, 0xf);
    BG_SCAN_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    BG_SCAN_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef BG_SCAN_STEP
    return v;
}

// largest magnitude of the 64 lanes' values, none of them NaN
__device__ __forceinline__ float wave_max_abs(float f)
{
    uint32_t v = __float_as_uint(fabsf(f));
#define BG_MAX_STEP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
    BG_MAX_STEP(0x111, 0xf);  // (as in wave_scan_u32)
    BG_MAX_STEP(0x112, 0xf);
    BG_MAX_STEP(0x114, 0xf);
    BG_MAX_STEP(0x118, 0xf);
    BG_MAX_STEP(0x142, 0xa);
    BG_MAX_STEP(0x143, 0xc);
#undef BG_MAX_STEP
    return __uint_as_float(__builtin_amdgcn_readlane(v, 63));
}

// A list of n counts, count(i), laid end to end: which entry place x falls into. Every wave finds out by itself. The first 64
// counts are asked for once.
struct Places {
    uint32_t first, upto, sum;  // this lane's of the first 64 counts, the sum up to it, the sum of all
};

template <typename F>
__device__ __forceinline__ Places places_of(uint32_t n, uint32_t lane, F count)
{
    Places p;
    p.first = lane < n ? count(lane) : 0;
    p.upto = wave_scan_u32(p.first);
    p.sum = __builtin_amdgcn_readlane(p.upto, 63);
    for (uint32_t i0 = 64; i0 < n; i0 += 64) {
        p.sum += __builtin_amdgcn_readlane(wave_scan_u32(i0 + lane < n ? count(i0 + lane) : 0), 63);
    }
    return p;
}

// x < p.sum; *before: the places in front of the entry
template <typename F>
__device__ __forceinline__ uint32_t entry_at(const Places &p, uint32_t n, uint32_t lane, uint32_t x, F count, uint32_t *before)
{
    uint32_t base = 0, c = p.first, upto = p.upto;
    for (uint32_t i0 = 0;;) {
        const uint32_t all = __builtin_amdgcn_readlane(upto, 63);
        if (x < base + all || i0 + 64 >= n) {
            const unsigned long long behind = __ballot(base + upto > x);
            const uint32_t at = behind ? (uint32_t)__builtin_ctzll(behind) : 63;
            *before = base + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(c, at);
            return min(i0 + at, n - 1);
        }
        base += all;
        i0 += 64;
        c = i0 + lane < n ? count(i0 + lane) : 0;
        upto = wave_scan_u32(c);
    }
}

// ---- operands of the matrix instructions ------------------------------------------------------------
// A 32-deep 16-bit operand: lane (i = lane % 16, g = lane / 16) holds eight contraction elements of row (column) i. Which
// eight of a head's DIM values step s of lane group g means is free as long as both operands agree (d_of): an int8 lane
// takes 16 neighbours for two steps, one wide load.
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

// power of two that brings a row with the largest magnitude `top` to [2^14, 2^15) -- inside fp16 with 38 binary orders
// below it -- and the exponent *e of its inverse. Zero, infinity and NaN stay as they are.
__device__ __forceinline__ float shift_into_f16(float top, int *e)
{
    if (!(top > 0.0f && top < INFINITY)) {
        *e = 0;
        return 1.0f;
    }
    int x;
    (void)frexpf(top, &x);  // top = f * 2^x, f in [0.5, 1)
    x = x < -100 ? -100 : x;
    *e = x - 15;
    return ldexpf(1.0f, 15 - x);
}

// the smallest power of two that is not below x, from kFirstUnit up to 2^126, the largest whose reciprocal is a normal number (and
// the largest step that a normal scale makes)
constexpr float kFirstUnit = 7.88860905e-31f;  // 2^-100
__device__ __forceinline__ float power_above(float x)
{
    const uint32_t u = (__float_as_uint(x) + 0x7fffffu) & 0x7f800000u;
    return fminf(fmaxf(__uint_as_float(u), kFirstUnit), 8.50705917e37f);
}

// what a part's outputs and sum are multiplied by before the former become multiples of 1 instead of `unit`: weights lie up to 2^15
// above the formula's, and fp32 has to hold their products with the largest values
template <int CT>
constexpr float kPartScale = CT == PT_I8 ? 0x1p-15f : 1.0f;

// four slots' factors from 4-byte aligned memory
__device__ __forceinline__ v4f load_scales(const float *p)
{
    typedef float v4f_a4 __attribute__((ext_vector_type(4), aligned(4)));
    return *(const v4f_a4 *)p;
}

template <int W>
struct Words;
template <>
struct Words<1> {
    uint32_t w[1];
};
template <>
struct Words<2> {
    uint32_t w[2];
};
template <>
struct Words<4> {
    uint32_t w[4];
};

// ONCE: nobody else reads it, past the caches (a read of 2 GiB goes at 7.0 TB/s so, at 6.2 through them)
template <bool ONCE, typename T>
__device__ __forceinline__ T load_as(const void *p)
{
    return ONCE ? __builtin_nontemporal_load((const T *)p) : *(const T *)p;
}

template <int W, bool ONCE>
__device__ __forceinline__ Words<W> load_words(const void *p)
{
    Words<W> r;
    if (W == 4) {
        const v4u v = load_as<ONCE, v4u>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            r.w[i] = v[i];
        }
    } else if (W == 2) {
        const v2u v = load_as<ONCE, v2u>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            r.w[i] = v[i];
        }
    } else {
        r.w[0] = load_as<ONCE, uint32_t>(p);
    }
    return r;
}

template <int W>
__device__ __forceinline__ Words<W> zero_words()
{
    Words<W> r;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        r.w[i] = 0;
    }
    return r;
}

// products in fp16: an fp16 cache, or an int8 one, whose values fp16 holds exactly
struct OperandF16 {
    typedef v8h V;
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    // a and b as sums of two fp16 parts (what is left is below 2^-21 of them); fp16 and bf16 values are all in the first
    static __device__ __forceinline__ void split2(float a, float b, uint32_t *hi, uint32_t *lo)
    {
        const auto r = __builtin_amdgcn_cvt_pkrtz(a, b);
        *hi = __builtin_bit_cast(uint32_t, r);
        *lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a - (float)r[0], b - (float)r[1]));
    }
    static __device__ __forceinline__ void split(const float *x, float up, V *hi, V *lo)
    {
        union {
            V v;
            uint32_t w[4];
        } h, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            split2(x[2 * i] * up, x[2 * i + 1] * up, &h.w[i], &l.w[i]);
        }
        *hi = h.v;
        *lo = l.v;
    }
};

struct OperandBf16 {
    typedef v8b V;
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split2(float x, float y, uint32_t *hi, uint32_t *lo)  // the upper halves are the truncated values
    {
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        *hi = __builtin_amdgcn_perm(b, a, 0x07060302);
        const float ra = x - __uint_as_float(a & 0xffff0000u), rb = y - __uint_as_float(b & 0xffff0000u);
        *lo = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302);
    }
    static __device__ __forceinline__ void split(const float *x, float up, V *hi, V *lo)
    {
        union {
            V v;
            uint32_t w[4];
        } h, l;
        (void)up;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            split2(x[2 * i], x[2 * i + 1], &h.w[i], &l.w[i]);
        }
        *hi = h.v;
        *lo = l.v;
    }
};

template <int CT>
struct Operand : OperandF16 {};
template <>
struct Operand<PT_BF16> : OperandBf16 {};

// What the cache holds -> operands. K: eight d of one key per step. V: DIM / 16 neighbouring d of eight keys (d = DIM / 16 * c
// + t for operand t), pairs of keys brought into one register.
template <int CT>
struct CacheOperand : Operand<CT> {
    typedef typename Operand<CT>::V V;
    typedef Words<4> Raw;
    template <int DIM>
    using RawV = Words<DIM / 32>;
    static constexpr int kRawK(int dim) { return dim / 32; }
    static __device__ __forceinline__ uint32_t d_of(uint32_t s, uint32_t g) { return 32 * s + 8 * g; }
    template <bool ONCE, int N>
    static __device__ __forceinline__ void load_k(const uint8_t *row, uint32_t g, Raw (&r)[N])
    {
#pragma unroll
        for (int s = 0; s < N; ++s) {
            r[s] = load_words<4, ONCE>(row + 2 * d_of(s, g));
        }
    }
    static __device__ __forceinline__ V k_operand(const Raw *r, int s) { return __builtin_bit_cast(V, r[s]); }
    template <bool ONCE, int DIM>
    static __device__ __forceinline__ RawV<DIM> load_v(const uint8_t *row, uint32_t c) { return load_words<DIM / 32, ONCE>(row + c * (DIM / 8)); }
    template <int DIM>
    static __device__ __forceinline__ RawV<DIM> zero_v() { return zero_words<DIM / 32>(); }
    template <int DIM>
    static __device__ __forceinline__ V v_operand(const RawV<DIM> *r, int t)
    {
        Words<4> w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w.w[i] = __builtin_amdgcn_perm(r[2 * i + 1].w[t / 2], r[2 * i].w[t / 2], t & 1 ? 0x07060302 : 0x05040100);
        }
        return __builtin_bit_cast(V, w);
    }
};

// Two bytes in the low halves of a word's two 16-bit places, of two's complement -> two fp16: with the sign bit flipped and
// 0x64 in front (biased) they read 1024 + 128 + value, exactly
__device__ __forceinline__ uint32_t biased_to_f16(uint32_t w)
{
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const v2h x = __builtin_bit_cast(v2h, w);
    return __builtin_bit_cast(uint32_t, x - (v2h){(_Float16)1152.0f, (_Float16)1152.0f});
}

__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t w)
{
    return biased_to_f16(w ^ 0x64806480u);
}

template <>
struct CacheOperand<PT_I8> : Operand<PT_I8> {
    typedef typename Operand<PT_I8>::V V;
    typedef Words<4> Raw;
    template <int DIM>
    using RawV = Words<DIM / 64>;
    static constexpr int kRawK(int dim) { return dim / 64; }
    static __device__ __forceinline__ uint32_t d_of(uint32_t s, uint32_t g) { return 64 * (s / 2) + 16 * g + 8 * (s % 2); }
    template <bool ONCE, int N>
    static __device__ __forceinline__ void load_k(const uint8_t *row, uint32_t g, Raw (&r)[N])
    {
#pragma unroll
        for (int s = 0; s < N; ++s) {
            r[s] = load_words<4, ONCE>(row + d_of(2 * s, g));
        }
    }
    static __device__ __forceinline__ V k_operand(const Raw *r, int s)
    {
        Words<4> w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w.w[i] = bytes_to_f16(__builtin_amdgcn_perm(0, r[s / 2].w[2 * (s % 2) + i / 2], i & 1 ? 0x0c030c02 : 0x0c010c00));
        }
        return __builtin_bit_cast(V, w);
    }
    template <bool ONCE, int DIM>
    static __device__ __forceinline__ RawV<DIM> load_v(const uint8_t *row, uint32_t c) { return load_words<DIM / 64, ONCE>(row + c * (DIM / 16)); }
    template <int DIM>
    static __device__ __forceinline__ RawV<DIM> zero_v() { return zero_words<DIM / 64>(); }
    template <int DIM>
    static __device__ __forceinline__ V v_operand(const RawV<DIM> *r, int t)
    {
        Words<4> w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // byte t % 4 of two keys
            w.w[i] = bytes_to_f16(__builtin_amdgcn_perm(r[2 * i + 1].w[t / 4], r[2 * i].w[t / 4], 0x0c040c00u + (uint32_t)(t % 4) * 0x00010001u));
        }
        return __builtin_bit_cast(V, w);
    }
};

// (activation type, cache type, head size) -> instantiation; the C-ABI layer refuses every other combination
template <template <int, int, int> class F, typename A>
hipError_t paged_dispatch(int act, int ct, uint32_t dim, const A &a, hipStream_t st)
{
#define BG_PAGED(X, C)                                                         \
    if (act == X && ct == C) {                                                 \
        return dim == 64 ? F<X, C, 64>::run(a, st) : F<X, C, 128>::run(a, st); \
    }
    BG_PAGED(PT_F32, PT_F16)
    BG_PAGED(PT_F32, PT_I8)
    BG_PAGED(PT_F16, PT_F16)
    BG_PAGED(PT_F16, PT_I8)
    BG_PAGED(PT_BF16, PT_BF16)
    BG_PAGED(PT_BF16, PT_I8)
#undef BG_PAGED
    return hipErrorInvalidValue;
}

}  // namespace bg
