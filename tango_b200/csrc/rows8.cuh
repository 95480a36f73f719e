// Device side of the 8-bit rows: a matrix cut into groups of neighbouring columns, each with int8 codes and one fp32 scale.
#pragma once
#include "common.cuh"

namespace tango {

constexpr float kSmallestNormal = 1.1754943508222875e-38f;      // 2^-126
constexpr float kRoundMagic = 12582912.f;                       // 1.5 * 2^23: adding it leaves round-to-even(t) in the low bits

// Two floats that one instruction works on.
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 both(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair o;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(o.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return o;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair o;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(o.v) : "l"(a.v), "l"(b.v));
    return o;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair o;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(o.v) : "l"(a.v), "l"(b.v));
    return o;
}

// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float o;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(o) : "f"(a), "f"(b), "f"(c));
    return o;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float o;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(a), "f"(b));
    return o;
}

// Scale of a group from its largest magnitude.  A group that holds an infinity or a NaN gets the scale NaN, so that its values
// come back as NaN, not as something else.
__device__ __forceinline__ float group_scale(float top) {
    if (!(top < INFINITY)) return __int_as_float(0x7fffffff);
    const float s = __fdiv_rn(top, 127.0f);
    return s < kSmallestNormal ? 0.f : s;
}
// About 1 / s; 0 for the scales 0 and NaN.
__device__ __forceinline__ float group_inverse(float s) { return s > 0.f ? __fdividef(1.0f, s) : 0.f; }

// N codes: x / s exactly rounded, ties to even.  x * inv is within 127 * 2^-21 of the quotient, which decides all but the values
// that close to a border between two codes.  For those x - q * s is exact in one fused operation (a multiple of half an ulp of
// s, at most about s / 2) and is doubled, exact too, to be compared with s (half of s is not exact for the smallest normal scales,
// where it is a subnormal number).  One question for all N (232965 x 602 fp32: 213 us; one for every
// four values 248), then, for the few, one for every four: bf16 quotients meet borders often (max / 2 lies on one), 205 -> 183 us
// with SiLU of 169343 x 601.  The codes come as floats whose bits hold them in the low byte.
template <int N>
__device__ __forceinline__ void round_nearest(const float *x, float s, float inv, float *b) {
    const Pair by = pair(inv, inv), magic = pair(kRoundMagic, kRoundMagic), minus = pair(-1.f, -1.f);
    float far[N / 4], farthest = 0.f;
#pragma unroll
    for (int k = 0; k < N; k += 4) {
        float d[4];
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const Pair v = pair(x[k + j], x[k + j + 1]), c = fma2(v, by, magic);
            const float2 e = both(fma2(v, by, fma2(c, minus, magic))), f = both(c);
            d[j] = e.x; d[j + 1] = e.y;
            b[k + j] = f.x; b[k + j + 1] = f.y;
        }
        far[k / 4] = max_abs3(max_abs3(d[0], d[1], d[2]), d[3], 0.f);
        farthest = k == 0 ? far[0] : max_or_nan(farthest, far[k / 4]);
    }
    if (farthest > 0.4999f) {
        const float below = __int_as_float(__float_as_int(s) - 1);      // of an odd code a half is enough
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            if (N > 4 && !(far[k / 4] > 0.4999f)) continue;
#pragma unroll
            for (int j = k; j < k + 4; ++j) {
                const float rest = fmaf(__fsub_rn(kRoundMagic, b[j]), s, x[j]);
                if (fabsf(rest + rest) > (__float_as_int(b[j]) & 1 ? below : s)) b[j] = __fadd_rn(b[j], copysignf(1.f, rest));
            }
        }
    }
}
template <int R>
__device__ __forceinline__ void encode_nearest(const float *x, float s, float inv, uint32_t *word) {
    float b[R * 4];
    round_nearest<R * 4>(x, s, inv, b);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t lo = __byte_perm(__float_as_uint(b[4 * r]), __float_as_uint(b[4 * r + 1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(b[4 * r + 2]), __float_as_uint(b[4 * r + 3]), 0x0040);
        word[r] = inv == 0.f ? 0u : __byte_perm(lo, hi, 0x5410);
    }
}

__device__ __forceinline__ float4 four(const float *x) { return make_float4(x[0], x[1], x[2], x[3]); }

// The other rounding modes: truncation, and the seeded stochastic stream keyed by the elements' flat indices: flat + i, and
// `behind` more for the first `turned`.
static __device__ __noinline__ uint32_t encode4_mode(float4 four, float s, int mode, uint64_t seed, uint64_t call, uint64_t flat,
                                                   int turned = 0, int behind = 0) {
    if (!(s > 0.f)) return 0u;
    const float x[4] = {four.x, four.y, four.z, four.w};       // by value: an address would keep the caller's values in memory
    const Philox ph{(uint32_t)seed, (uint32_t)(seed >> 32)};
    uint64_t blk = ~0ull;
    uint4 rnd = make_uint4(0, 0, 0, 0);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float u = mode == TANGO_ROUND_STOCHASTIC ? sr_uniform(ph, flat + i + (i < turned ? behind : 0), call, blk, rnd) : 0.f;
        word |= (uint32_t)(uint8_t)round_to_i8(__fdiv_rn(x[i], s), mode, u) << (8 * i);
    }
    return word;
}

// The four codes of a word as floats: the biased code lands in the mantissa of 2^23, exactly.
__device__ __forceinline__ void decode4(uint32_t word, Pair &lo, Pair &hi) {
    const uint32_t w = word ^ 0x80808080u;
    const Pair bias = pair(-8388736.f, -8388736.f);
    lo = add2(pair(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441))), bias);
    hi = add2(pair(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7442)), __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7443))), bias);
}

// Quotients of indices below 2^31 by a fixed divisor: floor(i * m / 2^(32 + shift)), with m rounded up.
struct FastDiv {
    uint32_t d, m, shift;
};
inline FastDiv fast_div(int64_t d) {
    FastDiv f{(uint32_t)d, 0, 0};
    if (d <= 1) return f;
    while ((1ull << (f.shift + 1)) < (uint64_t)d) ++f.shift;            // 2^shift < d <= 2^(shift + 1)
    f.m = (uint32_t)(((1ull << (32 + f.shift)) + (uint64_t)d - 1) / (uint64_t)d);
    return f;
}
__device__ __forceinline__ uint32_t quotient(uint32_t i, const FastDiv &f) { return f.d <= 1 ? i : __umulhi(i, f.m) >> f.shift; }

// Element types of the matrices: TANGO_FP32, TANGO_BF16, TANGO_FP16.  bf16 and fp16 results are rounded once, to nearest.
struct Bf16 { uint16_t bits; };
struct Fp16 { uint16_t bits; };
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ float to_float(Fp16 v) {
    float f;
    asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(v.bits));
    return f;
}
__device__ __forceinline__ void from_float(float v, float &o) { o = v; }
__device__ __forceinline__ void from_float(float v, Bf16 &o) { asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(o.bits) : "f"(v)); }
__device__ __forceinline__ void from_float(float v, Fp16 &o) { asm("cvt.rn.f16.f32 %0, %1;" : "=h"(o.bits) : "f"(v)); }

// Two neighbouring elements in a word.
template <class T> __device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi) {
    T a, b;
    a.bits = (uint16_t)w;
    b.bits = (uint16_t)(w >> 16);
    lo = to_float(a);
    hi = to_float(b);
}
template <> __device__ __forceinline__ void unpack2<Bf16>(uint32_t w, float &lo, float &hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
}
template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<Bf16>(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
template <> __device__ __forceinline__ uint32_t pack2<Fp16>(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

// VL elements at once, p aligned to them.
template <int BYTES> struct Word;
template <> struct Word<2> { typedef uint16_t T; };
template <> struct Word<4> { typedef uint32_t T; };
template <> struct Word<8> { typedef uint2 T; };
template <> struct Word<16> { typedef uint4 T; };
template <class T, int VL> union Pack {
    T e[VL];
    typename Word<VL * sizeof(T)>::T w;
    __device__ Pack() {}
};
// Four neighbouring elements, of which the first n exist (the others read as 0).
template <class T, int VL>
__device__ __forceinline__ void load4(const T *p, int n, float *v) {
#pragma unroll
    for (int i = 0; i < 4; i += VL) {
        Pack<T, VL> k;
        k.w = {};
        if (i + VL <= n) {
            k.w = __ldg(reinterpret_cast<const typename Word<VL * sizeof(T)>::T *>(p + i));
        } else if (VL > 1 && i < n) {
            for (int j = 0; j < VL - 1 && i + j < n; ++j) k.e[j] = p[i + j];
        }
#pragma unroll
        for (int j = 0; j < VL; ++j) v[i + j] = to_float(k.e[j]);
    }
}
template <class T, int VL>
__device__ __forceinline__ void store4(T *p, int n, const float *v) {
#pragma unroll
    for (int i = 0; i < 4; i += VL) {
        Pack<T, VL> k;
#pragma unroll
        for (int j = 0; j < VL; ++j) from_float(v[i + j], k.e[j]);
        if (i + VL <= n) {
            *reinterpret_cast<typename Word<VL * sizeof(T)>::T *>(p + i) = k.w;
        } else if (VL > 1 && i < n) {
            for (int j = 0; j < VL - 1 && i + j < n; ++j) p[i + j] = k.e[j];
        }
    }
}

}  // namespace tango
