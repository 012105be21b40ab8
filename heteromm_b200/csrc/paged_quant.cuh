// paged_quant.cuh — a paged cache held in 8 bits: its layout, and codes and scales to and
// from 16-bit values.
//
// Page arrays of bytes, free page / head strides.  Of each page and head one block: the
// codes [page_tokens][D], then a scale byte for each 32 values [page_tokens][D / 32].
//
//   value = code * 2^(s - 127)
//
// with s the smallest scale that holds the group: A = max |x|, e = least integer with
// A <= M 2^e (M = 448 for e4m3, 127 for int8), held to [-15 or -22, 7], s = e + 127;
// code = x 2^-e rounded to the nearest (ties to even), saturated at M.  A group with an
// infinity or NaN has s = 255 and codes of zero, and reads as NaN.  Scales are powers of two
// and at least 2^-15 (2^-22), at most 2^7, so that a value is a bf16 and an fp16 number
// exactly (a 4- or 8-bit significand; above 2^-25, at most 57,344): a product with it needs
// no second factor, and attention over the cache is that over a 16-bit cache of its values.
// A scale per 32 values costs 3% of the memory; one per head would be 1% and leave int8 with a
// few bits beside a large dimension.
#pragma once

#include <type_traits>

#include "paged_serve.cuh"

namespace hmm {
namespace serve {

enum Codec { CODEC_NONE, CODEC_E4M3, CODEC_I8 };   // NONE: 16-bit values as they are
constexpr int Q_GROUP = 32;

// Of a page array: where the scale bytes of a page and head begin, and a token's.
struct QuantRows {
    int64_t scales;   // page_tokens * D
    int per_token;    // D / 32
};

// ------------------------------------------------------------ to codes

// The scale byte of a group whose largest magnitude has the bits `top` (an infinity's or NaN's
// are the largest of all).  The exponent of A / M rounds up where A's significand is above M's:
// adding what M's lacks to the next power of two carries then.
template <int C>
__device__ __forceinline__ int scale_byte(uint32_t top) {
    constexpr uint32_t UP = C == CODEC_E4M3 ? 0x7fffffu - 0x600000u : 0x7fffffu - 0x7e0000u;   // 1.75, 127 / 64
    constexpr int POWER = C == CODEC_E4M3 ? 8 : 6, LOW = C == CODEC_E4M3 ? 127 - 15 : 127 - 22;
    if (top >= 0x7f800000u) return 255;
    return min(max((int)((top + UP) >> 23) - POWER, LOW), 127 + 7);
}

// Four codes, the first in the lowest byte, of values scaled already.
template <int C>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    if (C == CODEC_E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | (uint32_t)hi << 16;
    }
    auto code = [](float x) { return (uint32_t)__float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f)); };
    return __byte_perm(__byte_perm(code(a), code(b), 0x0040), __byte_perm(code(c), code(d), 0x0040), 0x5410);
}

// ------------------------------------------------------------ to 16-bit values

// Codes to pairs of T without arithmetic of fp32: of a word's four, the bytes 0 and 2
// (`even`) and 1 and 3 (`odd`), times a constant that multiplier() takes back.
//   e4m3: sign, 4 and 3 bits moved into T's fields: times 2^(7 - 127) (bf16) or 2^(7 - 15)
//   int8, bf16: 128 + the low seven bits, less 128 or, for a sign, 256: the value itself
//   int8, fp16: 4 + (n + 128) / 256 less 4.5: times 2^-8
template <typename T, int C>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& even, uint32_t& odd) {
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    if (C == CODEC_E4M3) {
        if (BF) {
            even = ((w << 4) & 0x07f007f0u) | ((w << 8) & 0x80008000u);
            odd = ((w >> 4) & 0x07f007f0u) | (w & 0x80008000u);
        } else {
            even = ((w << 7) & 0x3f803f80u) | ((w << 8) & 0x80008000u);
            odd = ((w >> 1) & 0x3f803f80u) | (w & 0x80008000u);
        }
    } else if (BF) {
        auto value = [](uint32_t x) {
            uint32_t r, a = (x & 0x007f007fu) | 0x43004300u, b = (x & 0x00800080u) | 0x43004300u;
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
            return r;
        };
        even = value(w);
        odd = value(w >> 8);
    } else {
        const uint32_t x = w ^ 0x80808080u;
        auto value = [](uint32_t a) {
            uint32_t r;
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x44804480u));
            return r;
        };
        even = value((x & 0x00ff00ffu) | 0x44004400u);
        odd = value(((x >> 8) & 0x00ff00ffu) | 0x44004400u);
    }
}

__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// The factors 2^(s - 127), and what widen() left, of two scale bytes (in the low bytes of the
// halves) as a pair of T: an infinity for s = 255, which makes NaN of codes of zero.  In fp16
// they are 2^-14 ... 2^15, normal numbers all.
template <typename T, int C>
__device__ __forceinline__ uint32_t multiplier(uint32_t s) {
    if (std::is_same<T, __nv_bfloat16>::value)
        return (C == CODEC_E4M3 ? min_u16x2(s + 0x00780078u, 0x00ff00ffu) : s) << 7;
    return min_u16x2(max_u16x2(s, 0x00690069u) - 0x00680068u, 0x001f001fu) << 10;
}

template <typename T>
__device__ __forceinline__ uint32_t mul_pair(uint32_t a, uint32_t b) {
    uint32_t d;
    if (std::is_same<T, __nv_bfloat16>::value)
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// The first two and the last two of a word's four values, from their even and odd pairs.
__device__ __forceinline__ uint32_t in_order_lo(uint32_t even, uint32_t odd) { return __byte_perm(even, odd, 0x5410); }
__device__ __forceinline__ uint32_t in_order_hi(uint32_t even, uint32_t odd) { return __byte_perm(even, odd, 0x7632); }

// One code's value times its scale, in fp32.
template <int C>
__device__ __forceinline__ float value_of(uint32_t code, uint32_t s) {
    const float scale = __uint_as_float(s != 0 ? s << 23 : 0x00400000u);   // 2^-127 is subnormal
    if (C == CODEC_I8) return (float)(int8_t)code * scale;
    return __uint_as_float((code & 0x80u) << 24 | (code & 0x7fu) << 20) * 0x1p120f * scale;
}

// Sixteen codes of one scale as values of O at dst.
template <typename O, int C>
__device__ __forceinline__ void store16(O* dst, const uint4& w, uint32_t s) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    if constexpr (std::is_same<O, float>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4*>(dst)[i] =
                make_float4(value_of<C>(u[i] & 255u, s), value_of<C>(u[i] >> 8 & 255u, s),
                            value_of<C>(u[i] >> 16 & 255u, s), value_of<C>(u[i] >> 24, s));
    } else {
        const uint32_t m = multiplier<O, C>(s | s << 16);
        uint32_t r[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t even, odd;
            widen<O, C>(u[i], even, odd);
            even = mul_pair<O>(even, m);
            odd = mul_pair<O>(odd, m);
            r[2 * i] = in_order_lo(even, odd);
            r[2 * i + 1] = in_order_hi(even, odd);
        }
        if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {   // a sector at once
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                         "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                         : "memory");
        } else {
            reinterpret_cast<uint4*>(dst)[0] = make_uint4(r[0], r[1], r[2], r[3]);
            reinterpret_cast<uint4*>(dst)[1] = make_uint4(r[4], r[5], r[6], r[7]);
        }
    }
}

// ------------------------------------------------------------ host helpers

// The sizes of a cache as those of one of 16-bit values.
inline hmm_paged_cache_t quant_dims(const hmm_paged_quant_t& c) {
    hmm_paged_cache_t d{};
    d.k = c.k;
    d.v = c.v;
    d.n_pages = c.n_pages;
    d.n_kv_heads = c.n_kv_heads;
    d.page_tokens = c.page_tokens;
    d.D = c.D;
    d.dtype = HMM_DTYPE_BF16;
    return d;
}

// Fills `b`, `k`, `v` (token strides: D) and `rows` from the ABI's descriptions, or returns the error.
hmm_status_t check_quant(const hmm_paged_quant_t* cache, const hmm_paged_batch_t* batch, Batch* b, Pages* k, Pages* v,
                         QuantRows* rows);

}  // namespace serve
}  // namespace hmm
