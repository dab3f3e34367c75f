// Device-side pieces of the 8-bit cache layout: the codes (e4m3 or int8), the page scale and the rotary angle.
//
// A page (16 cells) of one kv head has, for K and for V each, 16 x head_dim one-byte codes and ONE scale 2^e held as
// f32; the value is code * 2^e.  Powers of two because a page fills one token at a time: dividing by the scale and
// going over to a larger one are then exact up to the single rounding of the code itself, and every value is exact
// in f32 (and, int8's seven bits, in bf16).  They cost at most one bit of an int8 code against a free scale and none of an e4m3
// code, which is a floating number of its own.
#pragma once

#include <cuda_bf16.h>

#include "brc_device.cuh"

namespace brc {

constexpr uint32_t KV8_E4M3 = 1u, KV8_INT8 = 2u;
constexpr int KV8_EXP_MIN = -120, KV8_EXP_MAX = 120;   // 2^e and 2^-e are both normal f32

// Least e with amax <= top * 2^e, top = 448 = 1.75 * 2^8 (e4m3) or 127 = (2 - 2^-6) * 2^6 (int8), clamped.
template <uint32_t CODE>
__device__ __forceinline__ int kv8_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 127;
    const uint32_t m = b & 0x7fffffu;
    const int e = CODE == KV8_E4M3 ? x - 8 + (m > 0x600000u ? 1 : 0) : x - 6 + (m > 0x7e0000u ? 1 : 0);
    return min(max(e, KV8_EXP_MIN), KV8_EXP_MAX);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // |e| <= 126

// The exponent of a stored scale.  Anything but a power of two in range (a page never written) counts as the least.
__device__ __forceinline__ int kv8_scale_exponent(float scale) {
    const uint32_t b = __float_as_uint(scale);
    const int e = (int)(b >> 23) - 127;
    return (b & 0x807fffffu) == 0u && e >= KV8_EXP_MIN && e <= KV8_EXP_MAX ? e : KV8_EXP_MIN;
}

// Four f32 (already divided by the scale) -> four codes, lowest byte first: round to nearest even, saturating,
// NaN -> 0.
template <uint32_t CODE>
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d) {
    a = a == a ? a : 0.f;
    b = b == b ? b : 0.f;
    c = c == c ? c : 0.f;
    d = d == d ? d : 0.f;
    if (CODE == KV8_E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
    auto q = [](float x) { return (uint32_t)__float2int_rn(fminf(fmaxf(x, -127.f), 127.f)) & 0xffu; };
    return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
}

// The same for finite values whose magnitude the scale covers (none saturates): v * inv, inv = 2^-e.  int8: adding 1.5 * 2^23 to
// the exact product rounds it to an integer, ties to even, whose low byte is the code (the conversion instruction runs at
// a quarter of the rate).
template <uint32_t CODE>
__device__ __forceinline__ uint32_t kv8_encode4_finite(float a, float b, float c, float d, float inv) {
    if (CODE == KV8_E4M3) {
        uint32_t r;
        asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
            : "=r"(r) : "f"(a * inv), "f"(b * inv), "f"(c * inv), "f"(d * inv));
        return r;
    }
    const float m = 12582912.f;
    const uint32_t x = __float_as_uint(fmaf(a, inv, m)), y = __float_as_uint(fmaf(b, inv, m)), z = __float_as_uint(fmaf(c, inv, m)),
                   w = __float_as_uint(fmaf(d, inv, m));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// The four codes of a word as two pairs of exact binary16 numbers (bytes 0,1 and bytes 2,3).  int8: a byte with its sign bit flipped, under
// the exponent byte 0x64, is the binary16 number 1024 + 128 + code; subtracting 1152 is exact.
template <uint32_t CODE>
__device__ __forceinline__ void kv8_decode4(uint32_t w, uint32_t &p01, uint32_t &p23) {
    if (CODE == KV8_E4M3) {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(p01), "=r"(p23) : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), bias);
        p01 = *reinterpret_cast<const uint32_t *>(&x);
        p23 = *reinterpret_cast<const uint32_t *>(&y);
    }
}

template <uint32_t CODE>
__device__ __forceinline__ void kv8_decode4_f32(uint32_t w, float (&v)[4]) {
    uint32_t a, b;
    kv8_decode4<CODE>(w, a, b);
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&a)), y = __half22float2(*reinterpret_cast<const __half2 *>(&b));
    v[0] = x.x;
    v[1] = x.y;
    v[2] = y.x;
    v[3] = y.y;
}

// ---------------------------------------------------------------------------------------------
// rows of f32 / f16 / bf16 (dtype tags of breccia_kv.h: 0, 1, 2)
// ---------------------------------------------------------------------------------------------
template <int DT> struct elem;
template <> struct elem<0> { using t = float; static constexpr uint32_t size = 4; };
template <> struct elem<1> { using t = __half; static constexpr uint32_t size = 2; };
template <> struct elem<2> { using t = __nv_bfloat16; static constexpr uint32_t size = 2; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <int DT> __device__ __forceinline__ typename elem<DT>::t from_f32(float x);
template <> __device__ __forceinline__ float from_f32<0>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<1>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<2>(float x) { return __float2bfloat16_rn(x); }

// The larger of a magnitude, given as bits, and |x|; NaN wins (the bits of one are above those of infinity).
__device__ __forceinline__ uint32_t max_magnitude(uint32_t m, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(m)), "f"(fabsf(x)));
    return __float_as_uint(r);
}

// Eight consecutive elements as they lie in memory (`vec`: at a multiple of 16 bytes): half the registers of their f32 values for the
// 16-bit types.
template <int DT>
struct raw8 {
    static constexpr int WORDS = DT == 0 ? 8 : 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const typename elem<DT>::t *p, bool vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                w[i] = u.x;
                w[i + 1] = u.y;
                w[i + 2] = u.z;
                w[i + 3] = u.w;
            }
        } else if constexpr (DT == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(p[i]);
        } else {
            const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (DT == 0) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (DT == 1) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    // Largest magnitude so far, as bits: magnitudes order like unsigned integers, infinities above every finite one and NaN
    // above them.  16-bit types keep two running maxima in one word.
    __device__ __forceinline__ void top(uint32_t &m) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (DT == 0) m = max_magnitude(m, __uint_as_float(w[i]));
            else asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
        }
    }
    // `top`'s word as the bits of an f32
    static __device__ __forceinline__ uint32_t top_f32(uint32_t m) {
        if constexpr (DT == 0) return m;
        const uint32_t h = max(m >> 16, m & 0xffffu);
        if constexpr (DT == 2) return h << 16;
        return h > 0x7c00u ? 0x7fffffffu : __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    }
};

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == 1) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// ---------------------------------------------------------------------------------------------
// rotary angle
// ---------------------------------------------------------------------------------------------
// Turns per position as a 0.64 fixed-point fraction: pos * turns modulo 2^64 IS the fraction of a turn (whole turns
// fall off the top), off by at most pos * 2^-65, where an f32 angle of position 10^6 has lost 16 of its 24 bits.
// Read as a signed number it lies in [-1/2, 1/2) turns; times two that is sincospi's argument.  Sine, cosine and the factor
// in 64 bits and one rounding to f32: a pair is computed once for all heads of a token, and a wrong last bit of it
// shows as a neighbouring 8-bit code wherever a rotated key lies on a border.
// A negative position, as its 64-bit two's complement, turns backwards.
__device__ __forceinline__ float2 rope_cos_sin(uint64_t pos, uint64_t turns, double factor) {
    const int64_t f = (int64_t)(pos * turns);
    double s, c;
    sincospi((double)f * 0x1p-63, &s, &c);
    return make_float2((float)(c * factor), (float)(s * factor));
}

// ---------------------------------------------------------------------------------------------
// page tiles of a ragged batch
// ---------------------------------------------------------------------------------------------
// A call that covers cells pos0[s] .. pos0[s] + T(s) of each sequence works page by page.  How many pages a sequence
// touches depends on pos0, which only the device knows, so tiles get slots from the token counts alone: sequence s has
// the slots from cu[s] / 16 + 2 s up to those of s + 1.  T >= 1 tokens touch at most (T + 14) / 16 + 1 pages, and
// floor((a + T) / 16) - floor(a / 16) + 2 >= floor(T / 16) + 2 is never less; slots past the last page are idle.
struct page_tile {
    uint32_t seq, cell0, first, count, token0;   // page's first cell; first covered cell in it; covered cells; their first token
};

__host__ __device__ inline uint64_t tile_slots(uint32_t total_tokens, uint32_t n_seqs) { return (uint64_t)total_tokens / 16u + 2ull * n_seqs; }

// False: an idle slot.  Cells at or past max_pos_end are cut off (*cut reports the first such cell, else UINT32_MAX).
// Whole warps call it: the search for the sequence takes 32 steps at a time, a lane each (one load in front of the
// others for up to 32 sequences, two for up to 1024; one by one they would be five and ten).
__device__ __forceinline__ bool find_tile(uint64_t slot, const uint32_t *cu, uint32_t tokens_per_seq, uint32_t total, uint32_t n_seqs,
                                          const uint32_t *pos0, uint32_t max_pos_end, page_tile &t, uint32_t *cut) {
    auto begin = [&](uint32_t s) { return cu ? (uint64_t)min(cu[s], total) : (uint64_t)s * tokens_per_seq; };
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t lo = 0, hi = n_seqs;   // largest s in [lo, hi) whose slots begin at or before `slot`
    while (hi - lo > 1u) {
        const uint32_t step = (hi - lo + 31u) / 32u, s = lo + lane * step;
        const bool in = s < hi && begin(s) / 16u + 2ull * s <= slot;   // true up to some lane, false from there on
        const uint32_t last = max((uint32_t)__popc(__ballot_sync(0xffffffffu, in)), 1u) - 1u;
        lo += last * step;
        hi = min(hi, lo + step);
    }
    const uint64_t b = begin(lo), e = begin(lo + 1u);
    *cut = UINT32_MAX;
    if (e <= b || slot < b / 16u + 2ull * lo) return false;   // (the latter: tokens in front of cu[0], nobody's)
    const uint32_t p = pos0[lo];
    const uint64_t j = slot - (b / 16u + 2ull * lo);
    const uint64_t end_all = (uint64_t)p + (e - b);
    const uint64_t end = end_all < max_pos_end ? end_all : max_pos_end;
    if (j == 0 && end < end_all) *cut = p < max_pos_end ? max_pos_end : p;
    const uint64_t c0 = ((uint64_t)p / 16u + j) * 16u;
    if (c0 >= end || p >= end) return false;
    t.seq = lo;
    t.cell0 = (uint32_t)c0;
    t.first = c0 < p ? p - (uint32_t)c0 : 0u;
    t.count = (uint32_t)(end - c0 < 16u ? end - c0 : 16u) - t.first;
    t.token0 = (uint32_t)(b + (c0 + t.first - p));
    return true;
}

}  // namespace brc
