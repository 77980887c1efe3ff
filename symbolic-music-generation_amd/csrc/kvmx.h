// The quantised KV cache's number format and the device helpers that every kernel over it shares.
//
// A block is 32 consecutive elements of one head of one token: one scale byte e and 32 codes, value = code * 2^(e - 127).
// Codes are e4m3 numbers (BITS = 8, largest 448, a byte each) or e2m1 numbers (BITS = 4, largest 6, the even element in
// the low half of its byte). e is the smallest exponent at which the block's largest magnitude lies no further above the
// largest code than half a step (464 = 448 + 16 and 7 = 6 + 1, ties to even), so that no element is rounded by more than
// half a step of its own binade; it runs from 1 to the largest value at which every code is a finite float (246 / 252). (In 8
// bits that ends at 448 * 2^119 = 2.98e38, and bf16 at 3.39e38: the elements between become the former.)
// A block with an infinity or a NaN gets e = 255 and codes of zero and reads as NaN.
// gfx950 converts two codes per instruction in both directions, exactly (scaled conversions round to nearest even and
// saturate inside the range above), and every value is a bf16 number: the matrix instructions see the cache exactly.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
typedef __attribute__((ext_vector_type(2))) short s16x2;

template <int D, int BITS>
struct MX {
    static constexpr int RB = D * BITS / 8;    // bytes of a cached row's codes
    static constexpr int NB = D / 32;          // scale bytes of a cached row
};

// the two bf16 numbers of a dword (by value: clang's __builtin_bit_cast of a vector element reads element 0)
__device__ __forceinline__ bf16x2 mx_pair(unsigned w) { return __builtin_bit_cast(bf16x2, w); }

__device__ __forceinline__ float mx_scale(unsigned e) { return __uint_as_float(e << 23); }

// largest magnitude of 8 elements, as the 15 magnitude bits of a bf16 number (monotonic in the value; >= 0x7F80: Inf/NaN)
__device__ __forceinline__ unsigned mx_top8(bf16x8 x) {
    const u32x4 w = __builtin_bit_cast(u32x4, x);
    u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    return m[0] > m[1] ? m[0] : m[1];
}

// scale byte of a block whose largest magnitude has the bits `top`: the exponent field of top, one more when its
// fraction is above the edge (0.75 for e2m1: 7 = 1.75 * 4; 0.8125 for e4m3: 464 = 1.8125 * 256), less the largest
// code's exponent
template <int BITS>
__device__ __forceinline__ unsigned mx_exponent(unsigned top) {
    constexpr int EMAX = BITS == 4 ? 2 : 8, ROUND = BITS == 4 ? 127 - 96 : 127 - 104, MOST = BITS == 4 ? 252 : 246;
    const int e = (int)((top + ROUND) >> 7) - EMAX;
    return top >= 0x7F80u ? 255u : (unsigned)min(max(e, 1), MOST);
}

// codes of 8 elements of a block with scale byte e: one dword (BITS = 4) or two (BITS = 8)
template <int BITS>
__device__ __forceinline__ void mx_encode8(bf16x8 x, unsigned e, unsigned* out) {
    const float s = mx_scale(e == 255u ? 127u : e);
    const u32x4 w = __builtin_bit_cast(u32x4, x);
    if (BITS == 4) {
        unsigned c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, mx_pair(w[0]), s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, mx_pair(w[1]), s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, mx_pair(w[2]), s, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, mx_pair(w[3]), s, 3);
        out[0] = e == 255u ? 0u : c;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s16x2 c = {0, 0};
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, mx_pair(w[2 * h]), s, false);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, mx_pair(w[2 * h + 1]), s, true);
            // above 464 (only where e stands at its upper end) the conversion gives the NaN code 0x7F: 448 instead
            const unsigned v = __builtin_bit_cast(unsigned, c);
            const unsigned nan = ((v & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
            out[h] = e == 255u ? 0u : v - (nan >> 7);
        }
    }
}

// 8 elements from one dword (BITS = 4) or two (BITS = 8) of codes
template <int BITS>
__device__ __forceinline__ bf16x8 mx_decode8(const unsigned* c, float s) {
    u32x4 w;
    if (BITS == 4) {
        w[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[0], s, 0));
        w[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[0], s, 1));
        w[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[0], s, 2));
        w[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[0], s, 3));
    } else {
        w[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], s, false));
        w[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], s, true));
        w[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], s, false));
        w[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], s, true));
    }
    return __builtin_bit_cast(bf16x8, w);
}

// the 8 (BITS = 4) or 4 (BITS = 8) elements of one dword as fp32
template <int BITS>
__device__ __forceinline__ void mx_decode_f32(unsigned c, float s, float* out) {
    f32x2 t;
    if (BITS == 4) {
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0); out[0] = t[0]; out[1] = t[1];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1); out[2] = t[0]; out[3] = t[1];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2); out[4] = t[0]; out[5] = t[1];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3); out[6] = t[0]; out[7] = t[1];
    } else {
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, s, false); out[0] = t[0]; out[1] = t[1];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, s, true); out[2] = t[0]; out[3] = t[1];
    }
}

// exchanges inside a row of 16 lanes (no LDS traffic): lane i gets the value of lane ...
__device__ __forceinline__ int dpp_xor1(int v) { return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true); }
__device__ __forceinline__ int dpp_xor2(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true); }
__device__ __forceinline__ int dpp_xor7(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true); }   // 7 - i in 8
__device__ __forceinline__ int dpp_xor15(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true); }  // 15 - i
__device__ __forceinline__ float dppf_ror8(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true)); }
__device__ __forceinline__ float dppf_xor1(float v) { return __int_as_float(dpp_xor1(__float_as_int(v))); }
__device__ __forceinline__ float dppf_xor2(float v) { return __int_as_float(dpp_xor2(__float_as_int(v))); }
__device__ __forceinline__ float dppf_xor7(float v) { return __int_as_float(dpp_xor7(__float_as_int(v))); }
__device__ __forceinline__ float dppf_xor15(float v) { return __int_as_float(dpp_xor15(__float_as_int(v))); }

__device__ __forceinline__ float swz_xor4(float v) { return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 4 << 10 | 0x1F)); }

// sum / maximum over a row of 16 lanes, in every lane of it
__device__ __forceinline__ float row16_sum(float v) {
    v += dppf_xor1(v);
    v += dppf_xor2(v);
    v += dppf_xor7(v);
    return v + dppf_xor15(v);
}
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dppf_xor1(v));
    v = fmaxf(v, dppf_xor2(v));
    v = fmaxf(v, dppf_xor7(v));
    return fmaxf(v, dppf_xor15(v));
}
// over the wave
__device__ __forceinline__ float wave64_sum(float v) {
    v = row16_sum(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ float wave64_max(float v) {
    v = row16_max(v);
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
