// The decode step's own token, taken from the raw projection rows inside an attention kernel: per-head RMSNorm and
// rotation of one head row, shared by the attention over the bf16 cache (decode.hip) and over the quantised cache
// (attn_decode_mx.hip), so that both work on the same keys and queries bit for bit.
#pragma once
#include "common.h"

// The row of head `hh` of a projection output, normalised (g != null) and rotated: the arithmetic of
// decode_qkv_prep_kernel, lane for lane (D/16 lanes, two groups of 8 elements each); the bf16 results go to dst[D].
template <int D, bool IL>
__device__ __forceinline__ void prep_row(const bf16* __restrict__ src, const float* __restrict__ g,
                                         const float* __restrict__ cs_row, float eps, int sub, bf16* dst) {
    constexpr int LPR = D / 16;
    const int o1 = IL ? 16 * sub : 8 * sub;
    const int o2 = IL ? 16 * sub + 8 : D / 2 + 8 * sub;
    const bf16x8 r1 = *reinterpret_cast<const bf16x8*>(src + o1);
    const bf16x8 r2 = *reinterpret_cast<const bf16x8*>(src + o2);
    float a[16], o[16], c[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { a[e] = (float)r1[e]; a[8 + e] = (float)r2[e]; }
    const float* cp = cs_row + 16 * sub;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(cp + 2 * e);
        c[e] = v[0]; sn[e] = v[1]; c[e + 1] = v[2]; sn[e + 1] = v[3];
    }
    if (g != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss += a[e] * a[e];
        ss = group_sum<LPR>(ss);
        const float rs = rsqrtf(ss / (float)D + eps);
#pragma unroll
        for (int e = 0; e < 16; ++e) a[e] = g[e < 8 ? o1 + e : o2 + e - 8] * round_bf(a[e] * rs);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int pe = IL ? (e ^ 1) : (e ^ 8);
        const int ci = IL ? (e >> 1) : (e & 7);
        const bool second = IL ? (e & 1) : (e >= 8);
        o[e] = second ? (a[e] * c[ci] + a[pe] * sn[ci]) : (a[e] * c[ci] - a[pe] * sn[ci]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) { dst[o1 + e] = (bf16)o[e]; dst[o2 + e] = (bf16)o[8 + e]; }
}

// What the kernel needs to take the step's own token from the projection output instead of from prepared buffers
// (PREP instances): raw qkv rows, the norm gains, the rotary table.
struct DecodePrep {
    const bf16* qkv; long ld_in;
    const float* wq; const float* wk; const float* cs;
    const int* pos; float eps;
};
