// Single-token attention over the quantised KV cache (kvmx.h), and the decode step's form of it that takes the new token
// from the raw projection rows.
//
// Reference: the attention call with q_len = 1 (transformers models/qwen3/modeling_qwen3.py:252-279) after
// DynamicLayer.update (cache_utils.py:127-146); mgen_attn_decode / mgen_attn_decode_prep are the same over a bf16 cache.
//
//   s_j = scale * sum_d q_d K_jd,   o = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),   m = a running maximum
//
// Bound: HBM. A key and its value are 2 (D/2 + D/32) bytes in 4 bits, read once for all query heads of their kv head.
//
// One workgroup per (key split, kv head with up to 4 query heads, stream); a wave walks tiles of 16 keys. Lane (r, g),
// r = lane & 15, g = lane >> 4, takes the g-th quarter of key r's row: a tile is one contiguous run of memory and the
// quarter lies in one block, so a lane needs one scale byte per row.
//  * Scores on the matrix cores: the codes become bf16 fragments (exactly) as they come from memory; the reduction
//    index of fragment j runs over elements 8j .. 8j+7 of every quarter, a permutation that q shares. Query head i sits
//    in rows i, 4 + i, 8 + i, 12 + i of the other operand, so that every lane finds the scores of ITS key r for all heads
//    in its own accumulator: no exchange between lanes anywhere in the loop.
//  * Values on the vector unit: a lane's quarter of V_r as fp32, weighted into D/4 accumulators per head. Each lane keeps
//    the sum over its own keys; the 16 lanes of a row meet once, after the loop.
//  * The running maximum is one number per wave and head and moves only when a score exceeds it by more than 2^8 in the
//    weight (sums stay far inside fp32); then the sums are scaled. Weights, sums and outputs are fp32.
//  * Rows outside the split are never read: the loads go through buffer descriptors that end at the split's last key and
//    give zeros behind it (codes and scale: the value 0), and their weights are set to 0.
#include "kvmx.h"
#include "decode_prep.h"

namespace {

constexpr float MX_LOG2E = 1.4426950408889634f;
constexpr float MX_LOW = -3.0e38f;      // below every finite score that matters; not -inf, so that differences stay numbers
constexpr float MX_SLACK = 8.0f;

struct MXView {
    const unsigned char *k, *ks, *v, *vs;
    int max_len;
};

struct MXPrep {                          // the step's own token (PREP instances)
    const bf16* qkv;
    long ld_in;
    const float *wq, *wk, *cs;
    const int* pos;
    int npos;
    float eps;
};

typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t mx_rsrc(const unsigned char* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, (int)bytes, 0x00020000);
}

// a lane's quarter of a row: W dwords
template <int W>
__device__ __forceinline__ void mx_load(rsrc_t r, int off, unsigned* out) {
    if (W == 2) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
        out[0] = v[0]; out[1] = v[1];
    } else {
#pragma unroll
        for (int h = 0; h < W / 4; ++h) {
            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * h, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[4 * h + i] = v[i];
        }
    }
}

// PREP = 0: q is ready in `q` and the cache holds kv_len[b] keys. PREP = 1 (split-half pairs) / 2 (adjacent pairs): q,
// the new key and the new value come from the raw projection rows; the new row is quantised, takes the place of key
// kv_len[b] - 1 in the lanes that own it, and is written to the cache by the first head group.
// GC: query heads of the workgroup; U: tiles a wave has in flight; NW: waves
template <int D, int BITS, int GC, int PREP, int U, int NW>
__global__ __launch_bounds__(64 * NW) void attn_decode_mx_kernel(const bf16* __restrict__ q, long ld_q, MXView kv,
                                                                 const int* __restrict__ kv_len, int H, int KVH,
                                                                 int nsplit, float scale, float* __restrict__ part_ml,
                                                                 float* __restrict__ part_o, bf16* __restrict__ out,
                                                                 long ld_o, MXPrep pp) {
    constexpr int RB = MX<D, BITS>::RB, NB = MX<D, BITS>::NB;
    constexpr int W = RB / 16;            // dwords of a quarter row
    constexpr int NF = D / 32;            // bf16 fragments of a quarter row
    constexpr int ND = D / 4;             // elements of a quarter row
    __shared__ float sm_ml[NW * GC * 2];
    __shared__ __attribute__((aligned(16))) float sm_o[NW * GC * D];
    __shared__ __attribute__((aligned(16))) bf16 sm_new[PREP ? (GC + 2) * D : 8];   // q heads, new key, new value

    const int group = H / KVH, chunks = (group + GC - 1) / GC;
    const int split = blockIdx.x, kvh = blockIdx.y / chunks, chunk = blockIdx.y % chunks, b = blockIdx.z;
    const int h0 = kvh * group + chunk * GC, nh = min(GC, group - chunk * GC);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;

    int len = min(kv_len[b], kv.max_len);
    const int pos = PREP ? pp.pos[b] : 0;
    if (PREP && (pos < 0 || pos >= kv.max_len || pos >= pp.npos || kv_len[b] != pos + 1)) len = 0;
    if (len <= 0) {                       // a stream without keys: zeros
        for (int i = tid; i < nh * D; i += 64 * NW) {
            const int h = h0 + i / D;
            if (nsplit == 1) out[(long)b * ld_o + (long)h * D + i % D] = (bf16)0.f;
            else {
                const long pi = ((long)b * H + h) * nsplit + split;
                part_o[pi * D + i % D] = 0.f;
                if (i % D == 0) { part_ml[pi * 2] = 0.f; part_ml[pi * 2 + 1] = 1.f; }
            }
        }
        return;
    }
    const int per = ((len + nsplit - 1) / nsplit + 15) & ~15;
    const int k_beg = (int)min((long)split * per, (long)len), n = min(len - k_beg, per);     // keys of this split
    const int k_new = PREP ? len - 1 - k_beg : -1;                  // the new key, counted from k_beg

    if (PREP) {
        constexpr int L16 = D / 16;
        if (tid < (GC + 2) * L16) {
            const int which = tid / L16, s16 = tid % L16;
            const bf16* row = pp.qkv + (long)b * pp.ld_in;
            const float* csr = pp.cs + (long)pos * D;
            if (which < GC) {
                if (which < nh) prep_row<D, PREP == 2>(row + (long)(h0 + which) * D, pp.wq, csr, pp.eps, s16, sm_new + which * D);
            } else if (which == GC)
                prep_row<D, PREP == 2>(row + (long)(H + kvh) * D, pp.wk, csr, pp.eps, s16, sm_new + GC * D);
            else {
                const bf16* src = row + (long)(H + KVH + kvh) * D + 16 * s16;
                bf16* dst = sm_new + (GC + 1) * D + 16 * s16;
                *reinterpret_cast<bf16x8*>(dst) = *reinterpret_cast<const bf16x8*>(src);
                *reinterpret_cast<bf16x8*>(dst + 8) = *reinterpret_cast<const bf16x8*>(src + 8);
            }
        }
        __syncthreads();
    }

    // q: rows i, 4 + i, 8 + i, 12 + i of the operand hold head h0 + i (zeros from nh on)
    bf16x8 qf[NF];
    {
        const int i = r & 3;
        const bf16* src = PREP ? sm_new + i * D : q + (long)b * ld_q + (long)(h0 + i) * D;
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            qf[j] = bf16x8{};
            if (i < nh) qf[j] = *reinterpret_cast<const bf16x8*>(src + g * ND + 8 * j);
        }
    }
    const long slice = ((long)b * KVH + kvh) * kv.max_len;
    const unsigned nk = (unsigned)max(n, 0);
    const rsrc_t rk = mx_rsrc(kv.k + (slice + k_beg) * RB, nk * RB), rv = mx_rsrc(kv.v + (slice + k_beg) * RB, nk * RB);
    const rsrc_t rks = mx_rsrc(kv.ks + (slice + k_beg) * NB, nk * NB), rvs = mx_rsrc(kv.vs + (slice + k_beg) * NB, nk * NB);
    const int blk = g * NB / 4;           // block of this lane's quarter
    const float sl2 = scale * MX_LOG2E;

    float m[GC], l[GC], acc[GC][ND];
#pragma unroll
    for (int i = 0; i < GC; ++i) {
        m[i] = MX_LOW;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < ND; ++e) acc[i][e] = 0.f;
    }

    for (int base = wave * 16 * U; base < n; base += NW * 16 * U) {
        unsigned kk[U][W], vv[U][W], ke[U], ve[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = base + 16 * u + r;
            ke[u] = __builtin_amdgcn_raw_buffer_load_b8(rks, key * NB + blk, 0, 0);
            mx_load<W>(rk, key * RB + g * (RB / 4), kk[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = base + 16 * u + r;
            ve[u] = __builtin_amdgcn_raw_buffer_load_b8(rvs, key * NB + blk, 0, 0);
            mx_load<W>(rv, key * RB + g * (RB / 4), vv[u]);
        }
        if (PREP && k_new >= base && k_new < base + 16 * U) {       // (the same for all lanes of the wave)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (base + 16 * u + r != k_new) continue;
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    const bf16* row = sm_new + (GC + which) * D;
                    unsigned top = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        top = max(top, mx_top8(*reinterpret_cast<const bf16x8*>(row + 32 * blk + 8 * j)));
                    const unsigned e = mx_exponent<BITS>(top);
                    unsigned* c = which ? vv[u] : kk[u];
#pragma unroll
                    for (int j = 0; j < NF; ++j)
                        mx_encode8<BITS>(*reinterpret_cast<const bf16x8*>(row + g * ND + 8 * j), e, c + j * (BITS / 4));
                    (which ? ve : ke)[u] = e;
                    if (chunk == 0) {
                        unsigned char* codes = const_cast<unsigned char*>(which ? kv.v : kv.k) + (slice + pos) * RB + g * (RB / 4);
#pragma unroll
                        for (int j = 0; j < W; j += 2) *reinterpret_cast<u32x2*>(codes + 4 * j) = u32x2{c[j], c[j + 1]};
                        // (quarters that share a block write the same byte)
                        const_cast<unsigned char*>(which ? kv.vs : kv.ks)[(slice + pos) * NB + blk] = (unsigned char)e;
                    }
                }
            }
        }
        float s[U][GC], mx[GC];
#pragma unroll
        for (int i = 0; i < GC; ++i) mx[i] = MX_LOW;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float sc = mx_scale(ke[u]);
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NF; ++j)
                a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[j], mx_decode8<BITS>(kk[u] + j * (BITS / 4), sc), a, 0, 0, 0);
            const bool in = base + 16 * u + r < n;
#pragma unroll
            for (int i = 0; i < GC; ++i) {
                s[u][i] = in ? a[i] * sl2 : MX_LOW;
                mx[i] = fmaxf(mx[i], s[u][i]);
            }
        }
        bool grow = false;
#pragma unroll
        for (int i = 0; i < GC; ++i) grow |= mx[i] > m[i] + MX_SLACK;
        if (__any(grow)) {
#pragma unroll
            for (int i = 0; i < GC; ++i) {
                const float top = fmaxf(m[i], row16_max(mx[i]));
                const float alpha = __builtin_amdgcn_exp2f(m[i] - top);
                m[i] = top;
                l[i] *= alpha;
#pragma unroll
                for (int e = 0; e < ND; ++e) acc[i][e] *= alpha;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = base + 16 * u + r < n;
            const float sc = mx_scale(ve[u]);
#pragma unroll
            for (int i = 0; i < GC; ++i) {
                s[u][i] = in ? __builtin_amdgcn_exp2f(s[u][i] - m[i]) : 0.f;
                l[i] += s[u][i];
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                constexpr int PW = 32 / BITS;
                float f[PW];
                mx_decode_f32<BITS>(vv[u][w], sc, f);
#pragma unroll
                for (int i = 0; i < GC; ++i)
#pragma unroll
                    for (int e = 0; e < PW; ++e) acc[i][w * PW + e] = fmaf(s[u][i], f[e], acc[i][w * PW + e]);
            }
        }
    }

    // The 16 lanes of a row: sums over their keys, halving the elements a lane is responsible for at every step (lane r
    // ends up with elements r * ND/16 ... of quarter g). A step pairs lanes whose lower bits are mirrored; bits already
    // used stay equal.
#pragma unroll
    for (int i = 0; i < GC; ++i) {
        const float ls = row16_sum(l[i]);
        float t[ND];
#pragma unroll
        for (int e = 0; e < ND; ++e) t[e] = acc[i][e];
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const int half = ND >> (st + 1);
            const bool up = r & (8 >> st);
#pragma unroll
            for (int e = 0; e < half; ++e) {
                const float keep = up ? t[e + half] : t[e], give = up ? t[e] : t[e + half];
                t[e] = keep + (st == 0 ? dppf_xor15(give) : st == 1 ? dppf_xor7(give) : st == 2 ? dppf_xor3(give) : dppf_xor1(give));
            }
        }
        float* o = sm_o + (wave * GC + i) * D + g * ND + r * (ND / 16);
#pragma unroll
        for (int e = 0; e < ND / 16; ++e) o[e] = t[e];
        if (lane == 0) {
            sm_ml[(wave * GC + i) * 2] = m[i];
            sm_ml[(wave * GC + i) * 2 + 1] = ls;
        }
    }
    __syncthreads();
    for (int x = tid; x < nh * D; x += 64 * NW) {
        const int i = x / D, d = x % D;
        float M = MX_LOW;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_ml[(w * GC + i) * 2]);
        float L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm_ml[(w * GC + i) * 2] - M);
            L += sm_ml[(w * GC + i) * 2 + 1] * f;
            o += sm_o[(w * GC + i) * D + d] * f;
        }
        if (nsplit == 1) out[(long)b * ld_o + (long)(h0 + i) * D + d] = (bf16)(o / L);
        else {
            const long pi = ((long)b * H + h0 + i) * nsplit + split;
            part_o[pi * D + d] = o;
            if (d == 0) {
                part_ml[pi * 2] = M;
                part_ml[pi * 2 + 1] = L;
            }
        }
    }
}

template <int D>
__global__ void attn_decode_mx_merge_kernel(const float* __restrict__ part_ml, const float* __restrict__ part_o,
                                            int nsplit, int H, bf16* __restrict__ out, long ld_o) {
    const int h = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
    const long p0 = ((long)b * H + h) * nsplit;
    float M = MX_LOW;
    for (int s = 0; s < nsplit; ++s) M = fmaxf(M, part_ml[(p0 + s) * 2]);
    float L = 0.f, o = 0.f;
    for (int s = 0; s < nsplit; ++s) {
        const float f = __builtin_amdgcn_exp2f(part_ml[(p0 + s) * 2] - M);
        L += part_ml[(p0 + s) * 2 + 1] * f;
        o += part_o[(p0 + s) * D + t] * f;
    }
    out[(long)b * ld_o + (long)h * D + t] = (bf16)(o / L);
}

constexpr int MX_MAX_SPLITS = 64;

int heads_per_group(int H, int KVH) {
    const int group = H / KVH;
    return group == 1 ? 1 : group == 2 ? 2 : 4;
}

template <int D, int BITS, int GC, int PREP>
void launch(const void* q, long ld_q, MXView kv, const int* kv_len, void* out, long ld_o, float* ws, int B, int H,
            int KVH, int nsplit, float scale, MXPrep pp, hipStream_t stream) {
    constexpr int NW = 4, U = D * BITS / 8 == 128 ? 2 : 4;
    float* part_ml = ws;
    float* part_o = ws ? ws + (long)B * H * nsplit * 2 : nullptr;
    const int chunks = (H / KVH + GC - 1) / GC;
    hipLaunchKernelGGL((attn_decode_mx_kernel<D, BITS, GC, PREP, U, NW>), dim3(nsplit, KVH * chunks, B), dim3(64 * NW), 0,
                       stream, (const bf16*)q, ld_q, kv, kv_len, H, KVH, nsplit, scale, part_ml, part_o, (bf16*)out,
                       ld_o, pp);
    if (nsplit > 1)
        hipLaunchKernelGGL((attn_decode_mx_merge_kernel<D>), dim3(H, B), dim3(D), 0, stream, part_ml, part_o, nsplit, H,
                           (bf16*)out, ld_o);
}

template <int PREP>
int attend(const char* what, const void* q, long ld_q, const void* kc, const void* ks, const void* vc, const void* vs,
           const int* kv_len, void* out, long ld_o, float* ws, int B, int H, int KVH, int D, int max_len, int bits,
           int nsplit, float scale, MXPrep pp, hipStream_t stream) {
    MGEN_REQUIRE(kc && ks && vc && vs && kv_len && out, "%s: null pointer", what);
    MGEN_REQUIRE(B > 0 && B <= 65535 && H > 0 && KVH > 0 && H % KVH == 0 && max_len > 0,
                 "%s: bad sizes (B=%d H=%d KVH=%d max_len=%d)", what, B, H, KVH, max_len);
    MGEN_REQUIRE(D == 64 || D == 128, "%s: D=%d (64 or 128)", what, D);
    MGEN_REQUIRE(bits == 4 || bits == 8, "%s: bits=%d (4 or 8)", what, bits);
    MGEN_REQUIRE(H <= 65535, "%s: H=%d", what, H);
    MGEN_REQUIRE((long)max_len * D * bits / 8 < (1l << 31), "%s: max_len=%d is too long", what, max_len);
    MGEN_REQUIRE(nsplit >= 1 && nsplit <= MX_MAX_SPLITS, "%s: nsplit=%d (1 to %d)", what, nsplit, MX_MAX_SPLITS);
    MGEN_REQUIRE(nsplit == 1 || ws != nullptr, "%s: nsplit > 1 needs a workspace", what);
    MGEN_REQUIRE(ld_o >= (long)H * D, "%s: output rows overlap (ld_o below H * D)", what);
    MGEN_REQUIRE((((uintptr_t)kc | (uintptr_t)vc) & 15) == 0, "%s: codes must be 16-byte aligned", what);
    const MXView kv{(const unsigned char*)kc, (const unsigned char*)ks, (const unsigned char*)vc,
                    (const unsigned char*)vs, max_len};
#define LAUNCH(DD, BB)                                                                                                \
    do {                                                                                                              \
        switch (heads_per_group(H, KVH)) {                                                                            \
            case 1: launch<DD, BB, 1, PREP>(q, ld_q, kv, kv_len, out, ld_o, ws, B, H, KVH, nsplit, scale, pp, stream); break;  \
            case 2: launch<DD, BB, 2, PREP>(q, ld_q, kv, kv_len, out, ld_o, ws, B, H, KVH, nsplit, scale, pp, stream); break;  \
            default: launch<DD, BB, 4, PREP>(q, ld_q, kv, kv_len, out, ld_o, ws, B, H, KVH, nsplit, scale, pp, stream);        \
        }                                                                                                             \
    } while (0)
    if (D == 128) { if (bits == 4) LAUNCH(128, 4); else LAUNCH(128, 8); }
    else { if (bits == 4) LAUNCH(64, 4); else LAUNCH(64, 8); }
#undef LAUNCH
    return mgen_check_launch(what);
}

}  // namespace

// Key splits for a call whose longest stream has `longest` keys
extern "C" int mgen_attn_decode_mx_splits(int B, int H, int KVH, int D, int longest) {
    if (B <= 0 || KVH <= 0 || H < KVH || longest <= 0) return 1;
    const int GC = heads_per_group(H, KVH), chunks = (H / KVH + GC - 1) / GC;
    const long groups = (long)B * KVH * chunks;
    const long want = (1024 + groups - 1) / groups, most = (longest + 255) / 256;
    const long n = groups >= 1024 ? 1 : want < most ? want : most;
    return (int)(n < 1 ? 1 : n > MX_MAX_SPLITS ? MX_MAX_SPLITS : n);
}

// q [B][ld_q] (heads at h*D), out [B][ld_o] bf16; kv_len[b] = cached keys of stream b (0: the output row is zeros; values
// beyond max_len count as max_len). workspace: mgen_attn_decode_workspace(B, H, D, nsplit) floats for nsplit > 1
extern "C" int mgen_attn_decode_mx(const void* q, long ld_q, const void* k_codes, const void* k_scales,
                                   const void* v_codes, const void* v_scales, const int* kv_len, void* out, long ld_o,
                                   float* workspace, int B, int H, int KVH, int D, int max_len, int bits, int nsplit,
                                   float scale, hipStream_t stream) {
    MGEN_REQUIRE(q != nullptr, "mgen_attn_decode_mx: null pointer");
    MGEN_REQUIRE(ld_q % 8 == 0 && ((uintptr_t)q & 15) == 0, "mgen_attn_decode_mx: q must be 16-byte aligned, ld_q a multiple of 8");
    return attend<0>("mgen_attn_decode_mx", q, ld_q, k_codes, k_scales, v_codes, v_scales, kv_len, out, ld_o, workspace,
                     B, H, KVH, D, max_len, bits, nsplit, scale, MXPrep{}, stream);
}

// The decode step's attention straight from the projection rows (the bf16 cache's mgen_attn_decode_prep): qkv [B][ld_in]
// bf16 holds one new token per stream (H query heads, KVH key heads, KVH value heads). q and the new key get the per-head
// RMSNorm (wq/wk, both null: none) and the rotation by row pos[b] of cos_sin [npos][D/2][2]; the new key and value are
// quantised, written to cache slot pos[b] and take part in the softmax as they will be read later: the same bits as
// mgen_decode_qkv_prep's rows through mgen_kv_append_mx and mgen_attn_decode_mx. kv_len[b] = pos[b] + 1; a stream for
// which that does not hold, or whose pos[b] is outside [0, min(max_len, npos)), gets an output row of zeros and its cache
// is left as it was.
extern "C" int mgen_attn_decode_prep_mx(const void* qkv, long ld_in, const float* wq, const float* wk,
                                        const float* cos_sin, int npos, const int* pos, float eps, int interleaved,
                                        void* k_codes, void* k_scales, void* v_codes, void* v_scales, const int* kv_len,
                                        void* out, long ld_o, float* workspace, int B, int H, int KVH, int D,
                                        int max_len, int bits, int nsplit, float scale, hipStream_t stream) {
    MGEN_REQUIRE(qkv && cos_sin && pos, "mgen_attn_decode_prep_mx: null pointer");
    MGEN_REQUIRE((wq == nullptr) == (wk == nullptr), "mgen_attn_decode_prep_mx: wq and wk must both be given or both null");
    MGEN_REQUIRE(npos > 0, "mgen_attn_decode_prep_mx: npos=%d", npos);
    MGEN_REQUIRE(ld_in % 8 == 0 && ((uintptr_t)qkv & 15) == 0 && ((uintptr_t)cos_sin & 15) == 0,
                 "mgen_attn_decode_prep_mx: qkv and cos_sin must be 16-byte aligned, ld_in a multiple of 8");
    MGEN_REQUIRE(ld_in >= (long)(H + 2 * (long)KVH) * D, "mgen_attn_decode_prep_mx: ld_in below (H + 2 KVH) * D");
    const MXPrep pp{(const bf16*)qkv, ld_in, wq, wk, cos_sin, pos, npos, eps};
    if (interleaved)
        return attend<2>("mgen_attn_decode_prep_mx", nullptr, 0, k_codes, k_scales, v_codes, v_scales, kv_len, out, ld_o,
                         workspace, B, H, KVH, D, max_len, bits, nsplit, scale, pp, stream);
    return attend<1>("mgen_attn_decode_prep_mx", nullptr, 0, k_codes, k_scales, v_codes, v_scales, kv_len, out, ld_o,
                     workspace, B, H, KVH, D, max_len, bits, nsplit, scale, pp, stream);
}
