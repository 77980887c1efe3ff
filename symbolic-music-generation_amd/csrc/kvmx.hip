// KV cache in blocks of 32 elements with a shared power-of-two scale (e4m3 or e2m1 codes, kvmx.h): quantising rows as
// they are written, and reading them back. Both are bound by HBM: one pass, every byte moved once.
//
// Stands beside mgen_kv_append (the bf16 cache; DynamicLayer.update, transformers cache_utils.py:127-146).
#include "kvmx.h"

namespace {

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, division by invariant integers): q = (mulhi(n, m) + n) >> s
struct FastDiv {
    unsigned d, m, s;
};
inline FastDiv fast_div(unsigned d) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    return {d, (unsigned)((((1ull << s) - d) << 32) / d + 1), s};
}
__device__ __forceinline__ unsigned fdiv(unsigned n, FastDiv f) { return (__umulhi(n, f.m) + n) >> f.s; }

// The rows of one call, numbered tile by tile: up to a workgroup's worth of consecutive tokens of one head, then the next
// head, then the next tokens. A tile's cache rows are one contiguous run; neighbouring workgroups take the heads of the
// same tokens, so that the chip reads (writes) whole token rows at a time. (All tokens of a head first, as the cache lies,
// put every workgroup on the same 256-byte column of rows whose pitch is a multiple of the memory channels' period.)
struct MXRows {
    FastDiv tiles, heads;
    unsigned nrows, tokens;
    int shift;                  // tile = 1 << shift tokens
    int max_len;
    const int* pos0;
};

struct Row {
    bool there;
    long tok, head, slot;       // row of the token-major side, head in it, row of the cache
};

__device__ __forceinline__ Row locate(const MXRows& a, unsigned row) {
    const unsigned x = row >> a.shift, t = fdiv(x, a.heads), h = x - t * a.heads.d, b = fdiv(t, a.tiles);
    const unsigned i = ((t - b * a.tiles.d) << a.shift) + (row & ((1u << a.shift) - 1));
    if (i >= a.tokens) return {false, 0, 0, 0};
    const int p = (int)((unsigned)a.pos0[b] + i);
    return {p >= 0 && p < a.max_len, (long)b * a.tokens + i, (long)h, ((long)b * a.heads.d + h) * a.max_len + p};
}

// D/8 lanes per row of K and of V, 8 elements per lane; a block is 4 lanes, so its largest magnitude takes two exchanges
// inside a row of lanes. 32 x 2048 tokens of 8 heads x 128 in 4 bits: 67 us, 5.1 TB/s read and written (a copy: 4.6); with
// each head's tokens numbered first 85 us.
template <int D, int BITS>
__global__ __launch_bounds__(256) void kv_append_mx_kernel(const bf16* __restrict__ k_src, const bf16* __restrict__ v_src,
                                                           long ld_k, long ld_v, unsigned char* __restrict__ kc,
                                                           unsigned char* __restrict__ ks,
                                                           unsigned char* __restrict__ vc,
                                                           unsigned char* __restrict__ vs, MXRows a) {
    constexpr int LPR = D / 8, RPB = 256 / LPR, RB = MX<D, BITS>::RB, NB = MX<D, BITS>::NB;
    const int sub = threadIdx.x % LPR;
    for (unsigned row = blockIdx.x * RPB + threadIdx.x / LPR; row < a.nrows; row += gridDim.x * RPB) {
        const Row w = locate(a, row);
        if (!w.there) continue;                 // (all lanes of a row alike)
        const bf16x8 x[2] = {*reinterpret_cast<const bf16x8*>(k_src + w.tok * ld_k + w.head * D + sub * 8),
                             *reinterpret_cast<const bf16x8*>(v_src + w.tok * ld_v + w.head * D + sub * 8)};
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            unsigned top = mx_top8(x[which]);
            top = max(top, (unsigned)dpp_xor1((int)top));
            top = max(top, (unsigned)dpp_xor2((int)top));
            const unsigned e = mx_exponent<BITS>(top);
            unsigned c[2];
            mx_encode8<BITS>(x[which], e, c);
            unsigned char* codes = (which ? vc : kc) + w.slot * RB + sub * BITS;
            if (BITS == 4) *reinterpret_cast<unsigned*>(codes) = c[0];
            else *reinterpret_cast<u32x2*>(codes) = u32x2{c[0], c[1]};
            if ((sub & 3) == 0) (which ? vs : ks)[w.slot * NB + (sub >> 2)] = (unsigned char)e;
        }
    }
}

// The same numbering and lanes. The values go out past the caches (st_stream): the same tokens in 49 us, 6.9 TB/s; ordinary
// stores, each head's tokens first: 77 us.
template <int D, int BITS>
__global__ __launch_bounds__(256) void kv_read_mx_kernel(const unsigned char* __restrict__ kc,
                                                         const unsigned char* __restrict__ ks,
                                                         const unsigned char* __restrict__ vc,
                                                         const unsigned char* __restrict__ vs, bf16* __restrict__ k_dst,
                                                         bf16* __restrict__ v_dst, long ld_k, long ld_v, MXRows a) {
    constexpr int LPR = D / 8, RPB = 256 / LPR, RB = MX<D, BITS>::RB, NB = MX<D, BITS>::NB;
    const int sub = threadIdx.x % LPR;
    for (unsigned row = blockIdx.x * RPB + threadIdx.x / LPR; row < a.nrows; row += gridDim.x * RPB) {
        const Row w = locate(a, row);
        if (!w.there) continue;
        unsigned c[2][2], e[2];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const unsigned char* codes = (which ? vc : kc) + w.slot * RB + sub * BITS;
            if (BITS == 4) c[which][0] = *reinterpret_cast<const unsigned*>(codes);
            else {
                const u32x2 v = *reinterpret_cast<const u32x2*>(codes);
                c[which][0] = v[0];
                c[which][1] = v[1];
            }
            e[which] = (which ? vs : ks)[w.slot * NB + (sub >> 2)];
        }
#pragma unroll
        for (int which = 0; which < 2; ++which)
            st_stream(reinterpret_cast<bf16x8*>((which ? v_dst : k_dst) + w.tok * (which ? ld_v : ld_k) + w.head * D + sub * 8),
                      mx_decode8<BITS>(c[which], mx_scale(e[which])));
    }
}

// workgroups of 256 threads for the rows of a call (more rows than 2^20 of them hold: a workgroup takes several)
template <int D>
unsigned blocks_for(unsigned rows) {
    const unsigned n = (rows + 2048 / D - 1) / (2048 / D);
    return n < 1u << 20 ? n : 1u << 20;
}

// what the two calls check alike; fills the row numbering
int rows_of(const char* what, const void* k, const void* v, const void* kc, const void* ks, const void* vc,
            const void* vs, const int* pos0, long ld_k, long ld_v, int B, int n, int KVH, int D, int max_len, int bits,
            MXRows* a) {
    MGEN_REQUIRE(k && v && kc && ks && vc && vs && pos0, "%s: null pointer", what);
    MGEN_REQUIRE(B > 0 && n > 0 && KVH > 0 && max_len > 0, "%s: bad sizes (B=%d n=%d KVH=%d max_len=%d)", what, B, n,
                 KVH, max_len);
    MGEN_REQUIRE(D == 64 || D == 128, "%s: D=%d (64 or 128)", what, D);
    MGEN_REQUIRE(bits == 4 || bits == 8, "%s: bits=%d (4 or 8)", what, bits);
    MGEN_REQUIRE(ld_k % 8 == 0 && ld_v % 8 == 0, "%s: strides must be multiples of 8", what);
    MGEN_REQUIRE(ld_k >= (long)KVH * D && ld_v >= (long)KVH * D, "%s: rows overlap (stride below KVH * D)", what);
    MGEN_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)kc | (uintptr_t)vc) & 15) == 0,
                 "%s: rows and codes must be 16-byte aligned", what);
    MGEN_REQUIRE((((uintptr_t)ks | (uintptr_t)vs) & (D / 32 - 1)) == 0, "%s: scales must be aligned to a row (D / 32)", what);
    int shift = 0;              // a tile: at most the rows of a workgroup, no more than the tokens need
    while ((1 << shift) < 2048 / D && (1 << shift) < n) ++shift;
    const long tiles = ((long)n + (1 << shift) - 1) >> shift, per_stream = (tiles << shift) * KVH;      // (below 2^63)
    MGEN_REQUIRE(per_stream < (1l << 31) && B * per_stream < (1l << 31), "%s: too many rows (B=%d n=%d KVH=%d)", what, B, n, KVH);
    const long rows = B * per_stream;
    *a = {fast_div((unsigned)tiles), fast_div((unsigned)KVH), (unsigned)rows, (unsigned)n, shift, max_len, pos0};
    return MGEN_OK;
}

}  // namespace

#define MX_DISPATCH(LAUNCH)                                                             \
    do {                                                                                \
        if (D == 128) { if (bits == 4) LAUNCH(128, 4); else LAUNCH(128, 8); }           \
        else { if (bits == 4) LAUNCH(64, 4); else LAUNCH(64, 8); }                      \
    } while (0)

// k_src/v_src [B*n_new tokens][ld] bf16 (heads at h*D) into slots pos0[b] .. pos0[b] + n_new - 1 of stream b; a slot
// outside [0, max_len) is not written
extern "C" int mgen_kv_append_mx(const void* k_src, const void* v_src, long ld_k, long ld_v, void* k_codes,
                                 void* k_scales, void* v_codes, void* v_scales, const int* pos0, int B, int n_new,
                                 int KVH, int D, int max_len, int bits, hipStream_t stream) {
    MXRows a;
    if (int e = rows_of("mgen_kv_append_mx", k_src, v_src, k_codes, k_scales, v_codes, v_scales, pos0, ld_k, ld_v, B,
                        n_new, KVH, D, max_len, bits, &a))
        return e;
#define LAUNCH(DD, BB)                                                                                               \
    hipLaunchKernelGGL((kv_append_mx_kernel<DD, BB>), dim3(blocks_for<DD>(a.nrows)), dim3(256), 0,                    \
                       stream, (const bf16*)k_src, (const bf16*)v_src, ld_k, ld_v, (unsigned char*)k_codes,          \
                       (unsigned char*)k_scales, (unsigned char*)v_codes, (unsigned char*)v_scales, a)
    MX_DISPATCH(LAUNCH);
#undef LAUNCH
    return mgen_check_launch("mgen_kv_append_mx");
}

// the inverse: slots pos0[b] .. pos0[b] + n - 1 of stream b into k_dst/v_dst [B*n][ld] bf16; a row whose slot is outside
// [0, max_len) is left as it was
extern "C" int mgen_kv_read_mx(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                               const int* pos0, void* k_dst, void* v_dst, long ld_k, long ld_v, int B, int n, int KVH,
                               int D, int max_len, int bits, hipStream_t stream) {
    MXRows a;
    if (int e = rows_of("mgen_kv_read_mx", k_dst, v_dst, k_codes, k_scales, v_codes, v_scales, pos0, ld_k, ld_v, B, n,
                        KVH, D, max_len, bits, &a))
        return e;
#define LAUNCH(DD, BB)                                                                                               \
    hipLaunchKernelGGL((kv_read_mx_kernel<DD, BB>), dim3(blocks_for<DD>(a.nrows)), dim3(256), 0,                    \
                       stream, (const unsigned char*)k_codes, (const unsigned char*)k_scales,                        \
                       (const unsigned char*)v_codes, (const unsigned char*)v_scales, (bf16*)k_dst, (bf16*)v_dst,    \
                       ld_k, ld_v, a)
    MX_DISPATCH(LAUNCH);
#undef LAUNCH
    return mgen_check_launch("mgen_kv_read_mx");
}
