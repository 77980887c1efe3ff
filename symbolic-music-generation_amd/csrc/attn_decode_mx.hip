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
// One workgroup per (key split, kv head with up to 8 query heads, stream); its waves walk units of keys. A load instruction
// is one contiguous kilobyte of codes (MXTiles). Streams of different lengths: 256 x 8 heads x 128, 1 to 4096 keys in 4 bits
// 92 to 97 us (6.1 TB/s; as many keys in equal streams 91 to 98).
//
// One query head per kv head (MXOne), all on the vector unit. Scores: codes to bf16 pairs, two products and their sum per
// instruction, the 2, 4 or 8 lanes of a row add up. V: codes to fp32, weighted into the lane's own sums (its elements, over
// its own keys). Keys meet after the loop.
//   256 streams x 8 heads x 128: 2048 keys in 8 bits 163 us (6.8 TB/s), 4096 in 4 bits 170 to 189 by where its buffers lie
//   (6.7 to 6.1), 2048 in 4 bits 91 to 98 (6.2 to 5.8).
//
// Several query heads (MXHeads), on the matrix cores: units of 32 keys go straight to LDS, as codes, the next one on its way
// while one is worked on (in registers 16 to 32 of them would hold it, and a CU the fewer waves); lane (r, g), r = lane & 15,
// g = lane >> 4, takes the g-th quarter of rows r and 16 + r from there, and its codes become bf16 operand fragments of 8
// elements (exactly).
//  * Scores: the reduction runs over the elements in the order the lanes hold them, a permutation that q shares. The heads
//    are the columns (columns i and 8 + i hold the same head): lane (r, g) ends up with column r, keys 4g .. 4g+3, which is
//    the operand layout of the second product, so the weights never cross lanes.
//  * The second product reduces over keys, so a lane needs V by element, not by key: the matrix cores turn the tile around
//    (V fragment times a 0/1 selection of 16 of its 32 elements - one product per output, exact), a matrix instruction per
//    16 x 16 elements of a pipe that is mostly idle here. (Through a bf16 image in LDS instead, read transposed: the same.)
//    (The block-scaled instruction over 128 elements turns straight from the codes: 60 instructions a unit fewer, 25 to 26.5 us
//    at 16 streams of up to 8192 keys. For the scores it is too coarse: its sums are good to 2^-12 of the largest product.)
//  * Weights enter as two bf16 numbers, their rounded value in columns 0..7 and what that leaves in columns 8..15 (16 bits
//    of weight at the price of 8); the two rows are added at the end.
//  * A value block written with an infinity or a NaN enters as zeros and its elements of the result are set to NaN at the
//    end (0 * NaN in the turning product would reach the other elements).
// Bound on a full chip: in 4 bits the vector unit (250 instructions a unit: 74 % busy, the matrix pipe 35 %; a wave waits
// for its turn to issue 44 % of its time, for data 27 %), in 8 bits HBM (6.8 TB/s at 128 x 8192 keys with 4 heads per kv head;
// vector unit 42 %). Fewer but slower instructions in its place gave nothing: a unit is one dependent chain (scores, weights,
// turn, rounding, product), which is also what few streams of unequal lengths wait for. 256 streams x 8 kv heads x 128, 2048
// keys in 4 bits: 102 us with 4 heads per kv head (5.6 TB/s); of 2 x 64: 58. 40 streams of 1 to 4000 keys, 8 kv heads of 4 x
// 128, in 8 bits: 37 to 39 us (loads to registers, one unit at a time: 105, 67 and 51).
//
// Both: the running maximum of a head is shared by the wave and moves only when a score exceeds it by more than 2^8 in the
// weight; then the sums are scaled. Sums, maxima and outputs are fp32, divided at the end: finite while the values' magnitude
// times the number of keys is below 2^119 (2^8 in the weights, 2^127 in a sum). Rows outside the split
// are never read: the loads go through buffer descriptors that end at the split's last key and give zeros behind it (codes
// and scale: the value 0), and the weights of the last unit of keys are masked.
#include "kvmx.h"
#include "decode_prep.h"
#include "lds_dma.h"

namespace {

constexpr float MX_LOG2E = 1.4426950408889634f;
constexpr float MX_LOW = -3.0e38f;      // below every finite score that matters; not -inf, so that differences stay numbers
constexpr float MX_SLACK = 8.0f;
constexpr int MX_HEADS = 8;            // query heads of a workgroup
constexpr int MX_MAX_SPLITS = 64;      // (a lane of one wave each in the joining kernel)
constexpr int MX_PLACES = 1024;        // workgroups on the chip at a time
constexpr int MX_ORDERED = 512;        // streams that a workgroup puts in order
constexpr int MX_ORDER_KEYS = 1024;    // capacity from which on that pays
constexpr int MX_MIN_SPLIT = 256;      // keys below which a split is not worth a workgroup

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

// keys of stream b (0: none, or a step that does not fit)
template <int PREP>
__device__ __forceinline__ int mx_length(const int* kv_len, int max_len, const MXPrep& pp, int b) {
    const int len = kv_len[b];
    if (!PREP) return min(len, max_len);
    const int pos = pp.pos[b];
    return pos < 0 || pos >= max_len || pos >= pp.npos || len != pos + 1 ? 0 : len;
}
// The n streams from `first` on in the order of their keys, the longest first (to 1/256 of the longest one's; equal ones as
// they are numbered): the stream of rank `rank` among them, found bit by bit as the largest length that more than `rank`
// streams reach. Every lane of a wave calls it and gets the same answer.
__device__ __forceinline__ int mx_by_length(const int* kv_len, int max_len, int first, int n, int rank, int lane) {
    constexpr int NL = MX_ORDERED / 64;
    int key[NL];
    float longest = 1.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        key[i] = kv_len[first + min(i * 64 + lane, n - 1)];        // (without a branch: all of them under way together)
        key[i] = max(min(key[i], max_len), 0);
        longest = fmaxf(longest, (float)key[i]);
    }
    const float unit = 255.9f / wave64_max(longest);
#pragma unroll
    for (int i = 0; i < NL; ++i) key[i] = i * 64 + lane < n ? (int)((float)key[i] * unit) : -1;
    int at = 0, above = 0;                // streams of key at or more: above rank; of more than that: `above`
#pragma unroll 1
    for (int bit = 128; bit; bit >>= 1) {
        int k = 0;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (i * 64 < n) k += __popcll(__ballot(key[i] >= at + bit));
        if (k > rank) at += bit;
        else above = k;
    }
    rank -= above;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const bool in = key[i] == at;
        const unsigned long long m = __ballot(in);
        const int k = __popcll(m);
        if (rank < k) {
            const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0));
            return first + i * 64 + __ffsll(__ballot(in && before == rank)) - 1;
        }
        rank -= k;
    }
    return first;                         // (not reached: rank < n)
}
// keys of a split of a stream of len: short streams use fewer of the splits
__device__ __forceinline__ int mx_split(int len, int nsplit) {
    return nsplit == 1 ? len : max(((len + nsplit - 1) / nsplit + 31) & ~31, MX_MIN_SPLIT);
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t mx_rsrc(const unsigned char* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, (int)bytes, 0x00020000);
}

struct MXRsrc {                          // the split's keys: codes and scales of K and V
    rsrc_t k, ks, v, vs;
};
struct MXKeys {
    const unsigned char *k, *ks, *v, *vs;
};
struct MXNew {                           // the step's own key, the last of the stream's last split
    const bf16 *k, *v;                   // its rows in LDS
    unsigned char *kc, *ks, *vc, *vs;    // their place in the cache
    bool write, here;                    // this workgroup writes them; this split ends with it
};
// 16, 4 or 2 (zero-extended) bytes per lane from byte `from` of a buffer to 16 or 4 bytes per lane from LDS address dst on, past
// the caches (read once: the non-temporal hint is worth 8 to 10 %); waited for by hand, see lds_dma.h
template <int BYTES>
__device__ __forceinline__ void mx_dma(const u32x4& rsrc, int from, unsigned dst) {
    if (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                     : : "s"(dst), "v"(from), "s"(rsrc) : "memory", "m0");
    else if (BYTES == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                     : : "s"(dst), "v"(from), "s"(rsrc) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_ushort %1, %2, 0 offen lds"
                     : : "s"(dst), "v"(from), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ f32x4 mx_mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// scale byte of block blk of a bf16 row
template <int BITS>
__device__ __forceinline__ unsigned mx_block_exponent(const bf16* row, int blk) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, mx_top8(*reinterpret_cast<const bf16x8*>(row + 32 * blk + 8 * i)));
    return mx_exponent<BITS>(top);
}

// How a wave reads codes: T tiles of KPT consecutive keys, each one contiguous kilobyte: 16 bytes per lane, ED elements of
// one key inside one block, LR lanes a row. (Loads in the matrix cores' own layout - 16 neighbouring lanes in 16 rows - take
// the address unit a clock per cache line for 16 bytes of it, 16 bytes a clock and CU: 4.9 TB/s at 256 x 2048 keys.)
template <int D, int BITS, int T>
struct MXTiles {
    static constexpr int RB = MX<D, BITS>::RB, NB = MX<D, BITS>::NB;
    static constexpr int LR = RB / 16, KPT = 64 / LR;
    static constexpr int ED = 128 / BITS;             // elements of a lane
    static constexpr int WF = BITS / 4;               // dwords of 8 elements

    __device__ __forceinline__ static int key(int lane) { return lane / LR; }        // of a tile
    __device__ __forceinline__ static int elem(int lane) { return lane % LR * ED; }
    __device__ __forceinline__ static int block(int lane) { return elem(lane) / 32; }

    template <int AUX>
    __device__ __forceinline__ static void load(rsrc_t codes, int base, int lane, unsigned (&c)[T][4]) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(codes, (base + t * KPT) * RB + lane * 16, 0, AUX);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[t][i] = x[i];
        }
    }
    // the codes of the lane's elements of a bf16 row; with `write` to the cache too (the row's codes and scale bytes).
    // Returns the scale byte of the lane's block.
    __device__ __forceinline__ static unsigned encode(unsigned (&x)[4], int lane, const bf16* row, bool write,
                                                      unsigned char* codes, unsigned char* scales) {
        const unsigned e = mx_block_exponent<BITS>(row, block(lane));
#pragma unroll
        for (int j = 0; j < ED / 8; ++j)
            mx_encode8<BITS>(*reinterpret_cast<const bf16x8*>(row + elem(lane) + 8 * j), e, x + j * WF);
        if (write) {
            *reinterpret_cast<u32x4*>(codes + lane % LR * 16) = u32x4{x[0], x[1], x[2], x[3]};
            scales[block(lane)] = (unsigned char)e;                 // (lanes of a block write the same byte)
        }
        return e;
    }
};

// A core walks units of KPU keys with the softmax state of its wave.

// One query head
template <int D, int BITS>
struct MXOne {
    static constexpr int T = 4;
    typedef MXTiles<D, BITS, T> R;
    static constexpr int KPT = R::KPT, KPU = T * KPT, LR = R::LR, ED = R::ED, WF = R::WF, NB = R::NB;
    static constexpr int LDS = 0;                     // bytes of LDS a wave works in
    static constexpr int WAVES = 4;                   // a SIMD has to hold
    struct Unit {                                     // codes and scale bytes of K and of V
        unsigned k[T][4], v[T][4], ke[T], ve[T];
    };
    bf16x2 q[ED / 2];
    float m, l, acc[ED], sl2;
    int lane;
    MXRsrc src;                           // the split's codes and scales

    __device__ __forceinline__ void place(int lane_, char*) { lane = lane_; }
    __device__ __forceinline__ int key() const { return R::key(lane); }
    __device__ __forceinline__ void load(const MXRsrc& s, int base, Unit& u) const {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int at = (base + t * KPT + key()) * NB + R::block(lane);
            u.ke[t] = __builtin_amdgcn_raw_buffer_load_b8(s.ks, at, 0, 0);
            u.ve[t] = __builtin_amdgcn_raw_buffer_load_b8(s.vs, at, 0, 0);
        }
        // (read once: the non-temporal hint is worth 8 to 10 %)
        R::template load<2>(s.k, base, lane, u.k);
        R::template load<2>(s.v, base, lane, u.v);
    }
    // the step's own key t_new of the unit: K (codes c, scale bytes e) or V from its bf16 row
    __device__ __forceinline__ void patch(unsigned (&c)[T][4], unsigned (&e)[T], int t_new, const bf16* row, bool write,
                                          unsigned char* codes, unsigned char* scales) const {
        if (key() != t_new % KPT) return;
        unsigned x[4];
        const unsigned b = R::encode(x, lane, row, write, codes, scales);
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[t][i] = t == t_new / KPT ? x[i] : c[t][i];
            e[t] = t == t_new / KPT ? b : e[t];
        }
    }
    __device__ __forceinline__ void start(const bf16* src, int nh, float scale_log2e) {
        sl2 = scale_log2e;
#pragma unroll
        for (int j = 0; j < ED / 8; ++j) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(src + R::elem(lane) + 8 * j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned w = x[i];
                q[4 * j + i] = mx_pair(w);
            }
        }
        m = MX_LOW;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < ED; ++e) acc[e] = 0.f;
    }
    // LAST: the unit with the split's last key, `left` keys from its first on
    template <bool LAST>
    __device__ __forceinline__ void unit(const Unit& u, int left) {
        float s[T], mx = MX_LOW;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float sc = mx_scale(u.ke[t]);
            float d[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < ED / 8; ++j) {
                const u32x4 x = __builtin_bit_cast(u32x4, mx_decode8<BITS>(u.k[t] + j * WF, sc));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned w = x[i];
                    d[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(mx_pair(w), q[4 * j + i], d[i & 1], false);
                }
            }
            float a = d[0] + d[1];
            a += dppf_xor1(a);
            if (LR >= 4) a += dppf_xor2(a);
            if (LR >= 8) a += dppf_xor7(a);
            s[t] = a * sl2;
            if (LAST) s[t] = t * KPT + key() < left ? s[t] : MX_LOW;
            mx = fmaxf(mx, s[t]);
        }
        if (__any(mx > m + MX_SLACK)) {
            const float top = fmaxf(wave64_max(mx), m);
            const float alpha = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= alpha;
#pragma unroll
            for (int e = 0; e < ED; ++e) acc[e] *= alpha;
        }
#pragma unroll
        for (int t = 0; t < T; ++t) {
            float w = __builtin_amdgcn_exp2f(s[t] - m);
            if (LAST) w = t * KPT + key() < left ? w : 0.f;
            l += w;
            const float sc = mx_scale(u.ve[t]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                constexpr int PW = 32 / BITS;
                float f[PW];
                mx_decode_f32<BITS>(u.v[t][x], sc, f);
#pragma unroll
                for (int e = 0; e < PW; ++e) acc[x * PW + e] = fmaf(w, f[e], acc[x * PW + e]);
            }
        }
    }
    __device__ __forceinline__ void begin(const MXKeys& keys, int, int n) {
        src = {mx_rsrc(keys.k, n * R::RB), mx_rsrc(keys.ks, n * NB), mx_rsrc(keys.v, n * R::RB), mx_rsrc(keys.vs, n * NB)};
    }
    template <int NW>
    __device__ __forceinline__ void walk(int base, int n, const MXNew& fresh) {
        Unit u;
#pragma unroll 1
        for (; base + KPU < n; base += NW * KPU) {   // units before the one with the split's last key
            load(src, base, u);
            unit<false>(u, 0);
        }
        if (base < n) {
            load(src, base, u);
            if (fresh.here) {
                patch(u.k, u.ke, n - 1 - base, fresh.k, fresh.write, fresh.kc, fresh.ks);
                patch(u.v, u.ve, n - 1 - base, fresh.v, fresh.write, fresh.vc, fresh.vs);
            }
            unit<true>(u, n - base);
        }
    }
    // The wave's maximum, denominator and sums to ml[2] and o[D]. Lanes that hold the same elements (64 / LR keys) add up,
    // halving the elements a lane is responsible for at every step: a swap of half waves or of neighbouring rows of 16
    // lanes brings two elements' halves together, then exchanges inside a row.
    __device__ __forceinline__ void finish(float* ml, float* o, int nh) {
        l = wave64_sum(l);
        int from = lane % LR * ED;
#pragma unroll
        for (int e = 0; e < ED / 2; ++e) {
            const u32x2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[e]), __float_as_uint(acc[e + ED / 2]), false, false);
            acc[e] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
        }
        from += (lane >> 5 & 1) * (ED / 2);
#pragma unroll
        for (int e = 0; e < ED / 4; ++e) {
            const u32x2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[e]), __float_as_uint(acc[e + ED / 4]), false, false);
            acc[e] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
        }
        from += (lane >> 4 & 1) * (ED / 4);
#pragma unroll
        for (int st = 0; st < (LR == 8 ? 1 : LR == 4 ? 2 : 3); ++st) {
            const int half = ED >> (3 + st);
            const bool up = lane & (8 >> st);
#pragma unroll
            for (int e = 0; e < half; ++e) {
                const float keep = up ? acc[e + half] : acc[e], give = up ? acc[e] : acc[e + half];
                acc[e] = keep + (st == 0 ? dppf_ror8(give) : st == 1 ? swz_xor4(give) : dppf_xor2(give));
            }
            from += up ? half : 0;
        }
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[from + e] = acc[e];
        // the denominator: every lane of a row of the cache added the same weight
        if (lane == 0) {
            ml[0] = m;
            ml[1] = l / LR;
        }
    }
};

// Up to MX_HEADS query heads
template <int D, int BITS>
struct MXHeads {
    static constexpr int RB = MX<D, BITS>::RB, NB = MX<D, BITS>::NB;
    static constexpr int KPU = 32;
    typedef MXTiles<D, BITS, 1> R;
    static constexpr int T = KPU / R::KPT;            // loads of a unit's codes of K (of V)
    static constexpr int W = RB / 16;                 // dwords of a quarter row
    static constexpr int NF = D / 32;                 // fragments of 8 elements
    static constexpr int WF = BITS / 4;               // dwords of a fragment
    // a unit in LDS: codes of K and of V, a dword of scale bytes per key of K and of V; two a wave, one of them ahead
    static constexpr int IMG = KPU * RB, SLOT = 2 * IMG + 2 * 4 * KPU, LOADS = 2 * T + 2;
    static constexpr int LDS = 2 * SLOT;              // bytes of LDS a wave works in
    static constexpr int WAVES = RB == 128 ? 2 : 3;   // a SIMD has to hold (what LDS leaves)
    bf16x8 qf[NF], pick[2];
    float m, l, sl2, low;                 // of column r; low: the column takes the weights' remainders
    f32x4 acc[NF][2];                     // rows = columns of the scores, column r of selection c
    unsigned long long bad;               // lanes that met a value block of scale 255
    char* img;
    int lane, r, g;
    u32x4 rk, rks, rv, rvs;               // the split's codes and scales
    unsigned lds;                         // address of the wave's slots

    __device__ __forceinline__ void place(int lane_, char* image) {
        lane = lane_;
        r = lane & 15;
        g = lane >> 4;
        img = image;
        lds = __builtin_amdgcn_readfirstlane(lds_addr(image));
    }
    __device__ __forceinline__ static int elem_of(int j, int g) { return g * (D / 4) + 8 * j; }
    __device__ __forceinline__ int elem(int j) const { return elem_of(j, g); }
    __device__ __forceinline__ int block() const { return g * NB / 4; }
    // 16-byte chunk c of a row of the image, spread so that 16 rows' chunks lie on different banks
    __device__ __forceinline__ static int at(int row, int c) {
        return row * RB + 16 * (c ^ (RB == 128 ? row >> 1 & 7 : RB == 64 ? row >> 2 & 3 : row >> 3 & 1));
    }

    // unit [base, base + KPU) of the split on its way to a slot: each load a contiguous kilobyte, its chunks in the order of
    // the image; rows behind the split's last key arrive as zeros
    __device__ __forceinline__ void request(int base, int slot) const {
        const unsigned dst = lds + slot * SLOT;
        const int row = R::key(lane), c = lane % R::LR;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int from = (base + t * R::KPT + row) * RB + (at(t * R::KPT + row, c) & (RB - 1));
            mx_dma<16>(rk, from, dst + t * 1024);
            mx_dma<16>(rv, from, dst + IMG + t * 1024);
        }
        if (lane < KPU) {
            mx_dma<NB>(rks, (base + lane) * NB, dst + 2 * IMG);
            mx_dma<NB>(rvs, (base + lane) * NB, dst + 2 * IMG + 4 * KPU);
        }
    }
    __device__ __forceinline__ void begin(const MXKeys& keys, int base, int n) {
        rk = dma_rsrc(keys.k, n * RB);
        rks = dma_rsrc(keys.ks, n * NB);
        rv = dma_rsrc(keys.v, n * RB);
        rvs = dma_rsrc(keys.vs, n * NB);
        if (base < n) request(base, 0);
    }
    template <int NW>
    __device__ __forceinline__ void walk(int base, int n, const MXNew& fresh) {
        int slot = 0;
#pragma unroll 1
        for (; base < n; base += NW * KPU, slot ^= 1) {
            if (base + NW * KPU < n) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what was read from the slot that is filled again
                request(base + NW * KPU, slot ^ 1);
                dma_wait<LOADS>();
            } else dma_wait<0>();
            const int left = n - base;
            char* here = img + slot * SLOT;
            if (left > KPU) unit<false>(here, 0);
            else {
                if (fresh.here) {
                    patch(here, 0, left - 1, fresh.k, fresh.write, fresh.kc, fresh.ks);
                    patch(here, 1, left - 1, fresh.v, fresh.write, fresh.vc, fresh.vs);
                }
                unit<true>(here, left);
            }
        }
    }
    // key t_new of a unit, K (value = 0) or V, from its bf16 row
    __device__ __forceinline__ void patch(char* unit, int value, int t_new, const bf16* row, bool write,
                                          unsigned char* codes, unsigned char* scales) const {
        if (lane >= R::LR) return;
        unsigned x[4];
        const unsigned e = R::encode(x, lane, row, write, codes, scales);
        lds_write_b128(unit + value * IMG, at(t_new, lane), u32x4{x[0], x[1], x[2], x[3]});
        unit[2 * IMG + (value * KPU + t_new) * 4 + R::block(lane)] = (char)e;
    }
    // the lane's quarter of key 16 t + r, and its block's scale byte
    __device__ __forceinline__ unsigned quarter(const char* unit, int value, int t, unsigned (&out)[W]) const {
        const char* image = unit + value * IMG;
        const int row = 16 * t + r;
        if (W == 2) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(image + at(row, g >> 1) + 8 * (g & 1));
            out[0] = x[0];
            out[1] = x[1];
        } else {
#pragma unroll
            for (int h = 0; h < W / 4; ++h) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(image + at(row, g * (W / 4) + h));
#pragma unroll
                for (int i = 0; i < 4; ++i) out[4 * h + i] = x[i];
            }
        }
        return *reinterpret_cast<const unsigned char*>(unit + 2 * IMG + (value * KPU + row) * 4 + block());
    }

    __device__ __forceinline__ void start(const bf16* q, int nh, float scale_log2e) {
        sl2 = scale_log2e;
        low = r >> 3 ? 1.f : 0.f;
        m = MX_LOW;
        l = 0.f;
        bad = 0;
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            qf[j] = bf16x8{};
            if ((r & 7) < nh) qf[j] = *reinterpret_cast<const bf16x8*>(q + (r & 7) * D + elem(j));
        }
        // selection c: column r of the turned tile is element r & 7 of the fragment of lanes g = 2c + (r >> 3)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) pick[c][e] = (bf16)(g == 2 * c + (r >> 3) && e == (r & 7) ? 1.f : 0.f);
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[j][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    template <bool LAST>
    __device__ __forceinline__ void unit(const char* slot, int left) {
        float s[8];
        unsigned c[2][W], e[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) e[t] = quarter(slot, 0, t, c[t]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NF; ++j) a = mx_mfma(mx_decode8<BITS>(c[t] + j * WF, mx_scale(e[t])), qf[j], a);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[4 * t + i] = a[i] * sl2;
                if (LAST) s[4 * t + i] = 16 * t + 4 * g + i < left ? s[4 * t + i] : MX_LOW;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        if (__any(mx > m + MX_SLACK)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32, 64)), m);
            const float alpha = __builtin_amdgcn_exp2f(m - mx);
            m = mx;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float row = __shfl(alpha, 4 * g + i, 64);     // of the column that row 4g + i of the sums belongs to
#pragma unroll
                for (int j = 0; j < NF; ++j) {
                    acc[j][0][i] *= row;
                    acc[j][1][i] *= row;
                }
            }
        }
        bf16x8 p;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float w = __builtin_amdgcn_exp2f(s[i] - m);
            if (LAST) w = 16 * (i >> 2) + 4 * g + (i & 3) < left ? w : 0.f;
            l += w;
            p[i] = (bf16)fmaf(-low, round_bf(w), w);
        }
        float vs[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            e[t] = quarter(slot, 1, t, c[t]);
            bad |= __ballot(e[t] == 255u);
            vs[t] = e[t] == 255u ? 0.f : mx_scale(e[t]);
        }
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            const bf16x8 v0 = mx_decode8<BITS>(c[0] + j * WF, vs[0]), v1 = mx_decode8<BITS>(c[1] + j * WF, vs[1]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                const f32x4 t0 = mx_mfma(v0, pick[b], zero), t1 = mx_mfma(v1, pick[b], zero);   // keys 4g + i, column r
                bf16x8 x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = (bf16)t0[i];
                    x[4 + i] = (bf16)t1[i];
                }
                acc[j][b] = mx_mfma(p, x, acc[j][b]);
            }
        }
    }
    __device__ __forceinline__ void finish(float* ml, float* o, int nh) {
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0 && r < nh) {
            ml[2 * r] = m;
            ml[2 * r + 1] = l;
        }
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int from = 2 * c + (r >> 3);                  // lanes g the column's element came from
                const float nan = (bad >> (16 * from)) & 0xFFFFu ? __uint_as_float(0x7FC00000u) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {                       // rows 8 + i hold the remainders
                    const float x = acc[j][c][i] + __shfl_xor(acc[j][c][i], 32, 64) + nan;
                    if (4 * g + i < nh) o[(4 * g + i) * D + elem_of(j, from) + (r & 7)] = x;
                }
            }
    }
};

// PREP = 0: q is ready in `q` and the cache holds kv_len[b] keys. PREP = 1 (split-half pairs) / 2 (adjacent pairs): q,
// the new key and the new value come from the raw projection rows; the new row is quantised, takes the place of key
// kv_len[b] - 1 in the lanes that own it, and is written to the cache by the first head group.
template <int D, int BITS, int PREP, template <int, int> class Core, int NW>
__global__ __launch_bounds__(64 * NW, (Core<D, BITS>::WAVES)) void attn_decode_mx_kernel(const bf16* __restrict__ q, long ld_q, MXView kv,
                                                                 const int* __restrict__ kv_len, int H, int KVH,
                                                                 int nsplit, int first, float scale,
                                                                 float* __restrict__ part_ml,
                                                                 float* __restrict__ part_o, bf16* __restrict__ out,
                                                                 long ld_o, MXPrep pp) {
    typedef Core<D, BITS> C;
    constexpr int RB = MX<D, BITS>::RB, NB = MX<D, BITS>::NB, KPU = C::KPU;
    extern __shared__ __attribute__((aligned(16))) float smem[];

    const int group = H / KVH, chunks = (group + MX_HEADS - 1) / MX_HEADS;
    const int split = blockIdx.x, kvh = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
    int b = blockIdx.z;
    if (b >= first) b = __builtin_amdgcn_readfirstlane(mx_by_length(kv_len, kv.max_len, first, gridDim.z - first, b - first,
                                                                    threadIdx.x & 63));
    const int h0 = kvh * group + chunk * MX_HEADS, nh = min(MX_HEADS, group - chunk * MX_HEADS), hc = min(MX_HEADS, group);
    // LDS: q heads, new key and new value (PREP) and what the cores work in, which then give way to the waves' sums
    bf16* sm_q = reinterpret_cast<bf16*>(smem + NW * C::LDS / 4);    // [hc + 2][D]
    float* sm_o = smem;                              // [NW][hc][D]
    float* sm_ml = smem + NW * hc * D;               // [NW][hc][2]
    const int tid = threadIdx.x, wave = tid >> 6;
    C core;
    core.place(tid & 63, reinterpret_cast<char*>(smem) + wave * C::LDS);

    const int len = mx_length<PREP>(kv_len, kv.max_len, pp, b), pos = len - 1;       // (pos: of the new token, PREP)
    if (len <= 0) {                       // a stream without keys: zeros
        if (nsplit == 1)
#pragma unroll 1
            for (int i = tid; i < nh * D; i += 64 * NW) out[(long)b * ld_o + (long)h0 * D + i] = (bf16)0.f;
        return;
    }
    const int per = mx_split(len, nsplit);
    const int k_beg = (int)min((long)split * per, (long)len), n = min(len - k_beg, per);     // keys of this split
    if (n <= 0) return;

    const long slice = ((long)b * KVH + kvh) * kv.max_len;
    const long first_row = slice + k_beg;
    const MXKeys keys{kv.k + first_row * RB, kv.ks + first_row * NB, kv.v + first_row * RB, kv.vs + first_row * NB};
    const int base = wave * KPU;
    core.begin(keys, base, n);

    if (PREP) {
        constexpr int L16 = D / 16;
        const int s16 = tid % L16;
        const bf16* row = pp.qkv + (long)b * pp.ld_in;
        const float* csr = pp.cs + (long)pos * D;
#pragma unroll 1
        for (int which = tid / L16; which < nh + 2; which += 64 * NW / L16) {
            if (which < nh + 1) {
                const bool isq = which < nh;
                prep_row<D, PREP == 2>(row + (long)(isq ? h0 + which : H + kvh) * D, isq ? pp.wq : pp.wk, csr, pp.eps, s16,
                                       sm_q + (isq ? which : hc) * D);
            } else {
                const bf16* src = row + (long)(H + KVH + kvh) * D + 16 * s16;
                bf16* dst = sm_q + (hc + 1) * D + 16 * s16;
                *reinterpret_cast<bf16x8*>(dst) = *reinterpret_cast<const bf16x8*>(src);
                *reinterpret_cast<bf16x8*>(dst + 8) = *reinterpret_cast<const bf16x8*>(src + 8);
            }
        }
        __syncthreads();
    }
    core.start(PREP ? sm_q : q + (long)b * ld_q + (long)h0 * D, nh, scale * MX_LOG2E);
    // q has arrived before the walk: the compiler would wait for it inside, and with it for the units that are under way
    if (C::LDS) __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt(0)

    MXNew fresh{};
    if (PREP) {
        const long at = slice + pos;
        fresh = {sm_q + hc * D, sm_q + (hc + 1) * D, const_cast<unsigned char*>(kv.k) + at * RB,
                 const_cast<unsigned char*>(kv.ks) + at * NB, const_cast<unsigned char*>(kv.v) + at * RB,
                 const_cast<unsigned char*>(kv.vs) + at * NB, chunk == 0, k_beg + n == len};
    }
    core.template walk<NW>(base, n, fresh);

    if (PREP || C::LDS) __syncthreads();  // the sums overwrite both
    core.finish(sm_ml + wave * hc * 2, sm_o + wave * hc * D, nh);
    __syncthreads();
#pragma unroll 1
    for (int x = tid; x < nh * D; x += 64 * NW) {
        const int i = x / D, d = x % D;
        float M = MX_LOW;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_ml[(w * hc + i) * 2]);
        float L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm_ml[(w * hc + i) * 2] - M);
            L += sm_ml[(w * hc + i) * 2 + 1] * f;
            o += sm_o[(w * hc + i) * D + d] * f;
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

// Joins the splits of a stream's heads: one workgroup per (head, stream), D/4 lanes per split. Latency is all that counts
// here, so everything is requested at once, the splits that a short stream does not use among it (their memory belongs to
// the workspace; what it holds is not looked at).
template <int D, int PREP>
__global__ __launch_bounds__(256) void attn_decode_mx_merge_kernel(const float* __restrict__ part_ml,
                                                                   const float* __restrict__ part_o,
                                                                   const int* __restrict__ kv_len, int max_len,
                                                                   MXPrep pp, int nsplit, int H, bf16* __restrict__ out,
                                                                   long ld_o) {
    constexpr int L4 = D / 4, ROWS = 256 / L4, PER = MX_MAX_SPLITS / ROWS;
    __shared__ __attribute__((aligned(16))) f32x4 sums[ROWS][L4];
    const int h = blockIdx.x, b = blockIdx.y, t = threadIdx.x, row = t / L4, c = t % L4, lane = t & 63;
    const long p0 = ((long)b * H + h) * nsplit;
    f32x4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (i * ROWS + row < nsplit) x[i] = *reinterpret_cast<const f32x4*>(part_o + (p0 + i * ROWS + row) * D + 4 * c);
    float m = MX_LOW, l = 0.f;            // of split `lane`
    if (lane < nsplit) {
        m = part_ml[(p0 + lane) * 2];
        l = part_ml[(p0 + lane) * 2 + 1];
    }
    const int len = mx_length<PREP>(kv_len, max_len, pp, b);
    bf16* dst = out + (long)b * ld_o + (long)h * D;
    if (len <= 0) {
        if (t < D) dst[t] = (bf16)0.f;
        return;
    }
    const int per = mx_split(len, nsplit), used = (len + per - 1) / per;
    if (lane >= used) {
        m = MX_LOW;
        l = 0.f;
    }
    const float f = __builtin_amdgcn_exp2f(m - wave64_max(m)), w = f / wave64_sum(l * f);
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int s = i * ROWS + row;
        const float ws = __shfl(w, s, 64);
        if (s < used) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] += x[i][e] * ws;
        }
    }
    sums[row][c] = a;
    __syncthreads();
    if (t < D) {
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) o += sums[i][t >> 2][t & 3];
        dst[t] = (bf16)o;
    }
}

template <int D, int BITS, int PREP, template <int, int> class Core, int NW>
int launch(const char* what, const void* q, long ld_q, MXView kv, const int* kv_len, void* out, long ld_o, float* ws, int B, int H,
            int KVH, int nsplit, float scale, MXPrep pp, hipStream_t stream) {
    float* part_ml = ws;
    float* part_o = ws ? ws + (long)B * H * nsplit * 2 : nullptr;
    const int group = H / KVH, chunks = (group + MX_HEADS - 1) / MX_HEADS, hc = group < MX_HEADS ? group : MX_HEADS;
    const int loop = NW * Core<D, BITS>::LDS + (PREP ? (hc + 2) * D * 2 : 0), sums = NW * hc * (D + 2) * 4;
    const int lds = loop > sums ? loop : sums;
    // More workgroups than the chip holds: behind the streams that start at once (their order does not matter, and it would
    // show as latency) the longest go first, or a long one that starts last runs on alone. 256 x 8 heads x 128, lengths up
    // to 4096: 4 bits 103 us as numbered, 96 ordered, 8 bits 189 and 176; with 4 heads per kv head in 4 bits 115 and 105;
    // lengths up to 2048 in 8 bits 99 and 100; equal lengths of 4096 321 and 325. Short caches end before it pays (96 x 24
    // kv heads of 3 keys: one head each 7.0 and 10.1, four 16.6 and 19.9).
    // MX_PLACES is a round figure for all instances: by registers and LDS they hold from 512 workgroups (several heads in 8
    // bits, D = 128) to 1280 (one head), so where it is too high some streams that start late keep their place. With more than
    // MX_ORDERED streams behind the first ones nothing is ordered.
    const long groups = (long)KVH * chunks * nsplit, at_once = MX_PLACES / groups;
    const int first = kv.max_len >= MX_ORDER_KEYS && B > at_once && B - at_once <= MX_ORDERED ? (int)at_once : B;
    if (lds > 65536) {                    // more than the default 64 KiB of dynamic LDS: asked for once per kernel and device
        static bool asked[64] = {};
        int dev = 0;
        (void)hipGetDevice(&dev);
        dev = dev < 0 || dev > 63 ? 63 : dev;
        if (!asked[dev]) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_decode_mx_kernel<D, BITS, PREP, Core, NW>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
            if (e != hipSuccess) {
                mgen_set_error("%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
                return MGEN_ELAUNCH;
            }
            asked[dev] = true;
        }
    }
    hipLaunchKernelGGL((attn_decode_mx_kernel<D, BITS, PREP, Core, NW>), dim3(nsplit, KVH * chunks, B), dim3(64 * NW), lds,
                       stream, (const bf16*)q, ld_q, kv, kv_len, H, KVH, nsplit, first, scale, part_ml, part_o, (bf16*)out, ld_o,
                       pp);
    if (nsplit > 1)
        hipLaunchKernelGGL((attn_decode_mx_merge_kernel<D, PREP>), dim3(H, B), dim3(256), 0, stream, part_ml, part_o, kv_len,
                           kv.max_len, pp, nsplit, H, (bf16*)out, ld_o);
    return mgen_check_launch(what);
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
    MGEN_REQUIRE((((uintptr_t)ks | (uintptr_t)vs) & (D / 32 - 1)) == 0, "%s: scales must be aligned to a row (D / 32)", what);
    const MXView kv{(const unsigned char*)kc, (const unsigned char*)ks, (const unsigned char*)vc,
                    (const unsigned char*)vs, max_len};
    // Several heads: 8 waves where a CU gets one workgroup or none, 4 beyond. 8 and 4 waves, us: 32 x 8 kv heads of 4 x 128,
    // 2000 keys in 4 bits 17.5 and 20.2, in 8 bits 27.6 and 27.8; 16 streams of 700 10.3 and 10.9; 1 of 100003 keys in 64 splits
    // 25.4 and 25.1; 32 x 8 kv heads of 8, 4096 keys in 8 bits 49.9 and 47.9. Beyond: 40 streams of 1000 in 8 bits 24.1 and 21.1,
    // 200 x 8 kv heads of 8, up to 2000 keys 97 and 77, 96 x 24 of 4, 3 keys 26.4 and 16.6.
#define LAUNCH(DD, BB)                                                                                                 \
    do {                                                                                                               \
        if (H == KVH)                                                                                                  \
            return launch<DD, BB, PREP, MXOne, 4>(what, q, ld_q, kv, kv_len, out, ld_o, ws, B, H, KVH, nsplit, scale, pp, stream); \
        if ((long)B * KVH * ((H / KVH + MX_HEADS - 1) / MX_HEADS) * nsplit <= 256)                                     \
            return launch<DD, BB, PREP, MXHeads, 8>(what, q, ld_q, kv, kv_len, out, ld_o, ws, B, H, KVH, nsplit, scale, pp, stream); \
        return launch<DD, BB, PREP, MXHeads, 4>(what, q, ld_q, kv, kv_len, out, ld_o, ws, B, H, KVH, nsplit, scale, pp, stream);  \
    } while (0)
    if (D == 128) { if (bits == 4) LAUNCH(128, 4); else LAUNCH(128, 8); }
    if (bits == 4) LAUNCH(64, 4);
    LAUNCH(64, 8);
#undef LAUNCH
}

}  // namespace

// Key splits for a call whose longest stream has `longest` keys; never fewer for a longer one.
// Few workgroups: a power of two of splits (the chip's places divide evenly) that brings them to 512, to 1280 while each has
// 1024 keys, but no more than leave a workgroup's waves two rounds of keys (a limit that is no power of two: 5 for one
// stream x 8 heads x 128 of 1300 keys); where the second launch is worth its 3 us, from 8 rounds on. Measured, us: 1 stream
// x 8 heads x 128 in 8 bits, 4096 keys 33 in one split and 8.3 in 16, 512 keys 5.7 and 7.6. 16 streams of 8 kv heads x 128
// of up to 6000 keys, 4 heads each, 4 / 8 bits: 20.7 / 29.9 in 4 splits, 20.3 / 34.9 in 6, 21.3 / 34.6 in 8; up to 32768
// keys 79 / 119, 62 / 122, 59 / 116. 24 streams of up to 6000 keys, one head each, 26.5 / 38.7 in 2 splits, 19.8 / 33.7 in
// 4.
// From 256 workgroups on: one. One and two, at 1500 keys: 1536 workgroups of heads of 64 in 4 bits 28 and 38 us, in 8 bits 50
// and 52, of 128 96 and 99; at 6000 keys 347 and 355. One and four at 256 workgroups, 32 streams x 8 kv heads x 128: all of
// 16384 keys, 4 / 8 bits, 95 / 154 and 91 / 167, with 4 heads per kv head 93 / 167 and 100 / 172; all of 1500 14 / 20 and 15 / 22,
// 16 / 23 and 20 / 30. The longest stream is all that the rule goes by, and where the others are shorter splits would pay at
// such lengths: 1 to 16384 keys 94 / 147 and 59 / 110, with 4 heads 84 / 120 and 73 / 109; 1 to 4000 26 / 39 and 20 / 29, with 4
// heads 27 / 34 and 26 / 38; 100 streams of 1 to 16384 160 / 332 and 130 / 236.
extern "C" int mgen_attn_decode_mx_splits(int B, int H, int KVH, int D, int longest) {
    if (B <= 0 || KVH <= 0 || H < KVH || longest <= 0) return 1;
    const bool one = H == KVH;
    const long groups = (long)B * KVH * ((H / KVH + MX_HEADS - 1) / MX_HEADS);
    const int round = one && D == 64 ? 256 : 128;     // keys of a round of a workgroup's waves, taken at 8 bits
    const int rounds = (longest - 1) / round + 1;
    if (rounds < 8 || groups >= 256) return 1;
    int n = MX_MAX_SPLITS;
    while (n > 1 && (n * groups > 1280 || (n * groups > 512 && longest < 1024 * n))) n /= 2;
    return n < rounds / 2 ? n : rounds / 2;
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
