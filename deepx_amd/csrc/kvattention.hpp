// kvattention.hpp — attention of a ragged batch of rows over a paged cache in 8 bits.
//
// For one key head and one sequence the rows of all query heads that share it are one matrix Q [R, D], row r = i * G + g for
// query row i and head g of the G that share the key head.  With codes K', V' and page scales k_s, v_s, in base 2:
//     s_j = (Q K'^T)_j k_s(j) scale log2(e),     t_j = s_j + log2 v_s(j),     m = max t_j,     p_j = 2^(t_j - m),
//     O   = sum p_j V'_j,     l = sum p_j / v_s(j),     out = O / l,     lse = ln 2 (m + log2 l).
// Taking the value scale into the exponent keeps p in (0, 1] whatever the scales are, so that it can be rounded to f16 (held 2^15 times
// as large, or 2^7 times with 128-row tiles of 16-bit rows: normal down to 2^-29 or 2^-21 of the largest): 2^-11 of a term where bf16
// would lose 2^-8, on the same matrix instruction.  Codes are whole numbers below 2^8 or e4m3 values, exact in bf16 and in f16, and
// enter the products exactly; scales are applied to scores in fp32.  Q is exact too: bf16 rows multiply bf16 keys, f16 rows f16 keys;
// f32 rows are split into three bf16 parts (24 bits).
//
// A probability is held in two f16 parts, 22 bits, each one more product, but for 16-bit rows in the kernel for many rows.  There the
// second part costs a quarter of the time (four prompts of 3.3k-4.1k tokens, 32 / 8 heads of 128: 652 and 831 us), and bf16 results are
// 1.67e-3 from the exact value with one part, 1.66e-3 with two, which is their own rounding (f16: 2.8e-4 and 2.1e-4).  Under few rows it
// hides behind the codes' loads, 64 rows over 1k-16k tokens 213 us with one and 212 with two, f16 results 2.5e-4 and 2.1e-4 from the exact
// value; where the codes stay in the caches it costs 2 - 6 % (4 x 8 rows over 3k-6k tokens, 24 / 4 heads of 128: 24.3 and 25.2 us).
//
// Everything is computed transposed, S^T = K' Q^T and O^T = V'^T P^T, so that the tokens of a score tile are rows of the
// accumulator and a probability is already in the lane that feeds it to the second product: no exchange between lanes.
// Which token a row of the first product is, is free; it is chosen so that a lane holds 16 consecutive tokens — of one page,
// with one scale — and the matching piece of V' is 16 consecutive codes of one dimension in the cache's [dim][token] order.
//
// A page scale that is no finite number, or (where a mask cuts the tile) a NaN code among the values, must not reach rows
// that do not see the token, and 0 * NaN is NaN: such values are taken as zeros and the token's score becomes NaN for the
// rows that see it.  A key scale like that needs it as well: an infinite one makes scores of minus infinity, which weigh nothing.
#pragma once
#include <algorithm>
#include "kvcache.hpp"

namespace dxh {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct AttArgs {
    KvArgs kv;
    const char *q;
    char *out;
    int64_t q_row, q_head, o_row, o_head;
    float *lse, *part_o, *part_ml;  // partials: [slice][packed row][q head][dim] and [slice][packed row][q head][2]
    float scale;                    // scale * log2(e)
    int q_heads, group, causal, window, splits, min_tiles, row_tiles, tile_rows;
    int nt;  // few rows and pages of 64 tokens: the codes are read past the last-level cache
};

constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.4426950408889634f;
constexpr float kNone = -__builtin_inff();
constexpr float kLift = 15.f;        // probabilities are held 2^15 times as large: at most 2^15 in f16, whose largest number is 65504
// With 128-row tiles and one-part probabilities the reference of a row follows its maximum only when that has grown by more than
// kSlack (in powers of two): the output is then rescaled in few tiles, and a probability, held 2^(15 - kSlack) times as large, is
// still at most 2^15.
constexpr float kSlack = 8.f;
// A row's sum of (2^15 times) p / v_scale, kept 2^-9 times as large, is finite for 2^30 tokens of the smallest scale, 2^-92 (what is
// below is multiplied into the probabilities), and no less than 2^-123 for one token of the largest that written fp32 values get, 2^121.
// Of a caller's own scales up to 2^128 the reciprocal and the sum can be subnormal (with 128-row tiles down to 2^-130, 19 bits): the hardware's
// reciprocal and logarithm take them for zero and are given multiples of them (value_scale, lse_of).
constexpr float kTinyScale = 0x1p-92f, kSumUnit = 0x1p-9f, kSumLog = 9.f;

// ---- products ---------------------------------------------------------------------------------------------------------
// Kind: the 16-bit type of keys and queries; QP, PP: parts that hold a query value, a probability of the kernel for many rows
template <typename T> struct RowType { using Kind = __bf16; static constexpr int QP = 1, PP = 1; };
template <> struct RowType<f16_t> { using Kind = _Float16; static constexpr int QP = 1, PP = 1; };
template <> struct RowType<float> { using Kind = __bf16; static constexpr int QP = 3, PP = 2; };

template <typename Kind> __device__ __forceinline__ f32x4_t mma16(const u32x4 &a, const u32x4 &b, const f32x4_t &c) {
    if constexpr (std::is_same_v<Kind, __bf16>) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename Kind> __device__ __forceinline__ f32x16 mma32(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
    if constexpr (std::is_same_v<Kind, __bf16>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename Kind> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same_v<Kind, __bf16>) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}
// eight values -> N vectors of Kind whose sum they are, as far as N parts reach
template <typename Kind, int N> __device__ __forceinline__ void split_parts(float (&x)[8], u32x4 (&p)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = pack2<Kind>(x[2 * e], x[2 * e + 1]);
            p[k][e] = w;
            if (k + 1 < N) {
                if constexpr (std::is_same_v<Kind, __bf16>) {
                    x[2 * e] -= bits_to_float(w << 16);
                    x[2 * e + 1] -= bits_to_float(w & 0xffff0000u);
                } else {
                    const f16x2_t h = __builtin_bit_cast(f16x2_t, w);
                    x[2 * e] -= (float)h[0];
                    x[2 * e + 1] -= (float)h[1];
                }
            }
        }
}
// four codes (a dword) as Kind, exactly
template <typename Code, typename Kind> __device__ __forceinline__ void codes4(uint32_t c, uint32_t &lo, uint32_t &hi) {
    if constexpr (std::is_same_v<Code, CodeE4M3> && std::is_same_v<Kind, __bf16>) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true));
    } else if constexpr (std::is_same_v<Code, CodeE4M3>) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, true));
    } else if constexpr (std::is_same_v<Kind, _Float16>) {
        // 0x6400 + u is 1024 + u in f16, u = code + 128 < 256: exact, and so is the difference
        const uint32_t u = c ^ 0x80808080u;
        const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
    } else {
        float x[4];
        Code::decode(c, x);
        lo = pack2<Kind>(x[0], x[1]);
        hi = pack2<Kind>(x[2], x[3]);
    }
}
template <typename Code, typename Kind> __device__ __forceinline__ u32x4 codes8(uint32_t a, uint32_t b) {
    uint32_t w0, w1, w2, w3;
    codes4<Code, Kind>(a, w0, w1);
    codes4<Code, Kind>(b, w2, w3);
    return u32x4{w0, w1, w2, w3};
}
// bytes of `w` that are an e4m3 NaN, as 0x80 in each
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// 16 codes without their NaNs; bit j of the result: code j was one
__device__ __forceinline__ uint32_t drop_nans(u32x4 &v) {
    uint32_t found = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t b = nan_bytes(v[w]);
        v[w] &= ~((b >> 7) * 0xffu);
#pragma unroll
        for (int e = 0; e < 4; ++e) found |= ((b >> (8 * e + 7)) & 1u) << (4 * w + e);
    }
    return found;
}

// the larger of a lane's value and that of lane ^ 32
__device__ __forceinline__ float other_half_max(float x) {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(float_to_bits(x), float_to_bits(x), false, false));
    return __builtin_fmaxf(bits_to_float(r[0]), bits_to_float(r[1]));
}
__device__ __forceinline__ bool finite(float x) { return x - x == 0.f; }
// A value scale: its logarithm, its reciprocal, and the factor of the probabilities that go with it: 1 but for zero, tiny and
// negative scales.  One that is not finite counts as 1 here and makes the scores of its tokens NaN.
struct ValueScale { float log, inv, factor; };
__device__ __forceinline__ ValueScale value_scale(float vs) {
    if (!finite(vs)) vs = 1.f;
    const float mag = __builtin_fmaxf(__builtin_fabsf(vs), kTinyScale);
    return {__builtin_amdgcn_logf(mag), __builtin_amdgcn_rcpf(mag * 0x1p-32f) * 0x1p-32f, __builtin_fabsf(vs) >= kTinyScale ? __builtin_copysignf(1.f, vs) : vs * 0x1p92f};
}
// Where a scale is so much smaller than the largest that the row has seen so far that 2^(t - m) could be 0 while the token's share of l is not (a page of
// zeros beside one of huge values), the exponent keeps within kReach of that largest one's and the rest of the scale becomes a
// factor.  What it is a factor of is then below 2^-85 of the largest values.
constexpr float kReach = 85.f;
__device__ __forceinline__ bool out_of_reach(const ValueScale &v, float largest) { return v.log < largest - kReach; }
__device__ __forceinline__ void reach(ValueScale &v, float largest) {
    if (!out_of_reach(v, largest)) return;
    v.factor *= __builtin_amdgcn_exp2f(v.log - (largest - kReach));
    v.inv = __builtin_amdgcn_exp2f(kReach - largest);
    v.log = largest - kReach;
}
// 2^x, x <= 0, for a row whose reference moves.  Its sum holds 1 / scale of every token and may count although 2^x is less than any
// float (tokens of scale 2^-92 beside some of 2^60 that weigh the same): it is multiplied by 2^(x / 2) twice.
struct Shift {
    float half;
    __device__ __forceinline__ float all() const { return half * half; }
    __device__ __forceinline__ float sum(float l) const { return l * half * half; }
};
__device__ __forceinline__ Shift shift_of(float x) { return {__builtin_amdgcn_exp2f(0.5f * x)}; }

// ---- which tokens -------------------------------------------------------------------------------------------------------
// The tokens [lo, hi) that row i of a sequence sees; nothing for a row that is none or has no place in the cache.
struct Range { int lo, hi; };
__device__ __forceinline__ Range row_range(const AttArgs &a, const KvSeq &s, int i) {
    if (i >= s.n || s.begin + i < 0) return {0, 0};
    const int p = s.begin + i;
    const int hi = a.causal && p + 1 < s.length ? p + 1 : s.length;
    const int lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    return {lo < hi ? lo : hi, hi};
}
__device__ __forceinline__ bool sees(const Range &r, int token, int n) { return token < r.hi && token + n > r.lo; }  // any of n tokens
// 64-token tiles that rows i0 .. i1 of a sequence see between them: [first, last)
__device__ __forceinline__ void tile_range(const AttArgs &a, const KvSeq &s, int i0, int i1, int &first, int &last) {
    if (i1 >= s.n) i1 = s.n - 1;
    if (i0 + s.begin < 0) i0 = -s.begin;  // rows before token 0 see nothing
    first = last = 0;
    if (i0 > i1) return;
    const Range x = row_range(a, s, i0), y = row_range(a, s, i1);  // both ends grow with the row
    if (y.hi <= x.lo) return;
    first = x.lo / 64;
    last = (y.hi + 63) / 64;
}
// tiles in a slice when `tiles` of them are cut into at most a.splits slices: no fewer than a.min_tiles
__device__ __forceinline__ int slice_tiles(const AttArgs &a, int tiles) {
    const int each = (tiles + a.splits - 1) / a.splits;
    return each < a.min_tiles ? a.min_tiles : each;
}
// the part of [first, last) that slice `split` walks; false if there is none (slice 0 always has one, if empty)
__device__ __forceinline__ bool slice_of(const AttArgs &a, int split, int &first, int &last) {
    const int each = a.splits > 1 ? slice_tiles(a, last - first) : last - first, b = first + split * each;
    last = b + each < last ? b + each : last;
    first = b;
    return split == 0 || first < last;
}
// The table's entry for a token, read without a branch (past the last page: the last page's), and the page it stands for: -1 if
// the token is not below the length or the entry is none.  Loads go to page 0 then, which exists (a sequence of a cache without
// pages has length 0), and what they bring is masked.
__device__ __forceinline__ int entry_at(const AttArgs &a, int seq, int token) {
    const int slot = token >> a.kv.page_shift, at = slot < a.kv.pages_per_seq ? slot : a.kv.pages_per_seq - 1;
    const int64_t k = (int64_t)seq * a.kv.pages_per_seq + at;
    return a.kv.table ? a.kv.table[k] : (int)k;
}
__device__ __forceinline__ int page_of(const AttArgs &a, const KvSeq &s, int entry, int token) {
    return token < s.length && (unsigned)entry < (unsigned)a.kv.num_pages ? entry : -1;
}
// eight values of a row as Kind parts; zeros past the end of the head
template <typename T, int QP> __device__ __forceinline__ void load_query(const T *src, bool there, u32x4 (&q)[QP]) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (there) {
        constexpr int V = kVecBytes / (int)sizeof(T);
#pragma unroll
        for (int p = 0; p < 8 / V; ++p) {
            const vec_t<T, V> w = reinterpret_cast<const vec_t<T, V> *>(src)[p];
#pragma unroll
            for (int e = 0; e < V; ++e) x[p * V + e] = load_acc(w.v[e]);
        }
    }
    split_parts<typename RowType<T>::Kind, QP>(x, q);
}
template <typename T> __device__ __forceinline__ void store4(T *dst, float x0, float x1, float x2, float x3) {
    const float y[4] = {x0, x1, x2, x3};
    vec_t<T, 4> w;
    store_acc_vec<T, 4>(w, y);
    *reinterpret_cast<vec_t<T, 4> *>(dst) = w;
}
// `ref`: the power of two that l / kSumUnit and the output are counted in
__device__ __forceinline__ float lse_of(float ref, float l) {
    const bool small = l < 0x1p-100f;
    return l == 0.f ? kNone : kLn2 * (ref + kSumLog + (small ? __builtin_amdgcn_logf(l * 0x1p64f) - 64.f : __builtin_amdgcn_logf(l)));
}

// ---- few rows -------------------------------------------------------------------------------------------------------------
// One workgroup: 16 rows of one (sequence, key head), one slice of the tokens; its waves take the 64-token tiles in
// turn and meet at the end (four waves; eight where there is at most a workgroup a CU: one row over 777 tokens 9.5 -> 8.9 us).  Row 4g + r of 16-token score tile t is token 16g + 4t + r: lane group g holds tokens 16g .. 16g + 15,
// loads codes straight into the operands' registers (no LDS) and needs one page and one scale.  Bound by the bytes of the codes:
// 64 rows over 1k-16k tokens, 32 / 8 heads of 128 in e4m3, 211 us (5.5 TB/s); 4 rows over 131071 in int8, 53 us (5.0 TB/s).
template <typename T, typename Code, int SPANS, bool EXACT, bool ONE, bool NT, int WAVES>
static __global__ __launch_bounds__(WAVES * kWave, WAVES > 4 ? 2 : SPANS == 4 ? 1 : SPANS == 2 || RowType<T>::QP > 1 ? 2 : 3) void kvattention_rows_kernel(const AttArgs a) {
    using Kind = typename RowType<T>::Kind;
    constexpr int QP = RowType<T>::QP, PP = 2, DT = SPANS * 4;  // DT: 16-dimension tiles of the padded head
    __shared__ float meet_o[WAVES / 2][16][SPANS * 64 + 4];
    __shared__ float meet_m[WAVES][16], meet_l[WAVES][16];
    unsigned blk = blockIdx.x;
    const int split = blk % (unsigned)a.splits; blk /= (unsigned)a.splits;
    const int rt = blk % (unsigned)a.row_tiles; blk /= (unsigned)a.row_tiles;
    const int head = blk % (unsigned)a.kv.heads, seq = blk / (unsigned)a.kv.heads;
    const KvSeq s = kv_seq(a.kv, seq);
    const int G = a.group, rows = s.n * G, r0 = rt * 16;
    if (r0 >= rows) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int D = EXACT ? SPANS * 64 : a.kv.dim, P = a.kv.page_size;
    int tile, tile_end;
    tile_range(a, s, r0 / G, (r0 + 15) / G, tile, tile_end);
    if (!slice_of(a, split, tile, tile_end)) return;  // the joining launch knows

    // keys: row n of score tile t is token 16 (n / 4) + 4 t + n % 4; values and scales: tokens 16 g .. 16 g + 15
    const int kofs = 16 * (n >> 2), gofs = 16 * g;
    tile += wave;
    u32x4 kc[4][SPANS], vc[DT];
    int kentry = 0, gentry = 0, gp = -1;
    float ks = 0.f, vs = 0.f;
    // ONE: a tile lies in one page, whose number, address and scales are the same for all lanes and stay in scalar registers
    auto entries = [&](int t) __attribute__((always_inline)) {
        kentry = entry_at(a, seq, t * 64 + (ONE ? 0 : kofs));
        gentry = ONE ? kentry : entry_at(a, seq, t * 64 + gofs);
    };
    const int64_t page_bytes = (int64_t)a.kv.heads * P * D;
    const uint8_t *khead = a.kv.k + (int64_t)head * P * D, *vhead = a.kv.v + (int64_t)head * P * D;
    const uint32_t kin = ((kofs & (P - 1)) + (n & 3)) * D, vin = gofs & (P - 1);
    auto load_keys = [&](int t) __attribute__((always_inline)) {  // and the scales
        const int half = (t * 64) & (P - 1) & 64;  // the second half of a page of 128
        const int k = page_of(a, s, kentry, t * 64 + (ONE ? 0 : kofs));
        gp = ONE ? k : page_of(a, s, gentry, t * 64 + gofs);
        const uint8_t *src = khead + (k < 0 ? 0 : k) * page_bytes + half * D;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < SPANS; ++c) {
                const int d = c * 64 + g * 16;  // past the end of the head the query is zero: any key of the row will do
                const u32x4 *p = reinterpret_cast<const u32x4 *>(src + (kin + 4 * u * D + (EXACT || d < D ? d : 0)));
                kc[u][c] = ld_sel<NT>(p);
            }
        const int64_t at = (int64_t)(gp < 0 ? 0 : gp) * a.kv.heads + head;
        ks = a.kv.k_scale[at];
        vs = a.kv.v_scale[at];
    };
    auto load_values = [&](int t, int page) __attribute__((always_inline)) {
        const uint8_t *src = vhead + (page < 0 ? 0 : page) * page_bytes + ((t * 64) & (P - 1) & 64);
#pragma unroll
        for (int u = 0; u < DT; ++u) {
            const int d = u * 16 + n;  // dimensions past the end of the head are not stored
            const u32x4 *p = reinterpret_cast<const u32x4 *>(src + (vin + (EXACT || d < D ? d : n) * P));
            vc[u] = ld_sel<NT>(p);
        }
    };
    if (tile < tile_end) {
        entries(tile);
        load_keys(tile);
        load_values(tile, gp);
        entries(tile + WAVES);
    }

    // this lane's row
    const int r = r0 + n, i = r / G, h = head * G + (r - i * G);
    const bool real = r < rows;
    Range vis = row_range(a, s, i);
    if (!real) vis = {0, 0};
    u32x4 q[SPANS * 2][QP];
    {
        const T *src = (const T *)a.q + (s.first + i) * a.q_row + h * a.q_head;
#pragma unroll
        for (int c = 0; c < SPANS * 2; ++c) {  // span c / 2, half c % 2
            const int d = (c / 2) * 64 + g * 16 + (c % 2) * 8;
            load_query<T, QP>(src + d, real && d < D, q[c]);
        }
    }
    // a tile needs no masks when every real row sees all of it
    const int last_row = (r0 + 15 < rows ? r0 + 15 : rows - 1) / G;
    const int all_lo = row_range(a, s, last_row).lo, all_hi = row_range(a, s, r0 / G).hi;

    float m = kNone, l = 0.f, largest = kNone;  // largest: logarithm of a value scale that the row has seen
    f32x4_t o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    for (; tile < tile_end; tile += WAVES) {
        const int tok0 = tile * 64, gb = tok0 + gofs;
        ValueScale vsc = value_scale(vs);
        const bool cut = tok0 < all_lo || tok0 + 64 > all_hi;
        {
            float x = gp < 0 || (cut && !sees(vis, ONE ? tok0 : gb, ONE ? 64 : 16)) ? kNone : vsc.log;
            if constexpr (!ONE) {
                x = __builtin_fmaxf(x, __shfl_xor(x, 16));
                x = __builtin_fmaxf(x, __shfl_xor(x, 32));
            }
            largest = __builtin_fmaxf(largest, x);
            reach(vsc, largest);
        }
        const float mul = ks * a.scale;
        const bool none = gp < 0, fine = finite(vs) && finite(mul), more = tile + WAVES < tile_end;
        const bool odd = cut || __any(none || !fine);
        float sc[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < SPANS * 2; ++c) {
                const u32x4 k = codes8<Code, Kind>(kc[t][c / 2][(c % 2) * 2], kc[t][c / 2][(c % 2) * 2 + 1]);
#pragma unroll
                for (int p = 0; p < QP; ++p) acc = mma16<Kind>(k, q[c][p], acc);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[4 * t + e] = __builtin_fmaf(acc[e], mul, vsc.log);
        }
        // the keys' registers are free: the next tile's keys come while this one's values are used
        if (more) load_keys(tile + WAVES);
        if (odd) {
            uint32_t bad = fine ? 0u : 0xffffu;  // bit j: the score of token 16 g + j becomes NaN
            if constexpr (std::is_same_v<Code, CodeE4M3>) {
                uint32_t any = 0;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int w = 0; w < 4; ++w) any |= nan_bytes(vc[t][w]);
                if (__any(any != 0)) {
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        const uint32_t found = drop_nans(vc[t]);
                        if (EXACT || t * 16 < D) bad |= found;
                    }
#pragma unroll
                    for (int x = 1; x < 16; x <<= 1) bad |= __shfl_xor(bad, x, 16);
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (bad >> e & 1u) sc[e] = __builtin_nanf("");
                if (none || gb + e < vis.lo || gb + e >= vis.hi) sc[e] = kNone;
            }
        }
        float top = m;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = __builtin_fmaxf(top, sc[e]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float base = top == kNone ? 0.f : top;
        const Shift shift = shift_of(m - base);
        m = top;
        float sum = 0.f;
        u32x4 p[2][PP];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(sc[8 * u + e] - (base - kLift));
                sum += x[e];
                x[e] *= vsc.factor;
            }
            split_parts<_Float16, PP>(x, p[u]);
        }
        l = __builtin_fmaf(sum * kSumUnit, vsc.inv, shift.sum(l));
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            o[t] *= shift.all();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const u32x4 v = codes8<Code, _Float16>(vc[t][2 * u], vc[t][2 * u + 1]);
#pragma unroll
                for (int k = 0; k < PP; ++k) o[t] = mma16<_Float16>(v, p[u][k], o[t]);
            }
        }
        if (more) {
            load_values(tile + WAVES, gp);
            entries(tile + 2 * WAVES);
        }
    }

    // the waves meet: l over the lane groups, then everything relative to the common maximum, added in wave order
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) meet_m[wave][n] = m;
    __syncthreads();
    float top = meet_m[0][n];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = __builtin_fmaxf(top, meet_m[w][n]);
    const Shift mine = shift_of(m - (top == kNone ? 0.f : top));
    l = mine.sum(l);
    if (g == 0) meet_l[wave][n] = l;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] *= mine.all();
#pragma unroll
    for (int half = WAVES / 2; half >= 1; half >>= 1) {  // the upper half of the waves gives to the lower, until one is left
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4_t *>(&meet_o[wave - half][n][t * 16 + g * 4]) = o[t];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] += *reinterpret_cast<const f32x4_t *>(&meet_o[wave][n][t * 16 + g * 4]);
        __syncthreads();
    }
    if (wave != 0 || !real) return;
    l = meet_l[0][n];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) l += meet_l[w][n];
    const int64_t at = (s.first + i) * a.q_heads + h;
    if (a.splits > 1) {
        const int64_t slot = (int64_t)split * a.kv.rows * a.q_heads + at;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (t * 16 < D) *reinterpret_cast<f32x4_t *>(a.part_o + slot * D + t * 16 + g * 4) = o[t];
        if (g == 0) { a.part_ml[2 * slot] = top - kLift; a.part_ml[2 * slot + 1] = l; }
        return;
    }
    const float inv = l == 0.f ? 0.f : kSumUnit / l;
    T *dst = (T *)a.out + (s.first + i) * a.o_row + h * a.o_head;
#pragma unroll
    for (int t = 0; t < DT; ++t)
        if (t * 16 < D) store4<T>(dst + t * 16 + g * 4, o[t][0] * inv, o[t][1] * inv, o[t][2] * inv, o[t][3] * inv);
    if (g == 0 && a.lse) a.lse[at] = lse_of(top - kLift, l);
}

// ---- many rows ------------------------------------------------------------------------------------------------------------
// One workgroup: 32 rows a wave of one (sequence, key head); the waves share every 64-token tile, whose codes are turned into
// 16-bit operands once, on their way from registers (loaded a tile ahead) into LDS.  Scores: two 32-token products of 32x32x16;
// row 8b + 4h + r of one is token 16h + 4b + r, so lane half h holds 16 consecutive tokens of one page and feeds
// their probabilities to the second product as they are.  Rows of LDS are padded by 16 bytes: 16 lanes that read 16 bytes at
// one column of 16 rows meet 16 different bank groups.
// Bound by the vector pipe and what it cannot hide: causal prompts of 4 x 3.3k-4.1k tokens, 32 / 8 heads of 128, 636 us (765
// TFLOP/s), matrix pipe busy 31 %, vector pipe 48 % (2^x a third of that), waves waiting 29 %; 1.3 LDS instructions a product, whose bank
// conflicts add 0.8 cycles each.  Eight waves a workgroup, two
// buffers with one barrier a tile, an enforced alternation of matrix and vector instructions, and raised wave priority under
// the products were measured at 682, 672, 669 and 674 us.
// Heads over 128: two workgroups take half of the output's dimensions each and both compute the scores: half as much again in
// products, but a row's registers are fewer.  Four prompts of 2k-3k tokens, 16 / 4 heads of 256: 959 us with the head in one
// workgroup, 805 in two with one wave a SIMD, 535 with two (960, 740 where pages are of 16 tokens).  Two waves a SIMD leave 256 registers,
// of which these variants spill 44 to 68 (f32 rows, one wave, 512 registers: 27 to 76); that is part of
// those times.  So are the 6 to 16 that heads of 65 to 128 spill with a page number a lane.
constexpr int value_parts(int padded_dim) { return padded_dim > 128 ? 2 : 1; }
template <typename T, typename Code, int DP, bool EXACT, bool ONE, int WAVES>
static __global__ __launch_bounds__(WAVES * kWave, DP <= 64 || RowType<T>::QP == 1 ? 2 : 1) void kvattention_tiles_kernel(const AttArgs a) {
    using Kind = typename RowType<T>::Kind;
    constexpr int QP = RowType<T>::QP, PP = RowType<T>::PP, PARTS = value_parts(DP), DV = DP / PARTS, DT = DV / 32, THREADS = WAVES * kWave;
    constexpr int KPITCH = DP * 2 + 16, VPITCH = 64 * 2 + 16, KPIECES = (DP * 4 + THREADS - 1) / THREADS, VPIECES = (DV * 4 + THREADS - 1) / THREADS;
    constexpr float slack = PP == 1 ? kSlack : 0.f, lift = kLift - slack;
    __shared__ __attribute__((aligned(16))) unsigned char kl[64 * KPITCH], vl[DV * VPITCH];
    __shared__ uint32_t bad_tokens[2][2];
    // longest tiles of rows first; the tiles of one (sequence, head) stay on one XCD when there are a multiple of 8 pairs
    const unsigned pairs = (unsigned)a.kv.batch * a.kv.heads;
    unsigned blk = blockIdx.x;
    const int pair = blk % pairs; blk /= pairs;
    const int part = blk % PARTS; blk /= PARTS;
    const int split = blk % (unsigned)a.splits, rt = a.row_tiles - 1 - (int)(blk / (unsigned)a.splits);
    const int head = pair % a.kv.heads, seq = pair / a.kv.heads;
    const KvSeq s = kv_seq(a.kv, seq);
    const int G = a.group, rows = s.n * G, r0 = rt * (WAVES * 32);
    if (r0 >= rows) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h2 = lane >> 5;
    const int D = EXACT ? DP : a.kv.dim, P = a.kv.page_size;
    int tile, tile_end;
    tile_range(a, s, r0 / G, (r0 + WAVES * 32 - 1) / G, tile, tile_end);
    if (!slice_of(a, split, tile, tile_end)) return;

    // pieces of 16 codes that this thread brings: of the keys token kt, dimensions kd ..; of the values dimension v0 + vd, tokens vt ..
    const int v0 = part * DV, Dv = EXACT || D - v0 > DV ? DV : D - v0;
    int kt[KPIECES], kd[KPIECES], vd[VPIECES], vt[VPIECES];
    uint32_t kofs[KPIECES], vofs[VPIECES];  // where the pieces lie in a page of this head, for tiles that begin in a page's first 64 tokens
    bool kthere[KPIECES], vthere[VPIECES];  // others load piece 0 and drop it
    // a token of the piece's page: the same for a whole wave, whose pieces are 4, 8 or 16 tokens' keys and one block of tokens' values,
    // where the head fills its registers, so that page numbers and addresses are scalar
    int kpage[KPIECES], vpage[VPIECES];
    auto of_wave = [](int token) __attribute__((always_inline)) { return EXACT ? __builtin_amdgcn_readfirstlane(token) : token; };
#pragma unroll
    for (int j = 0; j < KPIECES; ++j) {
        const int id = threadIdx.x + j * THREADS, per = D / 16;
        kthere[j] = EXACT || id < 4 * D;
        const int x = kthere[j] ? id : 0;
        kt[j] = x / per;
        kd[j] = (x - kt[j] * per) * 16;
        kpage[j] = of_wave(kt[j]);
        kofs[j] = (kt[j] & (P - 1)) * D + kd[j];
    }
#pragma unroll
    for (int j = 0; j < VPIECES; ++j) {
        const int id = threadIdx.x + j * THREADS;
        vthere[j] = EXACT || id < 4 * Dv;
        const int x = vthere[j] ? id : 0;
        // lanes along the tokens where a page holds them all, else along the dimensions: one page a wave
        vd[j] = ONE ? x >> 2 : x % Dv;
        vt[j] = (ONE ? x & 3 : x / Dv) * 16;
        vpage[j] = of_wave(vt[j]);
        vofs[j] = (v0 + vd[j]) * P + (vt[j] & (P - 1));
    }
    if (threadIdx.x < 4) bad_tokens[threadIdx.x >> 1][threadIdx.x & 1] = 0;
    if (D < DP) {  // what pads the head stays zero
        for (int id = threadIdx.x; id < 64 * (DP - D) / 8; id += THREADS)
            *reinterpret_cast<u32x4 *>(kl + (id / ((DP - D) / 8)) * KPITCH + D * 2 + (id % ((DP - D) / 8)) * 16) = u32x4{0u, 0u, 0u, 0u};
        for (int id = threadIdx.x; id < (DV - Dv) * 8; id += THREADS)
            *reinterpret_cast<u32x4 *>(vl + (Dv + id / 8) * VPITCH + (id % 8) * 16) = u32x4{0u, 0u, 0u, 0u};
    }

    // this lane's row
    const int w0 = r0 + wave * 32, r = w0 + n, i = r / G, h = head * G + (r - i * G);
    const bool real = r < rows;
    Range vis = row_range(a, s, i);
    if (!real) vis = {0, 0};
    u32x4 q[DP / 16][QP];
    {
        const T *src = (const T *)a.q + (s.first + i) * a.q_row + h * a.q_head;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) load_query<T, QP>(src + c * 16 + h2 * 8, real && c * 16 < D, q[c]);
    }
    // tokens that any row of the wave sees, that all of them see; that all rows of the workgroup see
    Range any = {0, 0}, all = {0, 0}, group_all;
    {
        const int last = (r0 + WAVES * 32 < rows ? r0 + WAVES * 32 : rows) - 1, wlast = w0 + 31 < rows ? w0 + 31 : rows - 1;
        group_all = {row_range(a, s, last / G).lo, row_range(a, s, r0 / G).hi};
        if (w0 < rows) {
            const Range x = row_range(a, s, w0 / G), y = row_range(a, s, wlast / G);
            any = {x.lo, y.hi};
            all = {y.lo, x.hi};
        }
    }

    float m = kNone, l = 0.f, largest = kNone;  // largest: logarithm of a value scale that the row has seen
    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] = 0.f;

    // table entries two tiles ahead, codes and scales one.  ONE: a tile lies in one page, whose number, address and scales are the
    // same for all lanes and stay in scalar registers.
    constexpr int KE = ONE ? 1 : KPIECES, VE = ONE ? 1 : VPIECES, S = ONE ? 1 : 2;
    int kentry[KE], ventry[VE], sentry[S], sp[S];
    bool vnone[VE];  // values: the page is none
    u32x4 kc[KPIECES], vc[VPIECES];
    float ks_next[S], vs_next[S];
    auto entries = [&](int t) __attribute__((always_inline)) {
        if constexpr (ONE) {
            kentry[0] = entry_at(a, seq, t * 64);
        } else {
#pragma unroll
            for (int j = 0; j < KPIECES; ++j) kentry[j] = entry_at(a, seq, t * 64 + kpage[j]);
#pragma unroll
            for (int j = 0; j < VPIECES; ++j) ventry[j] = entry_at(a, seq, t * 64 + vpage[j]);
#pragma unroll
            for (int u = 0; u < 2; ++u) sentry[u] = entry_at(a, seq, t * 64 + u * 32 + h2 * 16);
        }
    };
    const int64_t page_bytes = (int64_t)a.kv.heads * P * D;
    const uint8_t *khead = a.kv.k + (int64_t)head * P * D, *vhead = a.kv.v + (int64_t)head * P * D;
    auto fetch = [&](int t) __attribute__((always_inline)) {
        const int half = (t * 64) & (P - 1) & 64;  // the second half of a page of 128
        if constexpr (ONE) {
            sp[0] = page_of(a, s, kentry[0], t * 64);
            vnone[0] = sp[0] < 0;
            const int page = sp[0] < 0 ? 0 : sp[0];
            const uint8_t *ksrc = khead + page * page_bytes + half * D, *vsrc = vhead + page * page_bytes + half;
#pragma unroll
            for (int j = 0; j < KPIECES; ++j) kc[j] = *reinterpret_cast<const u32x4 *>(ksrc + kofs[j]);
#pragma unroll
            for (int j = 0; j < VPIECES; ++j) vc[j] = *reinterpret_cast<const u32x4 *>(vsrc + vofs[j]);
        } else {
#pragma unroll
            for (int j = 0; j < KPIECES; ++j) {
                const int kp = page_of(a, s, kentry[j], t * 64 + kpage[j]);
                kc[j] = *reinterpret_cast<const u32x4 *>(khead + (kp < 0 ? 0 : kp) * page_bytes + (kofs[j] + half * D));
            }
#pragma unroll
            for (int j = 0; j < VPIECES; ++j) {
                const int vp = page_of(a, s, ventry[j], t * 64 + vpage[j]);
                vnone[j] = vp < 0;
                vc[j] = *reinterpret_cast<const u32x4 *>(vhead + (vp < 0 ? 0 : vp) * page_bytes + (vofs[j] + half));
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) sp[u] = page_of(a, s, sentry[u], t * 64 + u * 32 + h2 * 16);
        }
#pragma unroll
        for (int u = 0; u < S; ++u) {
            const int64_t at = (int64_t)(sp[u] < 0 ? 0 : sp[u]) * a.kv.heads + head;
            ks_next[u] = a.kv.k_scale[at];
            vs_next[u] = a.kv.v_scale[at];
        }
    };
    const int krow = (16 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3)) * KPITCH + h2 * 16, vrow = n * VPITCH + h2 * 32;
    auto clean = [&](int t) __attribute__((always_inline)) {  // e4m3: values without NaNs where a mask or a missing page could meet them
        if constexpr (std::is_same_v<Code, CodeE4M3>) {
            bool gone = false;
#pragma unroll
            for (int j = 0; j < VE; ++j) gone = gone || vnone[j];
            const bool cut = t * 64 < group_all.lo || t * 64 + 64 > group_all.hi;
            if (cut || __any(gone)) {
#pragma unroll
                for (int j = 0; j < VPIECES; ++j) {
                    if (!vthere[j]) continue;
                    if (vnone[ONE ? 0 : j]) vc[j] = u32x4{0u, 0u, 0u, 0u};
                    const uint32_t found = cut ? drop_nans(vc[j]) : 0u;
                    if (found) atomicOr(&bad_tokens[t & 1][vt[j] >> 5], found << (vt[j] & 16));
                }
            }
        }
    };
    // the codes in the registers as operands into LDS
    auto stage = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < KPIECES; ++j) {
            if (!kthere[j]) continue;
            u32x4 *dst = reinterpret_cast<u32x4 *>(kl + kt[j] * KPITCH + kd[j] * 2);
            dst[0] = codes8<Code, Kind>(kc[j][0], kc[j][1]);
            dst[1] = codes8<Code, Kind>(kc[j][2], kc[j][3]);
        }
#pragma unroll
        for (int j = 0; j < VPIECES; ++j) {
            if (!vthere[j]) continue;
            u32x4 *dst = reinterpret_cast<u32x4 *>(vl + vd[j] * VPITCH + vt[j] * 2);
            dst[0] = codes8<Code, _Float16>(vc[j][0], vc[j][1]);
            dst[1] = codes8<Code, _Float16>(vc[j][2], vc[j][3]);
        }
    };
    __syncthreads();  // the zeroed flags and pads
    if (tile < tile_end) {
        entries(tile);
        fetch(tile);
        entries(tile + 1);
    }
    for (; tile < tile_end; ++tile) {
        const int tok0 = tile * 64, slot = tile & 1;
        const unsigned char *kb = kl + krow, *vb = vl + vrow;
        clean(tile);
        stage();
        float ks[S], vs[S];
        int page[S];
#pragma unroll
        for (int u = 0; u < S; ++u) { ks[u] = ks_next[u] * a.scale; vs[u] = vs_next[u]; page[u] = sp[u]; }
        if (tile + 1 < tile_end) {
            fetch(tile + 1);
            entries(tile + 2);
        }
        __syncthreads();  // this tile is in LDS
        if (threadIdx.x < 2) bad_tokens[slot ^ 1][threadIdx.x] = 0;
        const bool cut = tok0 < group_all.lo || tok0 + 64 > group_all.hi;
        ValueScale vsc[S];
        bool plain = !cut;
#pragma unroll
        for (int u = 0; u < S; ++u) vsc[u] = value_scale(vs[u]);
        {
            float y[S];
#pragma unroll
            for (int u = 0; u < S; ++u) y[u] = page[u] < 0 ? kNone : vsc[u].log;
            if (cut) {
#pragma unroll
                for (int u = 0; u < S; ++u) y[u] = sees(vis, ONE ? tok0 : tok0 + u * 32 + h2 * 16, ONE ? 64 : 16) ? y[u] : kNone;
            }
            float x = __builtin_fmaxf(y[0], y[S - 1]);
            if constexpr (!ONE) x = other_half_max(x);
            largest = __builtin_fmaxf(largest, x);
        }
#pragma unroll
        for (int u = 0; u < S; ++u) {
            plain = plain && !__any(page[u] < 0 || !(ks[u] >= 0.f) || !finite(ks[u]) || !finite(vs[u]) || vsc[u].factor != 1.f || out_of_reach(vsc[u], largest));
        }
        f32x16 sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[u][e] = 0.f;
        auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    const u32x4 k = *reinterpret_cast<const u32x4 *>(kb + u * 32 * KPITCH + c * 32);
#pragma unroll
                    for (int p = 0; p < QP; ++p) sc[u] = mma32<Kind>(k, q[c][p], sc[u]);
                }
        };
        u32x4 p[2][2][PP];
        auto powers = [&](int u, float mul, float add, float factor) __attribute__((always_inline)) {
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][8 * v + e], mul, add));
                    sum += x[e];
                    x[e] *= factor;
                }
                split_parts<_Float16, PP>(x, p[u][v]);
            }
            l = __builtin_fmaf(sum * kSumUnit, vsc[ONE ? 0 : u].inv, l);
        };
        auto outputs = [&](int u) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(vb + t * 32 * VPITCH + u * 64 + v * 16);
#pragma unroll
                    for (int k = 0; k < PP; ++k) o[t] = mma32<_Float16>(x, p[u][v][k], o[t]);
                }
        };
        auto follow = [&](float top) __attribute__((always_inline)) {  // the row's reference after scores of at most `top`
            top = __builtin_fmaxf(m, top);
            const bool move = top > m + slack;
            if (__any(move)) {
                const float to = move ? top : m;
                const Shift shift = shift_of(m - (to == kNone ? 0.f : to));
                m = to;
                l = shift.sum(l);
#pragma unroll
                for (int t = 0; t < DT; ++t) o[t] *= shift.all();
            }
        };
        if (plain) {
            scores();
            float top = kNone;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float x = sc[u][0];
#pragma unroll
                for (int e = 1; e < 16; ++e) x = __builtin_fmaxf(x, sc[u][e]);
                top = __builtin_fmaxf(top, __builtin_fmaf(x, ks[ONE ? 0 : u], vsc[ONE ? 0 : u].log));  // ks >= 0: the largest product is the largest score
            }
            follow(other_half_max(top));
            powers(0, ks[0], vsc[0].log - (m - lift), 1.f);
            outputs(0);
            powers(1, ks[S - 1], vsc[S - 1].log - (m - lift), 1.f);
            outputs(1);
        } else {
            if (tok0 < any.hi && tok0 + 64 > any.lo) {
#pragma unroll
                for (int u = 0; u < S; ++u) reach(vsc[u], largest);
                scores();
                const uint32_t bads[2] = {bad_tokens[slot][0], bad_tokens[slot][1]};
                float top = kNone;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int su = ONE ? 0 : u;
                    const uint32_t bad = finite(ks[su]) && finite(vs[su]) ? bads[u] >> (16 * h2) : 0xffffu;
                    const int t0 = tok0 + u * 32 + h2 * 16;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float x = __builtin_fmaf(sc[u][e], ks[su], vsc[su].log);
                        if (bad >> e & 1u) x = __builtin_nanf("");
                        if (page[su] < 0 || t0 + e < vis.lo || t0 + e >= vis.hi) x = kNone;
                        sc[u][e] = x;
                        top = __builtin_fmaxf(top, x);
                    }
                }
                follow(other_half_max(top));
                const float base = m == kNone ? 0.f : m;
#pragma unroll
                for (int u = 0; u < 2; ++u) powers(u, 1.f, -(base - lift), vsc[ONE ? 0 : u].factor);
                outputs(0);
                outputs(1);
            }
        }
        __syncthreads();  // and is left by everybody
    }
    l += __shfl_xor(l, 32);
    if (!real) return;
    const int64_t at = (s.first + i) * a.q_heads + h;
    if (a.splits > 1) {
        const int64_t slot = (int64_t)split * a.kv.rows * a.q_heads + at;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int d = v0 + t * 32 + b * 8 + h2 * 4;
                if (d < D) *reinterpret_cast<f32x4_t *>(a.part_o + slot * D + d) = f32x4_t{o[t][4 * b], o[t][4 * b + 1], o[t][4 * b + 2], o[t][4 * b + 3]};
            }
        if (h2 == 0 && part == 0) { a.part_ml[2 * slot] = m - lift; a.part_ml[2 * slot + 1] = l; }
        return;
    }
    const float inv = l == 0.f ? 0.f : kSumUnit / l;
    T *dst = (T *)a.out + (s.first + i) * a.o_row + h * a.o_head;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int d = v0 + t * 32 + b * 8 + h2 * 4;
            if (d < D) store4<T>(dst + d, o[t][4 * b] * inv, o[t][4 * b + 1] * inv, o[t][4 * b + 2] * inv, o[t][4 * b + 3] * inv);
        }
    if (h2 == 0 && part == 0 && a.lse) a.lse[at] = lse_of(m - lift, l);
}

// ---- the slices of a row ------------------------------------------------------------------------------------------------
// Groups of dim / 4 lanes (rounded up to a power of two) add the slices of a packed row and query head, eight loads at a time, the first
// ones before the weights are known.  A slice's weight comes from its maximum and the common one: lane j of a group (of the wave,
// where there are more than kFewSlices) has those of slice j and j + 64.  Up to kFewSlices one group takes all slices of its own row;
// beyond, the groups of a workgroup share one row, every group every so many-th slice, and meet in LDS, where the sums are added
// in group order.  118 slices of 112 rows of 128: 6.6 us one slice after the other, 8.4 with a pass for the maximum first, 6.9 this way.
constexpr int kFewSlices = 16;
template <typename T>
static __global__ __launch_bounds__(kBlock) void kvattention_join_kernel(const AttArgs a) {
    __shared__ f32x4_t meet_o[kBlock];
    const int lanes = a.kv.dim <= 64 ? 16 : a.kv.dim <= 128 ? 32 : 64, groups = kBlock / lanes, group = threadIdx.x / lanes, d = (threadIdx.x % lanes) * 4;
    const bool shared = a.splits > kFewSlices, live = d < a.kv.dim;
    unsigned blk = shared ? blockIdx.x : blockIdx.x * groups + group;
    const int h = blk % (unsigned)a.q_heads; blk /= (unsigned)a.q_heads;
    const int i = blk % (unsigned)a.kv.max_rows, seq = blk / (unsigned)a.kv.max_rows;
    if (seq >= a.kv.batch) return;  // whole groups; in the shared form the grid is exact
    const KvSeq s = kv_seq(a.kv, seq);
    if (i >= s.n) return;
    const int r0 = (i * a.group + h % a.group) / a.tile_rows * a.tile_rows;
    int first, last;
    tile_range(a, s, r0 / a.group, (r0 + a.tile_rows - 1) / a.group, first, last);
    const int each = slice_tiles(a, last - first), used = last > first ? (last - first + each - 1) / each : 1;
    const int64_t at = (s.first + i) * a.q_heads + h, pitch = a.kv.rows * a.q_heads;
    const float *po = a.part_o + at * a.kv.dim + (live ? d : 0), *pm = a.part_ml + 2 * at;
    const int begin = shared ? group : 0, step = shared ? groups : 1, width = shared ? kWave : lanes, j = threadIdx.x % width;
    constexpr int kAhead = 8;
    f32x4_t v[kAhead], o = {0.f, 0.f, 0.f, 0.f};
    auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const int k = k0 + e * step;
            v[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (k < used) v[e] = *reinterpret_cast<const f32x4_t *>(po + k * pitch * a.kv.dim);
        }
    };
    load(begin);
    const bool one = j < used, two = shared && j + kWave < used;
    const float m0 = one ? pm[2 * j * pitch] : kNone, m1 = two ? pm[2 * (j + kWave) * pitch] : kNone;
    const float l0 = one ? pm[2 * j * pitch + 1] : 0.f, l1 = two ? pm[2 * (j + kWave) * pitch + 1] : 0.f;
    float top = __builtin_fmaxf(m0, m1);
    for (int x = width / 2; x > 0; x >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, x));
    const float base = top == kNone ? 0.f : top;
    const Shift w0 = shift_of(m0 - base), w1 = shift_of(m1 - base);
    float l = w0.sum(l0) + w1.sum(l1);
    for (int x = width / 2; x > 0; x >>= 1) l += __shfl_xor(l, x);
    for (int k0 = 0; k0 < used; k0 += kAhead * step) {  // the same number of times for all lanes that exchange weights
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {  // past the last slice: a finite weight of zeros
            const int k = k0 + begin + e * step;
            float w = __shfl(w0.all(), k, width);
            if (shared) {
                const float u = __shfl(w1.all(), k, width);
                w = k < kWave ? w : u;
            }
            o += v[e] * w;
        }
        if (k0 + kAhead * step < used) load(k0 + kAhead * step + begin);
    }
    if (shared) {  // the same for the whole workgroup
        meet_o[threadIdx.x] = o;
        __syncthreads();
        if (group > 0) return;
        for (int k = 1; k < groups; ++k) o += meet_o[k * lanes + threadIdx.x];
    }
    const float inv = l == 0.f ? 0.f : kSumUnit / l;
    if (live) store4<T>((T *)a.out + (s.first + i) * a.o_row + h * a.o_head + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (d == 0 && a.lse) a.lse[at] = lse_of(top, l);
}

// ---- launches -----------------------------------------------------------------------------------------------------------
constexpr int kWaves = 4, kTileRows = kWaves * 32;
template <typename T, typename Code, int SPANS, bool EXACT, bool ONE> void launch_one(const AttArgs &a, hipStream_t st) {
    const unsigned blocks = (unsigned)((int64_t)a.kv.batch * a.kv.heads * a.row_tiles * a.splits);
    if (a.tile_rows == 16) {
        if constexpr (ONE) {
            if (a.nt) { kvattention_rows_kernel<T, Code, SPANS, EXACT, ONE, true, 4><<<blocks, kBlock, 0, st>>>(a); return; }
        }
        if constexpr (SPANS <= 2) {
            if (blocks <= (unsigned)kCUs) { kvattention_rows_kernel<T, Code, SPANS, EXACT, ONE, false, 8><<<blocks, 8 * kWave, 0, st>>>(a); return; }
        }
        kvattention_rows_kernel<T, Code, SPANS, EXACT, ONE, false, 4><<<blocks, kBlock, 0, st>>>(a);
    } else {
        kvattention_tiles_kernel<T, Code, SPANS * 64, EXACT, ONE, kWaves><<<blocks * value_parts(SPANS * 64), kWaves * kWave, 0, st>>>(a);
    }
}
// Head sizes that fill their registers need no bounds in the loops, pages of at least 64 tokens no page number a lane.  Four prompts of
// 2k-3k tokens, 16 / 4 heads of 96, pages of 64: 174 us, with a page number a lane 261.
template <typename T, typename Code, int SPANS> void launch_dim(const AttArgs &a, hipStream_t st) {
    const bool exact = a.kv.dim == SPANS * 64, one = a.kv.page_size >= 64;
    if (exact && one) launch_one<T, Code, SPANS, true, true>(a, st);
    else if (exact) launch_one<T, Code, SPANS, true, false>(a, st);
    else if (one) launch_one<T, Code, SPANS, false, true>(a, st);
    else launch_one<T, Code, SPANS, false, false>(a, st);
}
template <typename T, typename Code> int kvattention_launch(const AttArgs &a, hipStream_t st) {
    if (a.kv.dim <= 64) launch_dim<T, Code, 1>(a, st);
    else if (a.kv.dim <= 128) launch_dim<T, Code, 2>(a, st);
    else launch_dim<T, Code, 4>(a, st);
    const int rc = launch_status();
    if (rc != DXH_OK || a.splits == 1) return rc;
    const int64_t rows = (int64_t)a.kv.batch * a.kv.max_rows * a.q_heads, at_once = a.splits > kFewSlices ? 1 : kBlock / (a.kv.dim <= 64 ? 16 : a.kv.dim <= 128 ? 32 : 64);
    kvattention_join_kernel<T><<<(unsigned)((rows + at_once - 1) / at_once), kBlock, 0, st>>>(a);
    return launch_status();
}

// one source file a row type: they compile side by side
int kvattention_f32(const AttArgs &a, bool i8, hipStream_t st);
int kvattention_f16(const AttArgs &a, bool i8, hipStream_t st);
int kvattention_bf16(const AttArgs &a, bool i8, hipStream_t st);

}  // namespace dxh
