// kvattention.hip — attention of a ragged batch of rows over a paged cache in 8 bits.
//
// For one key head and one sequence the rows of all query heads that share it are one matrix Q [R, D], row r = i * G + g for
// query row i and head g of the G that share the key head.  With K' = the key codes, one pass over the tokens keeps for every row
//     s_j = (Q K'^T)_j * k_scale(page of j) * scale * log2(e),     m = max s_j,  l = sum 2^(s_j - m),
//     O   = sum 2^(s_j - m) v_scale(page of j) V'_j;               out = O / l,  lse = ln 2 (m + log2 l).
// Codes are whole numbers below 2^8 or e4m3 values: both are exact in bf16, so they enter the matrix pipe exactly and the
// scales are applied to scores and probabilities in fp32.  A probability (with its v_scale) is rounded to bf16 for bf16 rows
// (2^-9 of each term, random signs: under the rounding of the result); f16 rows split Q and P into two bf16 parts and f32 rows
// into three (16 and 24 bits), each part one more product.
//
// Everything is computed transposed, S^T = K' Q^T and O^T = V'^T P^T, so that the tokens of a score tile are rows of the
// accumulator and a probability is already in the lane that feeds it to the second product.  Which token a row of the first
// product is, is free: row 4g + r of 16-token tile t of a 64-token block is token 16g + 4t + r.  Lane group g then holds the 16
// consecutive tokens 16g .. 16g + 15 — of one page, with one scale — and reads its values as 16 consecutive codes of one
// dimension: one 16-byte load from the [dim][token] order of the cache, no LDS and no exchange between lanes.
#include <algorithm>
#include "kvcache.hpp"

using namespace dxh;

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct AttArgs {
    KvArgs kv;
    const char *q;
    char *out;
    int64_t q_row, q_head, o_row, o_head;
    float *lse, *part_o, *part_ml;  // partials: [split][packed row][q head][dim] and [split][packed row][q head][2]
    float scale;                    // scale * log2(e)
    int q_heads, group, causal, window, splits, row_tiles;
};

constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.4426950408889634f;
constexpr float kNone = -__builtin_inff();

// number of bf16 parts that hold a value of T for the products
template <typename T> constexpr int kParts = std::is_same_v<T, bf16_t> ? 1 : std::is_same_v<T, f16_t> ? 2 : 3;

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t)); }
// eight values -> NP bf16 vectors whose sum they are (to 8 NP bits)
template <int NP> __device__ __forceinline__ void split_parts(float (&x)[8], bf16x8 (&p)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
            if (k + 1 < NP) {
                x[2 * e] -= bits_to_float(w[e] << 16);
                x[2 * e + 1] -= bits_to_float(w[e] & 0xffff0000u);
            }
        }
        p[k] = __builtin_bit_cast(bf16x8, w);
    }
}
// eight codes (two dwords) as bf16, exactly
template <typename Code> __device__ __forceinline__ bf16x8 codes_bf16(uint32_t a, uint32_t b) {
    u32x4 w;
    if constexpr (std::is_same_v<Code, CodeE4M3>) {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true));
    } else {
        float x[8];
        Code::decode(a, x);
        Code::decode(b, x + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
    }
    return __builtin_bit_cast(bf16x8, w);
}
// bytes of `w` that are an e4m3 NaN, as 0x80 in each
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The tokens [lo, hi) that row r of a sequence sees; nothing for a row that is none or has no place in the cache.
struct Range { int lo, hi; };
__device__ __forceinline__ Range row_range(const AttArgs &a, const KvSeq &s, int i) {
    const int p = s.begin + i;
    if (i >= s.n || p < 0) return {0, 0};
    const int hi = a.causal && p + 1 < s.length ? p + 1 : s.length;
    const int lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    return {lo < hi ? lo : hi, hi};
}
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
// the part of [first, last) that slice `split` of `splits` walks
__device__ __forceinline__ void slice_of(int splits, int split, int &first, int &last) {
    const int each = (last - first + splits - 1) / splits, b = first + split * each, e = b + each < last ? b + each : last;
    first = b;
    last = e;
}

// One workgroup: 16 rows of one (sequence, key head), one slice of the tokens; its four waves take every fourth 64-token tile.
template <typename T, typename Code, int SPANS>
__global__ __launch_bounds__(kBlock) void kvattention_kernel(const AttArgs a) {
    constexpr int NP = kParts<T>, DT = SPANS * 4;  // 16-dimension tiles of the padded head
    __shared__ float meet_o[2][16][SPANS * 64 + 4];
    __shared__ float meet_m[4][16], meet_l[4][16];
    unsigned blk = blockIdx.x;
    const int split = blk % (unsigned)a.splits; blk /= (unsigned)a.splits;
    const int rt = blk % (unsigned)a.row_tiles; blk /= (unsigned)a.row_tiles;
    const int head = blk % (unsigned)a.kv.heads, seq = blk / (unsigned)a.kv.heads;
    const KvSeq s = kv_seq(a.kv, seq);
    const int G = a.group, rows = s.n * G, r0 = rt * 16;
    if (r0 >= rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int D = a.kv.dim, P = a.kv.page_size;
    int tile, tile_end;
    tile_range(a, s, r0 / G, (r0 + 15) / G, tile, tile_end);
    slice_of(a.splits, split, tile, tile_end);
    if (a.splits > 1 && tile >= tile_end && split > 0) return;  // the joining launch knows

    // this lane's row
    const int r = r0 + n, i = r / G, h = head * G + (r - i * G);
    const bool real = r < rows;
    Range vis = row_range(a, s, i);
    if (!real) vis = {0, 0};
    bf16x8 q[SPANS * 2][NP];
    {
        const T *src = (const T *)a.q + (s.first + i) * a.q_row + h * a.q_head;
#pragma unroll
        for (int c = 0; c < SPANS * 2; ++c) {  // span c / 2, half c % 2
            const int d = (c / 2) * 64 + g * 16 + (c % 2) * 8;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.f;
            if (real && d < D) {
                constexpr int V = kVecBytes / (int)sizeof(T);
#pragma unroll
                for (int p = 0; p < 8 / V; ++p) {
                    const vec_t<T, V> w = *reinterpret_cast<const vec_t<T, V> *>(src + d + p * V);
#pragma unroll
                    for (int e = 0; e < V; ++e) x[p * V + e] = load_acc(w.v[e]);
                }
            }
            split_parts<NP>(x, q[c]);
        }
    }
    // a tile needs no masks when every real row sees all of it
    const int last_row = (r0 + 15 < rows ? r0 + 15 : rows - 1) / G;
    const Range first_vis = row_range(a, s, r0 / G), last_vis = row_range(a, s, last_row);
    const int all_lo = last_vis.lo, all_hi = first_vis.hi;

    float m = kNone, l = 0.f;
    f32x4_t o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    for (tile += wave; tile < tile_end; tile += 4) {
        const int tok0 = tile * 64;
        // keys: row n of score tile t is token 16 (n / 4) + 4 t + n % 4; values and scales: tokens 16 g .. 16 g + 15
        const int kb = tok0 + 16 * (n >> 2), gb = tok0 + 16 * g;
        const int64_t kp = kb < s.length ? kv_page(a.kv, seq, kb >> a.kv.page_shift) : -1;
        const int64_t gp = gb < s.length ? kv_page(a.kv, seq, gb >> a.kv.page_shift) : -1;
        u32x4 kc[4][SPANS], vc[DT];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < SPANS; ++c) {
                kc[t][c] = u32x4{0u, 0u, 0u, 0u};
                if (kp >= 0 && c * 64 + g * 16 < D)
                    kc[t][c] = *reinterpret_cast<const u32x4 *>(a.kv.k + ((kp * a.kv.heads + head) * P + ((kb & (P - 1)) + 4 * t + (n & 3))) * D + c * 64 + g * 16);
            }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            vc[t] = u32x4{0u, 0u, 0u, 0u};
            if (gp >= 0 && t * 16 < D) vc[t] = *reinterpret_cast<const u32x4 *>(a.kv.v + ((gp * a.kv.heads + head) * D + (t * 16 + n)) * P + (gb & (P - 1)));
        }
        const float ks = gp >= 0 ? a.kv.k_scale[gp * a.kv.heads + head] * a.scale : 0.f;
        const float vs = gp >= 0 ? a.kv.v_scale[gp * a.kv.heads + head] : 0.f;
        const bool masked = tok0 < all_lo || tok0 + 64 > all_hi || __any(gp < 0);

        float sc[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < SPANS * 2; ++c) {
                const bf16x8 k = codes_bf16<Code>(kc[t][c / 2][(c % 2) * 2], kc[t][c / 2][(c % 2) * 2 + 1]);
#pragma unroll
                for (int p = 0; p < NP; ++p) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[c][p], acc, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[4 * t + e] = acc[e] * ks;
        }
        if (masked) {
            if constexpr (std::is_same_v<Code, CodeE4M3>) {
                // 0 * NaN is NaN: a NaN among the values of a token becomes 0 here and makes the token's score NaN for the rows that see it
                uint32_t bad = 0, any = 0;  // bad: bit j = token 16 g + j
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int w = 0; w < 4; ++w) any |= nan_bytes(vc[t][w]);
                if (__any(any != 0)) {
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t b = nan_bytes(vc[t][w]);
                            vc[t][w] &= ~((b >> 7) * 0xffu);
#pragma unroll
                            for (int e = 0; e < 4; ++e) bad |= ((b >> (8 * e + 7)) & 1u) << (4 * w + e);
                        }
#pragma unroll
                    for (int x = 1; x < 16; x <<= 1) bad |= __shfl_xor(bad, x, 16);
#pragma unroll
                    for (int e = 0; e < 16; ++e) if (bad >> e & 1u) sc[e] = __builtin_nanf("");
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) if (gp < 0 || gb + e < vis.lo || gb + e >= vis.hi) sc[e] = kNone;
        }
        float top = m;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = __builtin_fmaxf(top, sc[e]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float base = top == kNone ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m - base);
        m = top;
        float sum = 0.f;
        bf16x8 p[2][NP];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = __builtin_amdgcn_exp2f(sc[8 * u + e] - base);
                sum += y;
                x[e] = sc[8 * u + e] == kNone ? 0.f : y * vs;  // whatever the scale of a page nobody sees is
            }
            split_parts<NP>(x, p[u]);
        }
        l = l * alpha + sum;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            if (t * 16 < D) {
                o[t] *= alpha;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const bf16x8 v = codes_bf16<Code>(vc[t][2 * u], vc[t][2 * u + 1]);
#pragma unroll
                    for (int k = 0; k < NP; ++k) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[u][k], o[t], 0, 0, 0);
                }
            }
        }
    }

    // the four waves meet: l over the lane groups, then everything relative to the common maximum, added in wave order
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) meet_m[wave][n] = m;
    __syncthreads();
    float top = meet_m[0][n];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = __builtin_fmaxf(top, meet_m[w][n]);
    const float base = top == kNone ? 0.f : top, mine = __builtin_amdgcn_exp2f(m - base);
    l *= mine;
    if (g == 0) meet_l[wave][n] = l;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] *= mine;
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {  // waves 2, 3 give to 0, 1; then 1 to 0
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
    l = (meet_l[0][n] + meet_l[1][n]) + (meet_l[2][n] + meet_l[3][n]);
    const int64_t at = (s.first + i) * a.q_heads + h;
    if (a.splits > 1) {
        const int64_t slot = (int64_t)split * a.kv.rows * a.q_heads + at;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (t * 16 < D) *reinterpret_cast<f32x4_t *>(a.part_o + slot * D + t * 16 + g * 4) = o[t];
        if (g == 0) { a.part_ml[2 * slot] = top; a.part_ml[2 * slot + 1] = l; }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *dst = (T *)a.out + (s.first + i) * a.o_row + h * a.o_head;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        if (t * 16 < D) {
            float y[4];
            vec_t<T, 4> w;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = o[t][e] * inv;
            store_acc_vec<T, 4>(w, y);
            *reinterpret_cast<vec_t<T, 4> *>(dst + t * 16 + g * 4) = w;
        }
    }
    if (g == 0 && a.lse) a.lse[at] = l == 0.f ? kNone : kLn2 * (top + __builtin_amdgcn_logf(l));
}

// Joins the slices of a row, in slice order: one workgroup of `dim` rounded up to 64 threads for each packed row slot of a sequence and head
template <typename T>
__global__ __launch_bounds__(kBlock) void kvattention_join_kernel(const AttArgs a) {
    unsigned blk = blockIdx.x;
    const int h = blk % (unsigned)a.q_heads; blk /= (unsigned)a.q_heads;
    const int i = blk % (unsigned)a.kv.max_rows, seq = blk / (unsigned)a.kv.max_rows;
    const KvSeq s = kv_seq(a.kv, seq);
    if (i >= s.n) return;
    const int r0 = (i * a.group + h % a.group) / 16 * 16;
    int first, last;
    tile_range(a, s, r0 / a.group, (r0 + 15) / a.group, first, last);
    const int each = (last - first + a.splits - 1) / a.splits, used = each > 0 ? (last - first + each - 1) / each : 1;
    const int64_t at = (s.first + i) * a.q_heads + h, pitch = a.kv.rows * a.q_heads;
    float top = kNone;
    for (int k = 0; k < used; ++k) top = __builtin_fmaxf(top, a.part_ml[2 * (at + k * pitch)]);
    const float base = top == kNone ? 0.f : top;
    float l = 0.f, o = 0.f;
    const int d = threadIdx.x;
    for (int k = 0; k < used; ++k) {
        const float w = __builtin_amdgcn_exp2f(a.part_ml[2 * (at + k * pitch)] - base);
        l = __builtin_fmaf(w, a.part_ml[2 * (at + k * pitch) + 1], l);
        if (d < a.kv.dim) o = __builtin_fmaf(w, a.part_o[(at + k * pitch) * a.kv.dim + d], o);
    }
    if (d < a.kv.dim) ((T *)a.out)[(s.first + i) * a.o_row + h * a.o_head + d] = store_acc<T>(l == 0.f ? 0.f : o * (1.f / l));
    if (d == 0 && a.lse) a.lse[at] = l == 0.f ? kNone : kLn2 * (top + __builtin_amdgcn_logf(l));
}

// How many slices the tokens of a sequence are cut into: enough workgroups for the card, but at least four 64-token tiles
// (one for each wave) a slice, counted on the longest sequence that the cache can hold.
int choose_splits(const KvArgs &kv, int q_heads, int64_t row_tiles) {
    const int64_t blocks = (int64_t)kv.batch * kv.heads * row_tiles, tiles = ((int64_t)kv.pages_per_seq * kv.page_size + 63) / 64;
    int64_t want = std::min<int64_t>((4 * kCUs + blocks - 1) / blocks, (tiles + 3) / 4);
    const int64_t row_bytes = kv.rows * q_heads * (kv.dim + 2) * 4;
    want = std::min<int64_t>(want, ((int64_t)256 << 20) / std::max<int64_t>(1, row_bytes));  // partial results of at most 256 MiB
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, 128));
}
size_t part_bytes(const KvArgs &kv, int q_heads, int splits) {
    return splits > 1 ? ((size_t)splits * kv.rows * q_heads * (kv.dim + 2) * sizeof(float) + 255) / 256 * 256 : 0;
}

int plan(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, int32_t q_heads, AttArgs &a) {
    a = AttArgs{};
    const int rc = kv_check(cache, rows, dtype, a.kv);
    if (rc != DXH_OK) return rc;
    if (q_heads < 1) return DXH_ERR_ARG;
    if (q_heads % a.kv.heads) return DXH_ERR_SHAPE;
    a.q_heads = q_heads;
    a.group = q_heads / a.kv.heads;
    a.splits = 1;
    if (kv_nothing(a.kv)) return DXH_OK;
    if ((int64_t)a.kv.max_rows * a.group > INT32_MAX - 64) return DXH_ERR_TOO_LARGE;
    a.row_tiles = (int)(((int64_t)a.kv.max_rows * a.group + 15) / 16);
    a.splits = choose_splits(a.kv, q_heads, a.row_tiles);
    if ((int64_t)a.kv.batch * a.kv.heads * a.row_tiles * a.splits > INT32_MAX || (int64_t)a.kv.batch * a.kv.max_rows * q_heads > INT32_MAX) return DXH_ERR_TOO_LARGE;
    return DXH_OK;
}

template <typename T, typename Code> int launch(const AttArgs &a, hipStream_t st) {
    const unsigned blocks = (unsigned)((int64_t)a.kv.batch * a.kv.heads * a.row_tiles * a.splits);
    switch ((a.kv.dim + 63) / 64) {
    case 1: kvattention_kernel<T, Code, 1><<<blocks, kBlock, 0, st>>>(a); break;
    case 2: kvattention_kernel<T, Code, 2><<<blocks, kBlock, 0, st>>>(a); break;
    case 3: kvattention_kernel<T, Code, 3><<<blocks, kBlock, 0, st>>>(a); break;
    default: kvattention_kernel<T, Code, 4><<<blocks, kBlock, 0, st>>>(a); break;
    }
    const int rc = launch_status();
    if (rc != DXH_OK || a.splits == 1) return rc;
    kvattention_join_kernel<T><<<(unsigned)((int64_t)a.kv.batch * a.kv.max_rows * a.q_heads), (a.kv.dim + 63) / 64 * 64, 0, st>>>(a);
    return launch_status();
}

}  // namespace

extern "C" {

int dxh_kvcache_attention_workspace_bytes(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, int32_t q_heads, size_t *bytes) {
    if (!bytes) return DXH_ERR_ARG;
    AttArgs a;
    const int rc = plan(cache, rows, dtype, q_heads, a);
    if (rc == DXH_OK) *bytes = part_bytes(a.kv, q_heads, a.splits);
    return rc;
}

int dxh_kvcache_attention(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, int32_t q_heads, const dxh_heads *q, const dxh_heads *out, float *lse,
                          float scale, int causal, int64_t window, void *workspace, size_t workspace_bytes, void *stream) {
    AttArgs a;
    int rc = plan(cache, rows, dtype, q_heads, a);
    if (rc != DXH_OK) return rc;
    if ((causal != 0 && causal != 1) || window < 0 || !(scale - scale == 0.f)) return DXH_ERR_ARG;
    const bool used = !kv_nothing(a.kv);
    const int es = dtype_size(dtype);
    if ((rc = kv_heads_check(q, es, used)) != DXH_OK || (rc = kv_heads_check(out, es, used)) != DXH_OK) return rc;
    if (!aligned(lse, 4)) return DXH_ERR_ALIGN;
    if (!used) return DXH_OK;
    const size_t need = part_bytes(a.kv, q_heads, a.splits);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256))) return DXH_ERR_WORKSPACE;
    a.q = (const char *)q->data; a.q_row = q->row_stride; a.q_head = q->head_stride;
    a.out = (char *)out->data; a.o_row = out->row_stride; a.o_head = out->head_stride;
    a.lse = lse;
    a.scale = scale * kLog2e;
    a.causal = causal;
    a.window = window > INT32_MAX ? 0 : (int)window;
    a.part_o = (float *)workspace;
    a.part_ml = a.part_o + (size_t)a.splits * a.kv.rows * q_heads * a.kv.dim;
    hipStream_t st = as_stream(stream);
    const bool i8 = cache->code == DXH_I8;
    switch (dtype) {
    case DXH_F32: return i8 ? launch<float, CodeI8>(a, st) : launch<float, CodeE4M3>(a, st);
    case DXH_F16: return i8 ? launch<f16_t, CodeI8>(a, st) : launch<f16_t, CodeE4M3>(a, st);
    default: return i8 ? launch<bf16_t, CodeI8>(a, st) : launch<bf16_t, CodeE4M3>(a, st);
    }
}

}  // extern "C"
