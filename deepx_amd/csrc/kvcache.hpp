// kvcache.hpp — what the kernels over a paged 8-bit cache share: which rows and tokens a sequence has, the codes.
//
// A cache holds value = code * scale, one scale for each page (page_size tokens of one sequence) and head; keys lie
// [page][head][token][dim], values [page][head][dim][token].  Everything read from the device arrays (offsets, lengths,
// page numbers) is clamped before it becomes an address.
#pragma once
#include "matmul_common.hpp"

namespace dxh {

struct KvArgs {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    const int32_t *table, *offsets, *lengths;
    int64_t num_pages, rows;
    int pages_per_seq, page_size, page_shift, heads, dim, batch, max_rows;
};

// The rows of sequence b: `n` of them (at most max_rows) from packed row `first` on, row i being the token at `begin` + i;
// `begin` is negative where a sequence has more rows than tokens.  `length`: the tokens that can be in the cache.
struct KvSeq { int64_t first; int n, begin, length; };
__device__ __forceinline__ KvSeq kv_seq(const KvArgs &a, int b) {
    KvSeq s;
    int64_t o0, o1;
    if (a.offsets) {
        o0 = a.offsets[b];
        o1 = a.offsets[b + 1];
        o0 = o0 < 0 ? 0 : o0 > a.rows ? a.rows : o0;
        o1 = o1 < o0 ? o0 : o1 > a.rows ? a.rows : o1;
    } else {
        o0 = (int64_t)b * a.max_rows;
        o1 = o0 + a.max_rows;  // the host has checked that batch * max_rows rows exist
    }
    const int64_t cap = (int64_t)a.pages_per_seq * a.page_size;
    const int len = a.lengths[b] < 0 ? 0 : a.lengths[b], all = (int)(o1 - o0);
    s.first = o0;
    s.n = all < a.max_rows ? all : a.max_rows;
    s.begin = len - all;
    s.length = len < cap ? len : (int)cap;
    return s;
}
// the page that holds tokens slot * page_size ... of sequence b, -1 if there is none
__device__ __forceinline__ int64_t kv_page(const KvArgs &a, int b, int slot) {
    if (slot < 0 || slot >= a.pages_per_seq) return -1;
    const int64_t at = (int64_t)b * a.pages_per_seq + slot, p = a.table ? (int64_t)a.table[at] : at;
    return p >= 0 && p < a.num_pages ? p : -1;
}

// ---- codes -------------------------------------------------------------------------------------------------------
struct CodeI8 {
    static constexpr float max = 127.f, inv_max = 1.f / 127.f;
    // four codes of a dword as fp32
    static __device__ __forceinline__ void decode(uint32_t w, float *x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)(w >> (8 * e));
    }
    static __device__ __forceinline__ uint32_t encode(const float *x) {  // values within +-max or NaN
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= ((uint32_t)(int)(x[e] == x[e] ? __builtin_rintf(x[e]) : 0.f) & 0xffu) << (8 * e);
        return w;
    }
};
struct CodeE4M3 {
    static constexpr float max = 448.f, inv_max = 1.f / 448.f;
    static __device__ __forceinline__ void decode(uint32_t w, float *x) {
        const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
    }
    static __device__ __forceinline__ uint32_t encode(const float *x) {
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false), true);
    }
};
// x * f into the codes' range, NaN kept
template <typename Code> __device__ __forceinline__ float code_value(float x, float f) {
    const float y = x * f;
    return y != y ? y : __builtin_fminf(__builtin_fmaxf(y, -Code::max), Code::max);
}

// ---- host checks ----------------------------------------------------------------------------------------------------
// Fills `a`; DXH_OK also when there is nothing to do (no batch or no rows).
inline int kv_check(const dxh_kvcache *c, const dxh_kvrows *r, int dtype, KvArgs &a) {
    if (!c || !r) return DXH_ERR_ARG;
    if (dtype != DXH_F32 && dtype != DXH_F16 && dtype != DXH_BF16) return DXH_ERR_DTYPE;
    if (c->code != DXH_I8 && c->code != DXH_F8E4M3) return DXH_ERR_DTYPE;
    if (c->num_pages < 0 || c->pages_per_seq < 0 || c->heads < 1 || r->batch < 0 || r->rows < 0 || r->max_rows < 0) return DXH_ERR_ARG;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return DXH_ERR_SHAPE;
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) return DXH_ERR_SHAPE;
    if (!c->page_table && c->num_pages < (int64_t)r->batch * c->pages_per_seq) return DXH_ERR_SHAPE;
    if (!r->offsets && r->rows < (int64_t)r->batch * r->max_rows) return DXH_ERR_SHAPE;
    // tokens are counted in 32 bits, a few tiles past the last one included
    if (r->rows > INT32_MAX || c->num_pages > INT32_MAX || (int64_t)c->pages_per_seq * c->page_size > ((int64_t)1 << 30)) return DXH_ERR_TOO_LARGE;
    if (!aligned(c->k, kVecBytes) || !aligned(c->v, kVecBytes) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->page_table, 4) ||
        !aligned(r->offsets, 4) || !aligned(r->lengths, 4)) return DXH_ERR_ALIGN;
    a = KvArgs{};
    a.k = (uint8_t *)c->k; a.v = (uint8_t *)c->v; a.k_scale = c->k_scale; a.v_scale = c->v_scale;
    a.table = c->page_table; a.offsets = r->offsets; a.lengths = r->lengths;
    a.num_pages = c->num_pages; a.rows = r->rows;
    a.pages_per_seq = c->pages_per_seq; a.page_size = c->page_size; a.heads = c->heads; a.dim = c->dim;
    a.page_shift = __builtin_ctz((unsigned)c->page_size);
    a.batch = r->batch; a.max_rows = r->max_rows;
    if (a.num_pages == 0) a.pages_per_seq = 0;  // no token has a place
    if (r->batch == 0 || r->rows == 0 || r->max_rows == 0) return DXH_OK;
    if (!r->lengths) return DXH_ERR_ARG;
    if (c->num_pages > 0 && c->pages_per_seq > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale || c->k == c->v || c->k_scale == c->v_scale)) return DXH_ERR_ARG;
    return DXH_OK;
}
// The product of counts that are each at most 2^63 - 1, or 2^63 - 1 if that is less
inline int64_t product(int64_t a) { return a; }
template <typename... More> int64_t product(int64_t a, int64_t b, More... more) {
    int64_t p;
    return product(__builtin_mul_overflow(a, b, &p) ? (a && b ? INT64_MAX : 0) : p, more...);
}
// a launch has fewer than 2^32 work items
inline bool launch_fits(int64_t blocks, int threads) { return blocks <= (int64_t)UINT32_MAX / threads; }
// does what a call writes, or writes into the cache, begin where something else that it reads or writes does
inline bool kv_meets(const KvArgs &a, const void *p) {
    return p && (p == a.k || p == a.v || p == a.k_scale || p == a.v_scale || p == a.table || p == a.offsets || p == a.lengths);
}
inline bool kv_nothing(const KvArgs &a) { return a.batch == 0 || a.rows == 0 || a.max_rows == 0; }
inline int kv_heads_check(const dxh_heads *h, int es, bool used) {
    if (!h || (used && !h->data)) return DXH_ERR_ARG;
    return aligned(h->data, kVecBytes) && (h->row_stride * es) % kVecBytes == 0 && (h->head_stride * es) % kVecBytes == 0 ? DXH_OK : DXH_ERR_ALIGN;
}

}  // namespace dxh
