// kvcache.hip — keys and values into a paged 8-bit cache, and back.
//
// One workgroup owns one page of one head, of the keys or of the values: the scale of a (page, head) comes from all new
// rows in it, and nobody else touches its codes, so a page is finished in one launch without atomics.
//   1. top = max |x| over the new rows of the page, 16-byte loads along a row, compared as the whole numbers that their bits
//      are (two at a time for 16-bit rows): an infinity or a NaN then shows as a top past the largest finite number, and only
//      such a page pays for clamps and NaN checks;
//   2. scale = max(top / max code, 2^-100), at least the old scale if older tokens of the sequence are in the page (an old scale that
//      is no finite number stays);
//   3. codes.  Keys: a lane makes 16 codes of one token.  Values lie with the tokens innermost: a lane makes 16 tokens of one
//      dimension, lanes along the dimensions, so that each of its 16 reads is one row of LDS (or one line of memory) for the
//      wave.  Older codes are only read when the scale grew, or where they share a 16-token piece with new ones.
// Reading back: keys 16 bytes of a row a lane; values turn in LDS, 32 tokens at a time, so that rows leave whole.
// Bound by the bytes of the rows: reading 16 sequences of 6k-8k tokens, 8 heads of 128, e4m3 into bf16, 134 us (5.2 TB/s); writing 32
// prompts of 333-2048 tokens, 2 heads of 64, f32 into int8, 14.8 us (3.4 TB/s).  A decode step (one row a sequence) is bound by its chain of
// loads, where the rows are, the page, its scale: 64 sequences, 8 heads of 128, 7.4 us.
#include <algorithm>
#include "kvcache.hpp"

using namespace dxh;

namespace {

struct RowsArgs {
    KvArgs kv;
    char *data[2];                     // rows of keys, of values
    int64_t row_stride[2], head_stride[2];  // elements
    int slots;                         // most pages that the rows of one sequence can touch
    int nt;                            // reading back: rows too many to be found in the last-level cache
};

__device__ __forceinline__ bool tile_of_block(const RowsArgs &a, int &which, int &head, int &slot, int &seq) {
    unsigned b = blockIdx.x;
    which = b & 1; b >>= 1;
    head = b % (unsigned)a.kv.heads; b /= (unsigned)a.kv.heads;
    slot = b % (unsigned)a.slots;
    seq = b / (unsigned)a.slots;
    return seq < a.kv.batch;
}

template <typename VT> __device__ __forceinline__ void store_row(VT *p, const VT &v, int nt) {
    if (nt) st_mode<3>(p, v); else *p = v;
}

template <int THREADS> __device__ __forceinline__ uint32_t block_max(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t u = __shfl_xor(v, o);
        v = u > v ? u : v;
    }
    if constexpr (THREADS > kWave) {
        __shared__ uint32_t meet[THREADS / kWave];
        __syncthreads();  // the last call's values have been read
        if (threadIdx.x % kWave == 0) meet[threadIdx.x / kWave] = v;
        __syncthreads();
        v = meet[0];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w) v = meet[w] > v ? meet[w] : v;
    }
    return v;
}

// max of |x| as bits, per 16-bit half for 16-bit rows
template <typename T> __device__ __forceinline__ uint32_t abs_max_bits(uint32_t m, uint32_t w) {
    if constexpr (sizeof(T) == 4) {
        w &= 0x7fffffffu;
        return w > m ? w : m;
    } else {
        typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, m), __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu)));
    }
}
// codes of four values: x * f, rounded.  FINITE: the values are no further than one rounding past the codes' range and no NaN
template <typename Code, bool FINITE> __device__ __forceinline__ uint32_t code4(const float (&x)[4], float f) {
    float y[4];
    if constexpr (!FINITE) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = code_value<Code>(x[e], f);
        return Code::encode(y);
    } else if constexpr (std::is_same_v<Code, CodeI8>) {
        // 1.5 2^23 has steps of 1: the sum rounds to nearest even and its low byte is the code
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = x[e] * f + 12582912.f;
        const uint32_t lo = __builtin_amdgcn_perm(float_to_bits(y[1]), float_to_bits(y[0]), 0x0c0c0400u), hi = __builtin_amdgcn_perm(float_to_bits(y[3]), float_to_bits(y[2]), 0x04000c0cu);
        return lo | hi;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = x[e] * f;
        return Code::encode(y);
    }
}

// The codes of tokens 0 .. t1 - 1 of a page, new from t0 on; x: the first new row
template <typename T, typename Code, int THREADS, bool FINITE>
__device__ __forceinline__ void write_codes(const T *x, int64_t pitch, uint8_t *codes, int which, int t0, int t1, int P, int D, bool grew, float inv, float again) {
    constexpr int V = kVecBytes / (int)sizeof(T);
    if (which == 0) {
        for (int i = threadIdx.x + (grew ? 0 : t0 * (D / 16)); i < t1 * (D / 16); i += THREADS) {
            const int t = i / (D / 16), d = (i - t * (D / 16)) * 16;
            u32x4 *dst = reinterpret_cast<u32x4 *>(codes + t * D + d);
            u32x4 w;
            if (t < t0) {
                w = *dst;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float y[4];
                    Code::decode(w[q], y);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = code_value<Code>(y[e], again);
                    w[q] = Code::encode(y);
                }
            } else {
                vec_t<T, V> r[16 / V];
#pragma unroll
                for (int q = 0; q < 16 / V; ++q) r[q] = *reinterpret_cast<const vec_t<T, V> *>(x + (t - t0) * pitch + d + q * V);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = load_acc(r[(4 * q + e) / V].v[(4 * q + e) % V]);
                    w[q] = code4<Code, FINITE>(y, inv);
                }
            }
            *dst = w;
        }
        return;
    }
    // pieces of 16 tokens from the first that holds a new one (or an older one whose code changes) to the last
    const int c0 = grew ? 0 : t0 / 16, c1 = (t1 + 15) / 16;
    for (int i = threadIdx.x; i < (c1 - c0) * D; i += THREADS) {
        const int c = c0 + i / D, d = i % D, t = c * 16;
        u32x4 *dst = reinterpret_cast<u32x4 *>(codes + d * P + t);
        const bool all_new = t >= t0 && t + 16 <= t1;
        u32x4 w = {0u, 0u, 0u, 0u};
        if (!all_new) w = *dst;
        // all 16 reads at once, those of tokens that are not new from the nearest new one
        T r[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) r[e] = x[((t + e < t0 ? t0 : t + e >= t1 ? t1 - 1 : t + e) - t0) * pitch + d];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = load_acc(r[4 * q + e]);
            uint32_t made = code4<Code, FINITE>(y, inv);
            if (!all_new) {
                float z[4];
                Code::decode(w[q], z);
                uint32_t stay = 0, redo = 0;  // codes that stay keep their bits (a NaN's payload, int8's -128)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int tt = t + 4 * q + e;
                    z[e] = code_value<Code>(z[e], again);
                    if (tt >= t1 || (tt < t0 && !grew)) stay |= 0xffu << (8 * e);
                    else if (tt < t0) redo |= 0xffu << (8 * e);
                }
                made = (made & ~(stay | redo)) | (w[q] & stay) | (Code::encode(z) & redo);
            }
            w[q] = made;
        }
        *dst = w;
    }
}

template <typename T, typename Code, int THREADS>
__global__ __launch_bounds__(THREADS) void kvcache_write_kernel(const RowsArgs a) {
    constexpr int V = kVecBytes / (int)sizeof(T);
    int which, head, slot, seq;
    if (!tile_of_block(a, which, head, slot, seq)) return;
    const KvSeq s = kv_seq(a.kv, seq);
    const int P = a.kv.page_size, D = a.kv.dim;
    slot += s.begin >> a.kv.page_shift;
    const int64_t start = (int64_t)slot * P;  // first token of the page; new ones are t0 .. t1 - 1 of it, older ones 0 .. t0 - 1
    const int t0 = (int)(s.begin > start ? s.begin - start : 0), t1 = (int)((int64_t)s.begin + s.n - start < P ? (int64_t)s.begin + s.n - start : P);
    if (t1 <= t0) return;
    // the table's entry comes beside the rows; only their codes need to know the page
    const int64_t entry_at = (int64_t)seq * a.kv.pages_per_seq + (slot < 0 ? 0 : slot < a.kv.pages_per_seq ? slot : a.kv.pages_per_seq - 1);
    const bool has_slot = slot >= 0 && slot < a.kv.pages_per_seq;
    const int64_t entry = !a.kv.table ? entry_at : a.kv.pages_per_seq > 0 ? (int64_t)a.kv.table[entry_at] : -1;
    const T *x = (const T *)a.data[which] + (s.first + (start + t0 - s.begin)) * a.row_stride[which] + head * a.head_stride[which];
    const int64_t pitch = a.row_stride[which];

    uint32_t bits = 0;
    const int per_row = D / V, pieces = (t1 - t0) * per_row;
#pragma unroll 4
    for (int i = threadIdx.x; i < pieces; i += THREADS) {
        const int r = i / per_row, d = (i - r * per_row) * V;
        const u32x4 q = *reinterpret_cast<const u32x4 *>(x + r * pitch + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) bits = abs_max_bits<T>(bits, q[e]);
    }
    if constexpr (sizeof(T) == 2) bits = (bits & 0xffffu) > (bits >> 16) ? bits & 0xffffu : bits >> 16;
    bits = block_max<THREADS>(bits);
    float top;
    if constexpr (sizeof(T) == 4) top = bits_to_float(bits);
    else top = load_acc(T{(uint16_t)bits});
    const bool all_finite = top - top == 0.f;
    if (!all_finite) {  // the largest that is no NaN
        float y = 0.f;
        for (int i = threadIdx.x; i < (t1 - t0) * D; i += THREADS) {
            const float v = __builtin_fabsf(load_acc(x[(i / D) * pitch + i % D]));
            y = v > y ? v : y;  // passes over a NaN; v_max_f32 of a signaling one is a NaN and would lose what came before
        }
        top = __builtin_fminf(bits_to_float(block_max<THREADS>(float_to_bits(y))), 3.4028234663852886e38f);
    }
    const int64_t page = has_slot && entry >= 0 && entry < a.kv.num_pages ? entry : -1;
    if (page < 0) return;  // the same for the whole workgroup
    const int64_t where = page * a.kv.heads + head;
    float *scale_at = (which ? a.kv.v_scale : a.kv.k_scale) + where;
    uint8_t *codes = (which ? a.kv.v : a.kv.k) + where * P * D;
    const float old = t0 > 0 ? *scale_at : 0.f;
    float scale = __builtin_fmaxf(top * Code::inv_max, 0x1p-100f);
    if (t0 > 0) scale = old - old == 0.f ? __builtin_fmaxf(scale, old) : old;  // the older tokens have no values: the page shows it
    const bool grew = t0 > 0 && scale > old;
    const float inv = 1.f / scale, again = old * inv;
    if (THREADS > kWave && t0 > 0) __syncthreads();  // every wave has the old scale
    if (all_finite) write_codes<T, Code, THREADS, true>(x, pitch, codes, which, t0, t1, P, D, grew, inv, again);
    else write_codes<T, Code, THREADS, false>(x, pitch, codes, which, t0, t1, P, D, grew, inv, again);
    if (threadIdx.x == 0) *scale_at = scale;
}

template <typename T, typename Code, int THREADS>
__global__ __launch_bounds__(THREADS) void kvcache_read_kernel(const RowsArgs a) {
    int which, head, slot, seq;
    if (!tile_of_block(a, which, head, slot, seq)) return;
    const KvSeq s = kv_seq(a.kv, seq);
    const int P = a.kv.page_size, D = a.kv.dim;
    slot += s.begin >> a.kv.page_shift;
    const int64_t start = (int64_t)slot * P;
    const int t0 = (int)(s.begin > start ? s.begin - start : 0), t1 = (int)((int64_t)s.begin + s.n - start < P ? (int64_t)s.begin + s.n - start : P);
    if (t1 <= t0) return;
    const int64_t page = kv_page(a.kv, seq, slot), pitch = a.row_stride[which];
    T *x = (T *)a.data[which] + (s.first + (start + t0 - s.begin)) * pitch + head * a.head_stride[which];
    const int64_t at = (page < 0 ? 0 : page) * a.kv.heads + head;
    const float scale = page < 0 ? 0.f : ((which ? a.kv.v_scale : a.kv.k_scale)[at]);
    const uint8_t *codes = (which ? a.kv.v : a.kv.k) + at * P * D;
    constexpr int V = kVecBytes / (int)sizeof(T);
    const int per_row = D / V;
    if (which == 0) {
        for (int i = threadIdx.x + t0 * per_row; i < t1 * per_row; i += THREADS) {  // V codes into 16 bytes of a row
            const int t = i / per_row, d = (i - t * per_row) * V;
            float y[V];
#pragma unroll
            for (int q = 0; q < V / 4; ++q) Code::decode(page >= 0 ? *reinterpret_cast<const uint32_t *>(codes + t * D + d + 4 * q) : 0u, y + 4 * q);
            vec_t<T, V> r;
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] *= scale;
            store_acc_vec<T, V>(r, y);
            store_row(reinterpret_cast<vec_t<T, V> *>(x + (t - t0) * pitch + d), r, a.nt);
        }
        return;
    }
    // 32 tokens at a time; a row of LDS is padded by a dword so that a lane's 16 stores down a column meet other banks than its neighbours' rows
    constexpr int PITCH = 256 + 4 / (int)sizeof(T);
    __shared__ __attribute__((aligned(16))) T turn[32 * PITCH];
    for (int t = t0 & ~31; t < t1; t += 32) {
        const int tokens = P - t < 32 ? 16 : 32;  // a page of 16 has no second piece
        for (int i = threadIdx.x; i < (tokens / 16) * D; i += THREADS) {
            const int d = tokens == 32 ? i >> 1 : i, c = tokens == 32 ? (i & 1) * 16 : 0;
            u32x4 w = {0u, 0u, 0u, 0u};
            if (page >= 0) w = *reinterpret_cast<const u32x4 *>(codes + d * P + t + c);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float y[4];
                Code::decode(w[q], y);
#pragma unroll
                for (int e = 0; e < 4; ++e) turn[(c + 4 * q + e) * PITCH + d] = store_acc<T>(y[e] * scale);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tokens * per_row; i += THREADS) {
            const int r = i / per_row, d = (i - r * per_row) * V, tt = t + r;
            vec_t<T, V> q;
#pragma unroll
            for (int e = 0; e < V; e += 4 / (int)sizeof(T))
                *reinterpret_cast<uint32_t *>(&q.v[e]) = *reinterpret_cast<const uint32_t *>(&turn[r * PITCH + d + e]);
            if (tt >= t0 && tt < t1) store_row(reinterpret_cast<vec_t<T, V> *>(x + (tt - t0) * pitch + d), q, a.nt);
        }
        __syncthreads();
    }
}

template <typename T, typename Code> int launch(const RowsArgs &a, bool write, hipStream_t st) {
    const int64_t blocks = product(2, a.kv.heads, a.slots, a.kv.batch);
    // a lane for every 16 codes of a page, as one new row can change the scale of all: one wave or four
    const bool wide = a.kv.page_size * a.kv.dim > 16 * kWave;
    if (!launch_fits(blocks, wide ? 256 : 64)) return DXH_ERR_TOO_LARGE;
    if (kv_meets(a.kv, a.data[0]) || kv_meets(a.kv, a.data[1])) return DXH_ERR_ARG;
    if (write) {
        if (wide) kvcache_write_kernel<T, Code, 256><<<(unsigned)blocks, 256, 0, st>>>(a);
        else kvcache_write_kernel<T, Code, 64><<<(unsigned)blocks, 64, 0, st>>>(a);
    } else {
        if (wide) kvcache_read_kernel<T, Code, 256><<<(unsigned)blocks, 256, 0, st>>>(a);
        else kvcache_read_kernel<T, Code, 64><<<(unsigned)blocks, 64, 0, st>>>(a);
    }
    return launch_status();
}

int rows_call(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, const dxh_heads *k, const dxh_heads *v, bool write, void *stream) {
    RowsArgs a{};
    int rc = kv_check(cache, rows, dtype, a.kv);
    if (rc != DXH_OK) return rc;
    const bool used = !kv_nothing(a.kv);
    for (int i = 0; i < 2; ++i) {
        const dxh_heads *h = i ? v : k;
        rc = kv_heads_check(h, dtype_size(dtype), used);
        if (rc != DXH_OK) return rc;
        a.data[i] = (char *)h->data;
        a.row_stride[i] = h->row_stride;
        a.head_stride[i] = h->head_stride;
    }
    if (!used) return DXH_OK;
    if (!write && a.data[0] == a.data[1]) return DXH_ERR_ARG;  // two results in one place
    // n rows that start anywhere in a page touch at most this many
    a.slots = (int)(((int64_t)a.kv.max_rows + a.kv.page_size - 2) / a.kv.page_size) + 1;
    a.nt = use_nt_store((size_t)product(2 * a.kv.rows, a.kv.heads, a.kv.dim * dtype_size(dtype)));
    hipStream_t st = as_stream(stream);
    const bool i8 = cache->code == DXH_I8;
    switch (dtype) {
    case DXH_F32: return i8 ? launch<float, CodeI8>(a, write, st) : launch<float, CodeE4M3>(a, write, st);
    case DXH_F16: return i8 ? launch<f16_t, CodeI8>(a, write, st) : launch<f16_t, CodeE4M3>(a, write, st);
    default: return i8 ? launch<bf16_t, CodeI8>(a, write, st) : launch<bf16_t, CodeE4M3>(a, write, st);
    }
}

}  // namespace

extern "C" {

int dxh_kvcache_write(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, const dxh_heads *k, const dxh_heads *v, void *stream) {
    return rows_call(cache, rows, dtype, k, v, true, stream);
}
int dxh_kvcache_read(const dxh_kvcache *cache, const dxh_kvrows *rows, int dtype, const dxh_heads *k, const dxh_heads *v, void *stream) {
    return rows_call(cache, rows, dtype, k, v, false, stream);
}

}  // extern "C"
