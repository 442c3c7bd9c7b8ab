// kvcache.hip — keys and values into a paged 8-bit cache, and back.
//
// One workgroup owns one page of one head, of the keys or of the values: the scale of a (page, head) comes from all new
// rows in it, and nobody else touches its codes, so a page is finished in one launch without atomics.
//   1. top = max |x| over the new rows of the page, 16-byte loads along a row;
//   2. scale = max(top / max code, 2^-100), at least the old scale if older tokens of the sequence are in the page;
//   3. codes.  Keys: a lane makes 16 codes of one token from 16 consecutive values.  Values lie with the tokens innermost:
//      a lane makes 16 tokens of one dimension, lanes along the dimensions, so that its 16 loads are each one line per
//      wave; both second readings come from L1 / L2.  Older codes are only read when the scale grew, or where they share
//      a 16-token piece with new ones.
// Bound by the bytes of the new rows; a decode step (one row a sequence) by its launch.
#include <algorithm>
#include "kvcache.hpp"

using namespace dxh;

namespace {

struct RowsArgs {
    KvArgs kv;
    char *data[2];                     // rows of keys, of values
    int64_t row_stride[2], head_stride[2];  // elements
    int slots;                         // most pages that the rows of one sequence can touch
};

__device__ __forceinline__ bool tile_of_block(const RowsArgs &a, int &which, int &head, int &slot, int &seq) {
    unsigned b = blockIdx.x;
    which = b & 1; b >>= 1;
    head = b % (unsigned)a.kv.heads; b /= (unsigned)a.kv.heads;
    slot = b % (unsigned)a.slots;
    seq = b / (unsigned)a.slots;
    return seq < a.kv.batch;
}

template <int THREADS> __device__ __forceinline__ float block_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, o));
    if constexpr (THREADS > kWave) {
        __shared__ float meet[THREADS / kWave];
        if (threadIdx.x % kWave == 0) meet[threadIdx.x / kWave] = v;
        __syncthreads();
        v = meet[0];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w) v = __builtin_fmaxf(v, meet[w]);
    }
    return v;
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
    const int64_t page = kv_page(a.kv, seq, slot);
    if (t1 <= t0 || page < 0) return;
    const T *x = (const T *)a.data[which] + (s.first + (start + t0 - s.begin)) * a.row_stride[which] + head * a.head_stride[which];
    const int64_t pitch = a.row_stride[which], at = page * a.kv.heads + head;
    float *scale_at = (which ? a.kv.v_scale : a.kv.k_scale) + at;
    uint8_t *codes = (which ? a.kv.v : a.kv.k) + at * P * D;
    const float old = t0 > 0 ? *scale_at : 0.f;

    float top = 0.f;
    const int per_row = D / V, pieces = (t1 - t0) * per_row;
#pragma unroll 4
    for (int i = threadIdx.x; i < pieces; i += THREADS) {
        const int r = i / per_row, d = (i - r * per_row) * V;
        const vec_t<T, V> q = *reinterpret_cast<const vec_t<T, V> *>(x + r * pitch + d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float y = __builtin_fabsf(load_acc(q.v[e]));
            top = y > top ? y : top;  // passes over a NaN; v_max_f32 of a signaling one is a NaN and would lose what came before
        }
    }
    top = __builtin_fminf(block_max<THREADS>(top), 3.4028234663852886e38f);
    float scale = __builtin_fmaxf(top * Code::inv_max, 0x1p-100f);
    if (t0 > 0) scale = __builtin_fmaxf(scale, old);
    const bool grew = t0 > 0 && scale > old;
    const float inv = 1.f / scale, again = old * inv;

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
                const T *src = x + (t - t0) * pitch + d;
                vec_t<T, V> r[16 / V];
#pragma unroll
                for (int q = 0; q < 16 / V; ++q) r[q] = reinterpret_cast<const vec_t<T, V> *>(src)[q];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = code_value<Code>(load_acc(r[(4 * q + e) / V].v[(4 * q + e) % V]), inv);
                    w[q] = Code::encode(y);
                }
            }
            *dst = w;
        }
    } else {
        // pieces of 16 tokens from the first that holds a new one (or an older one whose code changes) to the last
        const int c0 = grew ? 0 : t0 / 16, c1 = (t1 + 15) / 16;
        for (int i = threadIdx.x; i < (c1 - c0) * D; i += THREADS) {
            const int c = c0 + i / D, d = i % D, t = c * 16;
            u32x4 *dst = reinterpret_cast<u32x4 *>(codes + d * P + t);
            const bool all_new = t >= t0 && t + 16 <= t1;
            u32x4 w = {0u, 0u, 0u, 0u};
            // all 16 loads at once, those of tokens that are not new from the nearest new one
            T r[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int tt = t + e < t0 ? t0 : t + e >= t1 ? t1 - 1 : t + e;
                r[e] = x[(tt - t0) * pitch + d];
            }
            if (!all_new) w = *dst;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float y[4], z[4];
                if (!all_new) Code::decode(w[q], z);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int tt = t + 4 * q + e;
                    y[e] = code_value<Code>(load_acc(r[4 * q + e]), inv);
                    if (!all_new && !(tt >= t0 && tt < t1)) y[e] = grew && tt < t0 ? code_value<Code>(z[e], again) : z[e];
                }
                const uint32_t made = Code::encode(y);
                // codes that stay keep their bits (a NaN's payload, int8's -128)
                uint32_t mask = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int tt = t + 4 * q + e;
                    if (tt < t1 && (tt >= t0 || grew)) mask |= 0xffu << (8 * e);
                }
                w[q] = (w[q] & ~mask) | (made & mask);
            }
            *dst = w;
        }
    }
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
    if (which == 0) {
        for (int i = threadIdx.x + t0 * (D / 16); i < t1 * (D / 16); i += THREADS) {
            const int t = i / (D / 16), d = (i - t * (D / 16)) * 16;
            u32x4 w = {0u, 0u, 0u, 0u};
            if (page >= 0) w = *reinterpret_cast<const u32x4 *>(codes + t * D + d);
            T *dst = x + (t - t0) * pitch + d;
            float y[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) Code::decode(w[q], y + 4 * q);
            constexpr int V = kVecBytes / (int)sizeof(T);
#pragma unroll
            for (int q = 0; q < 16 / V; ++q) {
                float z[V];
                vec_t<T, V> r;
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = y[q * V + e] * scale;
                store_acc_vec<T, V>(r, z);
                reinterpret_cast<vec_t<T, V> *>(dst)[q] = r;
            }
        }
    } else {
        // as many dimensions a lane as make a dword of a row
        constexpr int N = 4 / (int)sizeof(T);
        const int c0 = t0 / 16, c1 = (t1 + 15) / 16;
        for (int i = threadIdx.x; i < (c1 - c0) * (D / N); i += THREADS) {
            const int c = c0 + i / (D / N), d = i % (D / N) * N, t = c * 16;
            float y[N][16];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                u32x4 w = {0u, 0u, 0u, 0u};
                if (page >= 0) w = *reinterpret_cast<const u32x4 *>(codes + (d + k) * P + t);
#pragma unroll
                for (int q = 0; q < 4; ++q) Code::decode(w[q], y[k] + 4 * q);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float z[N];
                vec_t<T, N> r;
#pragma unroll
                for (int k = 0; k < N; ++k) z[k] = y[k][e] * scale;
                store_acc_vec<T, N>(r, z);
                if (t + e >= t0 && t + e < t1) *reinterpret_cast<vec_t<T, N> *>(x + (t + e - t0) * pitch + d) = r;
            }
        }
    }
}

template <typename T, typename Code> int launch(const RowsArgs &a, bool write, hipStream_t st) {
    const int64_t blocks = (int64_t)2 * a.kv.heads * a.slots * a.kv.batch;
    if (blocks > INT32_MAX) return DXH_ERR_TOO_LARGE;
    // a wave is enough for the pieces of a few rows; a whole page of them goes to four
    const bool wide = std::min(a.kv.max_rows, a.kv.page_size) * a.kv.dim > 2048;
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
