// normrope.hip — RMS norm of each query / key head and its position rotation in one pass, and its gradients.
//
// One head of one row is D values x.  With the norm on, n_i = w_i x_i r, r = 1 / sqrt(mean(x^2) + eps); off, n = x.
// The first R values are rotated in pairs (a, b) = (i, i + R/2), or (2i, 2i + 1), by the angle whose cosine c_i and
// sine s_i the caller's tables hold for the row's position:
//     y_a = n_a c - n_b s,  y_b = n_b c + n_a s;      the others pass: y = n.
// The gradient goes back through the transposed rotation, g = R^T dy, and with h = w g:
//     dx = r h - x r^3 mean(h x),      dw = sum over rows and heads of g x r        (norm off: dx = g, no dw).
//
// Everything between the load and the store is fp32; a result is rounded once.  The kernels are bound by memory: a head
// is read once and written once, so a lane keeps a 16-byte piece of a head in registers and a power-of-two group of
// lanes (`lg`) holds the head: sums are cross-lane adds inside the group, and the other value of a pair is in the same lane
// (neighbouring pairs) or comes from lane +- R/2/V.  A lane group keeps its row while it walks over that row's heads, so the
// cosines and sines are loaded once per row and group, not once per head.  Measured: 16384 rows of 32 + 8 heads of 128 in bf16
// 62.9 us (5.5 TB/s); backward of 8192 such rows 49.5 us (5.2 TB/s).  Several heads' loads at once cost more in occupancy than
// they hide (two: 64.9, four: 87 us).
#include <algorithm>
#include "matmul_common.hpp"

using namespace dxh;

namespace {

constexpr int kMaxParts = DXH_NORMROPE_MAX_PARTS;

struct Part {
    const void *x, *y_in, *w;  // y_in: the gradient that comes in
    void *out;
    float *dw;
    int64_t x_row, x_head, y_row, y_head, o_row, o_head;
    int heads, norm, w_f32, groups;  // groups: lane groups that share one row of this part (a power of two)
};
struct Args {
    Part part[kMaxParts];
    const float *cos, *sin;
    const void *positions;
    int64_t rows, table_rows;
    int dim, rd, pos_i64, nt;  // nt: the results are too many bytes to be found in the last-level cache by whoever reads them
    float eps;
    float *partial;  // backward: [part][workgroup][dim]
};

// V consecutive values of a head as fp32
template <typename T> constexpr int kV = kVecBytes / (int)sizeof(T);
template <typename T> using Piece = vec_t<T, kV<T>>;
// A launch that stores more than the last-level cache is good for (use_nt_store) reads and writes past it: 16384 rows of 40
// heads of 128 in bf16, plain 71.5 us; stores nt 71.5; loads nt too 63.3; stores nt at agent scope 62.9.
template <typename T> __device__ __forceinline__ Piece<T> load_piece(const T *p, bool live, int nt) {
    Piece<T> r = {};
    if (live) r = nt ? ld_nt(reinterpret_cast<const Piece<T> *>(p)) : *reinterpret_cast<const Piece<T> *>(p);
    return r;
}
template <typename T> __device__ __forceinline__ void unpack(const Piece<T> &r, float (&x)[kV<T>]) {
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) x[e] = load_acc(r.v[e]);
}
template <typename T> __device__ __forceinline__ void load_vec(const T *p, float (&x)[kV<T>]) { unpack<T>(*reinterpret_cast<const Piece<T> *>(p), x); }
template <typename T> __device__ __forceinline__ void store_vec(T *p, const float (&x)[kV<T>], int nt) {
    Piece<T> r;
    store_acc_vec<T, kV<T>>(r, x);
    if (nt) st_mode<3>(reinterpret_cast<Piece<T> *>(p), r);
    else *reinterpret_cast<Piece<T> *>(p) = r;
}
template <typename T> __device__ __forceinline__ void load_weight(const Part &p, int d, float (&w)[kV<T>]) {
#pragma unroll
    for (int e = 0; e < kV<T>; ++e) w[e] = 1.f;
    if (!p.w) return;
    if (p.w_f32) {
        const float *f = (const float *)p.w + d;
#pragma unroll
        for (int e = 0; e < kV<T>; ++e) w[e] = f[e];
    } else {
        load_vec<T>((const T *)p.w + d, w);
    }
}
// A value of another lane by the vector pipe's own cross-lane paths: no LDS access, which the shuffles of a head (a sum and one
// value an element) would otherwise need about 12 of for 16 bytes.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return bits_to_float((uint32_t)__builtin_amdgcn_mov_dpp((int)float_to_bits(v), CTRL, 0xf, 0xf, true));
}
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kQuadReverse = 0x1b, kRowRor8 = 0x128, kRowMirror = 0x140, kHalfMirror = 0x141;
// The sum over a group of LG lanes, in every lane.  Lanes of a quad, then of eight, then of sixteen agree after a step, so that
// a mirror reaches the other half as well as an exclusive or would.
template <int LG> __device__ __forceinline__ float group_sum(float v) {
    v += dpp<kQuadXor1>(v);
    v += dpp<kQuadXor2>(v);
    if constexpr (LG >= 8) v += dpp<kHalfMirror>(v);
    if constexpr (LG >= 16) v += dpp<kRowMirror>(v);
    if constexpr (LG >= 32) v += __shfl_xor(v, 16);
    if constexpr (LG >= 64) v += __shfl_xor(v, 32);
    return v;
}
// 1 / sqrt(v).  The hardware's takes a subnormal v (eps 0 over values below 2^-63) for zero: it gets 2^64 v.
__device__ __forceinline__ float inv_sqrt(float v) {
    const bool small = v < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v);
    return small ? r * 0x1p32f : r;
}
// the value of lane ^ LG/2
template <int LG> __device__ __forceinline__ float other_half(float v) {
    if constexpr (LG == 4) return dpp<kQuadXor2>(v);
    else if constexpr (LG == 8) return dpp<kQuadReverse>(dpp<kHalfMirror>(v));
    else if constexpr (LG == 16) return dpp<kRowRor8>(v);
    else return __shfl_xor(v, LG / 2);
}

// How the values of a pair meet: kNear pairs (2i, 2i + 1) share a lane; kFar pairs (i, i + R/2) with R/2 a multiple of V
// are the same element of the lane R/2/V further, kHalf those of a head that is rotated whole and fills its lanes (the other
// lane is lane ^ LG/2); kAny is kFar with any even R: element by element through shuffles.
enum { kNear = 0, kFar = 1, kAny = 2, kHalf = 3 };

// cosine and sine of every element of this lane's piece and the sign its partner's product gets; elements past R: c = 1, s = 0
template <typename T, int MODE>
__device__ __forceinline__ void load_angles(const Args &a, int64_t row, int d, bool live, float (&c)[kV<T>], float (&s)[kV<T>]) {
    constexpr int V = kV<T>;
#pragma unroll
    for (int e = 0; e < V; ++e) { c[e] = 1.f; s[e] = 0.f; }
    if (a.rd == 0 || !live || d >= a.rd) return;
    int64_t p = row;
    if (a.positions) p = a.pos_i64 ? ((const int64_t *)a.positions)[row] : (int64_t)((const int32_t *)a.positions)[row];
    p = p < 0 ? 0 : p >= a.table_rows ? a.table_rows - 1 : p;
    const int half = a.rd / 2;
    const float *ct = a.cos + p * half, *st = a.sin + p * half;
    if constexpr (MODE == kFar || MODE == kHalf) {  // whole 16-byte pieces of the table
        const bool hi = d >= half;
        const int i = hi ? d - half : d;
#pragma unroll
        for (int e = 0; e < V; ++e) { c[e] = ct[i + e]; s[e] = hi ? st[i + e] : -st[i + e]; }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int j = d + e;
            if (j >= a.rd) continue;
            const bool hi = MODE == kNear ? (j & 1) : j >= half;
            const int i = MODE == kNear ? j >> 1 : hi ? j - half : j;
            c[e] = ct[i];
            s[e] = hi ? st[i] : -st[i];
        }
    }
}
// n rotated (or, with `back`, rotated back): y_e = n_e c_e + n_partner s_e below R, n_e past it (not n_e * 1 + 0 * partner:
// an infinity there stays one)
template <typename T, int MODE, int LG>
__device__ __forceinline__ void rotate(const Args &a, int d, const float (&n)[kV<T>], const float (&c)[kV<T>], const float (&s)[kV<T>], bool back, float (&y)[kV<T>]) {
    constexpr int V = kV<T>;
    const float sign = back ? -1.f : 1.f;
    const int half = a.rd / 2;
    if constexpr (MODE == kNear) {
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = d + e < a.rd ? __builtin_fmaf(n[e], c[e], sign * (n[e ^ 1] * s[e])) : n[e];
    } else if constexpr (MODE == kHalf) {
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = __builtin_fmaf(n[e], c[e], sign * (other_half<LG>(n[e]) * s[e]));
    } else if constexpr (MODE == kFar) {
        const int shift = half / V, me = d / V, from = d >= a.rd ? me : d >= half ? me - shift : me + shift;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float other = __shfl(n[e], from, LG);
            y[e] = d < a.rd ? __builtin_fmaf(n[e], c[e], sign * (other * s[e])) : n[e];
        }
    } else {
        float other[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int j = d + e, from = j >= a.rd ? j : j >= half ? j - half : j + half;
            // the partner is element from % V of lane from / V: one shuffle for each element it can be
            other[e] = 0.f;
#pragma unroll
            for (int q = 0; q < V; ++q) {
                const float v = __shfl(n[q], from / V, LG);
                if (from % V == q) other[e] = v;
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = d + e < a.rd ? __builtin_fmaf(n[e], c[e], sign * (other[e] * s[e])) : n[e];
    }
}

// grid: (workgroups along the rows, parts)
template <typename T, int LG, int MODE>
__global__ __launch_bounds__(kBlock) void normrope_kernel(const Args a) {
    constexpr int V = kV<T>, kGroups = kBlock / LG;
    const Part &p = a.part[blockIdx.y];
    const int group = (int)threadIdx.x / LG, d = ((int)threadIdx.x % LG) * V;
    const int sub = group % p.groups, slot = group / p.groups, slots = kGroups / p.groups;
    const bool live = d < a.dim;  // lanes past the end of the head keep zeros and take part in the shuffles
    float w[V];
    load_weight<T>(p, live ? d : 0, w);
    const float inv_dim = 1.f / (float)a.dim;
    for (int64_t row0 = (int64_t)blockIdx.x * slots; row0 < a.rows; row0 += (int64_t)gridDim.x * slots) {
        const int64_t row = row0 + slot;
        if (row >= a.rows) continue;  // whole lane groups leave together
        float c[V], s[V];
        load_angles<T, MODE>(a, row, d, live, c, s);
        for (int h = sub; h < p.heads; h += p.groups) {
            float x[V], y[V];
            unpack<T>(load_piece<T>((const T *)p.x + row * p.x_row + h * p.x_head + d, live, a.nt), x);
            if (p.norm) {
                float sq = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) sq = __builtin_fmaf(x[e], x[e], sq);
                const float r = inv_sqrt(__builtin_fmaf(group_sum<LG>(sq), inv_dim, a.eps));
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] *= r * w[e];
            }
            rotate<T, MODE, LG>(a, d, x, c, s, false, y);
            if (live) store_vec<T>((T *)p.out + row * p.o_row + h * p.o_head + d, y, a.nt);
        }
    }
}

// The same walk for the gradients.  A lane sums g x r of its piece over all rows and heads it meets; the lane groups of
// the workgroup meet in LDS and the sum goes to partial[part][workgroup][dim], which sum_partials_kernel adds in
// workgroup order: the same bits on every run, no atomics.
template <typename T, int LG, int MODE>
__global__ __launch_bounds__(kBlock) void normrope_backward_kernel(const Args a) {
    constexpr int V = kV<T>, kGroups = kBlock / LG;
    __shared__ float meet[kBlock * V];
    const Part &p = a.part[blockIdx.y];
    const int group = (int)threadIdx.x / LG, d = ((int)threadIdx.x % LG) * V;
    const int sub = group % p.groups, slot = group / p.groups, slots = kGroups / p.groups;
    const bool live = d < a.dim;
    float w[V], dw[V];
    load_weight<T>(p, live ? d : 0, w);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = 0.f;
    const float inv_dim = 1.f / (float)a.dim;
    for (int64_t row0 = (int64_t)blockIdx.x * slots; row0 < a.rows; row0 += (int64_t)gridDim.x * slots) {
        const int64_t row = row0 + slot;
        if (row >= a.rows) continue;
        float c[V], s[V];
        load_angles<T, MODE>(a, row, d, live, c, s);
        for (int h = sub; h < p.heads; h += p.groups) {
            float x[V], dy[V], g[V];
            unpack<T>(load_piece<T>((const T *)p.y_in + row * p.y_row + h * p.y_head + d, live, a.nt), dy);
            unpack<T>(load_piece<T>((const T *)p.x + row * p.x_row + h * p.x_head + d, live && p.norm, a.nt), x);
            rotate<T, MODE, LG>(a, d, dy, c, s, true, g);
            if (p.norm) {
                float sq = 0.f, hx = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sq = __builtin_fmaf(x[e], x[e], sq);
                    hx = __builtin_fmaf(g[e] * w[e], x[e], hx);
                }
                const float r = inv_sqrt(__builtin_fmaf(group_sum<LG>(sq), inv_dim, a.eps));
                const float q = group_sum<LG>(hx) * inv_dim * r * r;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    dw[e] = __builtin_fmaf(g[e], x[e] * r, dw[e]);
                    g[e] = r * __builtin_fmaf(-x[e], q, g[e] * w[e]);
                }
            }
            if (live) store_vec<T>((T *)p.out + row * p.o_row + h * p.o_head + d, g, a.nt);
        }
    }
    if (!p.dw) return;  // the same for the whole workgroup
#pragma unroll
    for (int e = 0; e < V; ++e) meet[(group * LG * V) + d + e] = dw[e];
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kBlock) {
        float t = 0.f;
        for (int g = 0; g < kGroups; ++g) t += meet[g * LG * V + i];
        a.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.dim + i] = t;
    }
}

// dw[i] = sum over n workgroups of partial[i]: 16 columns a workgroup, 64 lanes a column, each every 64th workgroup
constexpr int kSumLanes = 64;
__global__ __launch_bounds__(16 * kSumLanes) void sum_partials_kernel(const Args a, int n) {
    __shared__ float meet[16 * kSumLanes];
    const Part &p = a.part[blockIdx.y];
    if (!p.dw) return;
    const int col = blockIdx.x * 16 + threadIdx.x % 16, lane = threadIdx.x / 16;
    const float *src = a.partial + (int64_t)blockIdx.y * n * a.dim + col;
    float t = 0.f;
#pragma unroll 8
    for (int i = lane; i < n; i += kSumLanes) t += src[(int64_t)i * a.dim];  // dim is a multiple of 16: every column exists
    meet[threadIdx.x] = t;
    __syncthreads();
#pragma unroll
    for (int half = kSumLanes / 2; half > 0; half /= 2) {
        if (lane < half) meet[threadIdx.x] += meet[threadIdx.x + half * 16];
        __syncthreads();
    }
    if (lane == 0) p.dw[col] = meet[threadIdx.x];
}

// most workgroups along the rows, which bounds the workspace: 8192 rows of 40 heads of 128 in bf16 take 59.1 us at 512, 49.5 at 1024, 51.1 at 2048
constexpr int kBackwardMaxGroups = 1024;

bool heads_aligned(const dxh_heads &h, int es) {
    return aligned(h.data, kVecBytes) && (h.row_stride * es) % kVecBytes == 0 && (h.head_stride * es) % kVecBytes == 0;
}

// Every check of the two entry points; fills `a`.  DXH_OK with a.rows == 0: nothing to do.
int check(int dtype, const dxh_normrope_part *parts, int nparts, int64_t rows, int32_t dim, float eps, const dxh_rotary *rot, bool back, Args &a) {
    if (dtype != DXH_F32 && dtype != DXH_F16 && dtype != DXH_BF16) return DXH_ERR_DTYPE;
    if (!parts || nparts < 1 || nparts > kMaxParts || rows < 0 || !(eps >= 0.f)) return DXH_ERR_ARG;
    if (dim < 16 || dim > 256 || dim % 16) return DXH_ERR_SHAPE;
    a = Args{};
    a.rows = rows;
    a.dim = dim;
    a.eps = eps;
    if (rot && rot->dim != 0) {
        if (rot->dim < 0 || rot->dim > dim || rot->dim % 2) return DXH_ERR_SHAPE;
        if (rot->interleaved != 0 && rot->interleaved != 1) return DXH_ERR_ARG;
        if (rot->position_dtype != DXH_I32 && rot->position_dtype != DXH_I64) return DXH_ERR_DTYPE;
        if (rows > 0 && (!rot->cos || !rot->sin || rot->table_rows < 1)) return DXH_ERR_ARG;
        if (!aligned(rot->cos, 4) || !aligned(rot->sin, 4) || !aligned(rot->positions, dtype_size(rot->position_dtype))) return DXH_ERR_ALIGN;
        a.cos = rot->cos;
        a.sin = rot->sin;
        a.positions = rot->positions;
        a.table_rows = rot->table_rows;
        a.rd = rot->dim;
        a.pos_i64 = rot->position_dtype == DXH_I64;
    }
    const int es = dtype_size(dtype), v = kVecBytes / es;
    int lg = 4;
    while (lg * v < dim) lg *= 2;
    int64_t heads = 0;
    for (int i = 0; i < nparts; ++i) {
        const dxh_normrope_part &s = parts[i];
        Part &p = a.part[i];
        heads += s.heads > 0 ? s.heads : 0;
        if (s.heads < 0 || (s.norm != 0 && s.norm != 1)) return DXH_ERR_ARG;
        if (s.weight && s.weight_dtype != dtype && s.weight_dtype != DXH_F32) return DXH_ERR_DTYPE;
        const dxh_heads &out = back ? s.dx : s.y;
        if (rows > 0 && s.heads > 0) {
            if (!s.x.data || !s.y.data || !out.data) return DXH_ERR_ARG;
            if (!heads_aligned(s.x, es) || !heads_aligned(s.y, es) || !heads_aligned(out, es)) return DXH_ERR_ALIGN;
        }
        if (!aligned(s.weight, kVecBytes) || !aligned(s.dweight, 4)) return DXH_ERR_ALIGN;
        p.x = s.x.data; p.x_row = s.x.row_stride; p.x_head = s.x.head_stride;
        p.y_in = s.y.data; p.y_row = s.y.row_stride; p.y_head = s.y.head_stride;
        p.out = out.data; p.o_row = out.row_stride; p.o_head = out.head_stride;
        p.w = s.norm ? s.weight : nullptr;
        p.w_f32 = s.weight_dtype == DXH_F32;
        p.dw = back && s.norm ? s.dweight : nullptr;
        p.heads = s.heads;
        p.norm = s.norm;
        // one lane group per head while the rows alone do not fill the card, else about four heads a group
        const int most = kBlock / lg;
        int g = 1;
        while (g < most && g * (rows < 4 * kCUs ? 1 : 4) < s.heads) g *= 2;
        p.groups = g;
    }
    // a result may lie where its own inputs do, element on element, and nowhere else among what the launch touches
    auto shifted = [&](const Part &p, const void *in, int64_t row, int64_t head) { return p.out == in && ((rows > 1 && p.o_row != row) || (p.heads > 1 && p.o_head != head)); };
    for (int i = 0; i < nparts; ++i) {
        const Part &p = a.part[i];
        if (rows > 0 && p.heads && (shifted(p, p.x, p.x_row, p.x_head) || (back && shifted(p, p.y_in, p.y_row, p.y_head)))) return DXH_ERR_ARG;
    }
    for (int i = 0; i < nparts; ++i)
        for (int j = 0; j < nparts; ++j) {
            const Part &p = a.part[i], &q = a.part[j];
            if (rows == 0 || !p.heads) continue;
            if ((q.w && p.out == q.w) || (a.rd && (p.out == a.cos || p.out == a.sin || (a.positions && p.out == a.positions)))) return DXH_ERR_ARG;
            if (q.dw && p.out == q.dw) return DXH_ERR_ARG;
            if (i == j || !q.heads) continue;
            if (p.out == q.out || p.out == q.x || (back && p.out == q.y_in)) return DXH_ERR_ARG;
            if (p.dw && p.dw == q.dw) return DXH_ERR_ARG;
        }
    a.nt = use_nt_store((size_t)rows * heads * dim * es);
    return DXH_OK;
}
int slots_of(const Args &a, int nparts, int lg) {  // fewest rows that a workgroup of any part takes at once
    int s = kBlock / lg;
    for (int i = 0; i < nparts; ++i) s = std::min(s, kBlock / lg / a.part[i].groups);
    return s;
}
int backward_groups(const Args &a, int nparts, int lg) {
    const int64_t s = slots_of(a, nparts, lg);
    return (int)std::min<int64_t>(kBackwardMaxGroups, std::max<int64_t>(1, (a.rows + s - 1) / s));
}
int lanes_of(int dtype, int dim) {
    const int v = kVecBytes / dtype_size(dtype);
    int lg = 4;
    while (lg * v < dim) lg *= 2;
    return lg;
}

template <typename T, int LG> int launch(const Args &a, int nparts, const dxh_rotary *rot, bool back, unsigned groups, hipStream_t st) {
    const dim3 grid(groups, nparts);
    const bool near = a.rd == 0 || (rot && rot->interleaved), far = !near && (a.rd / 2) % kV<T> == 0, half = far && a.rd == a.dim && a.dim == LG * kV<T>;
    if (back) {
        if (near) normrope_backward_kernel<T, LG, kNear><<<grid, kBlock, 0, st>>>(a);
        else if (half) normrope_backward_kernel<T, LG, kHalf><<<grid, kBlock, 0, st>>>(a);
        else if (far) normrope_backward_kernel<T, LG, kFar><<<grid, kBlock, 0, st>>>(a);
        else normrope_backward_kernel<T, LG, kAny><<<grid, kBlock, 0, st>>>(a);
    } else {
        if (near) normrope_kernel<T, LG, kNear><<<grid, kBlock, 0, st>>>(a);
        else if (half) normrope_kernel<T, LG, kHalf><<<grid, kBlock, 0, st>>>(a);
        else if (far) normrope_kernel<T, LG, kFar><<<grid, kBlock, 0, st>>>(a);
        else normrope_kernel<T, LG, kAny><<<grid, kBlock, 0, st>>>(a);
    }
    return launch_status();
}
template <typename T> int launch_lanes(const Args &a, int nparts, const dxh_rotary *rot, bool back, int lg, unsigned groups, hipStream_t st) {
    switch (lg) {
    case 4: return launch<T, 4>(a, nparts, rot, back, groups, st);
    case 8: return launch<T, 8>(a, nparts, rot, back, groups, st);
    case 16: return launch<T, 16>(a, nparts, rot, back, groups, st);
    case 32: return launch<T, 32>(a, nparts, rot, back, groups, st);
    default: return launch<T, 64>(a, nparts, rot, back, groups, st);
    }
}
int launch_dtype(int dtype, const Args &a, int nparts, const dxh_rotary *rot, bool back, int lg, unsigned groups, hipStream_t st) {
    switch (dtype) {
    case DXH_F32: return launch_lanes<float>(a, nparts, rot, back, lg, groups, st);
    case DXH_F16: return launch_lanes<f16_t>(a, nparts, rot, back, lg, groups, st);
    default: return launch_lanes<bf16_t>(a, nparts, rot, back, lg, groups, st);
    }
}

}  // namespace

extern "C" {

int dxh_normrope(int dtype, const dxh_normrope_part *parts, int nparts, int64_t rows, int32_t dim, float eps, const dxh_rotary *rot, void *stream) {
    Args a;
    const int rc = check(dtype, parts, nparts, rows, dim, eps, rot, false, a);
    if (rc != DXH_OK || rows == 0) return rc;
    const int lg = lanes_of(dtype, dim);
    const int64_t s = slots_of(a, nparts, lg), groups = (rows + s - 1) / s;
    return launch_dtype(dtype, a, nparts, rot, false, lg, (unsigned)std::min<int64_t>(groups, (int64_t)1 << 22), as_stream(stream));
}

int dxh_normrope_backward_workspace_bytes(int dtype, const dxh_normrope_part *parts, int nparts, int64_t rows, int32_t dim, size_t *bytes) {
    if (!bytes) return DXH_ERR_ARG;
    if (dtype != DXH_F32 && dtype != DXH_F16 && dtype != DXH_BF16) return DXH_ERR_DTYPE;
    if (!parts || nparts < 1 || nparts > kMaxParts || rows < 0) return DXH_ERR_ARG;
    if (dim < 16 || dim > 256 || dim % 16) return DXH_ERR_SHAPE;
    bool any = false;
    for (int i = 0; i < nparts; ++i) any = any || (parts[i].dweight && parts[i].norm);
    *bytes = any && rows > 0 ? (size_t)nparts * kBackwardMaxGroups * dim * sizeof(float) : 0;
    return DXH_OK;
}

int dxh_normrope_backward(int dtype, const dxh_normrope_part *parts, int nparts, int64_t rows, int32_t dim, float eps, const dxh_rotary *rot,
                          void *workspace, size_t workspace_bytes, void *stream) {
    Args a;
    int rc = check(dtype, parts, nparts, rows, dim, eps, rot, true, a);
    if (rc != DXH_OK) return rc;
    size_t need = 0;
    rc = dxh_normrope_backward_workspace_bytes(dtype, parts, nparts, rows, dim, &need);
    if (rc != DXH_OK) return rc;
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return DXH_ERR_WORKSPACE;
    hipStream_t st = as_stream(stream);
    if (rows == 0) {  // a sum over nothing
        for (int i = 0; i < nparts; ++i)
            if (a.part[i].dw) {
                rc = dxh_constant(DXH_F32, a.part[i].dw, dim, dxh_scalar{0.0, 0}, stream);
                if (rc != DXH_OK) return rc;
            }
        return DXH_OK;
    }
    a.partial = (float *)workspace;
    const int lg = lanes_of(dtype, dim), groups = backward_groups(a, nparts, lg);
    rc = launch_dtype(dtype, a, nparts, rot, true, lg, (unsigned)groups, st);
    if (rc != DXH_OK || !need) return rc;
    sum_partials_kernel<<<dim3(dim / 16, nparts), 16 * kSumLanes, 0, st>>>(a, groups);
    return launch_status();
}

}  // extern "C"
