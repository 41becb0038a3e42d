// Layer norm for sm_100a, forward and backward with the reduction of the weight's and bias's gradients.
//
//   forward    mu = mean(x), v = mean((x - mu)^2), s = 1 / sqrt(v + eps);  y = (x - mu) * s * w[grp] + b[grp]
//   backward   xh = (x - mu) * s, u = dy * w[grp];  dx = s * (u - mean(u) - xh * mean(u * xh))
//              dw[grp] = sum over the group's rows of dy * xh,  db[grp] = sum over the group's rows of dy
//
// with grp = row / rows_per_group: one row of w and b for all rows (a plain affine layer norm), or one for each (batch,
// frame) group of rows as the adaLN blocks have it. Everything is computed and summed in float32 and rounded once, to
// the output's type.
//
// A row stays in registers: it is read once, its mean is summed, then the squares of the centred values (two sums over
// registers, so a mean far above the spread costs no digits). A thread owns fixed columns in every row of its block, so
// the column sums of the backward pass are plain register accumulators; a block writes them once per group as a row of
// partial sums, and reduce_partials adds those rows in a fixed order: the gradients are the same bits every time.
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx.

#include "wf_common.cuh"
#include "wf_rows.cuh"

#include <algorithm>

namespace wf {
namespace {

constexpr int kMaxThreads = 1024;

// the sum of v over the 32 lanes, in every lane
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// The sums of N values over the block's threads, in every thread (one warp: shuffles alone). `red` has room for
// 32 * N floats; two calls in a row take different buffers, so that one barrier a call is enough.
template <int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float *red, int warps) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if (warps == 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? red[i * 32 + lane] : 0.f);
}

// Where value j (0..7) of a thread's chunk c lies in the row. VEC: eight neighbours in one or two 16-byte accesses;
// else: neighbours lie in neighbouring threads, so that single-value accesses of a warp still share their sectors.
template <bool VEC>
__device__ __forceinline__ int column(int c, int j, int tid, int threads) {
    return VEC ? (c * threads + tid) * 8 + j : (c * 8 + j) * threads + tid;
}

template <int T, bool VEC>
__device__ __forceinline__ void load_chunk(float (&v)[8], const void *row, int c, int tid, int threads, int d) {
    if constexpr (VEC) {
        const int col = column<true>(c, 0, tid, threads);
        if (col < d) {
            load8<T>(v, row, col);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int col = column<false>(c, j, tid, threads);
            v[j] = col < d ? load1<T>(row, col) : 0.f;
        }
    }
}

template <int T, bool VEC>
__device__ __forceinline__ void store_chunk(const float (&v)[8], void *row, int c, int tid, int threads, int d) {
    if constexpr (VEC) {
        const int col = column<true>(c, 0, tid, threads);
        if (col < d) store8<T, true>(static_cast<char *>(row) + static_cast<size_t>(col) * dtype_size(T), v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int col = column<false>(c, j, tid, threads);
            if (col < d) store1<T>(row, col, v[j]);
        }
    }
}

struct NormArgs {
    const void *x, *w, *b;
    void *y;
    float *mean, *rstd;  // [rows], or null
    int64_t rows, ldx, ldy, rows_per_group;
    int d;
    float eps;
};

// One row a block (threads = the block), or one row a warp (blocks of several warps, threads = 32). NC chunks of 8
// values a thread.
template <int T, int W, int NC, bool VEC, bool WARP>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[2][32];
    const int threads = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int warps = WARP ? 1 : (blockDim.x >> 5);
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    for (int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
         row < a.rows; row += step) {
        const void *xr = row_of<T>(a.x, row, a.ldx);
        float x[NC][8];
        float s[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            load_chunk<T, VEC>(x[c], xr, c, tid, threads, a.d);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[0] += x[c][j];
        }
        team_sum<1>(s, red[0], warps);
        const float mean = s[0] * inv_d;
        float q[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] -= mean;
                if (column<VEC>(c, j, tid, threads) < a.d) q[0] = fmaf(x[c][j], x[c][j], q[0]);
            }
        team_sum<1>(q, red[1], warps);
        const float rstd = rsqrtf(fmaf(q[0], inv_d, a.eps));
        if (a.mean != nullptr && tid == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        const int64_t grp = a.w != nullptr || a.b != nullptr ? row / a.rows_per_group : 0;
        void *yr = row_of<T>(a.y, row, a.ldy);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float p[8];
            if (a.w != nullptr) {
                load_chunk<W, VEC>(p, row_of<W>(a.w, grp, a.d), c, tid, threads, a.d);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] *= rstd * p[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] *= rstd;
            }
            if (a.b != nullptr) {
                load_chunk<W, VEC>(p, row_of<W>(a.b, grp, a.d), c, tid, threads, a.d);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] += p[j];
            }
            store_chunk<T, VEC>(x[c], yr, c, tid, threads, a.d);
        }
    }
}

// Rows wider than a block's registers hold: the same sums with the row read again (from L2) for each of them.
template <int T, int W>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_wide_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[2][32];
    const int warps = blockDim.x >> 5;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const void *xr = row_of<T>(a.x, row, a.ldx);
        float s[1] = {0.f};
        for (int col = threadIdx.x; col < a.d; col += blockDim.x) s[0] += load1<T>(xr, col);
        team_sum<1>(s, red[0], warps);
        const float mean = s[0] * inv_d;
        float q[1] = {0.f};
        for (int col = threadIdx.x; col < a.d; col += blockDim.x) {
            const float v = load1<T>(xr, col) - mean;
            q[0] = fmaf(v, v, q[0]);
        }
        team_sum<1>(q, red[1], warps);
        const float rstd = rsqrtf(fmaf(q[0], inv_d, a.eps));
        if (a.mean != nullptr && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        const int64_t grp = row / a.rows_per_group;
        void *yr = row_of<T>(a.y, row, a.ldy);
        for (int col = threadIdx.x; col < a.d; col += blockDim.x) {
            float v = (load1<T>(xr, col) - mean) * rstd;
            if (a.w != nullptr) v *= load1<W>(row_of<W>(a.w, grp, a.d), col);
            if (a.b != nullptr) v += load1<W>(row_of<W>(a.b, grp, a.d), col);
            store1<T>(yr, col, v);
        }
    }
}

struct NormGradArgs {
    const void *x, *w, *dy;
    const float *mean, *rstd;
    void *dx;                 // or null
    float *part_w, *part_b;   // [groups * chunks, d] partial sums, or null
    int64_t rows, ldx, lddy, lddx;
    RowSplit split;
    int d;
};

// Block blockIdx.x takes one share of the rows (RowSplit). WARP: each warp of the block takes every warps-th row of
// the share and the warps' column sums are added at the end through shared memory.
template <int T, int W, int NC, bool VEC, bool WARP>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_grad_kernel(const __grid_constant__ NormGradArgs a) {
    __shared__ float red[2][64];
    __shared__ float col_red[WARP ? 8 * 32 * 8 : 1];  // WARP: one chunk of every warp (blocks of at most 8 warps)
    const int threads = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int warps = WARP ? 1 : (blockDim.x >> 5);
    const int row_step = WARP ? (blockDim.x >> 5) : 1, row_first = WARP ? (threadIdx.x >> 5) : 0;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    int buf = 0;
    for (int64_t grp = a.split.first_group(blockIdx.x), end = a.split.last_group(blockIdx.x); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.x, grp, lo, hi);
        float w[NC][8], dw[NC][8], db[NC][8];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (a.w != nullptr) load_chunk<W, VEC>(w[c], row_of<W>(a.w, grp, a.d), c, tid, threads, a.d);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dw[c][j] = db[c][j] = 0.f;
                if (a.w == nullptr) w[c][j] = 1.f;
            }
        }
        for (int64_t row = lo + row_first; row < hi; row += row_step) {
            const float mean = a.mean[row], rstd = a.rstd[row];
            float xh[NC][8], dy[NC][8];
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                load_chunk<T, VEC>(xh[c], row_of<T>(a.x, row, a.ldx), c, tid, threads, a.d);
                load_chunk<T, VEC>(dy[c], row_of<T>(a.dy, row, a.lddy), c, tid, threads, a.d);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    xh[c][j] = (xh[c][j] - mean) * rstd;  // dy is 0 past the row's end
                    db[c][j] += dy[c][j];
                    dw[c][j] = fmaf(dy[c][j], xh[c][j], dw[c][j]);
                    dy[c][j] *= w[c][j];
                    s[0] += dy[c][j];
                    s[1] = fmaf(dy[c][j], xh[c][j], s[1]);
                }
            }
            if (a.dx == nullptr) continue;
            team_sum<2>(s, red[buf], warps);
            buf ^= 1;
            const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) dy[c][j] = rstd * (dy[c][j] - m0 - xh[c][j] * m1);
                store_chunk<T, VEC>(dy[c], row_of<T>(a.dx, row, a.lddx), c, tid, threads, a.d);
            }
        }
        const int64_t part = a.split.partial_row(blockIdx.x, grp);
        for (int which = 0; which < 2; ++which) {
            float *dst = which ? a.part_b : a.part_w;
            if (dst == nullptr) continue;
            dst += part * a.d;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = which ? db[c][j] : dw[c][j];
                if constexpr (WARP) {
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < 8; ++j) col_red[(threadIdx.x >> 5) * 256 + j * 32 + tid] = v[j];
                    __syncthreads();
                    if (threadIdx.x < 32) {
                        for (int o = 1; o < static_cast<int>(blockDim.x >> 5); ++o)
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] += col_red[o * 256 + j * 32 + tid];
                        store_chunk<WF_F32, VEC>(v, dst, c, tid, threads, a.d);
                    }
                } else {
                    store_chunk<WF_F32, VEC>(v, dst, c, tid, threads, a.d);
                }
            }
        }
    }
}

// The backward pass of rows wider than a block's registers hold: dx row by row with the row read twice ...
template <int T, int W>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_grad_wide_kernel(const __grid_constant__ NormGradArgs a) {
    __shared__ float red[2][64];
    const int warps = blockDim.x >> 5;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    int buf = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, buf ^= 1) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        const void *xr = row_of<T>(a.x, row, a.ldx), *gr = row_of<T>(a.dy, row, a.lddy);
        const void *wr = a.w == nullptr ? nullptr : row_of<W>(a.w, row / a.split.rows_per_group, a.d);
        float s[2] = {0.f, 0.f};
        for (int col = threadIdx.x; col < a.d; col += blockDim.x) {
            const float u = load1<T>(gr, col) * (wr != nullptr ? load1<W>(wr, col) : 1.f);
            s[0] += u;
            s[1] = fmaf(u, (load1<T>(xr, col) - mean) * rstd, s[1]);
        }
        team_sum<2>(s, red[buf], warps);
        const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
        void *dr = row_of<T>(a.dx, row, a.lddx);
        for (int col = threadIdx.x; col < a.d; col += blockDim.x) {
            const float u = load1<T>(gr, col) * (wr != nullptr ? load1<W>(wr, col) : 1.f);
            store1<T>(dr, col, rstd * (u - m0 - (load1<T>(xr, col) - mean) * rstd * m1));
        }
    }
}

// ... and the column sums by themselves: block (x, y) sums columns 256 x .. 256 x + 255 over share y of the rows.
template <int T>
__global__ void __launch_bounds__(256) layer_norm_column_kernel(const __grid_constant__ NormGradArgs a) {
    const int col = blockIdx.x * 256 + threadIdx.x;
    wait_prior_grid();
    if (col >= a.d) return;
    for (int64_t grp = a.split.first_group(blockIdx.y), end = a.split.last_group(blockIdx.y); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.y, grp, lo, hi);
        float dw = 0.f, db = 0.f;
#pragma unroll 4
        for (int64_t row = lo; row < hi; ++row) {
            const float g = load1<T>(row_of<T>(a.dy, row, a.lddy), col);
            db += g;
            dw = fmaf(g, (load1<T>(row_of<T>(a.x, row, a.ldx), col) - a.mean[row]) * a.rstd[row], dw);
        }
        const int64_t at = a.split.partial_row(blockIdx.y, grp) * a.d + col;
        if (a.part_w != nullptr) a.part_w[at] = dw;
        if (a.part_b != nullptr) a.part_b[at] = db;
    }
}

// ------------------------------------------------------------------------------------------------------------- host
// Threads of a row and the way its values are dealt to them: at least 8 values a thread; a warp up to 256 values.
struct RowShape {
    bool warp, wide;
    int threads, nc;
};
RowShape row_shape(int d) {
    RowShape s;
    s.warp = d <= 256;
    const int need = (d + 7) / 8;
    s.threads = s.warp ? 32 : std::min(kMaxThreads, (need + 31) / 32 * 32);
    s.nc = (need + s.threads - 1) / s.threads;
    s.wide = s.nc > 2;
    return s;
}

bool vec_ok(const void *p, int64_t ld, int size) {
    return p == nullptr || (aligned_to(p, 16) && (ld * size) % 16 == 0);
}

template <int T, int W, int NC, bool VEC, bool WARP>
int launch_norm(const NormArgs &a, const RowShape &s, cudaStream_t stream) {
    constexpr auto kern = layer_norm_kernel<T, W, NC, VEC, WARP>;
    const int block = WARP ? 256 : s.threads;
    const int64_t need = WARP ? (a.rows + 7) / 8 : a.rows;
    const int grid = static_cast<int>(std::min<int64_t>(need, wave_ctas_at<kern>(block)));
    return launch_rows(kern, dim3(grid), block, stream, a);
}

template <int T, int W>
int dispatch_norm(const NormArgs &a, cudaStream_t stream) {
    const RowShape s = row_shape(a.d);
    if (s.wide) {
        constexpr auto kern = layer_norm_wide_kernel<T, W>;
        const int grid = static_cast<int>(std::min<int64_t>(a.rows, wave_ctas_at<kern>(kMaxThreads)));
        return launch_rows(kern, dim3(grid), kMaxThreads, stream, a);
    }
    const bool vec = a.d % 8 == 0 && vec_ok(a.x, a.ldx, dtype_size(T)) && vec_ok(a.y, a.ldy, dtype_size(T)) &&
                     vec_ok(a.w, a.d, dtype_size(W)) && vec_ok(a.b, a.d, dtype_size(W));
    if (s.warp) return vec ? launch_norm<T, W, 1, true, true>(a, s, stream) : launch_norm<T, W, 1, false, true>(a, s, stream);
    if (s.nc == 1) return vec ? launch_norm<T, W, 1, true, false>(a, s, stream) : launch_norm<T, W, 1, false, false>(a, s, stream);
    return vec ? launch_norm<T, W, 2, true, false>(a, s, stream) : launch_norm<T, W, 2, false, false>(a, s, stream);
}

template <int T, int W, int NC, bool VEC, bool WARP>
int launch_norm_grad(const NormGradArgs &a, const RowShape &s, cudaStream_t stream) {
    return launch_rows(layer_norm_grad_kernel<T, W, NC, VEC, WARP>, dim3(static_cast<unsigned>(a.split.blocks())),
                       WARP ? 256 : s.threads, stream, a);
}

template <int T, int W>
int dispatch_norm_grad(const NormGradArgs &a, cudaStream_t stream) {
    const RowShape s = row_shape(a.d);
    if (s.wide) {
        int rc = WF_OK;
        if (a.dx != nullptr) {
            constexpr auto kern = layer_norm_grad_wide_kernel<T, W>;
            const int grid = static_cast<int>(std::min<int64_t>(a.rows, wave_ctas_at<kern>(kMaxThreads)));
            rc = launch_rows(kern, dim3(grid), kMaxThreads, stream, a);
        }
        if (rc == WF_OK && (a.part_w != nullptr || a.part_b != nullptr))
            rc = launch_rows(layer_norm_column_kernel<T>, dim3((a.d + 255) / 256, static_cast<unsigned>(a.split.blocks())),
                             256, stream, a);
        return rc;
    }
    const bool vec = a.d % 8 == 0 && vec_ok(a.x, a.ldx, dtype_size(T)) && vec_ok(a.dy, a.lddy, dtype_size(T)) &&
                     vec_ok(a.dx, a.lddx, dtype_size(T)) && vec_ok(a.w, a.d, dtype_size(W)) && vec_ok(a.part_w, a.d, 4) &&
                     vec_ok(a.part_b, a.d, 4);
    if (s.warp) return vec ? launch_norm_grad<T, W, 1, true, true>(a, s, stream) : launch_norm_grad<T, W, 1, false, true>(a, s, stream);
    if (s.nc == 1) return vec ? launch_norm_grad<T, W, 1, true, false>(a, s, stream) : launch_norm_grad<T, W, 1, false, false>(a, s, stream);
    return vec ? launch_norm_grad<T, W, 2, true, false>(a, s, stream) : launch_norm_grad<T, W, 2, false, false>(a, s, stream);
}

bool norm_types_ok(int type, int w_type) {
    return (type == WF_F16 || type == WF_BF16 || type == WF_F32) && (w_type == type || w_type == WF_F32);
}

// the shares of the rows that the backward pass's blocks take
RowSplit norm_split(int64_t rows, int64_t rows_per_group, int d) {
    const RowShape s = row_shape(d);
    const int64_t wanted = s.wide ? std::max<int64_t>(1, 4ll * device_sm_count() * 256 / d)
                                  : static_cast<int64_t>(device_sm_count()) * (s.warp ? 8 : std::max(1, 2048 / s.threads));
    return make_split(rows, rows_per_group, wanted, s.warp ? 8 : 1);
}

}  // namespace
}  // namespace wf

extern "C" WF_API int wf_layer_norm(const wf_layer_norm_args *args, wf_stream_t stream) {
    using namespace wf;
    if (args == nullptr) return WF_ERR_ARG;
    const wf_layer_norm_args &g = *args;
    if (!norm_types_ok(g.type, g.w_type)) return WF_ERR_UNSUPPORTED;
    if (g.rows < 0 || g.d < 1 || g.d > (1 << 30) || g.rows_per_group < 1 || !(g.eps >= 0.f) || g.ldx < g.d || g.ldy < g.d)
        return WF_ERR_ARG;
    if ((g.mean == nullptr) != (g.rstd == nullptr)) return WF_ERR_ARG;
    if (g.rows == 0) return WF_OK;
    const int e = dtype_size(g.type), we = dtype_size(g.w_type);
    if (!g.x || !g.y || !aligned_to(g.x, e) || !aligned_to(g.y, e) || !aligned_to(g.w, we) || !aligned_to(g.b, we) ||
        !aligned_to(g.mean, 4) || !aligned_to(g.rstd, 4))
        return WF_ERR_ARG;
    const int rc = check_device();
    if (rc != WF_OK) return rc;
    const NormArgs a{g.x, g.w, g.b, g.y, g.mean, g.rstd, g.rows, g.ldx, g.ldy, g.rows_per_group, static_cast<int>(g.d), g.eps};
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (g.type == WF_F32) return dispatch_norm<WF_F32, WF_F32>(a, st);
    if (g.type == WF_BF16) return g.w_type == WF_F32 ? dispatch_norm<WF_BF16, WF_F32>(a, st) : dispatch_norm<WF_BF16, WF_BF16>(a, st);
    return g.w_type == WF_F32 ? dispatch_norm<WF_F16, WF_F32>(a, st) : dispatch_norm<WF_F16, WF_F16>(a, st);
}

extern "C" WF_API int64_t wf_layer_norm_backward_workspace(int64_t rows, int64_t d, int64_t rows_per_group) {
    using namespace wf;
    if (rows < 1 || d < 1 || d > (1 << 30) || rows_per_group < 1) return 0;
    return 2 * norm_split(rows, rows_per_group, static_cast<int>(d)).partial_rows() * d * static_cast<int64_t>(sizeof(float));
}

extern "C" WF_API int wf_layer_norm_backward(const wf_layer_norm_grad_args *args, wf_stream_t stream) {
    using namespace wf;
    if (args == nullptr) return WF_ERR_ARG;
    const wf_layer_norm_grad_args &g = *args;
    if (!norm_types_ok(g.type, g.w_type)) return WF_ERR_UNSUPPORTED;
    if (g.rows < 1 || g.d < 1 || g.d > (1 << 30) || g.rows_per_group < 1 || g.ldx < g.d || g.lddy < g.d ||
        (g.dx && g.lddx < g.d))
        return WF_ERR_ARG;
    const int e = dtype_size(g.type), we = dtype_size(g.w_type);
    if (!g.x || !g.dy || !g.mean || !g.rstd || !aligned_to(g.x, e) || !aligned_to(g.dy, e) || !aligned_to(g.dx, e) ||
        !aligned_to(g.w, we) || !aligned_to(g.dw, we) || !aligned_to(g.db, we) || !aligned_to(g.mean, 4) ||
        !aligned_to(g.rstd, 4))
        return WF_ERR_ARG;
    if (!g.dx && !g.dw && !g.db) return WF_OK;
    const RowSplit split = norm_split(g.rows, g.rows_per_group, static_cast<int>(g.d));
    const int64_t half = split.partial_rows() * g.d;
    if ((g.dw || g.db) && (!g.workspace || !aligned_to(g.workspace, 16) ||
                           g.workspace_bytes < 2 * half * static_cast<int64_t>(sizeof(float))))
        return WF_ERR_ARG;
    int rc = check_device();
    if (rc != WF_OK) return rc;
    float *part = static_cast<float *>(g.workspace);
    const NormGradArgs a{g.x, g.w, g.dy, g.mean, g.rstd, g.dx, g.dw ? part : nullptr, g.db ? part + half : nullptr, g.rows,
                         g.ldx, g.lddy, g.lddx, split, static_cast<int>(g.d)};
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (g.type == WF_F32) rc = dispatch_norm_grad<WF_F32, WF_F32>(a, st);
    else if (g.type == WF_BF16) rc = g.w_type == WF_F32 ? dispatch_norm_grad<WF_BF16, WF_F32>(a, st) : dispatch_norm_grad<WF_BF16, WF_BF16>(a, st);
    else rc = g.w_type == WF_F32 ? dispatch_norm_grad<WF_F16, WF_F32>(a, st) : dispatch_norm_grad<WF_F16, WF_F16>(a, st);
    if (rc != WF_OK) return rc;
    const int64_t parts = split.partials_per_group();
    return reduce_partials(PartialSum{a.part_w, g.dw, split.groups, parts}, PartialSum{a.part_b, g.db, split.groups, parts},
                           g.d, g.w_type, st);
}
