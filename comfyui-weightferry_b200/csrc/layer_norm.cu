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
// registers, so a mean far above the spread costs no digits). In the backward pass a thread owns fixed columns in every
// row of its block, so the column sums are plain register accumulators; a block writes them once per group as a row of
// partial sums, and reduce_partials adds those rows in a fixed order: the gradients are the same bits every time.
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx.

#include "wf_common.cuh"
#include "wf_pairs.cuh"
#include "wf_rows.cuh"
#include "wf_tcgen05.cuh"

#include <algorithm>

namespace wf {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kTeam = 8;  // CTAs of a team

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

// eight values of a row as they lie in memory (16-byte aligned): zeros past d
template <int T>
struct Raw8 {
    uint4 q[T == WF_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *row, int col, int d) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(row) + static_cast<int64_t>(col) * dtype_size(T));
#pragma unroll
        for (int i = 0; i < (T == WF_F32 ? 2 : 1); ++i) q[i] = col < d ? p[i] : make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void get(uint64_t (&v)[4]) const {
        if constexpr (T == WF_F32) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[2 * i] = pack_f2(__uint_as_float(q[i].x), __uint_as_float(q[i].y));
                v[2 * i + 1] = pack_f2(__uint_as_float(q[i].z), __uint_as_float(q[i].w));
            }
        } else {
            const uint32_t w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2<T>(w[i]);
                v[i] = pack_f2(f.x, f.y);
            }
        }
    }
};

// eight values, or four of float32, rounded to T, to column col of a row (16-byte aligned)
template <int T, int NP>
__device__ __forceinline__ void store_pairs(void *row, int col, const uint64_t (&v)[NP]) {
    static_assert(NP == 4 || (NP == 2 && T == WF_F32), "16 or 32 bytes");
    float f[2 * NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) unpack_f2(v[i], f[2 * i], f[2 * i + 1]);
    if constexpr (NP == 4) {
        store8<T, true>(static_cast<char *>(row) + static_cast<int64_t>(col) * dtype_size(T), f);
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(row) + col) = make_float4(f[0], f[1], f[2], f[3]);
    }
}

// the sum over aligned sets of LPR lanes, in each of them
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// The sums of N values (a power of 2) over the warp's lanes: lane l gets sum l / (32 / N). Each exchange halves the sums
// that a lane still carries, N + log2(32 / N) - 1 shuffles instead of 5 N.
template <int N>
__device__ __forceinline__ float lanes_sum_many(float (&v)[N], int lane) {
#pragma unroll
    for (int n = N / 2, o = 16; n > 0; n /= 2, o /= 2) {
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    }
    float s = v[0];
#pragma unroll
    for (int o = 16 / N; o > 0; o /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    return s;
}

// NV values a lane, 32 columns apart
template <int T, int NV>
__device__ __forceinline__ void load_lanes(float (&v)[NV], const void *row, int lane, int d) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = j * 32 + lane < d ? load1<T>(row, j * 32 + lane) : 0.f;
}

struct NormArgs {
    const void *x, *w, *b;
    void *y;
    float *mean, *rstd;  // [rows], or null
    int64_t rows, ldx, ldy, rows_per_group;
    int d;
    float eps;
};

// One row a block, NC chunks of 8 values a thread.
template <int T, int W, int NC, bool VEC>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[2][32];
    const int threads = blockDim.x, tid = threadIdx.x, warps = blockDim.x >> 5;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
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

// Narrow rows (up to 32 NV values) that 16-byte accesses do not fit, value by value: 8 / NV rows a warp at a time.
template <int T, int W, int NV>
__global__ void __launch_bounds__(256) layer_norm_warp_kernel(const __grid_constant__ NormArgs a) {
    constexpr int R = 8 / NV, L = 32 / R;  // lanes that hold the same sum
    const int lane = threadIdx.x & 31;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8 * R;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    for (int64_t row = (static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * R; row < a.rows; row += step) {
        float v[R][NV], s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            load_lanes<T, NV>(v[r], row_of<T>(a.x, row + r, a.ldx), lane, row + r < a.rows ? a.d : 0);
            s[r] = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) s[r] += v[r][j];
        }
        const float mean = lanes_sum_many<R>(s, lane) * inv_d;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float mu = __shfl_sync(0xFFFFFFFFu, mean, r * L);
            s[r] = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                v[r][j] -= mu;
                if (j * 32 + lane < a.d) s[r] = fmaf(v[r][j], v[r][j], s[r]);
            }
        }
        const float rstd = rsqrtf(fmaf(lanes_sum_many<R>(s, lane), inv_d, a.eps));
        if (a.mean != nullptr && (lane & (L - 1)) == 0 && row + lane / L < a.rows) {
            a.mean[row + lane / L] = mean;
            a.rstd[row + lane / L] = rstd;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float rs = __shfl_sync(0xFFFFFFFFu, rstd, r * L);
            if (row + r >= a.rows) continue;
            const int64_t grp = a.w != nullptr || a.b != nullptr ? (row + r) / a.rows_per_group : 0;
            const void *w = row_of<W>(a.w, grp, a.d), *b = row_of<W>(a.b, grp, a.d);
            void *y = row_of<T>(a.y, row + r, a.ldy);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = j * 32 + lane;
                if (col >= a.d) continue;
                float f = v[r][j] * rs;
                if (a.w != nullptr) f *= load1<W>(w, col);
                if (a.b != nullptr) f += load1<W>(b, col);
                store1<T>(y, col, f);
            }
        }
    }
}

// v * w + b with eight values of w and b (either may be null) from column col
template <int W>
__device__ __forceinline__ void affine(uint64_t (&v)[4], const void *w, const void *b, int col) {
    Raw8<W> raw;
    uint64_t p[4];
    if (w != nullptr) {
        raw.load(w, col, col + 8);
        raw.get(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = mul_f2(v[j], p[j]);
    }
    if (b != nullptr) {
        raw.load(b, col, col + 8);
        raw.get(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = add_f2(v[j], p[j]);
    }
}

// Narrow rows (up to 256 values) that 16-byte accesses fit: LPR lanes a row, 8 values a lane, 32 / LPR rows a warp.
template <int T, int W, int LPR>
__global__ void __launch_bounds__(256) layer_norm_narrow_kernel(const __grid_constant__ NormArgs a) {
    constexpr int RPW = 32 / LPR;
    const int lane = threadIdx.x & (LPR - 1), sub = (threadIdx.x & 31) / LPR, col = lane * 8;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    const bool in = col < a.d;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8 * RPW;
    wait_prior_grid();
    for (int64_t first = (static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * RPW; first < a.rows; first += step) {
        const int64_t row = first + sub;
        const bool on = row < a.rows;
        Raw8<T> x;
        x.load(row_of<T>(a.x, row, a.ldx), col, on ? a.d : 0);
        uint64_t v[4], s = 0, q = 0;  // +0, +0
        x.get(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) s = add_f2(s, v[j]);
        const float mean = lanes_sum<LPR>(sum_f2(s)) * inv_d;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = add_f2(v[j], pack_f2(-mean, -mean));
            if (in) q = fma_f2(v[j], v[j], q);
        }
        const float rstd = rsqrtf(fmaf(lanes_sum<LPR>(sum_f2(q)), inv_d, a.eps));
        if (!on || !in) continue;
        if (a.mean != nullptr && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = mul_f2(v[j], pack_f2(rstd, rstd));
        const int64_t grp = row / a.rows_per_group;
        affine<W>(v, a.w == nullptr ? nullptr : row_of<W>(a.w, grp, a.d), a.b == nullptr ? nullptr : row_of<W>(a.b, grp, a.d), col);
        store_pairs<T>(row_of<T>(a.y, row, a.ldy), col, v);
    }
}

// 16 bytes of T as pairs: 8 or 4 values
template <int T>
__device__ __forceinline__ void widen(uint64_t (&v)[T == WF_F32 ? 2 : 4], const uint4 &q) {
    if constexpr (T == WF_F32) {
        v[0] = pack_f2(__uint_as_float(q.x), __uint_as_float(q.y));
        v[1] = pack_f2(__uint_as_float(q.z), __uint_as_float(q.w));
    } else {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[i] = pack_f2(f.x, f.y);
        }
    }
}

// The values of w (or b) that belong to 16-byte piece `piece` of a row of T. Staged, a float32 row beside 16-bit values
// lies in two planes (a piece's first and second four values), so that neighbouring lanes read neighbouring 16 bytes.
template <int T, int W>
__device__ __forceinline__ void param_piece(uint64_t (&p)[T == WF_F32 ? 2 : 4], const uint4 *row, int piece, int pieces, bool staged) {
    if constexpr (T == W) {
        widen<T>(p, row[piece]);
    } else {
        uint64_t h[2];
        widen<WF_F32>(h, row[staged ? piece : 2 * piece]);
        p[0] = h[0], p[1] = h[1];
        widen<WF_F32>(h, row[staged ? pieces + piece : 2 * piece + 1]);
        p[2] = h[0], p[3] = h[1];
    }
}

// Many wider rows that 16-byte accesses fit: a team of WPR warps a row. Each thread copies its own 16-byte pieces of the
// team's next rows into a ring in shared memory (cp.async) and reads nobody else's, so that rows stream in without a
// barrier and without registers (a row held in registers, widened three times, needed 234 of them for 5120 values and
// left 8 warps an SM: 16384 x 5120 took 84 us where this takes 62). A block takes a run of rows (RowSplit) and keeps their
// group's w and b in shared memory: read from L2 for every row they cost more than x itself (16384 x 5120 bf16 in 16
// groups: 222 us). Groups of fewer than kStageRows rows are read from L2 all the same.
constexpr int kStageRows = 16;
template <int T, int W, int WPR>
__global__ void __launch_bounds__(256) layer_norm_stream_kernel(const __grid_constant__ NormArgs a,
                                                                const __grid_constant__ RowSplit split, int bufs, bool stage) {
    constexpr int NP = T == WF_F32 ? 2 : 4;           // pairs of a piece
    constexpr int TEAMS = 8 / WPR, LANES = 32 * WPR;
    extern __shared__ uint4 smem[];                   // w and b of the group (where staged), then a ring a team
    __shared__ float red[2][8];
    const int warp = threadIdx.x >> 5, team = warp / WPR, lane = threadIdx.x & (LANES - 1);
    const int pieces = a.d / (2 * NP), w_pieces = a.d * dtype_size(W) / 16;
    uint4 *sw = smem, *sb = smem + w_pieces;
    uint4 *ring = smem + (stage ? 2 * w_pieces : 0) + team * bufs * pieces;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    auto team_total = [&](float v, float *buf) {
        v = lanes_sum<32>(v);
        if constexpr (WPR > 1) {
            if ((threadIdx.x & 31) == 0) buf[warp] = v;
            asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(LANES) : "memory");
            v = 0.f;
#pragma unroll
            for (int i = 0; i < WPR; ++i) v += buf[team * WPR + i];
        }
        return v;
    };
    wait_prior_grid();
    for (int64_t grp = split.first_group(blockIdx.x), end = split.last_group(blockIdx.x); grp < end; ++grp) {
        int64_t lo, hi;
        split.rows_of(blockIdx.x, grp, lo, hi);
        auto fetch = [&](int64_t row, int buf) {  // one copy group a row, empty past the last
            if (row < hi) {
                const char *src = static_cast<const char *>(row_of<T>(a.x, row, a.ldx));
                for (int i = lane; i < pieces; i += LANES) copy16(ring + buf * pieces + i, src + 16 * i, true);
            }
            cp_async_commit();
        };
        int64_t ahead = lo + team;
        for (int i = 0; i < bufs - 1; ++i, ahead += TEAMS) fetch(ahead, i);
        const uint4 *w = a.w == nullptr ? nullptr : static_cast<const uint4 *>(row_of<W>(a.w, grp, a.d));
        const uint4 *b = a.b == nullptr ? nullptr : static_cast<const uint4 *>(row_of<W>(a.b, grp, a.d));
        if (stage) {
            __syncthreads();
            for (int i = threadIdx.x; i < w_pieces; i += 256) {
                const int at = T == W ? i : (i & 1) * pieces + (i >> 1);
                if (w != nullptr) sw[at] = w[i];
                if (b != nullptr) sb[at] = b[i];
            }
            __syncthreads();
            if (w != nullptr) w = sw;
            if (b != nullptr) b = sb;
        }
        int buf = 0, next = bufs - 1;
        for (int64_t row = lo + team; row < hi; row += TEAMS, ahead += TEAMS) {
            fetch(ahead, next);
            if (++next == bufs) next = 0;
            if (bufs == 2) cp_async_wait<1>();
            else if (bufs == 3) cp_async_wait<2>();
            else cp_async_wait<3>();
            const uint4 *x = ring + buf * pieces;
            if (++buf == bufs) buf = 0;
            uint64_t v[NP], s = 0, s1 = 0;  // +0, +0
#pragma unroll 4
            for (int i = lane; i < pieces; i += LANES) {
                widen<T>(v, x[i]);
#pragma unroll
                for (int j = 0; j < NP; j += 2) s = add_f2(s, v[j]), s1 = add_f2(s1, v[j + 1]);
            }
            const float mean = team_total(sum_f2(s) + sum_f2(s1), red[0]) * inv_d;
            const uint64_t shift = pack_f2(-mean, -mean);
            s = s1 = 0;
#pragma unroll 4
            for (int i = lane; i < pieces; i += LANES) {
                widen<T>(v, x[i]);
#pragma unroll
                for (int j = 0; j < NP; j += 2) {
                    const uint64_t c0 = add_f2(v[j], shift), c1 = add_f2(v[j + 1], shift);
                    s = fma_f2(c0, c0, s);
                    s1 = fma_f2(c1, c1, s1);
                }
            }
            const float rstd = rsqrtf(fmaf(team_total(sum_f2(s) + sum_f2(s1), red[1]), inv_d, a.eps));
            if (a.mean != nullptr && lane == 0) {
                a.mean[row] = mean;
                a.rstd[row] = rstd;
            }
            const uint64_t rs = pack_f2(rstd, rstd);
            uint4 *y = static_cast<uint4 *>(row_of<T>(a.y, row, a.ldy));
#pragma unroll 4
            for (int i = lane; i < pieces; i += LANES) {
                uint64_t p[NP];
                widen<T>(v, x[i]);
#pragma unroll
                for (int j = 0; j < NP; ++j) v[j] = mul_f2(add_f2(v[j], shift), rs);
                if (w != nullptr) {
                    param_piece<T, W>(p, w, i, pieces, stage);
#pragma unroll
                    for (int j = 0; j < NP; ++j) v[j] = mul_f2(v[j], p[j]);
                }
                if (b != nullptr) {
                    param_piece<T, W>(p, b, i, pieces, stage);
#pragma unroll
                    for (int j = 0; j < NP; ++j) v[j] = add_f2(v[j], p[j]);
                }
                float f[2 * NP];
#pragma unroll
                for (int j = 0; j < NP; ++j) unpack_f2(v[j], f[2 * j], f[2 * j + 1]);
                if constexpr (T == WF_F32) {
                    y[i] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
                } else {
                    store8<T, true>(y + i, f);
                }
            }
        }
        cp_async_wait<0>();
    }
}

// The sums of N values (a power of 2) over the block's threads, or (TEAM) over those of a cluster of kTeam CTAs: sum k in the
// lanes k, k + N, ... of every warp. One barrier; two calls in a row take different buffers. In a cluster every warp writes
// its sums to all CTAs (distributed shared memory): nothing is written after a barrier that a CTA leaves behind.
template <int N, bool TEAM>
__device__ __forceinline__ float block_sums(float (&v)[N], float (*red)[N], int warp, int lane, int warps) {
    constexpr int L = 32 / N;  // lanes that hold the same sum
    const float mine = lanes_sum_many<N>(v, lane);
    int all = warps;
    if constexpr (TEAM) {
        all = warps * kTeam;
        const uint32_t at = smem_u32(&red[cluster_rank() * warps + warp][lane / L]);
        for (int to = lane & (L - 1); to < kTeam; to += L)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_rank(at, to)), "f"(mine) : "memory");
        __syncwarp();
        cluster_sync();
    } else {
        if ((lane & (L - 1)) == 0) red[warp][lane / L] = mine;
        __syncthreads();
    }
    float t = 0.f;
    for (int i = lane / N; i < all; i += L) t += red[i][lane % N];
#pragma unroll
    for (int o = N; o < 32; o *= 2) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    return t;
}

// A row that 16-byte accesses do not fit, in shared memory: the aligned 16-byte pieces that it lies in are copied (cp.async),
// and values are read one by one from where its first byte falls in them. What a piece holds before the row is copied with
// it and never read (the piece holds a byte of the row, so it lies in its allocation); nothing past the row is read.
// Single values copied straight from HBM keep too few bytes in flight (16384 x 5119
// bf16: forward 186 us and backward 346, where these take 133 and 176).
__host__ __device__ inline int cover_bytes(int d, int type) { return (d * dtype_size(type) + 15) / 16 * 16 + 16; }
__device__ __forceinline__ int skew(const void *row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15); }
__device__ __forceinline__ void copy_cover(char *dst, const void *row, int bytes, int tid, int threads) {
    const int s = skew(row), n = s + bytes;
    const char *src = static_cast<const char *>(row) - s;
    for (int i = 16 * tid; i < n; i += 16 * threads)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + i)), "l"(src + i), "r"(min(16, n - i))
                     : "memory");
}

// The forward pass of rows of 257 to 16384 values that 16-byte accesses do not fit: eight values a thread, with their w and b
// in registers, R rows at a time through a ring of such copies; one barrier a sum. TEAM: a cluster of kTeam CTAs shares
// the rows, each CTA a run of columns.
constexpr int kRing = 3;
template <int T, int W, int R, int THREADS, int BLOCKS, bool TEAM>
__global__ void __launch_bounds__(THREADS, BLOCKS) layer_norm_unaligned_kernel(const __grid_constant__ NormArgs a,
                                                                               const __grid_constant__ RowSplit split, int block_cols) {
    extern __shared__ uint4 smem[];
    __shared__ float red[2][TEAM ? kTeam * THREADS / 32 : 32][R];
    const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
    const int64_t col0 = TEAM ? cluster_rank() * block_cols : 0, share = TEAM ? blockIdx.x / kTeam : blockIdx.x;
    const int d = TEAM ? min(block_cols, a.d - static_cast<int>(col0)) : a.d;  // this CTA's columns, from col0
    const int cover = cover_bytes(block_cols, T), bytes = d * dtype_size(T);
    char *ring = reinterpret_cast<char *>(smem);
    const float inv_d = 1.0f / static_cast<float>(a.d);
    auto x_row = [&](int64_t row) { return row_of<T>(a.x, row, a.ldx, col0); };
    if constexpr (TEAM) cluster_sync();  // every CTA of the team runs before another writes to its shared memory
    wait_prior_grid();
    for (int64_t grp = split.first_group(share), end = split.last_group(share); grp < end; ++grp) {
        int64_t lo, hi;
        split.rows_of(share, grp, lo, hi);
        auto fetch = [&](int64_t row, int slot) {
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (row + r < hi) copy_cover(ring + (slot * R + r) * cover, x_row(row + r), bytes, tid, threads);
            cp_async_commit();
        };
        for (int i = 0; i < kRing; ++i) fetch(lo + i * R, i);
        float w[8], b[8];
        if (a.w != nullptr) load_chunk<W, false>(w, row_of<W>(a.w, grp, a.d, col0), 0, tid, threads, d);
        if (a.b != nullptr) load_chunk<W, false>(b, row_of<W>(a.b, grp, a.d, col0), 0, tid, threads, d);
        cp_async_wait<kRing - 1>();
        __syncthreads();
        int slot = 0;
        for (int64_t row = lo; row < hi; row += R) {
            float v[R][8], s[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                load_chunk<T, false>(v[r], ring + (slot * R + r) * cover + skew(x_row(row + r)), 0, tid, threads, d);
                s[r] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) s[r] += v[r][j];
            }
            cp_async_wait<kRing - 2>();  // the next rows are here for this thread, and behind the barrier for all
            const float mean = block_sums<R, TEAM>(s, red[0], warp, lane, warps) * inv_d;
            fetch(row + kRing * R, slot);  // every thread has read this slot
            if (++slot == kRing) slot = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float mu = __shfl_sync(0xFFFFFFFFu, mean, r);
                s[r] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[r][j] -= mu;
                    if (column<false>(0, j, tid, threads) < d) s[r] = fmaf(v[r][j], v[r][j], s[r]);
                }
            }
            const float rstd = rsqrtf(fmaf(block_sums<R, TEAM>(s, red[1], warp, lane, warps), inv_d, a.eps));
            if (a.mean != nullptr && col0 == 0 && tid < R && row + tid < hi) {
                a.mean[row + tid] = mean;
                a.rstd[row + tid] = rstd;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float rs = __shfl_sync(0xFFFFFFFFu, rstd, r);
                if (row + r >= hi) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[r][j] *= rs;
                    if (a.w != nullptr) v[r][j] *= w[j];
                    if (a.b != nullptr) v[r][j] += b[j];
                }
                store_chunk<T, false>(v[r], row_of<T>(a.y, row + r, a.ldy, col0), 0, tid, threads, d);
            }
        }
    }
    cp_async_wait<0>();
}

struct NormGradArgs {
    const void *x, *w, *dy;
    const float *mean, *rstd;
    void *dx;                 // or null
    float *part_w, *part_b;   // [groups * chunks, d] partial sums, or null
    int64_t rows, ldx, lddy, lddx;
    RowSplit split;
    int d, block_cols;        // block_cols: d, or a team's columns of each CTA (a multiple of 8)
};

// The backward pass of rows that 16-byte accesses fit, V (8 or 4) values a thread of a block: R rows at a time, whose 2 R sums
// share one barrier (and their shuffles: lanes_sum_many). Each thread copies its own values of the next rows into a ring
// of kRing stages in shared memory (cp.async) and reads nobody else's: the loads run on behind the barrier.
// TEAM: a cluster of kTeam CTAs shares the rows, each CTA a run of a.block_cols columns: the wide kernels
// read x and dy once more.
template <int T, int W, int V, int R, int THREADS, int BLOCKS, bool TEAM>
__global__ void __launch_bounds__(THREADS, BLOCKS) layer_norm_grad_rows_kernel(const __grid_constant__ NormGradArgs a) {
    constexpr int H = V * dtype_size(T) / 16, NP = V / 2;  // 16-byte pieces and pairs of V values
    extern __shared__ uint4 smem[];                   // [kRing][R][x, dy][H][threads]
    __shared__ float red[2][TEAM ? kTeam * THREADS / 32 : 32][2 * R];
    const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
    const int rank = TEAM ? static_cast<int>(cluster_rank()) : 0, col = rank * a.block_cols + tid * V;
    const int64_t share = TEAM ? blockIdx.x / kTeam : blockIdx.x;
    const bool in = tid * V < a.block_cols && col < a.d;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    auto piece = [&](int stage, int r, int which, int h) { return smem + (((stage * R + r) * 2 + which) * H + h) * threads + tid; };
    auto get = [&](uint64_t (&v)[NP], int stage, int r, int which) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            uint64_t p[NP / H];
            widen<T>(p, *piece(stage, r, which, h));
#pragma unroll
            for (int j = 0; j < NP / H; ++j) v[h * (NP / H) + j] = p[j];
        }
    };
    int buf = 0;
    if constexpr (TEAM) cluster_sync();  // every CTA of the team runs before another writes to its shared memory
    wait_prior_grid();
    for (int64_t grp = a.split.first_group(share), end = a.split.last_group(share); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(share, grp, lo, hi);
        auto fetch = [&](int64_t row, int stage) {  // one copy group for R rows, zeros past the last
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const bool on = in && row + r < hi;
                const int64_t at = on ? row + r : 0;
                const int c = on ? col : 0;
                const char *x = static_cast<const char *>(row_of<T>(a.x, at, a.ldx)) + c * dtype_size(T);
                const char *g = static_cast<const char *>(row_of<T>(a.dy, at, a.lddy)) + c * dtype_size(T);
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    copy16(piece(stage, r, 0, h), x + 16 * h, on);
                    copy16(piece(stage, r, 1, h), g + 16 * h, on);
                }
            }
            cp_async_commit();
        };
        for (int i = 0; i < kRing - 1; ++i) fetch(lo + i * R, i);
        uint64_t w[NP], dw[NP], db[NP];
        const void *wr = row_of<W>(a.w, grp, a.d);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            dw[j] = db[j] = 0;  // +0, +0
            w[j] = a.w != nullptr && in ? pack_f2(load1<W>(wr, col + 2 * j), load1<W>(wr, col + 2 * j + 1)) : pack_f2(1.f, 1.f);
        }
        int stage = 0, next = kRing - 1;
        float scale[R], shift[R];  // of the rows at hand; the next ones are loaded a tile ahead
#pragma unroll
        for (int r = 0; r < R; ++r) {
            scale[r] = lo + r < hi ? a.rstd[lo + r] : 0.f;
            shift[r] = lo + r < hi ? a.mean[lo + r] : 0.f;
        }
        for (int64_t row = lo; row < hi; row += R) {
            fetch(row + (kRing - 1) * R, next);
            if (++next == kRing) next = 0;
            float scale1[R], shift1[R], s[2 * R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                scale1[r] = row + R + r < hi ? a.rstd[row + R + r] : 0.f;
                shift1[r] = row + R + r < hi ? a.mean[row + R + r] : 0.f;
            }
            cp_async_wait<kRing - 1>();
#pragma unroll
            for (int r = 0; r < R; ++r) {
                uint64_t v[NP], g[NP], s0 = 0, s1 = 0;
                get(v, stage, r, 0);
                get(g, stage, r, 1);
                const uint64_t rs = pack_f2(scale[r], scale[r]), mu = pack_f2(-shift[r], -shift[r]);
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const uint64_t xh = mul_f2(add_f2(v[j], mu), rs);  // dy is 0 outside
                    db[j] = add_f2(db[j], g[j]);
                    dw[j] = fma_f2(g[j], xh, dw[j]);
                    const uint64_t u = mul_f2(g[j], w[j]);
                    s0 = add_f2(s0, u);
                    s1 = fma_f2(u, xh, s1);
                }
                s[2 * r] = sum_f2(s0);
                s[2 * r + 1] = sum_f2(s1);
            }
            if (a.dx != nullptr) {
                const float t = block_sums<2 * R, TEAM>(s, red[buf], warp, lane, warps);
                buf ^= 1;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float m0 = __shfl_sync(0xFFFFFFFFu, t, 2 * r) * inv_d, m1 = __shfl_sync(0xFFFFFFFFu, t, 2 * r + 1) * inv_d;
                    if (!in || row + r >= hi) continue;
                    uint64_t v[NP], g[NP];
                    get(v, stage, r, 0);
                    get(g, stage, r, 1);
                    const uint64_t rs = pack_f2(scale[r], scale[r]), mu = pack_f2(-shift[r], -shift[r]);
                    const uint64_t a0 = pack_f2(-m0, -m0), a1 = pack_f2(-m1, -m1);
#pragma unroll
                    for (int j = 0; j < NP; ++j) {
                        const uint64_t xh = mul_f2(add_f2(v[j], mu), rs);
                        g[j] = mul_f2(rs, fma_f2(xh, a1, fma_f2(g[j], w[j], a0)));
                    }
                    store_pairs<T>(row_of<T>(a.dx, row + r, a.lddx), col, g);
                }
            }
            if (++stage == kRing) stage = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) scale[r] = scale1[r], shift[r] = shift1[r];
        }
        cp_async_wait<0>();
        const int64_t part = a.split.partial_row(share, grp) * a.d;
        if (a.part_w != nullptr && in) store_pairs<WF_F32>(a.part_w + part, col, dw);
        if (a.part_b != nullptr && in) store_pairs<WF_F32>(a.part_b + part, col, db);
    }
}

// The backward pass of narrow rows (up to 256 values) that 16-byte accesses fit: LPR lanes a row, 32 / LPR rows a warp, R
// of them at a time. At the end of a group the lanes that own the same columns, then the warps, add their column sums.
template <int T, int W, int LPR>
__global__ void __launch_bounds__(256, 3) layer_norm_grad_narrow_kernel(const __grid_constant__ NormGradArgs a) {
    constexpr int RPW = 32 / LPR, R = 2;
    __shared__ float col_red[8][16][LPR];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LPR - 1), sub = (threadIdx.x & 31) / LPR, col = lane * 8;
    const bool in = col < a.d;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    for (int64_t grp = a.split.first_group(blockIdx.x), end = a.split.last_group(blockIdx.x); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.x, grp, lo, hi);
        uint64_t w[4], dw[4], db[4];
        if (a.w != nullptr && in) {
            Raw8<W> raw;
            raw.load(row_of<W>(a.w, grp, a.d), col, a.d);
            raw.get(w);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            dw[j] = db[j] = 0;  // +0, +0
            if (a.w == nullptr || !in) w[j] = pack_f2(1.f, 1.f);
        }
        for (int64_t first = lo + warp * RPW * R; first < hi; first += 8 * RPW * R) {
            Raw8<T> x[R], dy[R];
            float scale[R], shift[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t row = first + r * RPW + sub;
                const bool on = row < hi;
                x[r].load(row_of<T>(a.x, row, a.ldx), col, on ? a.d : 0);
                dy[r].load(row_of<T>(a.dy, row, a.lddy), col, on ? a.d : 0);
                scale[r] = on ? a.rstd[row] : 0.f;
                shift[r] = on ? a.mean[row] : 0.f;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t row = first + r * RPW + sub;
                uint64_t v[4], g[4], s0 = 0, s1 = 0;
                x[r].get(v);
                dy[r].get(g);
                const uint64_t rs = pack_f2(scale[r], scale[r]), mu = pack_f2(-shift[r], -shift[r]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = mul_f2(add_f2(v[j], mu), rs);
                    db[j] = add_f2(db[j], g[j]);
                    dw[j] = fma_f2(g[j], v[j], dw[j]);
                    g[j] = mul_f2(g[j], w[j]);
                    s0 = add_f2(s0, g[j]);
                    s1 = fma_f2(g[j], v[j], s1);
                }
                if (a.dx == nullptr) continue;
                const float m0 = lanes_sum<LPR>(sum_f2(s0)) * inv_d, m1 = lanes_sum<LPR>(sum_f2(s1)) * inv_d;
                if (row >= hi || !in) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) g[j] = mul_f2(rs, fma_f2(v[j], pack_f2(-m1, -m1), add_f2(g[j], pack_f2(-m0, -m0))));
                store_pairs<T>(row_of<T>(a.dx, row, a.lddx), col, g);
            }
            __syncwarp();
        }
        if (a.part_w == nullptr && a.part_b == nullptr) continue;
        float sums[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unpack_f2(dw[j], sums[2 * j], sums[2 * j + 1]);
            unpack_f2(db[j], sums[8 + 2 * j], sums[9 + 2 * j]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
#pragma unroll
            for (int o = LPR; o < 32; o *= 2) sums[i] += __shfl_xor_sync(0xFFFFFFFFu, sums[i], o);
            if (sub == 0) col_red[warp][i][lane] = sums[i];
        }
        __syncthreads();
        const int64_t part = a.split.partial_row(blockIdx.x, grp) * a.d;
        for (int t = threadIdx.x; t < 16 * LPR; t += 256) {
            const int i = t / LPR, l = t % LPR, c = l * 8 + (i & 7);
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < 8; ++v) s += col_red[v][i][l];
            float *dst = i < 8 ? a.part_w : a.part_b;
            if (dst != nullptr && c < a.d) dst[part + c] = s;
        }
    }
}

// The same for narrow rows (up to 32 NV values) that 16-byte accesses do not fit, value by value: 8 / NV rows a warp at a time,
// and the warps' column sums are added at the end through shared memory.
template <int T, int W, int NV>
__global__ void __launch_bounds__(256) layer_norm_grad_warp_kernel(const __grid_constant__ NormGradArgs a) {
    constexpr int R = 8 / NV;
    __shared__ float col_red[8][NV][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    for (int64_t grp = a.split.first_group(blockIdx.x), end = a.split.last_group(blockIdx.x); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.x, grp, lo, hi);
        float w[NV], dw[NV], db[NV];
        if (a.w != nullptr) load_lanes<W, NV>(w, row_of<W>(a.w, grp, a.d), lane, a.d);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            dw[j] = db[j] = 0.f;
            if (a.w == nullptr) w[j] = 1.f;
        }
        for (int64_t row = lo + warp * R; row < hi; row += 8 * R) {
            float xh[R][NV], u[R][NV], s[2 * R], rstd[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int d = row + r < hi ? a.d : 0;
                const float mean = d ? a.mean[row + r] : 0.f;
                rstd[r] = d ? a.rstd[row + r] : 0.f;
                load_lanes<T, NV>(xh[r], row_of<T>(a.x, row + r, a.ldx), lane, d);
                load_lanes<T, NV>(u[r], row_of<T>(a.dy, row + r, a.lddy), lane, d);
                s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    xh[r][j] = (xh[r][j] - mean) * rstd[r];  // dy is 0 past the row's end
                    db[j] += u[r][j];
                    dw[j] = fmaf(u[r][j], xh[r][j], dw[j]);
                    u[r][j] *= w[j];
                    s[2 * r] += u[r][j];
                    s[2 * r + 1] = fmaf(u[r][j], xh[r][j], s[2 * r + 1]);
                }
            }
            if (a.dx == nullptr) continue;
            constexpr int L = 32 / (2 * R);
            const float mean_u = lanes_sum_many<2 * R>(s, lane) * inv_d;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float m0 = __shfl_sync(0xFFFFFFFFu, mean_u, 2 * r * L), m1 = __shfl_sync(0xFFFFFFFFu, mean_u, (2 * r + 1) * L);
                if (row + r >= hi) continue;
                void *dx = row_of<T>(a.dx, row + r, a.lddx);
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (j * 32 + lane < a.d) store1<T>(dx, j * 32 + lane, rstd[r] * (u[r][j] - m0 - xh[r][j] * m1));
            }
        }
        const int64_t part = a.split.partial_row(blockIdx.x, grp) * a.d;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float *dst = which ? a.part_b : a.part_w;
            if (dst == nullptr) continue;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NV; ++j) col_red[warp][j][lane] = which ? db[j] : dw[j];
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < a.d) {  // column 32 j + lane
                float v = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) v += col_red[i][warp][lane];
                dst[part + threadIdx.x] = v;
            }
        }
    }
}

// ... and for 257 to 8192 values: eight values a thread, R rows at a time through a ring of unaligned copies, one barrier for
// the rows' 2 R sums. TEAM: a cluster shares the rows.
template <int T, int W, int R, int THREADS, int BLOCKS, bool TEAM>
__global__ void __launch_bounds__(THREADS, BLOCKS) layer_norm_grad_unaligned_kernel(const __grid_constant__ NormGradArgs a) {
    extern __shared__ uint4 smem[];  // [kRing][R][x, dy][cover]
    __shared__ float red[2][TEAM ? kTeam * THREADS / 32 : 32][2 * R];
    const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = threads >> 5;
    const int64_t col0 = TEAM ? cluster_rank() * a.block_cols : 0, share = TEAM ? blockIdx.x / kTeam : blockIdx.x;
    const int d = TEAM ? min(a.block_cols, a.d - static_cast<int>(col0)) : a.d;  // this CTA's columns, from col0
    const int cover = cover_bytes(a.block_cols, T), bytes = d * dtype_size(T);
    auto x_row = [&](int64_t row) { return row_of<T>(a.x, row, a.ldx, col0); };
    auto dy_row = [&](int64_t row) { return row_of<T>(a.dy, row, a.lddy, col0); };
    char *ring = reinterpret_cast<char *>(smem);
    const float inv_d = 1.0f / static_cast<float>(a.d);
    int buf = 0;
    if constexpr (TEAM) cluster_sync();  // every CTA of the team runs before another writes to its shared memory
    wait_prior_grid();
    for (int64_t grp = a.split.first_group(share), end = a.split.last_group(share); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(share, grp, lo, hi);
        auto fetch = [&](int64_t row, int slot) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (row + r >= hi) break;
                char *dst = ring + (slot * R + r) * 2 * cover;
                copy_cover(dst, x_row(row + r), bytes, tid, threads);
                copy_cover(dst + cover, dy_row(row + r), bytes, tid, threads);
            }
            cp_async_commit();
        };
        for (int i = 0; i < kRing; ++i) fetch(lo + i * R, i);
        float w[8], dw[8], db[8];
        if (a.w != nullptr) load_chunk<W, false>(w, row_of<W>(a.w, grp, a.d, col0), 0, tid, threads, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            dw[j] = db[j] = 0.f;
            if (a.w == nullptr) w[j] = 1.f;
        }
        cp_async_wait<kRing - 1>();
        __syncthreads();
        int slot = 0;
        for (int64_t row = lo; row < hi; row += R) {
            float xh[R][8], u[R][8], s[2 * R], rstd[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const bool on = row + r < hi;  // else the slot holds older rows: count nothing
                const float mean = on ? a.mean[row + r] : 0.f;
                const char *x = ring + (slot * R + r) * 2 * cover;
                rstd[r] = on ? a.rstd[row + r] : 0.f;
                load_chunk<T, false>(xh[r], x + skew(x_row(row + r)), 0, tid, threads, on ? d : 0);
                load_chunk<T, false>(u[r], x + cover + skew(dy_row(row + r)), 0, tid, threads, on ? d : 0);
                s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    xh[r][j] = (xh[r][j] - mean) * rstd[r];  // dy is 0 past the row's end
                    db[j] += u[r][j];
                    dw[j] = fmaf(u[r][j], xh[r][j], dw[j]);
                    u[r][j] *= w[j];
                    s[2 * r] += u[r][j];
                    s[2 * r + 1] = fmaf(u[r][j], xh[r][j], s[2 * r + 1]);
                }
            }
            cp_async_wait<kRing - 2>();  // the next rows are here for this thread, and behind the barrier for all
            const float mean_u = block_sums<2 * R, TEAM>(s, red[buf], warp, lane, warps) * inv_d;
            buf ^= 1;
            fetch(row + kRing * R, slot);  // every thread has read this slot
            if (++slot == kRing) slot = 0;
            if (a.dx == nullptr) continue;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float m0 = __shfl_sync(0xFFFFFFFFu, mean_u, 2 * r), m1 = __shfl_sync(0xFFFFFFFFu, mean_u, 2 * r + 1);
                if (row + r >= hi) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) u[r][j] = rstd[r] * (u[r][j] - m0 - xh[r][j] * m1);
                store_chunk<T, false>(u[r], row_of<T>(a.dx, row + r, a.lddx, col0), 0, tid, threads, d);
            }
        }
        const int64_t part = a.split.partial_row(share, grp) * a.d + col0;
        if (a.part_w != nullptr) store_chunk<WF_F32, false>(dw, a.part_w + part, 0, tid, threads, d);
        if (a.part_b != nullptr) store_chunk<WF_F32, false>(db, a.part_b + part, 0, tid, threads, d);
    }
    cp_async_wait<0>();
}

// The backward pass of wider rows: dx row by row with the row read twice (the second time from L2) ...
template <int T, int W, bool VEC>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_grad_wide_kernel(const __grid_constant__ NormGradArgs a) {
    __shared__ float red[2][64];
    const int warps = blockDim.x >> 5, chunks = (a.d + 8 * static_cast<int>(blockDim.x) - 1) / (8 * static_cast<int>(blockDim.x));
    const float inv_d = 1.0f / static_cast<float>(a.d);
    wait_prior_grid();
    int buf = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, buf ^= 1) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        const void *xr = row_of<T>(a.x, row, a.ldx), *gr = row_of<T>(a.dy, row, a.lddy);
        const void *wr = a.w == nullptr ? nullptr : row_of<W>(a.w, row / a.split.rows_per_group, a.d);
        float s[2] = {0.f, 0.f}, x[8], g[8], w[8];
        for (int c = 0; c < chunks; ++c) {
            load_chunk<T, VEC>(x, xr, c, threadIdx.x, blockDim.x, a.d);
            load_chunk<T, VEC>(g, gr, c, threadIdx.x, blockDim.x, a.d);
            if (wr != nullptr) load_chunk<W, VEC>(w, wr, c, threadIdx.x, blockDim.x, a.d);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = wr != nullptr ? g[j] * w[j] : g[j];
                s[0] += u;
                s[1] = fmaf(u, (x[j] - mean) * rstd, s[1]);
            }
        }
        team_sum<2>(s, red[buf], warps);
        const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
        for (int c = 0; c < chunks; ++c) {
            load_chunk<T, VEC>(x, xr, c, threadIdx.x, blockDim.x, a.d);
            load_chunk<T, VEC>(g, gr, c, threadIdx.x, blockDim.x, a.d);
            if (wr != nullptr) load_chunk<W, VEC>(w, wr, c, threadIdx.x, blockDim.x, a.d);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = wr != nullptr ? g[j] * w[j] : g[j];
                g[j] = rstd * (u - m0 - (x[j] - mean) * rstd * m1);
            }
            store_chunk<T, VEC>(g, row_of<T>(a.dx, row, a.lddx), c, threadIdx.x, blockDim.x, a.d);
        }
    }
}

// ... and the column sums by themselves: block (x, y) sums 2048 columns from 2048 x over share y of the rows.
template <int T, bool VEC>
__global__ void __launch_bounds__(256) layer_norm_column_kernel(const __grid_constant__ NormGradArgs a) {
    wait_prior_grid();
    for (int64_t grp = a.split.first_group(blockIdx.y), end = a.split.last_group(blockIdx.y); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.y, grp, lo, hi);
        float dw[8], db[8], x[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[j] = db[j] = 0.f;
#pragma unroll 2
        for (int64_t row = lo; row < hi; ++row) {
            load_chunk<T, VEC>(x, row_of<T>(a.x, row, a.ldx), blockIdx.x, threadIdx.x, 256, a.d);
            load_chunk<T, VEC>(g, row_of<T>(a.dy, row, a.lddy), blockIdx.x, threadIdx.x, 256, a.d);
            const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                db[j] += g[j];
                dw[j] = fmaf(g[j], (x[j] - mean) * rstd, dw[j]);
            }
        }
        const int64_t at = a.split.partial_row(blockIdx.y, grp) * a.d;
        if (a.part_w != nullptr) store_chunk<WF_F32, VEC>(dw, a.part_w + at, blockIdx.x, threadIdx.x, 256, a.d);
        if (a.part_b != nullptr) store_chunk<WF_F32, VEC>(db, a.part_b + at, blockIdx.x, threadIdx.x, 256, a.d);
    }
}

// ------------------------------------------------------------------------------------------------------------- host
bool vec_ok(const void *p, int64_t ld, int size) {
    return p == nullptr || (aligned_to(p, 16) && (ld * size) % 16 == 0);
}

// threads of the backward pass's block: 16 bytes of a row each, or (float32 past 4096 values) 32
int grad_threads(int d, int type) {
    const int v = type == WF_F32 && d <= 4 * kMaxThreads ? 4 : 8;
    return ((d + v - 1) / v + 31) / 32 * 32;
}

// Whether a cluster shares the rows in the backward pass (and in the forward pass of rows that 16-byte accesses do not fit):
// rows too wide for one block, up to 2048 columns a CTA, in us against the wide kernels: 4096 x 12288 bf16 109 / 157 and
// float32 205 / 236, 4096 x 16384 152 / 190 and 302 / 286, 8192 x 9999 bf16 279 / 519. Past that a CTA has the SM to itself and the
// exchange stands in the open (4096 x 20480 bf16 332 / 230, 2000 x 17777 float32 249 / 188); below it one block is faster
// (8192 x 8192 bf16 117 / 96).
bool is_team(int d) { return d > 8 * kMaxThreads && d <= kTeam * 8 * 256; }
int team_columns(int d) { return (d + 8 * kTeam - 1) / (8 * kTeam) * 8; }

// a block's threads for 8 values each, or the most there are
int row_threads(int d) { return std::min(kMaxThreads, ((d + 7) / 8 + 31) / 32 * 32); }

template <int T, int W, int NC, bool VEC>
int launch_norm_block(const NormArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_kernel<T, W, NC, VEC>;
    const int block = row_threads(a.d), grid = static_cast<int>(std::min<int64_t>(a.rows, wave_ctas_at<kern>(block)));
    return launch_rows(kern, dim3(grid), block, stream, a);
}

template <int T, int W>
int launch_norm_wide(const NormArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_wide_kernel<T, W>;
    const int grid = static_cast<int>(std::min<int64_t>(a.rows, wave_ctas_at<kern>(kMaxThreads)));
    return launch_rows(kern, dim3(grid), kMaxThreads, stream, a);
}

template <int T, int W, int NV>
int launch_norm_warp(const NormArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_warp_kernel<T, W, NV>;
    constexpr int per_block = 8 * (8 / NV);
    const int grid = static_cast<int>(std::min<int64_t>((a.rows + per_block - 1) / per_block, wave_ctas_at<kern>(256)));
    return launch_rows(kern, dim3(grid), 256, stream, a);
}

// blocks an SM of a kernel whose block's threads hold some 100 registers each
int blocks_by_threads(int threads) { return std::max(1, std::min(8, 640 / threads)); }

template <auto KERN>
cudaError_t allow_smem(int bytes) {
    static std::atomic<bool> ready[64];  // any host thread may launch first
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) ready[dev].store(true, std::memory_order_release);
    return e;
}
constexpr int kMostSmem = 200 * 1024;  // beside the kernels' static shared memory

template <int T, int W, int R, int THREADS, int BLOCKS, bool TEAM>
int launch_norm_unaligned(const NormArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_unaligned_kernel<T, W, R, THREADS, BLOCKS, TEAM>;
    cudaError_t e = allow_smem<kern>(kMostSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int cols = TEAM ? team_columns(a.d) : a.d, threads = row_threads(cols), smem = kRing * R * cover_bytes(cols, T);
    const int per_sm = std::max(1, std::min(blocks_by_threads(threads), 220 * 1024 / (smem + 2048)));
    const RowSplit split = make_split(a.rows, a.rows_per_group, std::max(1, per_sm * device_sm_count() / (TEAM ? kTeam : 1)), R);
    e = launch_dependent_clusters(kern, dim3(static_cast<unsigned>(split.blocks() * (TEAM ? kTeam : 1))), TEAM ? kTeam : 0,
                                  threads, smem, stream, a, split, cols);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// Rows that 16-byte accesses do not fit. R rows at a time: as many as the registers of so many threads hold, half as many of
// float32 (the ring's room).
template <int T, int W>
int dispatch_norm_unaligned(const NormArgs &a, cudaStream_t stream) {
    if (a.d <= 32) return launch_norm_warp<T, W, 1>(a, stream);
    if (a.d <= 64) return launch_norm_warp<T, W, 2>(a, stream);
    if (a.d <= 128) return launch_norm_warp<T, W, 4>(a, stream);
    if (a.d <= 256) return launch_norm_warp<T, W, 8>(a, stream);
    constexpr int R = T == WF_F32 ? 2 : 4;
    if (a.d <= 8 * 256) return launch_norm_unaligned<T, W, R, 256, 2, false>(a, stream);
    if (a.d <= 8 * 640) return launch_norm_unaligned<T, W, R / 2, 640, 1, false>(a, stream);
    if (a.d <= 8 * kMaxThreads) return launch_norm_unaligned<T, W, 1, kMaxThreads, 1, false>(a, stream);
    if (is_team(a.d)) return launch_norm_unaligned<T, W, R, 256, 2, true>(a, stream);
    if (a.d <= 24 * kMaxThreads) return launch_norm_block<T, W, 3, false>(a, stream);
    return launch_norm_wide<T, W>(a, stream);
}

template <int T, int W, int LPR>
int launch_norm_narrow(const NormArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_narrow_kernel<T, W, LPR>;
    constexpr int per_block = 8 * (32 / LPR);
    const int grid = static_cast<int>(std::min<int64_t>((a.rows + per_block - 1) / per_block, wave_ctas_at<kern>(256)));
    return launch_rows(kern, dim3(grid), 256, stream, a);
}

// rings of 2 to 4 rows a team, for blocks of about 64 KB where a row is short enough
template <int T, int W, int WPR>
int launch_norm_stream(const NormArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_stream_kernel<T, W, WPR>;
    constexpr int most = kMostSmem;
    const int64_t row = static_cast<int64_t>(a.d) * dtype_size(T) * (8 / WPR), params = 2ll * a.d * dtype_size(W);
    const bool params_fit = params + 2 * row <= most;
    const int bufs = static_cast<int>(std::max<int64_t>(2, std::min<int64_t>(4, (64 * 1024 - (params_fit ? params : 0)) / row)));
    cudaError_t e = allow_smem<kern>(most);
    if (e != cudaSuccess) return static_cast<int>(e);
    const bool stage = (a.w != nullptr || a.b != nullptr) && params_fit && std::min(a.rows_per_group, a.rows) >= kStageRows;
    const int64_t smem = bufs * row + (stage ? params : 0);
    const int64_t resident = std::max<int64_t>(1, std::min<int64_t>(6, 220 * 1024 / (smem + 1024))) * device_sm_count();
    const RowSplit split = make_split(a.rows, a.rows_per_group, resident, 8 / WPR);
    e = launch_dependent(kern, dim3(static_cast<unsigned>(split.blocks())), 256, smem, stream, a, split, bufs, stage);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <int T, int W>
int dispatch_norm(const NormArgs &a, cudaStream_t stream) {
    const bool vec = a.d % 8 == 0 && vec_ok(a.x, a.ldx, dtype_size(T)) && vec_ok(a.y, a.ldy, dtype_size(T)) &&
                     vec_ok(a.w, a.d, dtype_size(W)) && vec_ok(a.b, a.d, dtype_size(W));
    if (!vec) return dispatch_norm_unaligned<T, W>(a, stream);
    const int chunks = a.d / 8;
    if (chunks <= 4) return launch_norm_narrow<T, W, 4>(a, stream);
    if (chunks <= 8) return launch_norm_narrow<T, W, 8>(a, stream);
    if (chunks <= 16) return launch_norm_narrow<T, W, 16>(a, stream);
    if (chunks <= 32) return launch_norm_narrow<T, W, 32>(a, stream);
    // Teams of warps where there are rows for them, else a row a block. Larger teams leave room for more rows in flight, at
    // a barrier a sum: 16384 x 2048 with teams of 1 / 2 / 4 27.4 / 31.1 / 43.7 us, 16384 x 5120 63.5 / 61.7 / 67.0, 8192 x 8192
    // with 2 / 4 / 8 55.4 / 50.8 / 55.3, 4096 x 12288 with 4 / 8 46.1 / 44.0.
    const int kb = (a.d * dtype_size(T) + 1023) / 1024;
    if (a.rows >= 4ll * device_sm_count()) {
        if (kb <= 8) return launch_norm_stream<T, W, 1>(a, stream);
        if (kb <= 12) return launch_norm_stream<T, W, 2>(a, stream);
        if (kb <= 20) return launch_norm_stream<T, W, 4>(a, stream);
        if (kb <= 80) return launch_norm_stream<T, W, 8>(a, stream);
    }
    if (a.d <= 8 * kMaxThreads) return launch_norm_block<T, W, 1, true>(a, stream);
    if (a.d <= 16 * kMaxThreads) return launch_norm_block<T, W, 2, true>(a, stream);
    if (a.d <= 24 * kMaxThreads) return launch_norm_block<T, W, 3, true>(a, stream);
    return launch_norm_wide<T, W>(a, stream);
}

template <int T, int W, bool VEC>
int launch_norm_grad_wide(const NormGradArgs &a, cudaStream_t stream) {
    int rc = WF_OK;
    if (a.dx != nullptr) {
        constexpr auto kern = layer_norm_grad_wide_kernel<T, W, VEC>;
        const int grid = static_cast<int>(std::min<int64_t>(a.rows, wave_ctas_at<kern>(kMaxThreads)));
        rc = launch_rows(kern, dim3(grid), kMaxThreads, stream, a);
    }
    if (rc == WF_OK && (a.part_w != nullptr || a.part_b != nullptr))
        rc = launch_rows(layer_norm_column_kernel<T, VEC>, dim3((a.d + 2047) / 2048, static_cast<unsigned>(a.split.blocks())),
                         256, stream, a);
    return rc;
}

template <int T, int W, int V, int R, int THREADS, int BLOCKS, bool TEAM>
int launch_norm_grad_rows(const NormGradArgs &a, int threads, cudaStream_t stream) {
    constexpr auto kern = layer_norm_grad_rows_kernel<T, W, V, R, THREADS, BLOCKS, TEAM>;
    constexpr int per_thread = kRing * R * 2 * V * dtype_size(T);
    cudaError_t e = allow_smem<kern>(THREADS * per_thread);
    if (e != cudaSuccess) return static_cast<int>(e);
    e = launch_dependent_clusters(kern, dim3(static_cast<unsigned>(a.split.blocks() * (TEAM ? kTeam : 1))), TEAM ? kTeam : 0,
                                  threads, static_cast<size_t>(threads) * per_thread, stream, a);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <int T, int W, int R, int THREADS, int BLOCKS, bool TEAM>
int launch_norm_grad_unaligned(const NormGradArgs &a, cudaStream_t stream) {
    constexpr auto kern = layer_norm_grad_unaligned_kernel<T, W, R, THREADS, BLOCKS, TEAM>;
    cudaError_t e = allow_smem<kern>(kMostSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    e = launch_dependent_clusters(kern, dim3(static_cast<unsigned>(a.split.blocks() * (TEAM ? kTeam : 1))), TEAM ? kTeam : 0,
                                  row_threads(a.block_cols), kRing * R * 2 * cover_bytes(a.block_cols, T), stream, a);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// R as in the forward pass
template <int T, int W>
int dispatch_norm_grad_unaligned(const NormGradArgs &a, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.split.blocks()));
    if (a.d <= 32) return launch_rows(layer_norm_grad_warp_kernel<T, W, 1>, grid, 256, stream, a);
    if (a.d <= 64) return launch_rows(layer_norm_grad_warp_kernel<T, W, 2>, grid, 256, stream, a);
    if (a.d <= 128) return launch_rows(layer_norm_grad_warp_kernel<T, W, 4>, grid, 256, stream, a);
    if (a.d <= 256) return launch_rows(layer_norm_grad_warp_kernel<T, W, 8>, grid, 256, stream, a);
    constexpr int R = T == WF_F32 ? 2 : 4;
    if (a.d <= 8 * 256) return launch_norm_grad_unaligned<T, W, R, 256, 2, false>(a, stream);
    if (a.d <= 8 * 640) return launch_norm_grad_unaligned<T, W, R / 2, 640, 1, false>(a, stream);
    if (a.d <= 8 * kMaxThreads) return launch_norm_grad_unaligned<T, W, 1, kMaxThreads, 1, false>(a, stream);
    if (is_team(a.d)) return launch_norm_grad_unaligned<T, W, R, 256, 2, true>(a, stream);
    return launch_norm_grad_wide<T, W, false>(a, stream);
}

template <int T, int W>
int dispatch_norm_grad(const NormGradArgs &a, cudaStream_t stream) {
    const bool vec = a.d % 8 == 0 && vec_ok(a.x, a.ldx, dtype_size(T)) && vec_ok(a.dy, a.lddy, dtype_size(T)) &&
                     vec_ok(a.dx, a.lddx, dtype_size(T)) && vec_ok(a.w, a.d, dtype_size(W)) && vec_ok(a.part_w, a.d, 4) &&
                     vec_ok(a.part_b, a.d, 4);
    if (!vec || (T == WF_F32 && is_team(a.d))) return dispatch_norm_grad_unaligned<T, W>(a, stream);
    if constexpr (T != WF_F32) {
        if (is_team(a.d)) return launch_norm_grad_rows<T, W, 8, 4, 256, 2, true>(a, grad_threads(a.block_cols, T), stream);
    }
    if (a.d > 8 * kMaxThreads) return launch_norm_grad_wide<T, W, true>(a, stream);
    const dim3 grid(static_cast<unsigned>(a.split.blocks()));
    if (a.d <= 32) return launch_rows(layer_norm_grad_narrow_kernel<T, W, 4>, grid, 256, stream, a);
    if (a.d <= 64) return launch_rows(layer_norm_grad_narrow_kernel<T, W, 8>, grid, 256, stream, a);
    if (a.d <= 128) return launch_rows(layer_norm_grad_narrow_kernel<T, W, 16>, grid, 256, stream, a);
    if (a.d <= 256) return launch_rows(layer_norm_grad_narrow_kernel<T, W, 32>, grid, 256, stream, a);
    constexpr int V = T == WF_F32 ? 4 : 8;  // 16 bytes a thread; float32 rows past 4096 values take 32
    const int threads = grad_threads(a.d, T);
    if constexpr (T == WF_F32) {
        if (a.d > V * kMaxThreads) return launch_norm_grad_rows<T, W, 8, 1, kMaxThreads, 1, false>(a, threads, stream);
    }
    if (threads <= 256) return launch_norm_grad_rows<T, W, V, 4, 256, 2, false>(a, threads, stream);
    if (threads <= 640) return launch_norm_grad_rows<T, W, V, 2, 640, 1, false>(a, threads, stream);
    return launch_norm_grad_rows<T, W, V, 1, kMaxThreads, 1, false>(a, threads, stream);
}

bool norm_types_ok(int type, int w_type) {
    return (type == WF_F16 || type == WF_BF16 || type == WF_F32) && (w_type == type || w_type == WF_F32);
}

// The shares of the rows that the backward pass's blocks take: about as many as are resident at once.
RowSplit norm_split(int64_t rows, int64_t rows_per_group, int d, int type) {
    const int64_t sms = device_sm_count();
    if (is_team(d)) return make_split(rows, rows_per_group, std::max<int64_t>(1, blocks_by_threads(row_threads(team_columns(d))) * sms / kTeam), 4);
    if (d > 8 * kMaxThreads) return make_split(rows, rows_per_group, std::max<int64_t>(1, 4 * sms * 2048 / d), 16);
    if (d <= 256) return make_split(rows, rows_per_group, 3 * sms, 16);
    return make_split(rows, rows_per_group, sms * blocks_by_threads(d % 8 == 0 ? grad_threads(d, type) : row_threads(d)), 4);
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

extern "C" WF_API int64_t wf_layer_norm_backward_workspace(int64_t rows, int64_t d, int64_t rows_per_group, int type) {
    using namespace wf;
    if (rows < 1 || d < 1 || d > (1 << 30) || rows_per_group < 1) return 0;
    return 2 * norm_split(rows, rows_per_group, static_cast<int>(d), type).partial_rows() * d * static_cast<int64_t>(sizeof(float));
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
    const RowSplit split = norm_split(g.rows, g.rows_per_group, static_cast<int>(g.d), g.type);
    const int64_t half = split.partial_rows() * g.d;
    const int d = static_cast<int>(g.d);
    if ((g.dw || g.db) && (!g.workspace || !aligned_to(g.workspace, 16) ||
                           g.workspace_bytes < 2 * half * static_cast<int64_t>(sizeof(float))))
        return WF_ERR_ARG;
    int rc = check_device();
    if (rc != WF_OK) return rc;
    float *part = static_cast<float *>(g.workspace);
    const NormGradArgs a{g.x, g.w, g.dy, g.mean, g.rstd, g.dx, g.dw ? part : nullptr, g.db ? part + half : nullptr, g.rows,
                         g.ldx, g.lddy, g.lddx, split, d, is_team(d) ? team_columns(d) : d};
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (g.type == WF_F32) rc = dispatch_norm_grad<WF_F32, WF_F32>(a, st);
    else if (g.type == WF_BF16) rc = g.w_type == WF_F32 ? dispatch_norm_grad<WF_BF16, WF_F32>(a, st) : dispatch_norm_grad<WF_BF16, WF_BF16>(a, st);
    else rc = g.w_type == WF_F32 ? dispatch_norm_grad<WF_F16, WF_F32>(a, st) : dispatch_norm_grad<WF_F16, WF_F16>(a, st);
    if (rc != WF_OK) return rc;
    const int64_t parts = split.partials_per_group();
    return reduce_partials(PartialSum{a.part_w, g.dw, split.groups, parts}, PartialSum{a.part_b, g.db, split.groups, parts},
                           g.d, g.w_type, st);
}
