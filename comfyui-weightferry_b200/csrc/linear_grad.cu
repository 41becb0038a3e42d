// The element-wise half of the dense linear layer's backward pass, one pass over dy and the kept z:
//
//   dh = g[row / rows_per_group] * dy,  dz = dh * act'(z)
//   db = sum over all rows of dz,  dg[grp] = sum over the group's rows of dy * act(z)
//
// dz is rounded to the layer's type, which the two products after it take (db is summed from the unrounded values);
// both sums are float32. A thread owns eight neighbouring columns and every eighth row of its block's share, so the
// sums stay in registers; a block writes them as a row of partial sums, which reduce_partials adds in a fixed order.
// Bound by HBM: dy and z in, dz out.

#include "wf_act.cuh"
#include "wf_linear.cuh"
#include "wf_rows.cuh"

namespace wf {
namespace {

constexpr int kGradCols = 256;  // columns of a block: 32 lanes x 8
constexpr int kGradRows = 8;    // rows in flight: one a warp

struct LinearGradArgs {
    const void *dy, *z, *gate;
    void *dz;                 // or null
    float *part_b;            // [blocks, n], or null
    float *part_g;            // [groups * chunks, n], or null
    int64_t lddy, ldz, lddz, n;
    RowSplit split;
    bool vec;
};

// z as it was kept: of the layer's type T, f16 or f32
template <int Z>
__device__ __forceinline__ void load_z(float (&v)[8], const LinearGradArgs &a, int64_t row, int64_t col, bool vec) {
    const void *zr = row_of<Z>(a.z, row, a.ldz);
    if (vec) {
        load8<Z>(v, zr, col);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = col + j < a.n ? load1<Z>(zr, col + j) : 0.f;
    }
}

// ZN: no z (no activation and no gradient of the gate)
template <int T, int Z, int ACT, bool ZN>
__global__ void __launch_bounds__(256) linear_grad_kernel(const __grid_constant__ LinearGradArgs a) {
    __shared__ float red[kGradRows][kGradCols];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kGradCols + lane * 8;
    const bool vec = a.vec && col + 8 <= a.n;
    wait_prior_grid();
    float db[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) db[j] = 0.f;
    auto reduce_to = [&](float (&v)[8], float *dst) {  // the warps' sums, to this block's columns of dst
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) red[warp][j * 32 + lane] = v[j];
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kGradRows; ++w) s += red[w][threadIdx.x];
        const int64_t at = static_cast<int64_t>(blockIdx.x) * kGradCols + (threadIdx.x & 31) * 8 + (threadIdx.x >> 5);
        if (at < a.n) dst[at] = s;
    };
    for (int64_t grp = a.split.first_group(blockIdx.y), end = a.split.last_group(blockIdx.y); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.y, grp, lo, hi);
        float g[8], dg[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = a.gate != nullptr && col + j < a.n ? load1<T>(row_of<T>(a.gate, grp, a.n), col + j) : 1.f;
            dg[j] = 0.f;
        }
#pragma unroll 2
        for (int64_t row = lo + warp; row < hi; row += kGradRows) {
            float dy[8], z[8];
            const void *yr = row_of<T>(a.dy, row, a.lddy);
            if (vec) {
                load8<T>(dy, yr, col);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) dy[j] = col + j < a.n ? load1<T>(yr, col + j) : 0.f;
            }
            if constexpr (!ZN) load_z<Z>(z, a, row, col, vec);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float h[2], slope[2] = {1.f, 1.f};
                if constexpr (!ZN) {
                    const float v[2] = {z[j], z[j + 1]};
                    act_slope2<ACT>(v, h, slope);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (!ZN) dg[j + i] = fmaf(dy[j + i], h[i], dg[j + i]);
                    dy[j + i] *= g[j + i] * slope[i];
                    db[j + i] += dy[j + i];
                }
            }
            if (a.dz != nullptr) {
                void *dr = row_of<T>(a.dz, row, a.lddz);
                if (vec) {
                    store8<T, true>(static_cast<uint16_t *>(dr) + col, dy);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col + j < a.n) store1<T>(dr, col + j, dy[j]);
                }
            }
        }
        if (a.part_g != nullptr) reduce_to(dg, a.part_g + a.split.partial_row(blockIdx.y, grp) * a.n);
    }
    if (a.part_b != nullptr) reduce_to(db, a.part_b + static_cast<int64_t>(blockIdx.y) * a.n);
}

RowSplit grad_split(int64_t m, int64_t n, int64_t rows_per_group) {
    const int64_t across = (n + kGradCols - 1) / kGradCols;
    const int64_t wanted = std::min<int64_t>(32768, std::max<int64_t>(1, 8ll * device_sm_count() / across));
    return make_split(m, rows_per_group, wanted, kGradRows);
}

template <int T, int Z, int ACT>
int launch_grad(const LinearGradArgs &a, cudaStream_t stream) {
    return launch_rows(linear_grad_kernel<T, Z, ACT, false>,
                       dim3(static_cast<unsigned>((a.n + kGradCols - 1) / kGradCols), static_cast<unsigned>(a.split.blocks())),
                       256, stream, a);
}

template <int T, int Z>
int dispatch_grad(const LinearGradArgs &a, int act, cudaStream_t stream) {
    switch (act) {
        case WF_ACT_RELU: return launch_grad<T, Z, WF_ACT_RELU>(a, stream);
        case WF_ACT_SILU: return launch_grad<T, Z, WF_ACT_SILU>(a, stream);
        case WF_ACT_GELU: return launch_grad<T, Z, WF_ACT_GELU>(a, stream);
        case WF_ACT_GELU_TANH: return launch_grad<T, Z, WF_ACT_GELU_TANH>(a, stream);
        default: return launch_grad<T, Z, WF_ACT_NONE>(a, stream);
    }
}

template <int T>
int dispatch_grad_type(const LinearGradArgs &a, int act, int z_type, cudaStream_t stream) {
    if (a.z == nullptr)
        return launch_rows(linear_grad_kernel<T, T, WF_ACT_NONE, true>,
                           dim3(static_cast<unsigned>((a.n + kGradCols - 1) / kGradCols),
                                static_cast<unsigned>(a.split.blocks())),
                           256, stream, a);
    if (z_type == WF_F32) return dispatch_grad<T, WF_F32>(a, act, stream);
    if (z_type == WF_F16) return dispatch_grad<T, WF_F16>(a, act, stream);
    return dispatch_grad<T, T>(a, act, stream);
}

}  // namespace

// rows of a group as the kernel takes them: all of them where no group matters
static int64_t grad_group(const wf_linear_grad_args &g) { return g.gate || g.dg ? g.rows_per_group : g.m; }

int64_t linear_grad_workspace(int64_t m, int64_t n, int64_t rows_per_group) {
    const RowSplit s = grad_split(m, n, rows_per_group);
    return (s.blocks() + s.partial_rows()) * n * static_cast<int64_t>(sizeof(float));
}

int linear_grad(const wf_linear_grad_args &g, void *dz, int64_t lddz, float *part, cudaStream_t stream) {
    const RowSplit split = grad_split(g.m, g.n, grad_group(g));
    const bool vec = aligned_to(g.dy, 16) && g.lddy % 8 == 0 && (!dz || (aligned_to(dz, 16) && lddz % 8 == 0)) &&
                     (!g.z || (aligned_to(g.z, 16) && g.ldz % 8 == 0));
    LinearGradArgs a{g.dy, g.z, g.gate, dz, g.db ? part : nullptr, g.dg ? part + split.blocks() * g.n : nullptr, g.lddy,
                     g.ldz, lddz, g.n, split, vec};
    const int rc = g.type == WF_BF16 ? dispatch_grad_type<WF_BF16>(a, g.act, g.z_type, stream)
                                     : dispatch_grad_type<WF_F16>(a, g.act, g.z_type, stream);
    if (rc != WF_OK) return rc;
    return reduce_partials(PartialSum{a.part_b, g.db, 1, split.blocks()},
                           PartialSum{a.part_g, g.dg, split.groups, split.partials_per_group()}, g.n, g.type, stream);
}

}  // namespace wf
