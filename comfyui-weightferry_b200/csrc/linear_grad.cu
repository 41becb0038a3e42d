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
#include "wf_pairs.cuh"
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
__device__ __forceinline__ void load_z(float (&v)[8], const LinearGradArgs &a, int64_t row, int64_t col) {
    const void *zr = row_of<Z>(a.z, row, a.ldz);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j < a.n ? load1<Z>(zr, col + j) : 0.f;
}

// Any width and alignment. ZN: no z (no activation and no gradient of the gate)
template <int T, int Z, int ACT, bool ZN>
__global__ void __launch_bounds__(256) linear_grad_kernel(const __grid_constant__ LinearGradArgs a) {
    __shared__ float red[kGradRows][kGradCols];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kGradCols + lane * 8;
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
#pragma unroll
            for (int j = 0; j < 8; ++j) dy[j] = col + j < a.n ? load1<T>(yr, col + j) : 0.f;
            if constexpr (!ZN) load_z<Z>(z, a, row, col);
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
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col + j < a.n) store1<T>(dr, col + j, dy[j]);
            }
        }
        if (a.part_g != nullptr) reduce_to(dg, a.part_g + a.split.partial_row(blockIdx.y, grp) * a.n);
    }
    if (a.part_b != nullptr) reduce_to(db, a.part_b + static_cast<int64_t>(blockIdx.y) * a.n);
}

// The same for eight columns that 16-byte accesses fit, without a gate of its own row group and its gradient where GATE is
// false. Each thread copies its own values of the next rows into a ring of kRing rows in shared memory (cp.async) and
// reads nobody else's: with the loads in registers instead, two rows ahead, the pass took 138 us on 8192 x 8192 where it
// now takes 77. ZN: no z (no activation and no gradient of the gate).
constexpr int kRing = 4;
template <int T, int Z, int ACT, bool ZN, bool GATE>
__global__ void __launch_bounds__(256, 3) linear_grad_vec_kernel(const __grid_constant__ LinearGradArgs a) {
    constexpr int ZP = ZN ? 0 : Z == WF_F32 ? 2 : 1, P = 1 + ZP;  // 16-byte pieces a row: dy, then z
    extern __shared__ uint4 ring[];                              // [kRing][P][256]; the column sums at the end
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kGradCols + lane * 8;
    const bool in = col < a.n;
    const int64_t c = in ? col : 0;
    wait_prior_grid();
    uint64_t db[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) db[j] = 0;  // +0, +0
    auto reduce_to = [&](const uint64_t (&v)[4], float *dst) {  // the warps' sums, to this block's columns of dst
        float *red = reinterpret_cast<float *>(ring);           // [8][kGradCols + 8]
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float lo, hi;
            unpack_f2(v[j], lo, hi);
            *reinterpret_cast<float2 *>(red + warp * (kGradCols + 8) + lane * 8 + 2 * j) = make_float2(lo, hi);
        }
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kGradRows; ++w) s += red[w * (kGradCols + 8) + tid];
        const int64_t at = static_cast<int64_t>(blockIdx.x) * kGradCols + tid;
        if (at < a.n) dst[at] = s;
        __syncthreads();
    };
    for (int64_t grp = a.split.first_group(blockIdx.y), end = a.split.last_group(blockIdx.y); grp < end; ++grp) {
        int64_t lo, hi;
        a.split.rows_of(blockIdx.y, grp, lo, hi);
        auto fetch = [&](int64_t row, int slot) {  // one copy group a row, empty past the last
            if (in && row < hi) {
                uint4 *dst = ring + slot * P * 256 + tid;
                copy16(dst, static_cast<const uint16_t *>(row_of<T>(a.dy, row, a.lddy)) + c);
                if constexpr (!ZN) {
                    const char *z = static_cast<const char *>(row_of<Z>(a.z, row, a.ldz)) + c * dtype_size(Z);
#pragma unroll
                    for (int p = 0; p < ZP; ++p) copy16(dst + (1 + p) * 256, z + 16 * p);
                }
            }
            cp_async_commit();
        };
        int64_t ahead = lo + warp;
        for (int i = 0; i < kRing - 1; ++i, ahead += kGradRows) fetch(ahead, i);
        uint64_t g[4], dg[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) dg[j] = 0;
        if (GATE && a.gate != nullptr) {
            float v[8];
            const void *gr = row_of<T>(a.gate, grp, a.n);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = load1<T>(gr, c + j);
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = pack_f2(v[2 * j], v[2 * j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = pack_f2(1.f, 1.f);
        }
        int slot = 0, next = kRing - 1;
        for (int64_t row = lo + warp; row < hi; row += kGradRows, ahead += kGradRows) {
            fetch(ahead, next);
            if (++next == kRing) next = 0;
            cp_async_wait<kRing - 1>();
            const uint4 *src = ring + slot * P * 256 + tid;
            if (++slot == kRing) slot = 0;
            if (!in) continue;
            const uint4 q = src[0];
            const uint32_t y[4] = {q.x, q.y, q.z, q.w};
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = unpack2<T>(y[j]);
                uint64_t dy = pack_f2(f.x, f.y), dz = dy;
                if constexpr (!ZN) {
                    float v[2], h[2], slope[2];
                    if constexpr (Z == WF_F32) {
                        const float2 z = reinterpret_cast<const float2 *>(src + (1 + j / 2) * 256)[j & 1];
                        v[0] = z.x, v[1] = z.y;
                    } else {
                        const float2 z = unpack2<Z>(reinterpret_cast<const uint32_t *>(src + 256)[j]);
                        v[0] = z.x, v[1] = z.y;
                    }
                    act_slope2<ACT>(v, h, slope);
                    if constexpr (GATE) dg[j] = fma_f2(dy, pack_f2(h[0], h[1]), dg[j]);
                    dz = mul_f2(dz, pack_f2(slope[0], slope[1]));
                }
                if constexpr (GATE) dz = mul_f2(dz, g[j]);
                db[j] = add_f2(db[j], dz);
                float o0, o1;
                unpack_f2(dz, o0, o1);
                out[j] = pack2<T>(o0, o1);
            }
            if (a.dz != nullptr)
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(row_of<T>(a.dz, row, a.lddz)) + c) =
                    make_uint4(out[0], out[1], out[2], out[3]);
        }
        if (GATE && a.part_g != nullptr) reduce_to(dg, a.part_g + a.split.partial_row(blockIdx.y, grp) * a.n);
    }
    if (a.part_b != nullptr) reduce_to(db, a.part_b + static_cast<int64_t>(blockIdx.y) * a.n);
    cp_async_wait<0>();
}

RowSplit grad_split(int64_t m, int64_t n, int64_t rows_per_group) {
    const int64_t across = (n + kGradCols - 1) / kGradCols;
    const int64_t wanted = std::min<int64_t>(32768, std::max<int64_t>(1, 6ll * device_sm_count() / across));
    return make_split(m, rows_per_group, wanted, kGradRows);
}

template <int T, int Z, int ACT, bool ZN, bool GATE>
int launch_grad_vec(const LinearGradArgs &a, dim3 grid, cudaStream_t stream) {
    constexpr int ring = kRing * (ZN ? 1 : Z == WF_F32 ? 3 : 2) * 256 * 16, red = kGradRows * (kGradCols + 8) * 4;
    constexpr auto kern = linear_grad_vec_kernel<T, Z, ACT, ZN, GATE>;
    const cudaError_t e = launch_dependent(kern, grid, 256, std::max(ring, red), stream, a);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <int T, int Z, int ACT, bool ZN>
int launch_grad(const LinearGradArgs &a, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((a.n + kGradCols - 1) / kGradCols), static_cast<unsigned>(a.split.blocks()));
    if (!a.vec) return launch_rows(linear_grad_kernel<T, Z, ACT, ZN>, grid, 256, stream, a);
    return a.gate != nullptr || a.part_g != nullptr ? launch_grad_vec<T, Z, ACT, ZN, true>(a, grid, stream)
                                                    : launch_grad_vec<T, Z, ACT, ZN, false>(a, grid, stream);
}

template <int T, int Z>
int dispatch_grad(const LinearGradArgs &a, int act, cudaStream_t stream) {
    switch (act) {
        case WF_ACT_RELU: return launch_grad<T, Z, WF_ACT_RELU, false>(a, stream);
        case WF_ACT_SILU: return launch_grad<T, Z, WF_ACT_SILU, false>(a, stream);
        case WF_ACT_GELU: return launch_grad<T, Z, WF_ACT_GELU, false>(a, stream);
        case WF_ACT_GELU_TANH: return launch_grad<T, Z, WF_ACT_GELU_TANH, false>(a, stream);
        default: return launch_grad<T, Z, WF_ACT_NONE, false>(a, stream);
    }
}

template <int T>
int dispatch_grad_type(const LinearGradArgs &a, int act, int z_type, cudaStream_t stream) {
    if (a.z == nullptr) return launch_grad<T, T, WF_ACT_NONE, true>(a, stream);
    if (z_type == WF_F32) return dispatch_grad<T, WF_F32>(a, act, stream);
    if (z_type == WF_F16) return dispatch_grad<T, WF_F16>(a, act, stream);
    return dispatch_grad<T, T>(a, act, stream);
}

}  // namespace

// rows of a group as the kernel takes them: all of them where no group matters
static int64_t grad_group(const wf_linear_grad_args &g) { return g.gate || g.dg ? g.rows_per_group : g.m; }

int64_t linear_grad_bytes(const wf_linear_grad_args &g) {
    const RowSplit s = grad_split(g.m, g.n, grad_group(g));
    return ((g.db ? s.blocks() : 0) + (g.dg ? s.partial_rows() : 0)) * g.n * static_cast<int64_t>(sizeof(float));
}

int64_t linear_grad_most_bytes(int64_t m, int64_t n, int64_t rows_per_group) {
    const RowSplit grouped = grad_split(m, n, rows_per_group), plain = grad_split(m, n, m);
    return std::max(grouped.blocks() + grouped.partial_rows(), plain.blocks()) * n * static_cast<int64_t>(sizeof(float));
}

int linear_grad(const wf_linear_grad_args &g, void *dz, int64_t lddz, float *part, cudaStream_t stream) {
    const RowSplit split = grad_split(g.m, g.n, grad_group(g));
    const bool vec = g.n % 8 == 0 && aligned_to(g.dy, 16) && g.lddy % 8 == 0 && (!dz || (aligned_to(dz, 16) && lddz % 8 == 0)) &&
                     (!g.z || (aligned_to(g.z, 16) && g.ldz % 8 == 0));
    LinearGradArgs a{g.dy, g.z, g.gate, dz, g.db ? part : nullptr, g.dg ? part + (g.db ? split.blocks() * g.n : 0) : nullptr, g.lddy,
                     g.ldz, lddz, g.n, split, vec};
    const int rc = g.type == WF_BF16 ? dispatch_grad_type<WF_BF16>(a, g.act, g.z_type, stream)
                                     : dispatch_grad_type<WF_F16>(a, g.act, g.z_type, stream);
    if (rc != WF_OK) return rc;
    return reduce_partials(PartialSum{a.part_b, g.db, 1, split.blocks()},
                           PartialSum{a.part_g, g.dg, split.groups, split.partials_per_group()}, g.n, g.type, stream);
}

}  // namespace wf
