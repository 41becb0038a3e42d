// The dense linear layer of 16-bit weights for sm_100a: matrix products on tcgen05 tensor cores with the bias, the
// activation and the gated residual in the epilogue, and the two products of its backward pass.
//
//   forward    z = x W^T + b,  y = r + g[row / rows_per_group] * act(z)        x [m, k], W [n, k]
//   backward   dx = dz W,  dW = dz^T x                                          dz [m, n] (linear_grad.cu)
//
// All three are D[i, j] = sum_c A[i, c] B[j, c] with A and B read as they lie in memory: an operand whose contraction
// index c is the contiguous one ("c-major": x and W of the forward pass, dz of dx) or whose row index is ("row-major":
// W of dx, dz and x of dW). The tensor core takes both from shared memory, so nothing is transposed first. Products are
// summed in float32 in tensor memory; the epilogue works in float32 and rounds once, to the output's type.

#include "wf_act.cuh"
#include "wf_linear.cuh"
#include "wf_rows.cuh"
#include "wf_tcgen05.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace wf {
namespace {

constexpr int BC = 64;  // contraction values of a stage: 128 bytes of 16-bit values, one swizzle row

__device__ int g_linear_status;  // 0 ok; 1 producer wait expired; 2 MMA wait expired; 3 epilogue wait expired

// What a pipeline wait needs to know beside its barrier: the CTA's abort flag, a word in mapped host memory that tells the
// host's next call, and the time limit.
struct Waits {
    volatile int *abort_flag, *alarm;
    uint64_t limit_ns;
};

// Wait for the phase of the given parity, at most limit_ns; gives up early when another role aborted. A try suspends for some
// microseconds, so that a limit shortened by a test is looked at after each.
__device__ __forceinline__ bool pipe_wait(uint32_t a, uint32_t parity, const Waits &w, int code) {
    if (mbar_try(a, parity)) return true;
    const uint64_t t0 = global_ns();
    const int tries = w.limit_ns < 1000000u ? 1 : 32;
    while (true) {
#pragma unroll 1
        for (int i = 0; i < tries; ++i)
            if (mbar_try(a, parity)) return true;
        if (*w.abort_flag) return false;
        if (global_ns() - t0 > w.limit_ns) {
            *w.abort_flag = 1;
            atomicCAS(&g_linear_status, 0, code);
            *w.alarm = code;
            return false;
        }
    }
}

// Shared-memory matrix descriptors, 128-byte swizzle, as two words: the high one is constant, the low one holds the
// address in 16 bytes, to which a stage or a step within it is a plain addition. One thread issues every MMA of a tile, so
// its instructions count: with descriptors put together from scratch (some 100 instructions a stage) a stage took 0.30 us
// however small its tile was.
//   c-major operand: rows 128 B apart, 8 rows 1024 B apart; 16 contraction indexes are the next 32 B
//   row-major operand: 64 rows (128 B) of one contraction index side by side, 8 contraction indexes 1024 B apart (stride
//     byte offset), the next 64 rows BC * 128 B on (leading byte offset); 16 contraction indexes are 2048 B
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride offset, version, 128-byte swizzle
template <bool ROWS>
__device__ __forceinline__ uint32_t desc_low(uint32_t addr) {  // the mask drops the CTA's rank in its cluster
    return ((addr >> 4) & 0x3FFFu) | ((ROWS ? BC * 128u >> 4 : 1u) << 16);
}
template <bool ROWS>
constexpr uint32_t kDescStep = ROWS ? 2048u >> 4 : 32u >> 4;

// instruction descriptor of kind::f16: D float32 (bits 4-5 = 1), A and B f16 (0) or bf16 (1) at bits 7-9 and 10-12,
// row-major A / B at bits 15 / 16, N >> 3 at bits 17-22, M >> 4 at bits 24-28
constexpr uint32_t f16_idesc(bool bf16, bool a_rows, bool b_rows, int m, int n) {
    return (1u << 4) | (static_cast<uint32_t>(bf16) << 7) | (static_cast<uint32_t>(bf16) << 10) |
           (static_cast<uint32_t>(a_rows) << 15) | (static_cast<uint32_t>(b_rows) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
#define WF_MMA_F16(GROUP)                                                             \
    asm volatile(                                                                     \
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"                               \
        "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t" \
        "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], da, db, %4, p;\n\t}"          \
        ::"r"(d_tmem), "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(accumulate) : "memory")
    if constexpr (PAIR) WF_MMA_F16("2");
    else WF_MMA_F16("1");
#undef WF_MMA_F16
}

// True in one lane of a converged warp. The roles that issue loads and MMAs run their loops in all lanes and only the
// issue itself in one: the compiler then knows loop counters, addresses and descriptors to be the same in every lane and
// keeps them in uniform registers, where those instructions want them. With the whole loop in lane 0, each MMA waited some
// 50 cycles for its operands to get there and each stage 340 more (547 cycles a stage, more than its MMAs take).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
// this thread's warp in its block, known to be the same in every lane
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x >> 5), 0); }

// tcgen05.ld of 16 consecutive columns of this thread's lane
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// What the epilogue does with z = D + bias: saved (for the backward pass) as keep says, then out = r + g * act(z).
enum { KEEP_NONE = 0, KEEP_F16 = 1, KEEP_F32 = 2, KEEP_SAME = 3 };
struct Epilogue {
    const void *bias;   // [n] or null
    const void *gate;   // [groups, n] or null
    const void *resid;  // [m, ld_resid] or null
    void *out;          // [m, ld_out]
    void *kept;         // [m, ld_kept] or null
    int *alarm;         // set when a wait runs out of time ...
    uint64_t wait_ns;   // ... and when that is
    int64_t ld_resid, ld_out, ld_kept, rows_per_group;
    int act, keep;
    bool vec;  // every pointer 8-byte aligned and every row pitch (n too, where it is one) a multiple of 4 values
    bool vec_bias;  // the pair kernel's: 16-byte accesses to the bias, whatever n is
};

// float32 -> f16, clamped to f16's range: the kept z is read by the slopes alone, which are constant out there, and
// f16's 11 bits keep a bf16 layer's gradients as exact as their own rounding. relu's slope steps at 0, so there no positive z
// may round to 0 (f16 ends at 2^-24, bf16 layers reach much further down).
__device__ __forceinline__ uint32_t pack2_sat(float a, float b, bool relu) {
    if (relu) {
        a = a > 0.f ? fmaxf(a, 0x1p-24f) : a;
        b = b > 0.f ? fmaxf(b, 0x1p-24f) : b;
    }
    uint32_t w;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}

template <int ACT, int R>
__device__ __forceinline__ void act4(float (&v)[R][4]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        act2<ACT>(v[r][0], v[r][1]);
        act2<ACT>(v[r][2], v[r][3]);
    }
}
template <int R>
__device__ __forceinline__ void apply_act4(int kind, float (&v)[R][4]) {
    switch (kind) {
        case WF_ACT_RELU: act4<WF_ACT_RELU>(v); break;
        case WF_ACT_SILU: act4<WF_ACT_SILU>(v); break;
        case WF_ACT_GELU: act4<WF_ACT_GELU>(v); break;
        case WF_ACT_GELU_TANH: act4<WF_ACT_GELU_TANH>(v); break;
        default: break;
    }
}

// Four values of a row: neighbours in one 8-byte access, or (VEC false) 32 columns apart, so that a warp's single-value
// accesses share their sectors; those at and past n as 0
template <int T, bool VEC>
__device__ __forceinline__ void load4(float (&v)[4], const void *row, int col, int n) {
    if constexpr (VEC) {
        const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(row) + col);
        const float2 a = unpack2<T>(q.x), b = unpack2<T>(q.y);
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = col + 32 * i < n ? load1<T>(row, col + 32 * i) : 0.f;
    }
}
template <int T, bool VEC>
__device__ __forceinline__ void store4(void *row, int col, int n, const float (&v)[4]) {
    if constexpr (VEC) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(row) + col) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + 32 * i < n) store1<T>(row, col + 32 * i, v[i]);
    }
}

// The epilogue of four outputs (load4's columns) in each of R rows (row, row + step, ...; those from row_end on are left out).
// Several rows share each of its branches, and their chains of loads and arithmetic overlap.
template <int T, bool VEC, int R>
__device__ __forceinline__ void finish4(const Epilogue &e, float (&v)[R][4], int row, int step, int row_end, int col, int n) {
    constexpr int C = VEC ? 1 : 32;
    float o[R][4];
    if (e.bias != nullptr) {
        load4<T, VEC>(o[0], e.bias, col, n);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] += o[0][i];
    }
    if (e.keep != KEEP_NONE) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int at = row + r * step;
            if (at >= row_end) continue;
            if (e.keep == KEEP_F16) {
                const bool relu = e.act == WF_ACT_RELU;
                const uint32_t w[2] = {pack2_sat(v[r][0], v[r][1], relu), pack2_sat(v[r][2], v[r][3], relu)};
                uint16_t *dst = static_cast<uint16_t *>(e.kept) + at * e.ld_kept + col;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + C * i < n) dst[C * i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
            } else if (e.keep == KEEP_F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + C * i < n) static_cast<float *>(e.kept)[at * e.ld_kept + col + C * i] = v[r][i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + C * i < n) store1<T>(row_of<T>(e.kept, at, e.ld_kept), col + C * i, v[r][i]);
            }
        }
    }
    if (e.act != WF_ACT_NONE) apply_act4(e.act, v);
    if (e.gate != nullptr) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (row + r * step < row_end) load4<T, VEC>(o[r], row_of<T>(e.gate, (row + r * step) / e.rows_per_group, n), col, n);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] *= o[r][i];
    }
    if (e.resid != nullptr) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (row + r * step < row_end) load4<T, VEC>(o[r], row_of<T>(e.resid, row + r * step, e.ld_resid), col, n);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] += o[r][i];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (row + r * step < row_end) store4<T, VEC>(row_of<T>(e.out, row + r * step, e.ld_out), col, n, v[r]);
}

// Value by value, out of line: the loop around the epilogue has to stay small (see linear_tile_kernel). Rows t, t + step, ...
// of the tile's sums, whose row 0 and column 0 are row0 and j0 of D.
template <int T, int R, int COLS>
__device__ __noinline__ void finish4_any(const Epilogue &e, const float *sums, int t, int step, int t_end, int row0, int j0, int n) {
    const int lane = threadIdx.x & 31;
    float v[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[r][i] = t + r * step < t_end ? sums[(t + r * step) * COLS + lane + 32 * i] : 0.f;
    finish4<T, false, R>(e, v, row0 + t, step, row0 + t_end, j0 + lane, n);
}

// ------------------------------------------------------------------------------------------------ few-rows kernel
// One 128-column x NT-row tile of D for each cluster of S CTAs. The columns j (the layer's output features) take the
// tensor core's 128 lanes and the few rows i its N, so a product of a handful of rows reads the weight once and wastes
// no more than NT - m rows. The CTAs of a cluster share the contraction, and their float32 parts are added through
// distributed shared memory in rank order (the same bits every time): with few tiles every SM still reads weights. Warp
// 4 loads tiles by TMA into a ring, warp 5 issues the MMAs, warps 0-3 move the accumulator to shared memory, and all
// eight warps finish the CTA's share of the rows.
constexpr int TILE_J = 128;
constexpr int TILE_THREADS = 256;
template <int NT>
struct TileShape {
    static constexpr int p_bytes = TILE_J * BC * 2, q_bytes = NT * BC * 2, stage = p_bytes + q_bytes;
    static constexpr int shallow = NT <= 32 ? 5 : NT <= 64 ? 4 : 3;  // stages: about 100 KB, two CTAs an SM ...
    static constexpr int deep = 2 * shallow;                         // ... or all of it
    static constexpr int smem(int stages) { return stages * stage + 1024 + 16 * deep + 16; }
    static constexpr int tmem_cols = NT < 32 ? 32 : NT;
    static_assert(NT * TILE_J * 4 <= shallow * stage, "the float32 tile reuses the ring");
};

template <bool P_ROWS, bool Q_ROWS, int NT, int T>
__global__ void __launch_bounds__(TILE_THREADS)
linear_tile_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ Epilogue epi, int m, int n, int c, int tiles_q, int split,
                   int stages) {
    using S = TileShape<NT>;
    constexpr uint32_t idesc = f16_idesc(T == WF_BF16, P_ROWS, Q_ROWS, TILE_J, NT);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + stages * S::stage);
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;
    const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(bars), empty0 = full0 + 8 * stages,
                   done = empty0 + 8 * stages;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int tile = blockIdx.x / split;
    const int j0 = tile / tiles_q * TILE_J, i0 = tile % tiles_q * NT;
    const int steps = (c + BC - 1) / BC;
    const int c_lo = static_cast<int>(static_cast<int64_t>(steps) * rank / split);
    const int c_hi = static_cast<int>(static_cast<int64_t>(steps) * (rank + 1) / split);

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&s_tmem_base)), "r"(S::tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem_base;
    wait_prior_grid();
    const Waits waits{&s_abort, epi.alarm, epi.wait_ns};

    if (warp == 4) {
        int stage = 0;
        uint32_t phase = 0;
        int issued = 0;
        for (int s = c_lo; s < c_hi; ++s, ++issued) {
            if (!__all_sync(0xFFFFFFFFu, pipe_wait(empty0 + 8 * stage, phase ^ 1u, waits, 1))) break;
            const uint32_t bar = full0 + 8 * stage, p = ring0 + stage * S::stage, q = p + S::p_bytes;
            if (elect_one()) {
                mbar_expect_tx(bar, S::stage);
                if constexpr (P_ROWS) {
                    for (int h = 0; h < TILE_J / 64; ++h) tma_load_2d(p + h * BC * 128, &map_p, j0 + 64 * h, s * BC, bar);
                } else {
                    tma_load_2d(p, &map_p, s * BC, j0, bar);
                }
                if constexpr (Q_ROWS) {
                    for (int h = 0; h < NT / 64; ++h) tma_load_2d(q + h * BC * 128, &map_q, i0 + 64 * h, s * BC, bar);
                } else {
                    tma_load_2d(q, &map_q, s * BC, i0, bar);
                }
            }
            __syncwarp();
            if (++stage == stages) stage = 0, phase ^= 1u;
        }
        // every load has landed before the CTA leaves or reuses the ring: only the last use of a stage can be
        // outstanding, and only after an abort
        for (int s = 0; s < stages && s < issued; ++s)
            mbar_drain_wait(full0 + 8 * s, static_cast<uint32_t>((issued - 1 - s) / stages) & 1u);
        __syncwarp();
    } else if (warp == 5) {
        const uint32_t p0 = desc_low<P_ROWS>(ring0), q0 = desc_low<Q_ROWS>(ring0 + S::p_bytes);
        int stage = 0;
        uint32_t phase = 0;
        for (int s = c_lo; s < c_hi; ++s) {
            if (!__all_sync(0xFFFFFFFFu, pipe_wait(full0 + 8 * stage, phase, waits, 2))) break;
            const uint32_t p = p0 + stage * (S::stage >> 4), q = q0 + stage * (S::stage >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < BC / 16; ++k)
                    mma_f16<false>(tmem, p + k * kDescStep<P_ROWS>, q + k * kDescStep<Q_ROWS>, idesc, s > c_lo || k > 0);
                mma_commit(empty0 + 8 * stage);
            }
            __syncwarp();
            if (++stage == stages) stage = 0, phase ^= 1u;
        }
        if (elect_one()) mma_commit(done);  // the accumulator is complete
        __syncwarp();
        mbar_drain_wait(done, 0);
        __syncwarp();
    } else if (warp < 4) {
        // lane w * 32 + l of tensor memory is column j0 + 32 w + l
        const bool ok = __all_sync(0xFFFFFFFFu, pipe_wait(done, 0, waits, 3) && !*waits.abort_flag);
        fence_after();
        if (ok) {  // the NT rows to part[row][column]
            float *part = reinterpret_cast<float *>(ring) + warp * 32 + lane;
            constexpr int STEP = NT < 32 ? 16 : 32;
#pragma unroll
            for (int t = 0; t < NT; t += STEP) {
                uint32_t r[STEP];
                if constexpr (STEP == 16) {
                    tmem_ld16(tmem + (static_cast<uint32_t>(warp * 32) << 16), r);
                } else {
                    tmem_ld32(tmem + (static_cast<uint32_t>(warp * 32) << 16) + t, r);
                    tmem_wait32(r);
                }
#pragma unroll
                for (int u = 0; u < STEP; ++u) part[(t + u) * TILE_J] = __uint_as_float(r[u]);
            }
        }
    }
    fence_before();
    __syncthreads();
    if (*waits.abort_flag) {  // settled: every role has stopped. The tile's sums become NaN, here and in the CTAs that add these parts
        for (int i = threadIdx.x; i < NT * TILE_J; i += TILE_THREADS) reinterpret_cast<float *>(ring)[i] = __int_as_float(0x7FFFFFFF);
        __syncthreads();
    }
    if (split > 1) cluster_sync();
    fence_after();
    if (warp == 5)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::tmem_cols) : "memory");
    // This CTA finishes rows t_lo .. t_hi of the tile, a row a warp, four columns a lane: it adds their parts, in rank
    // order, to its own copy, then runs the epilogue over them. The sums are unrolled (distributed shared memory is far
    // away); the epilogue is one copy of its code, four rows through each of its branches: with one row at a time, or
    // unrolled into the sums, 128 rows took 6.5 to 7.6 us.
    const int t_lo = NT * rank / split, t_hi = min(NT * (rank + 1) / split, m - i0), col = j0 + lane * 4;
    constexpr int WARPS = TILE_THREADS / 32;
    auto add_parts = [&](auto parts) {
        constexpr int S = decltype(parts)::value, R = S == 8 ? 2 : 4;
        uint32_t base[S];
#pragma unroll
        for (int r = 0; r < S; ++r) base[r] = map_to_rank(ring0, r);
        for (int t = t_lo + warp; t < t_hi; t += R * WARPS) {
            float4 p[R][S];
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int r = 0; r < S; ++r) {
                    p[i][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (t + i * WARPS < t_hi)
                        p[i][r] = ld_cluster4(base[r] + static_cast<uint32_t>((t + i * WARPS) * TILE_J + lane * 4) * 4u);
                }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (t + i * WARPS >= t_hi) continue;
#pragma unroll
                for (int r = 1; r < S; ++r)
                    p[i][0].x += p[i][r].x, p[i][0].y += p[i][r].y, p[i][0].z += p[i][r].z, p[i][0].w += p[i][r].w;
                reinterpret_cast<float4 *>(ring)[(t + i * WARPS) * (TILE_J / 4) + lane] = p[i][0];
            }
        }
    };
    if (split == 2) add_parts(std::integral_constant<int, 2>{});
    else if (split == 4) add_parts(std::integral_constant<int, 4>{});
    else if (split == 8) add_parts(std::integral_constant<int, 8>{});
    // No CTA leaves while another reads its part. Every read above has been waited for here, because its value has been
    // stored: a read that nobody waits for (of a row past t_hi, say) could still be under way when the CTA that it reads
    // has left, an illegal access.
    if (split > 1) cluster_sync();
    const float4 *sums = reinterpret_cast<const float4 *>(ring);
    constexpr int R = 4;
    if (epi.vec && (n % 4 == 0 || j0 + TILE_J <= n)) {  // the whole warp, or none of it
        if (col >= n) return;
#pragma unroll 1
        for (int t = t_lo + warp; t < t_hi; t += R * WARPS) {
            float v[R][4];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 q = sums[min(t + r * WARPS, NT - 1) * (TILE_J / 4) + lane];
                v[r][0] = q.x, v[r][1] = q.y, v[r][2] = q.z, v[r][3] = q.w;
            }
            finish4<T, true, R>(epi, v, i0 + t, WARPS, i0 + t_hi, col, n);
        }
    } else {
#pragma unroll 1
        for (int t = t_lo + warp; t < t_hi; t += R * WARPS)
            finish4_any<T, R, TILE_J>(epi, reinterpret_cast<const float *>(ring), t, WARPS, t_hi, i0, j0, n);
    }
}

// ------------------------------------------------------------------------------------------------- many-rows kernel
// One 256 x 256 tile of D for each pair of CTAs (a cluster of 2 on neighbouring SMs), persistent. tcgen05.mma
// cta_group::2 (M = 256, N = 256, K = 16), issued by one thread of the even CTA, reads rows 0..127 of the A tile and
// columns 0..127 of the B tile from the even CTA's shared memory and the other halves from the odd CTA's; each CTA's
// tensor memory holds its 128 rows x 256 columns, twice, so that the next tile's MMAs run while this one is written out.
// Warp 8 loads (six 32 KB stages), warp 9 of the even CTA issues, warps 0..7 are the epilogue: a warp takes 32 rows and
// 128 columns of the accumulator in chunks of 32 x 64 (32 x 32 where z is kept, too), which leave through a swizzled buffer
// and one TMA store each (plain stores where the output's pitch or base is not a multiple of 16 bytes). Chunks of 32 x 32
// for y alone: 8192 x 512 x 8192 63.9 against 58.9 us; a stage given up for a second wide buffer: 8192 x 2048 x 8192 with
// silu and z 214 against 197.
// What bounds it: a stage is 512 cycles of MMAs and 32 KB an SM, 64 bytes a cycle -- what an SM takes in from L2 (56 to
// 60 measured) -- and in long runs the board's power. A 256 x 128 tile (24 KB for 256 cycles) was no faster anywhere:
// 2048^3 30.5 against 20.6 us, 8192 x 256 x 2048 24.4 against 20.8.
constexpr int BN = 256;
constexpr int PAIR_THREADS = 320;
constexpr int PAIR_EPI_THREADS = 256;
constexpr int PAIR_HALF = 128 * BC * 2;            // 16 KB: this CTA's 128 rows of A or columns of B
constexpr int PAIR_STAGE = 2 * PAIR_HALF;
constexpr int PAIR_STAGES = 6;
constexpr int WARP_OUT = 4096;                     // output chunks of an epilogue warp: 32 rows of 64 columns of y, or of 32 of y
                                                   // and 32 of the kept z
constexpr int PAIR_SMEM = PAIR_STAGES * PAIR_STAGE + 8 * WARP_OUT + 1024 + 256;
constexpr int chunk_cols(bool keep) { return keep ? 32 : 64; }
constexpr int kBand = 8;                           // tile rows of a band of the tile order

// Value by value and out of line, for rows that 16-byte accesses do not fit.
__device__ __noinline__ void load32_any(uint32_t (&w)[16], const uint16_t *row, int col, int n) {
    for (int i = 0; i < 16; ++i) {
        const int c = col + 2 * i;
        const uint32_t lo = c < n ? row[c] : 0u, hi = c + 1 < n ? row[c + 1] : 0u;
        w[i] = lo | (hi << 16);
    }
}

// 32 neighbouring 16-bit values of a row in 16 registers, those at and past n as 0; vec: 16-byte aligned, n % 8 == 0
__device__ __forceinline__ void load32(uint32_t (&w)[16], const void *row, int col, int n, bool vec) {
    if (vec) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (col + 8 * q < n) v = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(row) + col + 8 * q));
            w[4 * q] = v.x, w[4 * q + 1] = v.y, w[4 * q + 2] = v.z, w[4 * q + 3] = v.w;
        }
    } else {
        uint32_t any[16];
        load32_any(any, static_cast<const uint16_t *>(row), col, n);
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = any[i];
    }
}

template <int ACT>
__device__ __forceinline__ void act32(float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) act2<ACT>(v[i], v[i + 1]);
}

// An output chunk of a warp in shared memory: 32 rows of CW columns, sent off with one TMA store (which clips what lies
// outside), or row by row. 16-byte piece j of row r lies at piece j ^ (r & 7) (CW = 64: 128-byte swizzle) or
// j ^ ((r >> 1) & 3) (CW = 32: 64-byte swizzle).
struct ChunkOut {
    const CUtensorMap *map;
    void *out;
    int64_t ld;
    uint32_t buf;
    bool tma;
};

template <int CW>
__device__ __forceinline__ uint32_t piece_at(uint32_t buf, uint32_t row, uint32_t piece) {
    return buf + 2u * CW * row + 16u * (piece ^ (CW == 64 ? row & 7u : (row >> 1) & 3u));
}

// 32 columns (this lane's row in p), half h of the chunk; the buffer's last store has been read
template <int CW>
__device__ __forceinline__ void put32(const ChunkOut &o, const uint32_t (&p)[16], int h, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at<CW>(o.buf, lane, 4 * h + j)), "r"(p[4 * j]),
                     "r"(p[4 * j + 1]), "r"(p[4 * j + 2]), "r"(p[4 * j + 3])
                     : "memory");
}

// the chunk's values one by one, a row at a time: rows and columns past the output's are left alone
template <int CW>
__device__ __noinline__ void send_any(uint16_t *out, int64_t ld, uint32_t buf, int lane, int rows, int cols) {
    for (int c = lane; c < cols; c += 32)
        for (int r0 = 0; r0 < rows; r0 += 8) {  // eight rows in flight
            uint16_t v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v[r]) : "r"(piece_at<CW>(buf, r0 + r, c >> 3) + 2u * (c & 7)) : "memory");
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r0 + r < rows) out[(r0 + r) * ld + c] = v[r];
        }
}

template <int CW>
__device__ __forceinline__ void send_chunk(const ChunkOut &o, int lane, int row0, int col0, int m, int n) {
    if (o.tma) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(o.map, o.buf, col0, row0);
            bulk_commit();
        }
    } else {
        __syncwarp();
        send_any<CW>(static_cast<uint16_t *>(o.out) + row0 * o.ld + col0, o.ld, o.buf, lane, min(32, m - row0), min(CW, n - col0));
        __syncwarp();
    }
}

// what one epilogue warp knows of its 32 rows
struct Warp32 {
    int lane, row0, m, n;
    const void *gate, *resid; // this lane's rows (null: none, or a row past m)
    ChunkOut y, z;
};

// 32 columns of the warp's rows, half h of a chunk of 64 (KEEP: a chunk of their own)
template <int T, bool FULL, bool KEEP>
__device__ __forceinline__ void finish_half(float (&v)[32], Warp32 &w, const Epilogue &e, const uint32_t (&b)[16],
                                            const uint32_t (&g)[16], const uint32_t (&res)[16], int col0, int h) {
    uint32_t p[16];
    if constexpr (FULL) {
        if (e.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 f = unpack2<T>(b[i]);
                v[2 * i] += f.x;
                v[2 * i + 1] += f.y;
            }
        }
        if constexpr (KEEP) {
            if (e.keep == KEEP_F32) {
                const int row = w.row0 + w.lane;
                if (row < w.m) {
                    float *dst = static_cast<float *>(e.kept) + row * e.ld_kept + col0;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (col0 + i < w.n) dst[i] = v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    p[i] = e.keep == KEEP_F16 ? pack2_sat(v[2 * i], v[2 * i + 1], e.act == WF_ACT_RELU) : pack2<T>(v[2 * i], v[2 * i + 1]);
                // z's last store has been read; y's may go on, and is the last one where y leaves by TMA at all
                if (w.lane == 0) w.y.tma ? bulk_wait_read1() : bulk_wait_read_all();
                __syncwarp();
                put32<32>(w.z, p, 0, w.lane);
                send_chunk<32>(w.z, w.lane, w.row0, col0, w.m, w.n);
            }
        }
        switch (e.act) {
            case WF_ACT_RELU: act32<WF_ACT_RELU>(v); break;
            case WF_ACT_SILU: act32<WF_ACT_SILU>(v); break;
            case WF_ACT_GELU: act32<WF_ACT_GELU>(v); break;
            case WF_ACT_GELU_TANH: act32<WF_ACT_GELU_TANH>(v); break;
            default: break;
        }
        if (w.gate != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 f = unpack2<T>(g[i]);
                v[2 * i] *= f.x;
                v[2 * i + 1] *= f.y;
            }
        }
        if (e.resid != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 f = unpack2<T>(res[i]);
                v[2 * i] += f.x;
                v[2 * i + 1] += f.y;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    if constexpr (KEEP) {
        if (w.lane == 0) w.z.tma ? bulk_wait_read1() : bulk_wait_read_all();  // the same for y
        __syncwarp();
        put32<32>(w.y, p, 0, w.lane);
        send_chunk<32>(w.y, w.lane, w.row0, col0, w.m, w.n);
    } else {
        if (h == 0) {
            if (w.lane == 0) bulk_wait_read_all();
            __syncwarp();
        }
        put32<64>(w.y, p, h, w.lane);
        if (h == 1) send_chunk<64>(w.y, w.lane, w.row0, col0 - 32, w.m, w.n);
    }
}

// After a wait that ran out of time: NaN in an epilogue warp's rows of every tile that it has not written, and in the kept z's.
__device__ __noinline__ void fill_nan(const Epilogue &e, int tile, int n_clusters, int m, int n, int band, int rank, int quarter, int half) {
    const int tiles_m = (m + 255) / 256, tiles_n = (n + BN - 1) / BN, lane = threadIdx.x & 31;
    for (; tile < tiles_m * tiles_n; tile += n_clusters) {
        int mi, ni;
        tile_coords(tile, tiles_m, tiles_n, band, mi, ni);
        const int row0 = mi * 256 + rank * 128 + quarter * 32, col0 = ni * BN + half * (BN / 2);
        for (int row = row0; row < min(row0 + 32, m); ++row)
            for (int col = col0 + lane; col < min(col0 + BN / 2, n); col += 32) {
                static_cast<uint16_t *>(e.out)[row * e.ld_out + col] = 0x7FFF;  // bf16's and f16's
                if (e.keep == KEEP_F32) static_cast<uint32_t *>(e.kept)[row * e.ld_kept + col] = 0x7FFFFFFFu;
                else if (e.keep != KEEP_NONE) static_cast<uint16_t *>(e.kept)[row * e.ld_kept + col] = 0x7FFF;
            }
    }
}

// FULL: the forward pass's epilogue; else D is rounded and stored. KEEP: z is kept
template <bool A_ROWS, bool B_ROWS, int T, bool FULL, bool KEEP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_kept,
                   const __grid_constant__ Epilogue epi, int m, int n, int c, int band, bool tma_out, bool tma_kept) {
    constexpr uint32_t idesc = f16_idesc(T == WF_BF16, A_ROWS, B_ROWS, 256, BN);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *out_chunks = ring + PAIR_STAGES * PAIR_STAGE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(out_chunks + 8 * WARP_OUT);
    // full (used in the even CTA) and empty of each stage, tmem_full[0..1], tmem_empty[0..1] (even CTA), drain
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;
    __shared__ int s_issued[2];  // stage loads issued by this CTA's producer; [1] in the even CTA: the odd CTA's
    const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(bars), empty0 = full0 + 8 * PAIR_STAGES,
                   tfull0 = empty0 + 8 * PAIR_STAGES, tempty0 = tfull0 + 16, drain = tempty0 + 16;
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), peer = rank ^ 1u;
    const int tiles_m = (m + 255) / 256, tiles_n = (n + BN - 1) / BN, n_tiles = tiles_m * tiles_n;
    const int steps = (c + BC - 1) / BC;
    const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        s_abort = 0;
        s_issued[0] = s_issued[1] = 0;
        for (int s = 0; s < PAIR_STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull0 + 8 * b, 1);
            mbar_init(tempty0 + 8 * b, 2 * PAIR_EPI_THREADS);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&s_tmem_base)), "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_before();
    cluster_sync();  // barriers initialised and tensor memory allocated in both CTAs
    fence_after();
    const uint32_t tmem = s_tmem_base;
    wait_prior_grid();
    const Waits waits{&s_abort, epi.alarm, epi.wait_ns};

    if (warp == 8) {
        if (elect_one()) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_b)) : "memory");
        }
        __syncwarp();
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = cluster_id; tile < n_tiles && ok; tile += n_clusters) {
            int mi, ni;
            tile_coords(tile, tiles_m, tiles_n, band, mi, ni);
            const int i0 = mi * 256 + static_cast<int>(rank) * 128, j0 = ni * BN + static_cast<int>(rank) * (BN / 2);
            for (int s = 0; s < steps; ++s) {
                if (!__all_sync(0xFFFFFFFFu, pipe_wait(empty0 + 8 * stage, phase ^ 1u, waits, 1))) { ok = false; break; }
                const uint32_t bar = (full0 + 8 * stage) & kPeerBitMask;  // the even CTA's
                const uint32_t a = ring0 + stage * PAIR_STAGE, b = a + PAIR_HALF;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full0 + 8 * stage, 2 * PAIR_STAGE);
                    if constexpr (A_ROWS) {
                        tma_load_2d_pair(a, &map_a, i0, s * BC, bar);
                        tma_load_2d_pair(a + BC * 128, &map_a, i0 + 64, s * BC, bar);
                    } else {
                        tma_load_2d_pair(a, &map_a, s * BC, i0, bar);
                    }
                    if constexpr (B_ROWS) {
                        tma_load_2d_pair(b, &map_b, j0, s * BC, bar);
                        tma_load_2d_pair(b + BC * 128, &map_b, j0 + 64, s * BC, bar);
                    } else {
                        tma_load_2d_pair(b, &map_b, s * BC, j0, bar);
                    }
                }
                __syncwarp();
                ++issued;
                if (++stage == PAIR_STAGES) stage = 0, phase ^= 1u;
            }
        }
        // the count goes to the even CTA, whose full barriers count both CTAs' bytes: it drains (below)
        if (lane == 0) {
            if (rank == 0) {
                s_issued[0] = issued;
            } else {
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank(smem_u32(&s_issued[1]), 0)), "r"(issued)
                             : "memory");
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        if (rank == 0) {
            const uint32_t empty_peer = map_to_rank(empty0, peer), tfull_peer = map_to_rank(tfull0, peer);
            const uint32_t a0 = desc_low<A_ROWS>(ring0), b0 = desc_low<B_ROWS>(ring0 + PAIR_HALF);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int tile = cluster_id; tile < n_tiles && ok; tile += n_clusters) {
                if (!__all_sync(0xFFFFFFFFu, pipe_wait(tempty0 + 8 * acc, acc_phase ^ 1u, waits, 2))) break;
                fence_after();
                const uint32_t d = tmem + static_cast<uint32_t>(acc * BN);
                for (int s = 0; s < steps; ++s) {
                    if (!__all_sync(0xFFFFFFFFu, pipe_wait(full0 + 8 * stage, phase, waits, 2))) { ok = false; break; }
                    const uint32_t a = a0 + stage * (PAIR_STAGE >> 4), b = b0 + stage * (PAIR_STAGE >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BC / 16; ++k)
                            mma_f16<true>(d, a + k * kDescStep<A_ROWS>, b + k * kDescStep<B_ROWS>, idesc, s > 0 || k > 0);
                        mma_commit_pair(empty0 + 8 * stage);
                        mma_commit_pair(empty_peer + 8 * stage);
                    }
                    __syncwarp();
                    if (++stage == PAIR_STAGES) stage = 0, phase ^= 1u;
                }
                if (!ok) break;
                if (elect_one()) {
                    mma_commit_pair(tfull0 + 8 * acc);
                    mma_commit_pair(tfull_peer + 8 * acc);
                }
                __syncwarp();
                if (++acc == 2) acc = 0, acc_phase ^= 1u;
            }
            if (elect_one()) mma_commit_pair(drain);
            __syncwarp();
            mbar_drain_wait(drain, 0);
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t tempty_leader = map_to_rank(tempty0, 0);
        Warp32 w;
        w.lane = lane, w.m = m, w.n = n;
        w.y = ChunkOut{&map_out, epi.out, epi.ld_out, smem_u32(out_chunks + warp * WARP_OUT), tma_out};
        w.z = ChunkOut{&map_kept, epi.kept, epi.ld_kept, w.y.buf + WARP_OUT / 2, tma_kept};
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int tile = cluster_id; tile < n_tiles; tile += n_clusters) {
            int mi, ni;
            tile_coords(tile, tiles_m, tiles_n, band, mi, ni);
            w.row0 = mi * 256 + static_cast<int>(rank) * 128 + quarter * 32;
            const int col0 = ni * BN + half * (BN / 2), row = w.row0 + lane;
            const bool in = row < m;
            w.gate = FULL && epi.gate != nullptr && in ? row_of<T>(epi.gate, row / epi.rows_per_group, n) : nullptr;
            w.resid = FULL && epi.resid != nullptr && in ? row_of<T>(epi.resid, row, epi.ld_resid) : nullptr;
            if (FULL && w.resid != nullptr && epi.vec && col0 < n)  // the row's span to L2 while the MMAs run
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                             ::"l"(static_cast<const uint16_t *>(w.resid) + col0), "r"(static_cast<uint32_t>(min(BN / 2, n - col0)) * 2u)
                             : "memory");
            if (!__all_sync(0xFFFFFFFFu, pipe_wait(tfull0 + 8 * acc, acc_phase, waits, 3))) {
                fill_nan(epi, tile, n_clusters, m, n, band, static_cast<int>(rank), quarter, half);
                break;
            }
            fence_after();
            const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BN + half * (BN / 2));
            uint32_t r[32], b[16], g[16], res[16];
            tmem_ld32(taddr, r);
            // one copy of the chunk's code (unrolled four times, with every activation inside, it outgrew the
            // instruction cache: 266 against 137 us for a gelu layer of 8192 x 512 x 8192)
#pragma unroll 1
            for (int q = 0; q < BN / 64; ++q) {
                // in flight together with the accumulator's columns
                if (FULL && epi.bias != nullptr) load32(b, epi.bias, col0 + 32 * q, n, epi.vec || (epi.vec_bias && col0 + 32 * (q + 1) <= n));
                if (FULL && w.gate != nullptr) load32(g, w.gate, col0 + 32 * q, n, epi.vec);
                if (FULL && epi.resid != nullptr) {
                    if (w.resid != nullptr) {
                        load32(res, w.resid, col0 + 32 * q, n, epi.vec);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) res[i] = 0u;
                    }
                }
                tmem_wait32(r);
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                if (q < BN / 64 - 1) {
                    tmem_ld32(taddr + 32 * (q + 1), r);  // in flight while this half is finished
                } else {  // the accumulator is in registers: it may be overwritten
                    fence_before();
                    mbar_arrive_cluster(tempty_leader + 8 * acc);
                }
                finish_half<T, FULL, KEEP>(v, w, epi, b, g, res, col0 + 32 * q, q & 1);
            }
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
        if (lane == 0) bulk_wait_read_all();
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs stopped issuing; the odd CTA's load count is in the even CTA's s_issued[1]
    if (rank == 0 && warp == 8 && lane == 0) {
        // Every stage load either CTA issued lands before either CTA leaves: only a stage's last use can be outstanding,
        // and after an abort one CTA may have issued a use that the other did not (its bytes are then made up for).
        const int n_even = s_issued[0], n_odd = s_issued[1], last = max(n_even, n_odd);
        for (int s = 0; s < PAIR_STAGES && s < last; ++s) {
            const int u = s + ((last - 1 - s) / PAIR_STAGES) * PAIR_STAGES;
            const uint32_t bar = full0 + 8 * s;
            if (u >= n_even)
                mbar_expect_tx(bar, PAIR_STAGE);
            else if (u >= n_odd)
                mbar_complete_tx(bar, PAIR_STAGE);
            mbar_drain_wait(bar, static_cast<uint32_t>(u / PAIR_STAGES) & 1u);
        }
    }
    cluster_sync();  // no CTA leaves (or frees tensor memory) while loads into it or the pair's MMAs may still run
    fence_after();
    if (warp == 9)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
}

// ------------------------------------------------------------------------------------------------------------- host
// a 16-bit matrix of `rows` rows of `cols` values, `ld` apart, as boxes of box_rows x 64 values with 128-byte swizzle
// and zeros outside
int operand_map(CUtensorMap *map, const void *base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeTiled enc = encoder();
    if (enc == nullptr) return WF_ERR_DEVICE;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? WF_OK : WF_ERR_ARG;
}

// D [m, n] = A B^T: a is [m, c] (or [c, m] where it is row-major), b is [n, c] (or [c, n])
struct Product {
    const void *a, *b;
    int64_t lda, ldb, m, n, c;
};

template <bool A_ROWS, bool B_ROWS, int NT, int T>
int launch_tile(const Product &p, const Epilogue &e, int split, bool deep, int dev, cudaStream_t stream) {
    using S = TileShape<NT>;
    constexpr auto kern = linear_tile_kernel<B_ROWS, A_ROWS, NT, T>;
    static std::atomic<bool> ready[64];  // any host thread may launch first
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e0 = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem(S::deep));
        if (e0 != cudaSuccess) return static_cast<int>(e0);
        ready[dev].store(true, std::memory_order_release);
    }
    CUtensorMap mp, mq;
    int rc = B_ROWS ? operand_map(&mp, p.b, p.c, p.n, p.ldb, BC) : operand_map(&mp, p.b, p.n, p.c, p.ldb, TILE_J);
    if (rc == WF_OK) rc = A_ROWS ? operand_map(&mq, p.a, p.c, p.m, p.lda, BC) : operand_map(&mq, p.a, p.m, p.c, p.lda, NT);
    if (rc != WF_OK) return rc;
    const int64_t tiles_q = (p.m + NT - 1) / NT, tiles = (p.n + TILE_J - 1) / TILE_J * tiles_q;
    if (tiles * split > (1ll << 31) - 1) return WF_ERR_ARG;
    const int stages = deep ? S::deep : S::shallow;
    const cudaError_t err = launch_dependent_clusters(
        kern, dim3(static_cast<unsigned>(tiles * split)), split > 1 ? split : 0, TILE_THREADS, S::smem(stages), stream, mp, mq, e,
        static_cast<int>(p.m), static_cast<int>(p.n), static_cast<int>(p.c), static_cast<int>(tiles_q), split, stages);
    return static_cast<int>(err != cudaSuccess ? err : cudaGetLastError());
}

// a 16-bit [rows, cols] output as boxes of 32 rows x 64 or 32 values, swizzled over a box's row
int output_map(CUtensorMap *map, void *base, int64_t rows, int64_t cols, int64_t ld, int box_cols) {
    EncodeTiled enc = encoder();
    if (enc == nullptr) return WF_ERR_DEVICE;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), 32};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? WF_OK : WF_ERR_ARG;
}

bool vec8_ok(const void *p, int64_t ld) { return p == nullptr || (aligned_to(p, 16) && ld % 8 == 0); }

template <bool A_ROWS, bool B_ROWS, int T, bool KEEP>
int launch_pair(const Product &p, const Epilogue &e0, int dev, cudaStream_t stream) {
    constexpr bool full = !A_ROWS && !B_ROWS;
    constexpr auto kern = linear_pair_kernel<A_ROWS, B_ROWS, T, full, KEEP>;
    constexpr int smem = PAIR_SMEM;
    static std::atomic<int> clusters[64];  // resident pairs; any host thread may launch first
    if (clusters[dev].load(std::memory_order_acquire) == 0) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return static_cast<int>(e);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * device_sm_count());
        cfg.blockDim = dim3(PAIR_THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
        if (e != cudaSuccess) return static_cast<int>(e);
        clusters[dev].store(std::max(n, 1), std::memory_order_release);
    }
    Epilogue e = e0;
    // 16-byte accesses to the bias, the gate and the residual
    e.vec_bias = vec8_ok(e.bias, 0);
    e.vec = p.n % 8 == 0 && vec8_ok(e.bias, 0) && vec8_ok(e.gate, p.n) && vec8_ok(e.resid, e.ld_resid);
    // A TMA store clips at whole 16-byte pieces: behind a row of n values it writes zeros up to the next multiple of 8 (as
    // measured). y's neighbours are the caller's; z's rows have room for it where their pitch is that multiple.
    const bool tma_out = p.n % 8 == 0 && vec8_ok(e.out, e.ld_out);
    const bool tma_kept = (e.keep == KEEP_F16 || e.keep == KEEP_SAME) && vec8_ok(e.kept, e.ld_kept) &&
                          (p.n % 8 == 0 || e.ld_kept == (p.n + 7) / 8 * 8);
    CUtensorMap ma, mb, mo = {}, mk = {};
    int rc = A_ROWS ? operand_map(&ma, p.a, p.c, p.m, p.lda, BC) : operand_map(&ma, p.a, p.m, p.c, p.lda, 128);
    if (rc == WF_OK) rc = B_ROWS ? operand_map(&mb, p.b, p.c, p.n, p.ldb, BC) : operand_map(&mb, p.b, p.n, p.c, p.ldb, BN / 2);
    if (rc == WF_OK && tma_out) rc = output_map(&mo, e.out, p.m, p.n, e.ld_out, chunk_cols(KEEP));
    if (rc == WF_OK && tma_kept) rc = output_map(&mk, e.kept, p.m, p.n, e.ld_kept, chunk_cols(KEEP));
    if (rc != WF_OK) return rc;
    const int64_t tiles = ((p.m + 255) / 256) * ((p.n + BN - 1) / BN);
    if (tiles > (1ll << 30)) return WF_ERR_ARG;
    const int grid = 2 * static_cast<int>(std::min<int64_t>(tiles, clusters[dev].load(std::memory_order_acquire)));
    const cudaError_t err = launch_dependent(kern, dim3(grid), PAIR_THREADS, smem, stream, ma, mb, mo, mk, e,
                                             static_cast<int>(p.m), static_cast<int>(p.n), static_cast<int>(p.c),
                                             kBand, tma_out, tma_kept);
    return static_cast<int>(err != cudaSuccess ? err : cudaGetLastError());
}

// Which kernel and shape take a product: the one of the least estimated time, from what one B200 measured (graphs of
// calls over operands that do not stay in L2; the estimates are within some 15 %).
//   tile kernel (NT rows, S CTAs to a tile): a CTA takes 3.8 us, 13 ns a row of its epilogue, and its contraction steps. A
//     step takes 0.19 us, 7.2 ns a KB of its operands, or the ring's share of a 1.2 us round trip; CTAs that share an SM
//     share that rate. More than two CTAs an SM come in rounds. Sharing a tile costs 1.2 us of cluster barriers and the
//     parts' way through distributed shared memory at 3.3 TB/s. Nothing is faster than the operands' bytes at 6 TB/s.
//   pair kernel: 8.9 us and 0.275 us a step for the first 74 tiles (somewhat less for a step or two), and for each further
//     74 0.3 us a step, or 4.2 us where the epilogue is longer.
// Measured on both sides of the choice, in us (tile NT, S / pair): 333 x 1024 x 5120 128, 1 9.6 / 13.8; 1024 x 2048 x 2048
// 128, 1 13.0 / 18.2; 512 x 5120 x 5120 128, 1 35.1 / 33.2; 5000 x 72 x 2048 128, 1 18.3 / 16.5; 8192 x 256 x 2048 128, 1 26.5 /
// 20.5. Among tiles: 128 x 2048 x 2048 64, 4 8.5, 128, 1 12.3, 16, 8 23; 8192 rows to a 256 x 256 gradient 64, 8 10.2, 64, 1 29.
struct Plan {
    int nt, split;  // nt 0: the pair kernel
    bool deep;
    double us;
};

Plan tile_plan(const Product &p, int nt, int split, int sms) {
    const double steps = static_cast<double>((p.c + BC * split - 1) / (BC * split));
    const double ctas = static_cast<double>((p.n + TILE_J - 1) / TILE_J * ((p.m + nt - 1) / nt)) * split;
    const bool deep = split == 1 && ctas <= sms;
    const int stages = (nt <= 32 ? 5 : nt <= 64 ? 4 : 3) * (deep ? 2 : 1);
    const double shared = ctas > sms ? std::min(2.0, 1.0 + 1.5 * std::sqrt(ctas / sms - 1.0)) : 1.0;
    const double step = std::max(std::max(0.19, (16 + nt / 8.0) * 0.0072) * shared, 1.2 / stages);
    double cta = 3.8 + steps * step + 0.013 * std::min<double>(nt, static_cast<double>(p.m)) / split;
    if (split > 1) cta += 1.2 + nt * 512.0 * (split - 1) / split * std::min(ctas, 2.0 * sms) / 3.3e6;
    const double bytes = 2.0 * (static_cast<double>(p.m) * p.c + static_cast<double>(p.n) * p.c + static_cast<double>(p.m) * p.n);
    return {nt, split, deep, std::max(cta * std::ceil(ctas / (2.0 * sms)), bytes / 6.0e6 + 4.0)};
}

Plan make_plan(const Product &p, int least_nt) {
    static const int forced = env_digit("WEIGHTFERRY_LINEAR_PAIR", 2);  // 0 / 1: the tile / the pair kernel only
    const int sms = device_sm_count();
    const double tiles = static_cast<double>((p.m + 255) / 256) * ((p.n + BN - 1) / BN), steps = static_cast<double>((p.c + BC - 1) / BC);
    Plan best{0, 1, false, 8.9 + 0.275 * steps - 0.2 * std::max(0.0, 8.0 - steps) +
                               (std::ceil(tiles / (sms / 2)) - 1.0) * std::max(0.3 * steps, 4.2)};
    if (forced == 1) return best;
    if (forced == 0) best.us = 1e30;
    for (int nt = least_nt; nt <= 128; nt *= 2) {
        for (int split = 1; split <= 8 && (split == 1 || split <= steps); split *= 2) {
            const Plan t = tile_plan(p, nt, split, sms);
            if (t.us < best.us) best = t;
        }
        if (p.m <= nt) break;  // wider tiles would hold nothing more
    }
    return best;
}

template <bool A_ROWS, bool B_ROWS, int T>
int dispatch(const Product &p, const Epilogue &e, cudaStream_t stream) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return WF_ERR_DEVICE;
    const Plan plan = make_plan(p, A_ROWS ? 64 : 16);  // a row-major operand comes in swizzle rows of 64
    switch (plan.nt) {
        case 0:
            if constexpr (!A_ROWS && !B_ROWS)
                if (e.keep != KEEP_NONE) return launch_pair<A_ROWS, B_ROWS, T, true>(p, e, dev, stream);
            return launch_pair<A_ROWS, B_ROWS, T, false>(p, e, dev, stream);
        case 64: return launch_tile<A_ROWS, B_ROWS, 64, T>(p, e, plan.split, plan.deep, dev, stream);
        case 128: return launch_tile<A_ROWS, B_ROWS, 128, T>(p, e, plan.split, plan.deep, dev, stream);
        default: break;
    }
    if constexpr (!A_ROWS) {
        if (plan.nt == 16) return launch_tile<A_ROWS, B_ROWS, 16, T>(p, e, plan.split, plan.deep, dev, stream);
        if (plan.nt == 32) return launch_tile<A_ROWS, B_ROWS, 32, T>(p, e, plan.split, plan.deep, dev, stream);
    }
    return WF_ERR_ARG;
}

// what TMA asks of an operand: a 16-byte aligned base and row pitch
bool operand_ok(const void *p, int64_t cols, int64_t ld) {
    return p != nullptr && aligned_to(p, 16) && ld >= cols && ld % 8 == 0;
}

bool sizes_ok(int64_t m, int64_t n, int64_t k) {
    constexpr int64_t most = 1ll << 30;
    return m >= 0 && n >= 0 && k >= 1 && m <= most && n <= most && k <= most;
}

bool vec4_ok(const void *p, int64_t ld) { return p == nullptr || (aligned_to(p, 8) && ld % 4 == 0); }

int64_t dz_bytes(int64_t m, int64_t n) { return m * ((n + 7) / 8 * 8) * 2; }

Epilogue plain_epilogue(void *out, int64_t ld) {
    return Epilogue{nullptr, nullptr, nullptr, out, nullptr, nullptr, 0, 0, ld, 0, 1, WF_ACT_NONE, KEEP_NONE, false};
}

// A word of each device in mapped host memory, set by a kernel whose wait ran out of time and looked at by every call: no
// call is needed to learn of it. Allocated by the first call, which a stream capture may surround.
int *alarm_words() {
    static int *words = [] {
        int *p = nullptr;
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (cudaHostAlloc(reinterpret_cast<void **>(&p), 64 * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (p != nullptr) std::fill(p, p + 64, 0);
        return p;
    }();
    return words;
}

std::atomic<uint64_t> g_wait_ns{kWaitLimitNs};  // wf_linear_set_wait_limit

// the current device's word, or the status that refuses the call
int alarm_of_device(int **word) {
    int dev = 0;
    cudaGetDevice(&dev);
    int *words = alarm_words();
    if (dev < 0 || dev >= 64 || words == nullptr) return WF_ERR_DEVICE;
    *word = words + dev;
    return *static_cast<volatile int *>(*word) != 0 ? WF_ERR_EXPIRED : WF_OK;
}

template <bool A_ROWS, bool B_ROWS>
int run_product(const Product &p, Epilogue e, int type, cudaStream_t stream) {
    e.vec = vec4_ok(e.bias, 0) && vec4_ok(e.gate, p.n) && vec4_ok(e.resid, e.ld_resid) && vec4_ok(e.out, e.ld_out) &&
            (e.keep != KEEP_SAME || vec4_ok(e.kept, e.ld_kept));
    int rc = check_device();
    if (rc == WF_OK) rc = alarm_of_device(&e.alarm);
    if (rc != WF_OK) return rc;
    e.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
    return type == WF_BF16 ? dispatch<A_ROWS, B_ROWS, WF_BF16>(p, e, stream) : dispatch<A_ROWS, B_ROWS, WF_F16>(p, e, stream);
}

}  // namespace
}  // namespace wf

extern "C" WF_API int wf_linear(const wf_linear_args *args, wf_stream_t stream) {
    using namespace wf;
    if (args == nullptr) return WF_ERR_ARG;
    const wf_linear_args &a = *args;
    if (a.type != WF_BF16 && a.type != WF_F16) return WF_ERR_UNSUPPORTED;
    if (a.act < WF_ACT_NONE || a.act > WF_ACT_GELU_TANH) return WF_ERR_UNSUPPORTED;
    if (!sizes_ok(a.m, a.n, a.k)) return WF_ERR_ARG;
    if (a.m == 0 || a.n == 0) return WF_OK;
    if (!operand_ok(a.x, a.k, a.ldx) || !operand_ok(a.w, a.k, a.ldw) || !a.y || a.ldy < a.n || a.rows_per_group < 1 ||
        (a.resid && a.ld_resid < a.n) || !aligned_to(a.y, 2) || !aligned_to(a.bias, 2) || !aligned_to(a.gate, 2) ||
        !aligned_to(a.resid, 2))
        return WF_ERR_ARG;
    int keep = KEEP_NONE;
    if (a.z != nullptr) {
        if (a.z_type != WF_F32 && a.z_type != WF_F16 && a.z_type != a.type) return WF_ERR_UNSUPPORTED;
        if (a.ldz < a.n || !aligned_to(a.z, dtype_size(a.z_type))) return WF_ERR_ARG;
        // an f16 layer's own type is the slope's f16 too, where there is an activation: z past f16's range would be infinite
        // otherwise, and the slope of infinity NaN
        keep = a.z_type == WF_F32 ? KEEP_F32 : a.z_type == WF_F16 && (a.type != WF_F16 || a.act != WF_ACT_NONE) ? KEEP_F16 : KEEP_SAME;
    }
    const Product p{a.x, a.w, a.ldx, a.ldw, a.m, a.n, a.k};
    const Epilogue e{a.bias, a.gate, a.resid, a.y, a.z, nullptr, 0, a.ld_resid, a.ldy, a.ldz, a.rows_per_group, a.act, keep, false};
    return run_product<false, false>(p, e, a.type, reinterpret_cast<cudaStream_t>(stream));
}

namespace wf {
namespace {
// Whether a backward pass writes dz: the products read dy itself where dz is dy and TMA can read it.
bool makes_dz(const wf_linear_grad_args &a) {
    return (a.dx || a.dw) && (a.act != WF_ACT_NONE || a.gate || !operand_ok(a.dy, a.n, a.lddy));
}
int64_t backward_bytes(const wf_linear_grad_args &a) { return (makes_dz(a) ? dz_bytes(a.m, a.n) : 0) + linear_grad_bytes(a); }
}  // namespace
}  // namespace wf

extern "C" WF_API int64_t wf_linear_backward_workspace(int64_t m, int64_t n, int64_t rows_per_group) {
    using namespace wf;
    if (!sizes_ok(m, n, 1) || m < 1 || n < 1 || rows_per_group < 1) return 0;
    return dz_bytes(m, n) + linear_grad_most_bytes(m, n, rows_per_group);
}

extern "C" WF_API int64_t wf_linear_backward_needs(const wf_linear_grad_args *args) {
    using namespace wf;
    if (args == nullptr || !sizes_ok(args->m, args->n, 1) || args->m < 1 || args->n < 1 || args->rows_per_group < 1) return 0;
    return backward_bytes(*args);
}

extern "C" WF_API int wf_linear_backward(const wf_linear_grad_args *args, wf_stream_t stream) {
    using namespace wf;
    if (args == nullptr) return WF_ERR_ARG;
    const wf_linear_grad_args &a = *args;
    if (a.type != WF_BF16 && a.type != WF_F16) return WF_ERR_UNSUPPORTED;
    if (a.act < WF_ACT_NONE || a.act > WF_ACT_GELU_TANH) return WF_ERR_UNSUPPORTED;
    if (a.z != nullptr && a.z_type != WF_F32 && a.z_type != WF_F16 && a.z_type != a.type) return WF_ERR_UNSUPPORTED;
    if (!sizes_ok(a.m, a.n, a.k) || a.m < 1 || a.n < 1 || a.rows_per_group < 1 || !a.dy || a.lddy < a.n ||
        !aligned_to(a.dy, 2) || (a.z && (a.ldz < a.n || !aligned_to(a.z, dtype_size(a.z_type)))) ||
        ((a.act != WF_ACT_NONE || a.dg) && !a.z) || !aligned_to(a.gate, 2) || !aligned_to(a.db, 2) || !aligned_to(a.dg, 2))
        return WF_ERR_ARG;
    if (a.dx && (!operand_ok(a.w, a.k, a.ldw) || a.lddx < a.k || !aligned_to(a.dx, 2))) return WF_ERR_ARG;
    if (a.dw && (!operand_ok(a.x, a.k, a.ldx) || a.lddw < a.k || !aligned_to(a.dw, 2))) return WF_ERR_ARG;
    if (!a.dx && !a.dw && !a.db && !a.dg) return WF_OK;
    const bool make_dz = makes_dz(a);
    if ((make_dz || a.db || a.dg) && (!a.workspace || !aligned_to(a.workspace, 16) || a.workspace_bytes < backward_bytes(a)))
        return WF_ERR_ARG;
    int rc = check_device();
    int *word = nullptr;
    if (rc == WF_OK) rc = alarm_of_device(&word);  // before the first launch, not between two
    if (rc != WF_OK) return rc;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const void *dz = a.dy;
    int64_t lddz = a.lddy;
    if (make_dz || a.db || a.dg) {
        if (make_dz) {
            dz = a.workspace;
            lddz = (a.n + 7) / 8 * 8;
        }
        float *part = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + (make_dz ? dz_bytes(a.m, a.n) : 0));
        rc = linear_grad(a, make_dz ? a.workspace : nullptr, lddz, part, st);
        if (rc != WF_OK) return rc;
    }
    if (a.dx) {
        const Product p{dz, a.w, lddz, a.ldw, a.m, a.k, a.n};
        rc = run_product<false, true>(p, plain_epilogue(a.dx, a.lddx), a.type, st);
        if (rc != WF_OK) return rc;
    }
    if (a.dw) {
        const Product p{dz, a.x, lddz, a.ldx, a.n, a.k, a.m};
        rc = run_product<true, true>(p, plain_epilogue(a.dw, a.lddw), a.type, st);
    }
    return rc;
}

extern "C" WF_API int wf_linear_set_wait_limit(uint64_t limit_ns) {
    wf::g_wait_ns.store(limit_ns == 0 ? wf::kWaitLimitNs : std::min<uint64_t>(limit_ns, wf::kWaitLimitNs));
    return WF_OK;
}

extern "C" WF_API int wf_linear_status(int *status) {
    if (status == nullptr) return WF_ERR_ARG;
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, wf::g_linear_status, sizeof(int));
    if (e != cudaSuccess) return static_cast<int>(e);
    if (v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(wf::g_linear_status, &zero, sizeof(int));
        int *word = nullptr;
        if (wf::alarm_of_device(&word) == WF_ERR_EXPIRED) *word = 0;
    }
    *status = v;
    return WF_OK;
}
