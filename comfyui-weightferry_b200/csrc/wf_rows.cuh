// Helpers of the kernels that work on rows of f16 / bf16 / f32 values (layer norm, the dense linear layer's gradients):
// typed loads and stores, the split of grouped rows over blocks, and the sum of the blocks' partial column sums.
#pragma once

#include <algorithm>

#include "wf_common.cuh"
#include "wf_launch.cuh"

namespace wf {

// Consecutive groups of rows_per_group rows (the last one may be shorter) dealt to blocks: where there are fewer groups
// than blocks, `chunks` blocks share a group (each takes `chunk_rows` of its rows); else a block takes `per_block` whole
// groups. Either way each block adds up the rows of one group at a time and a group's sum has `chunks` parts.
struct RowSplit {
    int64_t rows, rows_per_group, groups, per_block, chunks, chunk_rows;

    __host__ __device__ int64_t blocks() const {
        return chunks > 1 ? groups * chunks : (groups + per_block - 1) / per_block;
    }
    __host__ __device__ int64_t partials_per_group() const { return chunks; }
    __host__ __device__ int64_t partial_rows() const { return groups * chunks; }
    __device__ int64_t first_group(int64_t block) const { return chunks > 1 ? block / chunks : block * per_block; }
    __device__ int64_t last_group(int64_t block) const {
        return chunks > 1 ? block / chunks + 1 : min((block + 1) * per_block, groups);
    }
    __device__ int64_t partial_row(int64_t block, int64_t group) const { return chunks > 1 ? block : group; }
    __device__ void rows_of(int64_t block, int64_t group, int64_t &lo, int64_t &hi) const {
        const int64_t end = min((group + 1) * rows_per_group, rows);
        lo = group * rows_per_group + (chunks > 1 ? block % chunks * chunk_rows : 0);
        hi = chunks > 1 ? min(lo + chunk_rows, end) : end;
    }
};

// `wanted` blocks (about), at least min_rows rows to a block that shares its group
inline RowSplit make_split(int64_t rows, int64_t rows_per_group, int64_t wanted, int64_t min_rows) {
    RowSplit s;
    s.rows = rows;
    s.rows_per_group = std::min(rows_per_group, rows);
    s.groups = (rows + s.rows_per_group - 1) / s.rows_per_group;
    s.per_block = std::max<int64_t>(1, (s.groups + wanted - 1) / wanted);
    s.chunks = std::max<int64_t>(1, std::min(wanted / s.groups, (s.rows_per_group + min_rows - 1) / min_rows));
    s.chunk_rows = (s.rows_per_group + s.chunks - 1) / s.chunks;
    s.chunks = (s.rows_per_group + s.chunk_rows - 1) / s.chunk_rows;
    return s;
}

// A column sum whose parts blocks have written: out[g, c] = sum over p < parts of part[g * parts + p, c] for g < groups.
// A null out: no such sum.
struct PartialSum {
    const float *part;
    void *out;
    int64_t groups, parts;
};
// Up to two of them over d columns in one launch: float32 in a fixed order, rounded once to `type`.
int reduce_partials(const PartialSum &s0, const PartialSum &s1, int64_t d, int type, cudaStream_t stream);

namespace {

inline bool aligned_to(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// a row of a matrix, from column col0 on
template <int T>
__device__ __forceinline__ const void *row_of(const void *base, int64_t row, int64_t ld, int64_t col0 = 0) {
    return static_cast<const char *>(base) + (row * ld + col0) * dtype_size(T);
}
template <int T>
__device__ __forceinline__ void *row_of(void *base, int64_t row, int64_t ld, int64_t col0 = 0) {
    return static_cast<char *>(base) + (row * ld + col0) * dtype_size(T);
}

template <int T>
__device__ __forceinline__ float load1(const void *row, int64_t col) {
    if constexpr (T == WF_F32) return static_cast<const float *>(row)[col];
    else if constexpr (T == WF_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(row)[col]);
    else return __half2float(static_cast<const __half *>(row)[col]);
}
template <int T>
__device__ __forceinline__ void store1(void *row, int64_t col, float v) {
    if constexpr (T == WF_F32) static_cast<float *>(row)[col] = v;
    else if constexpr (T == WF_BF16) static_cast<__nv_bfloat16 *>(row)[col] = __float2bfloat16_rn(v);
    else static_cast<__half *>(row)[col] = __float2half_rn(v);
}

// the sum of v over the 32 lanes, in every lane
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// two 16-bit values of a word as float32
template <int T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (T == WF_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// 16 bytes from global to shared memory past the registers (cp.async; zeros where `on` is false)
__device__ __forceinline__ void copy16(void *dst, const void *src, bool on = true) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src), "r"(on ? 16 : 0)
                 : "memory");
}

// ... and the pair of float32 values rounded to the type
template <int T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (T == WF_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
// eight values from column col of a row (16-byte aligned)
template <int T>
__device__ __forceinline__ void load8(float (&v)[8], const void *row, int64_t col) {
    if constexpr (T == WF_F32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(row) + col);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(row) + col);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// resident blocks of KERN on the whole device at `threads` threads: unlike wave_ctas, for kernels that are launched
// with several block sizes (one cached count for each multiple of a warp)
template <auto KERN>
int wave_ctas_at(int threads) {
    static std::atomic<int> occ[64][33];
    int dev = 0;
    cudaGetDevice(&dev);
    const int w = threads / 32;
    int o = (dev >= 0 && dev < 64) ? occ[dev][w].load(std::memory_order_relaxed) : 0;
    if (o == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&o, KERN, threads, 0) != cudaSuccess || o < 1) o = 1;
        if (dev >= 0 && dev < 64) occ[dev][w].store(o, std::memory_order_relaxed);
    }
    return o * device_sm_count();
}

template <typename Kern, typename Args>
int launch_rows(Kern kern, dim3 grid, int threads, cudaStream_t stream, const Args &args) {
    const cudaError_t e = launch_dependent(kern, grid, threads, 0, stream, args);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace
}  // namespace wf
