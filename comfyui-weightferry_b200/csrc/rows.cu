// The sum of partial column sums (see wf_rows.cuh) and the copy of rows to an aligned row pitch.

#include "wf_rows.cuh"

namespace wf {
namespace {

struct ReduceArgs {
    PartialSum sum[2];
    int64_t d;
};

// Block (x, y, z): columns 32 x .. 32 x + 31 of groups y, y + gridDim.y, ... of sum z. Warp w takes parts w,
// w + warps, ..., then a tree adds the warps' sums: a fixed order for a given shape. A few MB at most; bound by latency:
// 8 to 32 warps by the number of parts.
template <int T>
__global__ void __launch_bounds__(1024) reduce_partials_kernel(const __grid_constant__ ReduceArgs a) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    const PartialSum &sum = a.sum[blockIdx.z];
    wait_prior_grid();
    for (int64_t g = blockIdx.y; g < sum.groups; g += gridDim.y) {
        float s = 0.f;
        if (col < a.d)
#pragma unroll 8
            for (int64_t p = warp; p < sum.parts; p += warps) s += sum.part[(g * sum.parts + p) * a.d + col];
        red[warp][lane] = s;
        __syncthreads();
        for (int c = warp; c < 32; c += warps) {  // a warp adds the sums of a column
            const float t = warp_sum(lane < warps ? red[lane][c] : 0.f);
            if (lane == 0 && blockIdx.x * 32ll + c < a.d) store1<T>(row_of<T>(sum.out, g, a.d), blockIdx.x * 32ll + c, t);
        }
        __syncthreads();
    }
}

}  // namespace

int reduce_partials(const PartialSum &s0, const PartialSum &s1, int64_t d, int type, cudaStream_t stream) {
    if (s0.out == nullptr && s1.out == nullptr) return WF_OK;
    ReduceArgs a{{s0.out != nullptr ? s0 : s1, s1}, d};
    const bool both = s0.out != nullptr && s1.out != nullptr;
    const int64_t groups = both ? std::max(s0.groups, s1.groups) : a.sum[0].groups;
    const dim3 grid(static_cast<unsigned>((d + 31) / 32), static_cast<unsigned>(std::min<int64_t>(groups, 32768)), both ? 2 : 1);
    const int64_t parts = both ? std::max(s0.parts, s1.parts) : a.sum[0].parts;
    const int threads = parts >= 512 ? 1024 : parts >= 200 ? 512 : 256;
    if (type == WF_F32) return launch_rows(reduce_partials_kernel<WF_F32>, grid, threads, stream, a);
    if (type == WF_BF16) return launch_rows(reduce_partials_kernel<WF_BF16>, grid, threads, stream, a);
    return launch_rows(reduce_partials_kernel<WF_F16>, grid, threads, stream, a);
}

namespace {

struct CopyRows {
    const uint16_t *src;
    uint16_t *dst;
    int64_t rows, cols, lds, ldd;
};
struct CopyRowsArgs {
    CopyRows job[2];
};

// Rows of 16-bit values to another row pitch (job blockIdx.y): a warp a piece of 256 values, neighbouring values in
// neighbouring lanes (the source may have any 2-byte alignment).
__global__ void __launch_bounds__(256) copy_rows_kernel(const __grid_constant__ CopyRowsArgs args) {
    const CopyRows &a = args.job[blockIdx.y];
    const int64_t per = (a.cols + 255) / 256;  // pieces of a row
    const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
    wait_prior_grid();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < a.rows * per; i += step) {
        const int64_t row = i / per, col = i % per * 256 + (threadIdx.x & 31);
        const uint16_t *s = a.src + row * a.lds + col;
        uint16_t *d = a.dst + row * a.ldd + col;
        uint16_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + 32 * j < a.cols) v[j] = s[32 * j];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + 32 * j < a.cols) d[32 * j] = v[j];
    }
}

int copy_job(CopyRows &job, const wf_copy_rows &c) {
    if (c.rows < 0 || c.cols < 0 || c.ld_src < c.cols || c.ld_dst < c.cols) return WF_ERR_ARG;
    if (c.rows > 0 && c.cols > 0 && (!c.src || !c.dst || !aligned_to(c.src, 2) || !aligned_to(c.dst, 2))) return WF_ERR_ARG;
    job = CopyRows{static_cast<const uint16_t *>(c.src), static_cast<uint16_t *>(c.dst), c.cols > 0 ? c.rows : 0, c.cols, c.ld_src,
                   c.ld_dst};
    return WF_OK;
}

}  // namespace
}  // namespace wf

extern "C" WF_API int wf_copy_rows16(const wf_copy_rows *copies, int n_copies, wf_stream_t stream) {
    using namespace wf;
    if (copies == nullptr || n_copies < 1 || n_copies > 2) return WF_ERR_ARG;
    CopyRowsArgs a = {};
    int64_t pieces = 0;
    for (int i = 0; i < n_copies; ++i) {
        const int rc = copy_job(a.job[i], copies[i]);
        if (rc != WF_OK) return rc;
        pieces = std::max(pieces, a.job[i].rows * ((a.job[i].cols + 255) / 256));
    }
    if (pieces == 0) return WF_OK;
    const int rc = check_device();
    if (rc != WF_OK) return rc;
    const int grid = static_cast<int>(std::min<int64_t>((pieces + 7) / 8, wave_ctas_at<copy_rows_kernel>(256)));
    return launch_rows(copy_rows_kernel, dim3(grid, n_copies), 256, reinterpret_cast<cudaStream_t>(stream), a);
}
