// What the two halves of the dense linear layer's backward pass share.
#pragma once

#include "wf_common.cuh"

namespace wf {

// bytes of partial sums of linear_grad, and the most that any choice of results takes
int64_t linear_grad_bytes(const wf_linear_grad_args &g);
int64_t linear_grad_most_bytes(int64_t m, int64_t n, int64_t rows_per_group);
// The element-wise half: dz (may be null) [m, n] with pitch lddz, and g.db and g.dg (may be null) by way of `part`. The
// caller has checked g.
int linear_grad(const wf_linear_grad_args &g, void *dz, int64_t lddz, float *part, cudaStream_t stream);

}  // namespace wf
