// lin_small.cuh — the one-launch orthogonalisation of matrices whose smaller side is at most 128.
#pragma once

#include "lin_common.cuh"

namespace lin {

// Whether an m x n matrix fits one cluster's shared memory.
bool small_supported(int64_t m, int64_t n, bool split);
// momentum == nullptr: out = orthogonalize(x); else the optimiser step on out. No workspace.
int launch_small(const linalg_matrix* x, const linalg_matrix* momentum, const linalg_matrix* out,
                 int64_t batch, int64_t m, int64_t n, double beta, int nesterov, float decay,
                 float rate, int steps, const float* coefficients, float eps, bool split,
                 cudaStream_t q);
cudaError_t prepare_small_ortho();

}  // namespace lin
