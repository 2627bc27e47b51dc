// lin_mid.cuh — the one-launch orthogonalisation of matrices with both sides up to 256.
#pragma once

#include "lin_common.cuh"

namespace lin {

// Whether an m x n matrix fits a CTA pair's shared memory (and not one CTA's: lin_small.cuh).
bool mid_supported(int64_t m, int64_t n, bool split);
// As launch_small (half precision only).
int launch_mid_ortho(const linalg_matrix* x, const linalg_matrix* momentum,
                     const linalg_matrix* out, int64_t batch, int64_t m, int64_t n, double beta,
                     int nesterov, float decay, float rate, int steps, const float* coefficients,
                     float eps, cudaStream_t q);
cudaError_t prepare_mid_ortho();

}  // namespace lin
