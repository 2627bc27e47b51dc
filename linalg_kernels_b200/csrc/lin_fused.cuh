// lin_fused.cuh — a batch's Newton-Schulz iteration in one launch, a CTA pair per matrix.
#pragma once

#include "lin_common.cuh"

namespace lin {

struct FusedCall {
  int64_t batch, m, n;
  const void* x0;  // fp16 start values, rows ldx apart, matrices x_plane apart
  void* x;         // fused_pairs(batch) * 2 such matrices
  void* squares;   // fused_pairs(batch) * 2 squares of the smaller side, rows lds apart
  int64_t ldx, lds, x_plane, s_plane;
  float scale;     // X's (G has its square, B 1)
  int steps;
  const float* coefficients;
  bool muon;  // out <- decay * out - rate * result, else out <- result
  void* out;
  int64_t ldo, out_stride;
  int out_type;
  float decay, rate;
};

// Pairs a launch uses (each needs its own X and squares).
int fused_pairs(int64_t batch);
bool fused_better(int64_t batch, int64_t m, int64_t n);
int launch_fused(const FusedCall& f, cudaStream_t q);
cudaError_t prepare_fused();

}  // namespace lin
