// lin_common.cuh — shared declarations of the half-precision tensor-core products
// (lin_gemm.cu), the Newton-Schulz orthogonalisation (lin_ortho.cu) and the grouped products
// (lin_grouped.cu). C ABI: include/linalg_b200.h.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/linalg_b200.h"
#include "chol_common.cuh"

namespace lin {

using chol::griddep_launch;
using chol::griddep_wait;

// What the epilogue of a product does with alpha * acc (+ beta * C).
enum Epilogue : int {
  kStore16 = 0,  // rounded to 16 bits (the operands' type), masked to the output's rows
  kPlanes = 1,   // fp16 plane(s) of the iteration's workspace, C from such planes, mirrored when
                 // symmetric
  kFinal = 2,    // the caller's matrix: bf16, fp16 or fp32
  kMuon = 3,     // the caller's weights: w <- decay * w - rate * value
};

// Which index of the product is ragged.
enum Mode : int {
  kBatch = 0,    // a batch of equal products
  kRaggedM = 1,  // rows of A and of the output grouped by offsets; B per group
  kRaggedK = 2,  // the summed index grouped by offsets; the output per group
};

// One operand: `rows` x `cols` elements of 16 bits, the columns contiguous, rows `ld` apart,
// `count` such matrices `stride` elements apart (all of them multiples of 8, base 16-byte
// aligned). `mn_major`: the contiguous index is the output's (M or N) and not the summed one.
struct Operand {
  const void* base;
  int64_t rows, cols, ld, count, stride;
  bool mn_major;
};

struct Product {
  Operand a, b;
  int mode = kBatch;
  int epilogue = kStore16;
  bool bf16 = false;  // operand type: bf16 or fp16
  bool split = false; // two planes (high, low) per matrix in both operands: three products
  bool symmetric = false;
  int64_t m = 0, n = 0, k = 0, batch = 1;
  float alpha = 1.f, beta = 0.f;
  float diag = 0.f;  // kPlanes: added to the diagonal
  // kPlanes: C and the output are fp16 planes; matrix i, plane p at
  // base + (i * planes + p) * plane elements, rows ldc / ldo apart
  const void* c = nullptr;
  int64_t ldc = 0, c_plane = 0;
  void* out = nullptr;
  int64_t ldo = 0, out_stride = 0;
  int out_type = 0;  // LINALG_BF16 / LINALG_FP16 / LINALG_FP32
  float decay = 1.f, rate = 0.f;  // kMuon
  // ragged modes
  const void* offsets = nullptr;
  int offsets64 = 0;
  int64_t total_rows = 0;
  int fill = 0;  // kRaggedM: rows of no group are set to zero (otherwise left as they are)
};

constexpr int kMaxGroups = 1024;

// Newton-Schulz in fp16 (one plane, or two with split): the scales of X and of B; G has X's squared.
__host__ __device__ constexpr float x_scale(bool split) { return split ? 64.f : 32.f; }
__host__ __device__ constexpr float b_scale(bool split) { return split ? 2048.f : 1.f; }

int launch_product(const Product& p, cudaStream_t q);
cudaError_t prepare_products();

// Checks the device once (sm_100) and sets the kernels' shared-memory limits.
int prepare_device(int dev);
int prepare_current();
// SMs of the device that this thread's call runs on (prepare_current sets it).
int sm_count();
void use_sm_count(int sms);

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}

}  // namespace lin
