// lin_elem.cuh — element access of the orthogonalisation's first and last passes: caller matrices
// of any supported type and alignment, eight columns at a time.
#pragma once

#include "lin_common.cuh"

namespace lin {

struct Matrix {
  void* data;
  int64_t ld, stride;
  int type;
  int vec;  // rows of 8 elements can be accessed 16 bytes at a time
};

inline Matrix device_matrix(const linalg_matrix* x) {
  Matrix d{x->data, x->ld, x->stride, x->type, 0};
  const int per16 = x->type == LINALG_FP32 ? 4 : 8;
  d.vec = reinterpret_cast<uintptr_t>(x->data) % 16 == 0 && x->ld % per16 == 0 &&
          x->stride % per16 == 0;
  return d;
}
// Which instance reads (in: 1 bf16 with a momentum of fp32 or none, 2 fp32 with fp32 or none, 3 bf16
// with bf16) or writes (out: 1 bf16, 2 fp32) the matrices in whole aligned chunks of eight columns;
// 0: the one for any types, alignment and number of columns.
inline int input_path(const Matrix& x, const Matrix* momentum, int64_t n) {
  if (n % 8 || !x.vec || (momentum != nullptr && !momentum->vec)) return 0;
  const int m = momentum == nullptr ? LINALG_FP32 : momentum->type;
  if (x.type == LINALG_BF16) return m == LINALG_FP32 ? 1 : (m == LINALG_BF16 ? 3 : 0);
  return x.type == LINALG_FP32 && m == LINALG_FP32 ? 2 : 0;
}
inline int output_path(const Matrix& x, int64_t n) {
  if (n % 8 || !x.vec) return 0;
  return x.type == LINALG_BF16 ? 1 : (x.type == LINALG_FP32 ? 2 : 0);
}

template <typename T>
__device__ __forceinline__ void store8t(T* p, float (&v)[8], int count, bool vec) {
  alignas(16) T h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    h[j] = from_float<T>(v[j]);
    v[j] = to_float(h[j]);  // what the array now holds
  }
  if (vec && count == 8) {
#pragma unroll
    for (int j = 0; j < int(sizeof(T)) / 2; ++j)
      reinterpret_cast<uint4*>(p)[j] = reinterpret_cast<const uint4*>(h)[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) p[j] = h[j];
  }
}
__device__ __forceinline__ void store_any(const Matrix& x, int64_t at, float (&v)[8], int count) {
  if (x.type == LINALG_BF16)
    store8t(static_cast<__nv_bfloat16*>(x.data) + at, v, count, x.vec);
  else if (x.type == LINALG_FP16)
    store8t(static_cast<__half*>(x.data) + at, v, count, x.vec);
  else
    store8t(static_cast<float*>(x.data) + at, v, count, x.vec);
}

__device__ __forceinline__ float load_one(const Matrix& x, int64_t at) {
  if (x.type == LINALG_FP32) return static_cast<const float*>(x.data)[at];
  if (x.type == LINALG_BF16) return to_float(static_cast<const __nv_bfloat16*>(x.data)[at]);
  return to_float(static_cast<const __half*>(x.data)[at]);
}

// Eight columns as loaded: the conversion comes later, so that several loads are in flight at a
// time. `T` an element type: whole aligned chunks; `Any`: a matrix of any type, alignment and
// number of columns.
struct Any {};
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const Matrix& x, int64_t at, int) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(x.data) + at);
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) w[i] = p[i];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const T* h = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(h[j]);
  }
  // v: as rounded to the array's type on return
  static __device__ __forceinline__ void put(const Matrix& x, int64_t at, float (&v)[8], int) {
    store8t(static_cast<T*>(x.data) + at, v, 8, true);
  }
};
template <>
struct Eight<Any> {
  float w[8];
  __device__ __forceinline__ void load(const Matrix& x, int64_t at, int count) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < count ? load_one(x, at + j) : 0.f;
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = w[j];
  }
  static __device__ __forceinline__ void put(const Matrix& x, int64_t at, float (&v)[8],
                                             int count) {
    store_any(x, at, v, count);
  }
};

// The factor F of X = F * u, F = scale / (norm + eps), as a power of two near its square root (x)
// times the rest (y): F alone passes FP32's range for norms of subnormals and for the largest
// ones, (u * x) * y does not. Not finite: the matrix holds a NaN or an infinity (or norm + eps
// is zero).
__device__ __forceinline__ float2 start_factor(double squares, float scale, float eps) {
  const double f = double(scale) / (sqrt(squares) + double(eps));
  if (!isfinite(f) || !isfinite(squares)) {
    const float nan = __int_as_float(0x7fc00000);
    return make_float2(nan, nan);
  }
  const int k = ilogb(f) / 2;
  return make_float2(float(ldexp(1.0, k)), float(ldexp(f, -k)));
}
__device__ __forceinline__ float start_scaled(float u, float2 f) { return (u * f.x) * f.y; }

}  // namespace lin
