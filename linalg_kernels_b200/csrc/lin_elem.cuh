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

template <typename T>
__device__ __forceinline__ void load8t(const T* p, float (&v)[8], int count, bool vec) {
  if (vec && count == 8) {
    alignas(16) T h[8];
#pragma unroll
    for (int j = 0; j < int(sizeof(T)) / 2; ++j)
      reinterpret_cast<uint4*>(h)[j] = reinterpret_cast<const uint4*>(p)[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(h[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < count ? to_float(p[j]) : 0.f;
  }
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
__device__ __forceinline__ void load_any(const Matrix& x, int64_t at, float (&v)[8], int count) {
  if (x.type == LINALG_BF16)
    load8t(static_cast<const __nv_bfloat16*>(x.data) + at, v, count, x.vec);
  else if (x.type == LINALG_FP16)
    load8t(static_cast<const __half*>(x.data) + at, v, count, x.vec);
  else
    load8t(static_cast<const float*>(x.data) + at, v, count, x.vec);
}
__device__ __forceinline__ void store_any(const Matrix& x, int64_t at, float (&v)[8], int count) {
  if (x.type == LINALG_BF16)
    store8t(static_cast<__nv_bfloat16*>(x.data) + at, v, count, x.vec);
  else if (x.type == LINALG_FP16)
    store8t(static_cast<__half*>(x.data) + at, v, count, x.vec);
  else
    store8t(static_cast<float*>(x.data) + at, v, count, x.vec);
}

// Eight columns as loaded: the conversion comes later, so that several loads are in flight at a
// time (a load is waited for where its register is used).
struct Raw8 {
  uint32_t w[8];  // 16-bit types: four words
};
__device__ __forceinline__ void load_raw(const Matrix& x, int64_t at, int count, Raw8& r) {
  if (x.vec && count == 8) {
    const uint4* p = x.type == LINALG_FP32
                         ? reinterpret_cast<const uint4*>(static_cast<const float*>(x.data) + at)
                         : reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x.data) + at);
    const uint4 a = p[0];
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    if (x.type == LINALG_FP32) {
      const uint4 b = p[1];
      r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
    }
  } else if (x.type == LINALG_FP32) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      r.w[j] = j < count ? static_cast<const uint32_t*>(x.data)[at + j] : 0u;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t* p = static_cast<const uint16_t*>(x.data) + at + 2 * j;
      const uint32_t lo = 2 * j < count ? p[0] : 0, hi = 2 * j + 1 < count ? p[1] : 0;
      r.w[j] = lo | (hi << 16);
    }
  }
}
__device__ __forceinline__ float bits_to_float(uint32_t w, int type) {  // one element, low bits
  if (type == LINALG_FP32) return __uint_as_float(w);
  if (type == LINALG_BF16) return __uint_as_float(w << 16);
  return __half2float(__ushort_as_half(uint16_t(w)));
}
__device__ __forceinline__ void convert_raw(const Raw8& r, int type, float (&v)[8]) {
  if (type == LINALG_FP32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r.w[j]);
  } else if (type == LINALG_BF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(r.w[j] << 16);
      v[2 * j + 1] = __uint_as_float(r.w[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = *reinterpret_cast<const __half2*>(&r.w[j]);
      v[2 * j] = __low2float(h);
      v[2 * j + 1] = __high2float(h);
    }
  }
}
__device__ __forceinline__ uint32_t load_one(const Matrix& x, int64_t at) {
  return x.type == LINALG_FP32 ? static_cast<const uint32_t*>(x.data)[at]
                               : uint32_t(static_cast<const uint16_t*>(x.data)[at]);
}
__device__ __forceinline__ void store_one(const Matrix& x, int64_t at, float v) {
  if (x.type == LINALG_FP32)
    static_cast<float*>(x.data)[at] = v;
  else if (x.type == LINALG_BF16)
    static_cast<__nv_bfloat16*>(x.data)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(x.data)[at] = __float2half_rn(v);
}

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
