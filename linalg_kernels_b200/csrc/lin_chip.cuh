// lin_chip.cuh — what the on-chip Newton-Schulz kernels share: clusters, fp16 tiles in shared memory
// (128-byte-swizzled blocks of 64 columns), conversions.
#pragma once

#include <cuda.h>

#include "chol_tc_ptx.cuh"
#include "lin_elem.cuh"

namespace lin {
namespace chip {

using namespace chol::tcx;
using chol::fence_proxy_async_smem;
using chol::smem_u32;

constexpr int kBlockBytes = 128 * 128;  // 128 rows x 64 fp16 columns

__device__ __forceinline__ uint32_t rank_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void sync_cluster() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ double ld_remote_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_remote16(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void st_remote_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void mma_half(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// X as B operand of B X: N = its columns (contiguous), K = its rows. The next 64 columns are one
// block further, the next 8 rows 1024 bytes.
__device__ __forceinline__ uint64_t desc_cols(const void* tile) {
  const uint32_t addr = smem_u32(tile);
  uint64_t d = 0;
  d |= uint64_t((addr >> 4) & 0x3FFF);
  d |= uint64_t(kBlockBytes >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
// fp16 operands, FP32 sums, M = 128.
__device__ __forceinline__ uint32_t idesc_half(int n, int b_mn_major) {
  return (1u << 4) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// Byte offset of the 16-byte chunk holding columns c .. c + 7 of row r.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return uint32_t(c >> 6) * kBlockBytes + uint32_t(r) * 128 + ((uint32_t(c >> 3) & 7) ^ (r & 7)) * 16;
}

// Eight values to fp16 (and the remainder plane): shared-memory chunks of 16 bytes. Saturating: an
// infinity in one matrix would reach the others of its tile as 0 * inf in B X. (Coefficients that
// could take a matrix there are refused, lin_ortho.cu: 65504 stands for singular values of G of 16
// in full precision and 64 in half.)
__device__ __forceinline__ uint32_t half2_sat(float a, float b) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <bool SPLIT>
__device__ __forceinline__ void round8v(const float (&v)[8], uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = half2_sat(v[2 * j], v[2 * j + 1]);
    if (SPLIT) {
      const __half2 x = *reinterpret_cast<const __half2*>(&h[j]);
      l[j] = half2_sat(v[2 * j] - __low2float(x), v[2 * j + 1] - __high2float(x));
    }
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  if (SPLIT) lo = make_uint4(l[0], l[1], l[2], l[3]);
}
// v += f * (eight fp16 values)
__device__ __forceinline__ void add8(float (&v)[8], uint4 w, float f) {
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = __half22float2(h[j]);
    const float2 r = chol::ffma2(make_float2(f, f), x, make_float2(v[2 * j], v[2 * j + 1]));
    v[2 * j] = r.x;
    v[2 * j + 1] = r.y;
  }
}

// k / d for the divisor whose rounded-up 2^32 / d is given; exact while k * d < 2^32.
__device__ __forceinline__ int div_by(int k, uint32_t reciprocal, int d) {
  return d == 1 ? k : int(__umulhi(uint32_t(k), reciprocal));
}
// Sum of squares of eight values, in FP32 (of scaled values where a square could leave its range)
// and handed on in FP64: converting every element costs more than everything else here.
__device__ __forceinline__ double squares8(const float (&u)[8], int count) {
  float top = 0.f, s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) {
      top = fmaxf(top, fabsf(u[j]));
      s = fmaf(u[j], u[j], s);
    }
  if (s != s || top == 0.f || (top > 0x1p-40f && top < 0x1p50f)) return double(s);
  if (isinf(top)) return double(top);
  const int k = ilogbf(top) / 2;
  const float f = ldexpf(1.f, -k);
  s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) s = fmaf(u[j] * f * f, u[j] * f * f, s);
  return ldexp(double(s), 4 * k);
}

}  // namespace chip
}  // namespace lin
