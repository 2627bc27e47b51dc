// lin_tile.cuh — the parts of a CTA pair's 256 x BN tile that the half-precision kernels share:
// stage layout, barriers, TMA and tcgen05 wrappers, and the epilogue of a 32 x 32 piece.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "chol_tc_ptx.cuh"
#include "lin_common.cuh"

namespace lin {

// Tensor map of an operand; boxes of 64 columns x box_rows (64 x 64 when MN-major). (lin_gemm.cu)
bool make_operand_map(CUtensorMap* map, const Operand& o, bool bf16, int box_rows);

namespace tile {

using namespace chol::tcx;
using chol::fence_proxy_async_smem;
using chol::smem_u32;

constexpr int kBlockK = 64;     // 16-bit elements of K per stage: one 128-byte swizzle row
constexpr int kTileM = 256;     // rows of a pair's tile
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kEpiLd = 33;      // staging row stride in floats: conflict-free by row and by column
constexpr int kChunk = 4;       // split: K blocks per drained accumulator

template <int BN>
struct Cfg {
  static constexpr int STAGES = BN == 256 ? 6 : 8;
  static constexpr int A_BYTES = 128 * kBlockK * 2;
  static constexpr int B_BYTES = BN / 2 * kBlockK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int EPI = kEpiWarps * 16 * kEpiLd * 4;  // half a piece per warp
  static constexpr int TABLE = 2 * (kMaxGroups + 4) * 4;  // group starts and first tiles
  static constexpr size_t SMEM = size_t(STAGES) * STAGE + EPI + 512 + TABLE + 1024;
  static constexpr int TMEM_COLS = 2 * BN;
};

// ------------------------------- device helpers ---------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void arrive_leader(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait at cluster scope.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* status) {
  if (try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 0;; ++it) {
    if (try_wait_cluster(bar, parity)) return true;
    if ((it & 255u) == 255u && global_ns() - t0 > kWaitLimitNs) {
      atomicExch(status, CHOL_ERR_WAIT_TIMEOUT);
      return false;
    }
  }
}
// A copy of a pair: the barrier may be the other CTA's (a shared::cluster address).
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y,
                                              int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}
// MN-major operand, 128-byte swizzle: boxes of 64 MN elements x 64 K rows (8 KB), the next box
// 64 MN elements further; groups of 8 K rows 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc_mn(const void* smem_tile) {
  const uint32_t addr = smem_u32(smem_tile);
  uint64_t d = 0;
  d |= uint64_t((addr >> 4) & 0x3FFF);
  d |= uint64_t(8192 >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}

// 32-byte accesses: a lane holds 32 columns of one row, so each access is one whole sector.
__device__ __forceinline__ void ldg32(const void* p, uint32_t* r) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void stg32(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (sizeof(T) == 4) {
    return 0;
  } else {
    alignas(4) T h[2] = {from_float<T>(a), from_float<T>(b)};
    return *reinterpret_cast<const uint32_t*>(h);
  }
}
template <typename T>
__device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) {
  const T* h = reinterpret_cast<const T*>(&w);
  a = to_float(h[0]);
  b = to_float(h[1]);
}

// 32 columns of a row in 32-byte accesses.
template <typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[32]) {
  constexpr int N = 32 * int(sizeof(T)) / 4;  // words
  uint32_t r[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    r[j] = sizeof(T) == 4 ? __float_as_uint(v[j]) : pack<T>(v[(2 * j) & 31], v[(2 * j + 1) & 31]);
#pragma unroll
  for (int j = 0; j < N; j += 8) stg32(reinterpret_cast<uint32_t*>(p) + j, r + j);
}
template <typename T>
__device__ __forceinline__ void load_row(const T* p, float (&v)[32]) {
  constexpr int N = 32 * int(sizeof(T)) / 4;
  uint32_t r[N];
#pragma unroll
  for (int j = 0; j < N; j += 8) ldg32(reinterpret_cast<const uint32_t*>(p) + j, r + j);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (sizeof(T) == 4)
      v[j] = __uint_as_float(r[j]);
    else
      unpack<T>(r[j], v[2 * j], v[2 * j + 1]);
  }
}
template <typename T>
__device__ __forceinline__ void write_row(T* p, float (&v)[32], bool weights, float decay,
                                          float rate) {
  if (weights) {
    float w[32];
    load_row(p, w);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = fmaf(-rate, v[j], decay * w[j]);
  }
  store_row(p, v);
}
// One column of a 32 x 32 piece's row (any alignment, any number of columns).
template <typename T>
__device__ __forceinline__ void write_one(T* p, float v, bool weights, float decay, float rate) {
  if (weights) v = fmaf(-rate, v, decay * to_float(*p));
  *p = from_float<T>(v);
}

// What a warp does with a 32 x 32 piece of accumulators (a lane holds 32 columns of one row):
// alpha * acc + beta * C, to the output. All pointers are those of one matrix (or group).
struct Piece {
  const __half* c;  // fp16 plane(s), rows ldc apart; 32-byte aligned rows
  int64_t ldc, c_plane;
  float alpha, beta;
  void* out;  // kPlanes: plane 0, rows on 32-byte boundaries; else the caller's element (0, 0)
  int64_t ldo, out_plane;
  int out_type, out_vec;  // out_vec: rows of the caller's matrix start on 32-byte boundaries
  float decay, rate;      // kMuon
  int rows, n;            // rows and columns of the output
};

// C of one piece, this lane's row (whole pieces only; loaded ahead of their use).
template <int EPI, bool SPLIT>
__device__ __forceinline__ void load_c(const Piece& g, int row, int gc0,
                                       uint32_t (&cw)[SPLIT ? 2 : 1][16]) {
  if (EPI == kStore16 || g.beta == 0.f || row >= g.rows || gc0 + 32 > g.n) return;
  const __half* cp = g.c + int64_t(row) * g.ldc + gc0;
#pragma unroll
  for (int p = 0; p < (SPLIT ? 2 : 1); ++p) {
    ldg32(cp + p * g.c_plane, cw[p]);
    ldg32(cp + p * g.c_plane + 16, cw[p] + 8);
  }
}

// `mirror`: a symmetric result's tile below the diagonal is written to its transposed place too.
// `stage`: 16 rows of kEpiLd floats of this warp's own.
template <int EPI, bool SPLIT>
__device__ __forceinline__ void finish_piece(const Piece& g, float (&v)[32], int lane, int row_base,
                                             int gc0, const uint32_t (&cw)[SPLIT ? 2 : 1][16],
                                             bool mirror, float* stage) {
  constexpr int P = SPLIT ? 2 : 1;
  if (gc0 >= g.n || row_base >= g.rows) return;
  const int row = row_base + lane;
  const int cols = g.n - gc0 < 32 ? g.n - gc0 : 32;
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] *= g.alpha;
  if (EPI != kStore16 && g.beta != 0.f) {
    if (cols == 32) {
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float c0, c1;
          unpack<__half>(cw[p][j], c0, c1);
          v[2 * j] = fmaf(g.beta, c0, v[2 * j]);
          v[2 * j + 1] = fmaf(g.beta, c1, v[2 * j + 1]);
        }
    } else if (row < g.rows) {
      const __half* cp = g.c + int64_t(row) * g.ldc + gc0;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < cols)
          for (int p = 0; p < P; ++p)
            v[j] = fmaf(g.beta, __half2float(cp[p * g.c_plane + j]), v[j]);
    }
  }
  if (EPI == kPlanes) {
    // rows of the workspace are padded to whole 32-byte sectors
    __half* o = static_cast<__half*>(g.out);
#pragma unroll
    for (int p = 0; p < P; ++p, o += g.out_plane) {
      uint32_t h[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) h[j] = pack<__half>(v[2 * j], v[2 * j + 1]);
      if (row < g.rows) {
        __half* q0 = o + int64_t(row) * g.ldo + gc0;
        if (cols == 32) {
          stg32(q0, h);
          stg32(q0 + 16, h + 8);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)  // the pad after an odd last column exists
            if (2 * j < cols) reinterpret_cast<uint32_t*>(q0)[j] = h[j];
        }
      }
      if (mirror) {
        // the transposed piece (its columns all exist): neighbouring lanes exchange halves, so that
        // an even lane writes column 2j and an odd one column 2j + 1 of two rows
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, h[j], 1);
          const uint32_t two = (lane & 1) ? __byte_perm(other, h[j], 0x7632)
                                          : __byte_perm(h[j], other, 0x5410);
          const int r = row & ~1;
          if (r < g.rows)
            *reinterpret_cast<uint32_t*>(o + int64_t(gc0 + 2 * j + (lane & 1)) * g.ldo + r) = two;
        }
      }
      if (SPLIT && p == 0) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float c0, c1;
          unpack<__half>(h[j], c0, c1);
          v[2 * j] -= c0;
          v[2 * j + 1] -= c1;
        }
      }
    }
    return;
  }
  constexpr bool kWeights = EPI == kMuon;
  if (cols == 32 && g.out_vec) {
    if (row < g.rows) {
      const int64_t at = int64_t(row) * g.ldo + gc0;
      if (g.out_type == LINALG_BF16)
        write_row(static_cast<__nv_bfloat16*>(g.out) + at, v, kWeights, g.decay, g.rate);
      else if (g.out_type == LINALG_FP16)
        write_row(static_cast<__half*>(g.out) + at, v, kWeights, g.decay, g.rate);
      else if (EPI != kStore16)
        write_row(static_cast<float*>(g.out) + at, v, kWeights, g.decay, g.rate);
    }
    return;
  }
  // rows that do not start on sectors, or the last columns: through shared memory, half a piece at
  // a time, so that a warp writes along a row
#pragma unroll 1
  for (int h = 0; h < 32; h += 16) {
    if ((lane & 16) == h) {
#pragma unroll
      for (int j = 0; j < 32; ++j) stage[(lane & 15) * kEpiLd + j] = v[j];
    }
    __syncwarp();
    const int left = g.rows - row_base - h, rows = left < 16 ? left : 16;
    if (lane < cols) {
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const float x = stage[r * kEpiLd + lane];
        const int64_t at = int64_t(row_base + h + r) * g.ldo + gc0 + lane;
        if (g.out_type == LINALG_BF16)
          write_one(static_cast<__nv_bfloat16*>(g.out) + at, x, kWeights, g.decay, g.rate);
        else if (g.out_type == LINALG_FP16)
          write_one(static_cast<__half*>(g.out) + at, x, kWeights, g.decay, g.rate);
        else if (EPI != kStore16)
          write_one(static_cast<float*>(g.out) + at, x, kWeights, g.decay, g.rate);
      }
    }
    __syncwarp();
  }
}

}  // namespace tile
}  // namespace lin
