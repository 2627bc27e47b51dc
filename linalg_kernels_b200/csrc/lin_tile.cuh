// lin_tile.cuh — the parts of a CTA pair's 256 x BN tile that the half-precision kernels share:
// stage layout, barriers, TMA and tcgen05 wrappers, and the epilogue of a 32 x 32 piece.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "chol_tc_ptx.cuh"
#include "lin_common.cuh"

namespace lin {

// Tensor map of an operand; boxes of 64 columns x box_rows (64 x 64 when MN-major). (lin_gemm.cu)
bool make_operand_map(CUtensorMap* map, const Operand& o, bool bf16, int box_rows);
// Map of an output's (or C's) boxes: 64 columns x 32 rows, or 32 x 64 unswizzled for mirrored ones.
bool make_output_map(CUtensorMap* map, const Operand& o, bool bf16, bool mirrored);

namespace tile {

using namespace chol::tcx;
using chol::fence_proxy_async_smem;
using chol::smem_u32;

constexpr int kBlockK = 64;     // 16-bit elements of K per stage: one 128-byte swizzle row
constexpr int kTileM = 256;     // rows of a pair's tile
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kEpiLd = 33;      // staging row stride in floats: conflict-free by row and by column

constexpr int kBoxBytes = 32 * 128;  // one warp's 32 rows x 64 columns of 16 bits

// BUFS: boxes of staging per epilogue warp. TABLE: bytes for the group tables. PLANES: of each
// operand in a stage.
template <int BN, int BUFS, int TABLE_BYTES, int PLANES>
struct Cfg {
  static constexpr int STAGES = PLANES == 2 ? 3 : (BN == 512 ? 4 : (BN == 256 ? 5 : 6));
  static constexpr int A_PLANE = 128 * kBlockK * 2;
  static constexpr int B_PLANE = BN / 2 * kBlockK * 2;
  static constexpr int A_BYTES = PLANES * A_PLANE;
  static constexpr int B_BYTES = PLANES * B_PLANE;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int EPI = kEpiWarps * BUFS * kBoxBytes;
  static constexpr int TABLE = TABLE_BYTES;
  static constexpr size_t SMEM = size_t(STAGES) * STAGE + EPI + 512 + TABLE + 1024;
  static constexpr int TMEM_COLS = BN == 512 ? 512 : 2 * BN;  // 512: one tile's, in two halves
  static_assert(SMEM <= 227 * 1024, "shared memory");
};
constexpr int kTableBytes = 2 * (kMaxGroups + 4) * 4;  // group starts and first tiles

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
// The same without ordering memory: for a drained accumulator, whose reads tcgen05.wait::ld and
// tcgen05.fence::before_thread_sync have ordered (a release costs ~1000 cycles here).
__device__ __forceinline__ void arrive_leader_relaxed(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}
// The limit of a wait that spans `blocks` K blocks: 2 us each, five times what one takes where the loads'
// latency paces it (356 ns), on top of the usual limit, which 5.6 million blocks alone would reach.
__device__ __forceinline__ uint64_t limit_of(int64_t blocks) {
  return kWaitLimitNs + uint64_t(blocks) * 2000;
}
// Bounded wait at cluster scope.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* status,
                                         uint64_t limit = kWaitLimitNs) {
  if (try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 0;; ++it) {
    if (try_wait_cluster(bar, parity)) return true;
    if ((it & 255u) == 255u && global_ns() - t0 > limit) {
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
// Two values in one word (one instruction).
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (sizeof(T) == 4) {
    return 0;
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
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

// The group tables, by one warp. start[0 .. groups]: first rows, clamped to [0, rows] and to the
// largest before them.
__device__ __forceinline__ void group_starts(int* start, const void* offsets, int offsets64,
                                             int groups, int rows) {
  const int lane = threadIdx.x & 31;
  int high = 0;
  for (int e0 = 0; e0 <= groups; e0 += 32) {
    const int e = e0 + lane;
    int64_t v = 0;
    if (e <= groups)
      v = offsets64 ? static_cast<const int64_t*>(offsets)[e]
                    : int64_t(static_cast<const int32_t*>(offsets)[e]);
    v = v < 0 ? 0 : (v > rows ? rows : v);
    int x = int(v);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d && y > x) x = y;
    }
    if (x < high) x = high;
    if (e <= groups) start[e] = x;
    high = __shfl_sync(0xffffffffu, x, 31);
  }
  __syncwarp();
}
// first[0 .. n]: first tiles of the groups (of tile_rows rows by tiles_n column tiles) and, with
// fill, of two more: the rows behind the last group and those before the first.
__device__ __forceinline__ void group_tiles(int* first, const int* start, int groups, int fill,
                                            int rows, int tile_rows, int tiles_n) {
  const int lane = threadIdx.x & 31;
  const int n = groups + (fill ? 2 : 0);
  int base = 0;
  for (int e0 = 0; e0 < n; e0 += 32) {
    const int e = e0 + lane;
    int count = 0;
    if (e < groups)
      count = start[e + 1] - start[e];
    else if (e < n)
      count = e == groups ? rows - start[groups] : start[0];
    const int tiles = (count + tile_rows - 1) / tile_rows * tiles_n;
    int x = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (e < n) first[e] = base + x - tiles;
    base += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) first[n] = base;
}

// What an epilogue warp does with its accumulators (a lane holds columns of one row):
// alpha * acc (+ beta * C) (+ diag on the diagonal), to the output. Results and C pass through
// shared memory in boxes of 32 rows x 64 columns that TMA copies: a lane's own 32-byte accesses
// reach half a sector a cycle per SM, 4096 cycles for a 128 x 256 half tile, and took longer
// than its MMAs (b640n512 3.4 ms).
struct Out {
  float alpha, beta, diag;
  int rows, n;  // rows and columns of the output
  // boxes (TMA): plane p of the output at z + p; C likewise; `y`: row 0's coordinate
  const CUtensorMap *map, *mirror, *c_map;
  int z, z_c, y;
  int boxes;  // the output is written by boxes (else, and where a box would pass the rows: below)
  // the caller's matrix, any alignment
  void* out;
  int64_t ldo;
  int type, vec;  // vec: rows start on 32-byte boundaries
  int weights;    // out <- decay * out - rate * value
  float decay, rate;
};

__device__ __forceinline__ void store_box(const CUtensorMap* map, const void* src, int x, int y,
                                          int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(y), "r"(z), "r"(smem_u32(src))
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// This thread's box stores have read shared memory / have written global memory.
__device__ __forceinline__ void boxes_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
// The same but for the newest `newer` (0, 1 or 2).
__device__ __forceinline__ void boxes_read_but(int newer) {
  if (newer == 0)
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  else if (newer == 1)
    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
  else
    asm volatile("cp.async.bulk.wait_group.read 2;" ::: "memory");
}
__device__ __forceinline__ void boxes_written() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// 16-byte chunk c of row r of a box (128-byte rows, 128-byte swizzle).
__device__ __forceinline__ uint4* box_chunk(uint8_t* box, int r, int c) {
  return reinterpret_cast<uint4*>(box + r * 128 + ((c ^ (r & 7)) << 4));
}

// 32 columns of this lane's row straight to the caller's matrix.
template <typename T>
__device__ __forceinline__ void write_direct(const Out& g, float (&v)[32], int lane, int row_base,
                                             int gc0, float* stage) {
  const int row = row_base + lane;
  const int cols = g.n - gc0 < 32 ? g.n - gc0 : 32;
  T* out = static_cast<T*>(g.out);
  if (cols == 32 && g.vec) {
    if (row < g.rows)
      write_row(out + int64_t(row) * g.ldo + gc0, v, g.weights, g.decay, g.rate);
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
      for (int r = 0; r < rows; ++r)
        write_one(out + int64_t(row_base + h + r) * g.ldo + gc0 + lane, stage[r * kEpiLd + lane],
                  g.weights, g.decay, g.rate);
    }
    __syncwarp();
  }
}

// The epilogue of one warp's 32 rows x COLS columns (a multiple of 64).
template <int COLS, int BUFS, bool SPLIT>
struct WarpEpilogue {
  static constexpr int BOXES = COLS / 64;
  static_assert(!SPLIT || (BOXES == 1 && BUFS == 2), "planes take a buffer each");
  // Consecutive boxes use different buffers (buf(b), b = 0 .. BOXES - 1 over and over): one's stores may
  // still read its buffer while the next is filled. With a single box per tile it is buffer 0 every
  // time, however many there are.
  static constexpr bool ALTERNATE = BUFS == 2 && BOXES == 2;
  uint8_t* bufs;        // BUFS boxes of this warp, 1024-byte aligned
  uint64_t* c_bar;      // [2] this warp's
  uint32_t c_phase;     // bit b: parity of the next wait on c_bar[b]
  int lane;
  int newest = 0;       // stores of the box before (ALTERNATE: from the other buffer)

  __device__ __forceinline__ uint8_t* buf(int b) const { return bufs + (b % BUFS) * kBoxBytes; }

  // C's boxes, ahead of the accumulator (needs a buffer per box). The last tile's results may have
  // passed through these buffers by ordinary stores with no copy behind them (write_direct): every
  // lane orders its own before TMA writes there.
  __device__ __forceinline__ void load_c(const Out& g, int row_base, int col0) {
    if (g.beta == 0.f) return;
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      boxes_read();
#pragma unroll
      for (int b = 0; b < (SPLIT ? 2 : BOXES); ++b) {
        mbar_expect_tx(&c_bar[b], kBoxBytes);
        tma_load_3d(buf(b), g.c_map, col0 + (SPLIT ? 0 : b * 64), g.y + row_base,
                    g.z_c + (SPLIT ? b : 0), &c_bar[b]);
      }
    }
  }
  // Waits for what load_c asked for.
  __device__ __forceinline__ bool wait_c(const Out& g, int b, int* status) {
    if (g.beta == 0.f) return true;
    const bool ok = mbar_wait(&c_bar[b], c_phase >> b & 1u, status);
    c_phase ^= 1u << b;
    return __all_sync(0xffffffffu, ok);
  }

  // Whether this warp's rows go out by boxes.
  __device__ __forceinline__ bool by_box(const Out& g, int row_base) const {
    return g.boxes && (g.boxes == 2 || row_base + 32 <= g.rows);
  }

  // One box's values, rounded, into its buffer: get(h, v) gives accumulators of columns 32 h ..
  // 32 h + 31 of this lane's row. with_c: the buffer holds C.
  template <bool HAS_C, typename Get>
  __device__ __forceinline__ void fill(const Out& g, int b, int row_base, int gc0, bool with_c,
                                       const Get& get, uint32_t (&packed)[32]) {
    uint8_t* hi = buf(b);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[32];
      get(h, v);
      const float2 alpha = make_float2(g.alpha, g.alpha), beta = make_float2(g.beta, g.beta);
      if (with_c) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 w = *box_chunk(hi, lane, h * 4 + c);
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&ws[e]));
            float* p = v + c * 8 + 2 * e;
            const float2 t = chol::ffma2(beta, x, make_float2(0.f, 0.f));
            const float2 r = chol::ffma2(alpha, make_float2(p[0], p[1]), t);
            p[0] = r.x;
            p[1] = r.y;
          }
        }
      } else if (g.alpha != 1.f) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 r = chol::ffma2(alpha, make_float2(v[j], v[j + 1]), make_float2(0.f, 0.f));
          v[j] = r.x;
          v[j + 1] = r.y;
        }
      }
      if (HAS_C && g.diag != 0.f && gc0 + 32 * h == row_base) {  // the same for the whole warp
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += j == lane ? g.diag : 0.f;
      }
      if (!HAS_C && g.type == LINALG_BF16) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          packed[h * 16 + j] = pack<__nv_bfloat16>(v[2 * j], v[2 * j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) packed[h * 16 + j] = pack<__half>(v[2 * j], v[2 * j + 1]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int o = h * 16 + c * 4;
        *box_chunk(hi, lane, h * 4 + c) =
            make_uint4(packed[o], packed[o + 1], packed[o + 2], packed[o + 3]);
      }
    }
  }

  // The transposed box, 64 rows of 64 bytes, in place of one that has been read: neighbouring lanes
  // exchange halves, so that an even lane writes row 2j and an odd one row 2j + 1, two columns
  // each.
  __device__ __forceinline__ void transpose(uint8_t* box, const uint32_t* packed) {
    uint32_t* t = reinterpret_cast<uint32_t*>(box);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, packed[j], 1);
      t[(2 * j + (lane & 1)) * 16 + (lane >> 1)] = (lane & 1)
                                                       ? __byte_perm(other, packed[j], 0x7632)
                                                       : __byte_perm(packed[j], other, 0x5410);
    }
  }

  // One box (64 columns from gc0) to memory by TMA.
  template <bool HAS_C, typename Get>
  __device__ __forceinline__ bool box(const Out& g, int b, int row_base, int gc0, bool mirror,
                                      int* status, const Get& get) {
    bool ok = true;
    if (HAS_C) {
      ok = wait_c(g, b, status);
      if (!ok) return false;
    }
    if (gc0 >= g.n || row_base >= g.rows) {
      newest = 0;
      return true;
    }
    const bool with_c = HAS_C && g.beta != 0.f;
    if (!with_c) {
      if (lane == 0) boxes_read_but(ALTERNATE ? newest : 0);
      __syncwarp();
    }
    newest = mirror ? 2 : 1;
    uint8_t* hi = buf(b);
    uint32_t packed[32];
    fill<HAS_C>(g, b, row_base, gc0, with_c, get, packed);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      store_box(g.map, hi, gc0, g.y + row_base, g.z);
    }
    if (HAS_C && mirror) {
      if (lane == 0) boxes_read();
      __syncwarp();
      transpose(hi, packed);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        store_box(g.mirror, hi, row_base, gc0, g.z);
      }
    }
    return true;
  }

  // SPLIT: sum = alpha * sum + beta * C, of the boxes that load_c has asked for (alpha may be zero).
  __device__ __forceinline__ bool add_c(const Out& g, float (&sum)[2][32], int* status) {
    if (g.beta == 0.f) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[h][j] *= g.alpha;
      return true;
    }
    bool ok = wait_c(g, 0, status);
    ok = wait_c(g, 1, status) && ok;
    if (!ok) return false;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 a = *box_chunk(buf(0), lane, h * 4 + c), b = *box_chunk(buf(1), lane, h * 4 + c);
        const uint32_t as[4] = {a.x, a.y, a.z, a.w}, bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&as[e]));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&bs[e]));
          float* p = sum[h] + c * 8 + 2 * e;
          p[0] = fmaf(g.beta, x.x + y.x, g.alpha * p[0]);
          p[1] = fmaf(g.beta, x.y + y.y, g.alpha * p[1]);
        }
      }
    return true;
  }

  // SPLIT: add_c's result as two planes, 64 columns from gc0. Nothing but the sums stays in registers
  // (with packed copies they went to local memory, 2200 cycles for each drain); only the instances
  // that write the caller's matrix spill, 72 bytes, and 32 in the optimiser step.
  __device__ __forceinline__ void planes(const Out& g, int row_base, int gc0, bool mirror,
                                         const float (&sum)[2][32]) {
    if (gc0 >= g.n || row_base >= g.rows) return;
    uint8_t *hi = buf(0), *lo = buf(1);
    if (lane == 0) boxes_read();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t h[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = sum[c >> 2][(c & 3) * 8 + 2 * e];
        const float y = sum[c >> 2][(c & 3) * 8 + 2 * e + 1];
        h[e] = pack<__half>(x, y);
        float a, b;
        unpack<__half>(h[e], a, b);
        l[e] = pack<__half>(x - a, y - b);
      }
      *box_chunk(hi, lane, c) = make_uint4(h[0], h[1], h[2], h[3]);
      *box_chunk(lo, lane, c) = make_uint4(l[0], l[1], l[2], l[3]);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      store_box(g.map, hi, gc0, g.y + row_base, g.z);
      store_box(g.map, lo, gc0, g.y + row_base, g.z + 1);
    }
    if (!mirror) return;
    if (lane == 0) boxes_read();
    __syncwarp();
#pragma unroll 1
    for (int p = 0; p < 2; ++p) {
      uint8_t* box = p ? lo : hi;
      uint32_t packed[32];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 w = *box_chunk(box, lane, c);
        packed[4 * c] = w.x, packed[4 * c + 1] = w.y;
        packed[4 * c + 2] = w.z, packed[4 * c + 3] = w.w;
      }
      __syncwarp();
      transpose(box, packed);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) store_box(g.mirror, box, row_base, gc0, g.z + p);
    }
  }

  // 32 columns from gc0 straight to the caller's matrix (SPLIT: as add_c left them).
  __device__ __forceinline__ void direct(const Out& g, int row_base, int gc0, float (&v)[32]) {
    if (gc0 >= g.n || row_base >= g.rows) return;
    if (lane == 0) boxes_read();
    __syncwarp();
    float* stage = reinterpret_cast<float*>(bufs);
    if constexpr (!SPLIT) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= g.alpha;
    }
    if (g.type == LINALG_BF16)
      write_direct<__nv_bfloat16>(g, v, lane, row_base, gc0, stage);
    else if (g.type == LINALG_FP16)
      write_direct<__half>(g, v, lane, row_base, gc0, stage);
    else
      write_direct<float>(g, v, lane, row_base, gc0, stage);
  }
};

}  // namespace tile
}  // namespace lin
