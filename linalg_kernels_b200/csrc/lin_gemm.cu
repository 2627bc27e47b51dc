// lin_gemm.cu — half-precision products on CTA pairs (tcgen05, cta_group::2), the engine of the
// Newton-Schulz iteration and of the grouped products.
//
//   D = alpha * A B + beta * C,   A: M x K, B: K x N, both bf16 or both fp16, sums in FP32
//
// Each operand is read in the order it is stored in: "K-major" (the summed index contiguous) or
// "MN-major" (the output's index contiguous), so X X^T, X^T X, S X, X S, x W, dy W^T and
// x^T dy all run without a transposed copy.
//
// A pair of CTAs computes one 256 x BN tile (BN = 512, 256 or 128): each CTA holds 128 rows of A,
// BN/2 rows of B and 128 x BN of the accumulator. The pair shares B, so a CTA writes and reads 32 KB of
// shared memory per 64 of K at BN = 256 instead of 48 KB; at 512 cycles of tensor work
// that is 128 bytes a cycle, what shared memory can give (one CTA alone would need 192).
//
// BN = 512 (large products without C): both accumulators hold halves of one tile, D0 and D1, and a
// CTA loads 48 KB per 64 of K for 1024 cycles of tensor work instead of 32 KB for 512.
//
//   warp 0       TMA producer: 128-byte-swizzled boxes of A and B into a ring of stages. Both CTAs'
//                copies report to the full barrier of the pair's first CTA.
//   warp 1       the first CTA's lane 0 issues tcgen05.mma (M256 x BN x K16); the commits free the
//                stage in both CTAs.
//   warp 2       TMEM allocation; with a ragged K, where a group ends inside a 16-wide slab: once its
//                CTA's part of the last block has landed, zeroes the slab's rows that belong to
//                the next group (they may hold anything, NaN included). (Passing every stage
//                through this warp cost the weight gradient of 16384 rows 398 us, against 250.)
//   warps 4..11  epilogue, overlapped with the next tile (two accumulators; at BN = 512 with the
//                last blocks' MMAs into D1 and the next tile's first into D0): TMEM -> registers ->
//                boxes in shared memory -> TMA stores (lin_tile.cuh).
//
// The grid is persistent: one pair per two SMs, tiles round-robin. Groups' sizes are read from
// device memory by every CTA, so the host needs no synchronisation.
//
// `split`: FP32 accuracy. An operand is a pair of fp16 planes, x = hi + lo (22 bits), and the
// product is lo hi + hi lo + hi hi (lo lo, < 2^-22, is dropped), all three from one stage that holds
// both planes of both operands. The accumulator rounds toward zero at every MMA, an error that
// grows with the number of steps, so it is drained into registers (rounded to nearest) after each K
// block, the small terms summed first: 4 full-size steps per drain. (Error of the iteration
// against 64 bits, 3 x 1001 x 601: 4.5e-6 with a drain per 256 of K, 2.3e-6 per 128, 1.4e-6 per 64,
// where FP32 products have 3.0e-6.)
//
// Every wait is bounded (2 s of %globaltimer, and 2 us more for each K block that it spans); one that
// runs out records CHOL_ERR_WAIT_TIMEOUT in the library's status word and ends the launch.
#include <mutex>

#include "lin_tile.cuh"

namespace lin {

namespace {

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

bool resolve_encode() {
  std::call_once(g_encode_once, []() {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  return g_encode != nullptr;
}

}  // namespace

namespace {
bool encode(CUtensorMap* map, const Operand& o, bool bf16, uint32_t box_cols, uint32_t box_rows,
            CUtensorMapSwizzle swizzle) {
  if (!resolve_encode()) return false;
  if ((reinterpret_cast<uintptr_t>(o.base) & 15) || o.ld % 8 || (o.count > 1 && o.stride % 8))
    return false;
  cuuint64_t dims[3] = {cuuint64_t(o.cols), cuuint64_t(o.rows), cuuint64_t(o.count)};
  cuuint64_t strides[2] = {cuuint64_t(o.ld) * 2,
                           cuuint64_t(o.count > 1 ? o.stride : o.ld * o.rows) * 2};
  cuuint32_t box[3] = {box_cols, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return g_encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(o.base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
}  // namespace

bool make_operand_map(CUtensorMap* map, const Operand& o, bool bf16, int box_rows) {
  return encode(map, o, bf16, tile::kBlockK, o.mn_major ? tile::kBlockK : box_rows,
                CU_TENSOR_MAP_SWIZZLE_128B);
}
bool make_output_map(CUtensorMap* map, const Operand& o, bool bf16, bool mirrored) {
  return mirrored ? encode(map, o, bf16, 32, 64, CU_TENSOR_MAP_SWIZZLE_NONE)
                  : encode(map, o, bf16, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
}

namespace {

using namespace tile;

constexpr int kBand = 8;  // row tiles per band of the tile order

struct Args {
  int m, n, k, batch;
  int tiles_m, tiles_n, per_matrix;
  int symmetric;
  float alpha, beta, diag;
  int boxes;  // the output through boxes: 1 inside the rows of a group only, 2 everywhere
  void* out;
  int64_t ldo, out_stride;
  int out_type;
  int out_vec;  // rows of the output start on 32-byte sectors
  float decay, rate;
  const void* offsets;
  int offsets64;
  int total_rows;
  int fill;
  uint32_t idesc;
};

struct Tile {
  int index;      // matrix or group
  int tm, tn;
  int row0;       // first row of A (and of the output) of the group; 0 for kBatch
  int rows;       // rows of the output in this matrix or group
  int k0, k_len;  // the summed range
};

// The tiles of a launch, in the order every role walks them.
template <int MODE>
struct Walker {
  const Args& g;
  const int* start;  // kRagged*: first row of each group (and one past the last)
  const int* first;  // kRaggedM: first tile of each group
  int groups;        // kRaggedM: with the rows of no group
  int cursor;
  __device__ __forceinline__ Walker(const Args& args, const int* s, const int* f, int n)
      : g(args), start(s), first(f), groups(n), cursor(0) {}
  __device__ __forceinline__ int total() const {
    return MODE == kRaggedM ? first[groups] : g.per_matrix * g.batch;
  }
  __device__ __forceinline__ void at(int t, Tile& w) {
    if (MODE == kRaggedM) {
      while (t >= first[cursor + 1]) ++cursor;
      const int e = cursor;
      w.row0 = e <= g.batch ? start[e] : 0;  // group batch: the rows behind the last group;
      const int end = e <= g.batch ? (e < g.batch ? start[e + 1] : g.total_rows) : start[0];
      w.rows = end - w.row0;                 // group batch + 1: those before the first
      w.index = e;
      w.k0 = 0;
      w.k_len = e < g.batch ? g.k : 0;
      band(t - first[e], (w.rows + kTileM - 1) / kTileM, w);
      return;
    }
    w.index = t / g.per_matrix;
    const int r = t - w.index * g.per_matrix;
    w.row0 = 0;
    w.rows = g.m;
    w.k0 = 0;
    w.k_len = g.k;
    if (MODE == kRaggedK) {
      w.k0 = start[w.index];
      w.k_len = start[w.index + 1] - w.k0;
    }
    if (g.symmetric) {
      // in the same bands: the columns left of the band's triangle, then the triangle by rows (a step
      // of 8192 x 8192: 2057 -> 1963 us, by rows alone each 74 tiles read all of X)
      const int top = row_of(r) / kBand * kBand, left = g.symmetric * top;
      int t = r - row_first(top);
      const int h = g.tiles_m - top < kBand ? g.tiles_m - top : kBand;
      if (t < h * left) {
        w.tn = t / h;
        w.tm = top + t - w.tn * h;
      } else {
        t -= h * left;
        w.tm = row_of(t);
        w.tn = left + t - row_first(w.tm);
        w.tm += top;
      }
    } else {
      band(r, g.tiles_m, w);
    }
  }
  // Of a symmetric result, row tile tm holds its tiles up to the diagonal: ratio (tm + 1) of them
  // (the last row fewer, if its last ones lie outside); g.symmetric = ratio = 256 / BN.
  __device__ __forceinline__ int row_first(int tm) const {  // tiles in the rows above
    return g.symmetric * (tm * (tm + 1) / 2);
  }
  __device__ __forceinline__ int row_of(int r) const {
    int tm = int((sqrtf(8.f * float(r / g.symmetric) + 1.f) - 1.f) * 0.5f);
    while (row_first(tm) > r) --tm;
    while (row_first(tm + 1) <= r) ++tm;
    return tm;
  }
  // Bands of 8 row tiles, down each column of a band: the tiles in flight at a time then read
  // about as many rows of A as of B (8192^3 by offsets: 882 -> 842 us, 840 -> 777 with B MN-major).
  __device__ __forceinline__ void band(int r, int tiles_m, Tile& w) const {
    const int b = r / (kBand * g.tiles_n);
    r -= b * kBand * g.tiles_n;
    const int h = tiles_m - b * kBand < kBand ? tiles_m - b * kBand : kBand;
    w.tn = r / h;
    w.tm = b * kBand + r - w.tn * h;
  }
};

// Epilogue buffers per warp: two hold C's boxes (and the two planes) of a batch's products; ragged
// products have no C and need the group tables' space.
template <int BN, int MODE>
constexpr int kBuffers = BN == 512 ? 1 : (MODE == kBatch || BN == 128 ? 2 : 1);
constexpr int kWideGroups = 124;  // groups whose tables fit beside BN = 512's stages
template <int BN>
constexpr int kTableEntries = (BN == 512 ? kWideGroups : kMaxGroups) + 4;
template <int BN, int MODE, bool SPLIT>
using ProductCfg = Cfg<BN, kBuffers<BN, MODE>, MODE == kBatch ? 0 : 2 * kTableEntries<BN> * 4,
                       SPLIT ? 2 : 1>;

template <int BN, bool AMN, bool BMN, int MODE, int EPI, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a,
                   const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_out,
                   const __grid_constant__ CUtensorMap map_mirror,
                   const __grid_constant__ CUtensorMap map_c, const Args g, int* status) {
  using C = ProductCfg<BN, MODE, SPLIT>;
  constexpr int S = C::STAGES;
  constexpr int kBufs = kBuffers<BN, MODE>;
  constexpr bool WIDE = BN == 512;
  constexpr int HALVES = WIDE ? 2 : 1;  // accumulators of one tile
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* epi = smem + size_t(S) * C::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + size_t(S) * C::STAGE + C::EPI);
  uint64_t* full = bars;             // [S] first CTA: a stage of both CTAs has landed
  uint64_t* landed = bars + S;       // [S] kRaggedK: this CTA's part of a group's last block landed
  uint64_t* empty = bars + 2 * S;    // [S] the MMAs have read the stage
  uint64_t* tfull = bars + 3 * S;    // [2] accumulator ready
  uint64_t* tempty = tfull + 2;      // [2] first CTA: accumulator drained by both CTAs
  uint64_t* clean = tempty + 2;      // [S] kRaggedK, first CTA: the other CTA's part is clean
  uint64_t* c_bars = clean + S;      // [2 * kEpiWarps] C's boxes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(c_bars + 2 * kEpiWarps);
  int* start = reinterpret_cast<int*>(smem + size_t(S) * C::STAGE + C::EPI + 512);
  int* first = start + kTableEntries<BN>;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&landed[s], 1);
      mbar_init(&clean[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * kEpiWarps);
    }
    for (int b = 0; b < 2 * kEpiWarps; ++b) mbar_init(&c_bars[b], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(uint32_t(C::TMEM_COLS))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  griddep_wait();  // before any read of what earlier kernels wrote
  if (MODE != kBatch && warp == 0) {
    group_starts(start, g.offsets, g.offsets64, g.batch, g.total_rows);
    if (MODE == kRaggedM)
      group_tiles(first, start, g.batch, g.fill, g.total_rows, kTileM, g.tiles_n);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  griddep_launch();
  const uint32_t tmem = *tmem_slot;
  const int pair = int(blockIdx.x >> 1), pairs = int(gridDim.x >> 1);
  Walker<MODE> walk(g, start, first, MODE == kRaggedM ? g.batch + (g.fill ? 2 : 0) : 0);
  const int total = walk.total();
  Tile w;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      uint32_t kt = 0;
      uint32_t tails = 0;  // stages whose last copy reports to landed
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs) {
        walk.at(t, w);
        const int num_k = (w.k_len + kBlockK - 1) / kBlockK;
        const int a_row = w.row0 + w.tm * kTileM + int(rank) * 128;
        const int b_row = w.tn * BN + int(rank) * (WIDE ? 128 : BN / 2);
        constexpr int planes = SPLIT ? 2 : 1;
        const int za = MODE == kBatch ? w.index * planes : 0;
        const int zb = MODE == kRaggedK ? 0 : w.index * planes;
        for (int kb = 0; kb < num_k; ++kb, ++kt) {
          const int s = int(kt % S);
          if (kt >= uint32_t(S) && !wait_bar(&empty[s], ((kt / S) & 1u) ^ 1u, status)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + size_t(s) * C::STAGE;
          uint8_t* sb = sa + C::A_BYTES;
          uint32_t bar;
          if (MODE == kRaggedK && kb == num_k - 1 && (w.k_len & 15)) {
            mbar_expect_tx(&landed[s], C::STAGE);  // warp 2 reports the stage
            bar = smem_u32(&landed[s]);
            tails |= 1u << s;
          } else {
            if (rank == 0) mbar_expect_tx(&full[s], 2 * C::STAGE);
            bar = leader_addr(&full[s]);
            tails &= ~(1u << s);
          }
          const int kx = w.k0 + kb * kBlockK;
#pragma unroll
          for (int p = 0; p < planes; ++p) {
            uint8_t* pa = sa + p * C::A_PLANE;
            uint8_t* pb = sb + p * C::B_PLANE;
            if (AMN) {
              tma_load_pair(pa, &map_a, a_row, kx, za + p, bar);
              tma_load_pair(pa + 8192, &map_a, a_row + 64, kx, za + p, bar);
            } else {
              tma_load_pair(pa, &map_a, kx, a_row, za + p, bar);
            }
#pragma unroll
            for (int d = 0; d < HALVES; ++d) {
              const int row = b_row + d * 256;
              if (BMN) {
                tma_load_pair(pb + d * 16384, &map_b, row, kx, zb + p, bar);
                if (BN >= 256) tma_load_pair(pb + d * 16384 + 8192, &map_b, row + 64, kx, zb + p, bar);
              } else {
                tma_load_pair(pb + d * 16384, &map_b, kx, row, zb + p, bar);
              }
            }
          }
        }
      }
      if (!ok && rank == 0) {
        // copies still in flight write this pair's shared memory: give them time to land (those of
        // a last block are waited for by warp 2)
        for (uint32_t j = kt < uint32_t(S) ? 0 : kt - S; j < kt; ++j)
          if (!(tails >> (j % S) & 1u)) wait_bar(&full[j % S], (j / S) & 1u, status);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (first CTA) ----------------
    if (rank == 0 && lane == 0) {
      uint32_t kt = 0, round = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs) {
        walk.at(t, w);
        const int num_k = (w.k_len + kBlockK - 1) / kBlockK;
        if (num_k == 0) continue;
        if constexpr (WIDE) {
          // The first blocks are summed into D0 while the epilogue
          // still drains the last tile's D1, and the last blocks into D0 before D1, so that the
          // epilogue starts on D0 under D1's MMAs: as many blocks as there are stages.
          auto ready = [&](int kb) {
            ok = ok && wait_bar(&full[(kt + kb) % S], ((kt + kb) / S) & 1u, status);
            tc_fence_after();
            return ok;
          };
          auto block = [&](int kb, int d) {
            const uint8_t* sa = smem + size_t((kt + kb) % S) * C::STAGE;
            const uint8_t* sb = sa + C::A_BYTES + d * 16384;
            const uint64_t da = AMN ? sw128_desc_mn(sa) : sw128_desc(sa);
            const uint64_t db = BMN ? sw128_desc_mn(sb) : sw128_desc(sb);
            const int left = w.k_len - kb * kBlockK;
            const int slabs = left >= kBlockK ? kBlockK / 16 : (left + 15) / 16;
#pragma unroll
            for (int kk = 0; kk < kBlockK / 16; ++kk) {
              if (kk >= slabs) break;
              mma_pair(tmem + d * 256u, da + uint64_t(kk * (AMN ? 2048 : 32) / 16),
                       db + uint64_t(kk * (BMN ? 2048 : 32) / 16), g.idesc, (kb | kk) ? 1u : 0u);
            }
          };
          auto drained = [&](int d) {
            if (round > 0) ok = ok && wait_bar(&tempty[d], (round - 1) & 1u, status);
            tc_fence_after();
          };
          const int lead = num_k < S ? num_k : S;
          const int tail = num_k - S > lead ? num_k - S : lead;
          drained(0);
          for (int kb = 0; kb < lead && ok; ++kb)
            if (ready(kb)) block(kb, 0);
          if (ok && tail == num_k) commit_pair(&tfull[0]);
          drained(1);
          for (int kb = 0; kb < lead && ok; ++kb) {
            block(kb, 1);
            commit_pair(&empty[(kt + kb) % S]);
          }
          for (int kb = lead; kb < tail && ok; ++kb)
            if (ready(kb)) {
              block(kb, 0);
              block(kb, 1);
              commit_pair(&empty[(kt + kb) % S]);
            }
          for (int kb = tail; kb < num_k && ok; ++kb)
            if (ready(kb)) block(kb, 0);
          if (ok && tail < num_k) commit_pair(&tfull[0]);
          for (int kb = tail; kb < num_k && ok; ++kb) {
            block(kb, 1);
            commit_pair(&empty[(kt + kb) % S]);
          }
          if (ok) commit_pair(&tfull[1]);
          kt += uint32_t(num_k);
          ++round;
          continue;
        }
        const int rounds = SPLIT ? num_k : 1;  // split: an accumulator per K block
        for (int r = 0; r < rounds && ok; ++r, ++round) {
          const uint32_t buf = round & 1u;
          if (round >= 2 && !wait_bar(&tempty[buf], ((round >> 1) & 1u) ^ 1u, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem + buf * uint32_t(BN);
          for (int kb = SPLIT ? r : 0; kb < (SPLIT ? r + 1 : num_k); ++kb, ++kt) {
            const int s = int(kt % S);
            if (!wait_bar(&full[s], (kt / S) & 1u, status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint8_t* sa = smem + size_t(s) * C::STAGE;
            const uint8_t* sb = sa + C::A_BYTES;
            const int left = w.k_len - kb * kBlockK;  // the last block: only its 16-wide slabs
            const int slabs = left >= kBlockK ? kBlockK / 16 : (left + 15) / 16;
#pragma unroll
            for (int c = SPLIT ? 0 : 2; c < 3; ++c) {  // lo hi, hi lo, hi hi
              const uint8_t* pa = sa + (c == 0 ? C::A_PLANE : 0);
              const uint8_t* pb = sb + (c == 1 ? C::B_PLANE : 0);
              const uint64_t da = AMN ? sw128_desc_mn(pa) : sw128_desc(pa);
              const uint64_t db = BMN ? sw128_desc_mn(pb) : sw128_desc(pb);
#pragma unroll
              for (int kk = 0; kk < kBlockK / 16; ++kk) {
                if (kk >= slabs) break;
                mma_pair(acc, da + uint64_t(kk * (AMN ? 2048 : 32) / 16),
                         db + uint64_t(kk * (BMN ? 2048 : 32) / 16), g.idesc,
                         SPLIT ? (c | kk ? 1u : 0u) : (kb | kk ? 1u : 0u));
              }
            }
            commit_pair(&empty[s]);
          }
          if (ok) commit_pair(&tfull[buf]);
        }
      }
    }
  } else if (warp == 2) {
    // ---------------- kRaggedK: the last block of a group that ends inside a 16-wide slab --------
    if (MODE == kRaggedK) {
      uint32_t kt = 0, landed_phase = 0, clean_phase = 0;  // bit s: parity of the next wait
      int64_t span = 0;  // K blocks loaded since the last wait
      bool ok = true;
      for (int t = pair; t < total && ok; t += pairs) {
        walk.at(t, w);
        const int num_k = (w.k_len + kBlockK - 1) / kBlockK;
        kt += uint32_t(num_k);
        span += num_k;
        if ((w.k_len & 15) == 0) continue;
        const int s = int((kt - 1) % S);
        ok = wait_bar(&landed[s], landed_phase >> s & 1u, status, limit_of(span));
        span = 0;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        landed_phase ^= 1u << s;
        // the K rows from the group's end to the end of their slab are read by the MMA: zero them
        const int left = w.k_len - (num_k - 1) * kBlockK;
        const int count = ((left + 15) & ~15) - left;
        uint8_t* sa = smem + size_t(s) * C::STAGE;
        constexpr int boxes = C::STAGE / 8192;  // A's two, then B's
        for (int j = lane; j < boxes * count * 8; j += 32) {
          const int box = j / (count * 8), r = j - box * count * 8;
          *reinterpret_cast<uint4*>(sa + box * 8192 + (left + (r >> 3)) * 128 + (r & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (rank != 0) {
          if (lane == 0) arrive_leader(leader_addr(&clean[s]));
        } else {
          ok = wait_bar(&clean[s], clean_phase >> s & 1u, status);
          ok = __all_sync(0xffffffffu, ok);
          clean_phase ^= 1u << s;
          if (lane == 0 && ok) arrive_leader(leader_addr(&full[s]));
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------- epilogue ----------------
    const int q = warp & 3, half = (warp - 4) >> 2;  // TMEM lane quarter; half of the columns
    constexpr int kCols = WIDE ? 128 : BN / 2;  // of one accumulator
    using Epi = WarpEpilogue<kCols, kBufs, SPLIT>;
    Epi ep{epi + (warp - 4) * kBufs * kBoxBytes, c_bars + 2 * (warp - 4), 0u, lane};
    uint32_t round = 0;
    constexpr int P = SPLIT ? 2 : 1;
    Out o;
    o.alpha = g.alpha, o.beta = EPI == kPlanes || SPLIT ? g.beta : 0.f;
    o.diag = EPI == kPlanes ? g.diag : 0.f;
    o.n = g.n;
    o.map = &map_out, o.mirror = &map_mirror, o.c_map = &map_c;
    o.boxes = EPI == kMuon ? 0 : g.boxes;
    o.ldo = g.ldo, o.type = EPI == kPlanes ? LINALG_FP16 : g.out_type, o.vec = g.out_vec;
    o.weights = EPI == kMuon, o.decay = g.decay, o.rate = g.rate;
    for (int t = pair; t < total; t += pairs) {
      walk.at(t, w);
      const int num_k = (w.k_len + kBlockK - 1) / kBlockK;
      const int row_base = w.tm * kTileM + int(rank) * 128 + q * 32;  // within the matrix or group
      const int col0 = w.tn * BN + half * kCols;
      const bool mirror = EPI == kPlanes && g.symmetric && w.tm * kTileM > w.tn * BN + BN - 1;
      o.rows = w.rows;
      o.z = MODE == kRaggedM ? 0 : w.index * (EPI == kPlanes ? P : 1);
      o.z_c = w.index * P;
      o.y = w.row0;
      const int size = EPI != kPlanes && g.out_type == LINALG_FP32 ? 4 : 2;
      o.out = static_cast<char*>(g.out) + (int64_t(MODE == kRaggedM ? 0 : w.index) * g.out_stride +
                                           int64_t(w.row0) * g.ldo) * size;
      constexpr bool kC = EPI == kPlanes;  // C, the diagonal, mirrored tiles
      const bool by_box = ep.by_box(o, row_base);
      if (num_k == 0) {  // nothing to sum: zeros (rows of no group, a group without rows)
        auto zeros = [](int, float (&v)[32]) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        };
#pragma unroll 1
        for (int i = 0; i < HALVES * kCols; i += 64) {
          const int c = i < kCols ? i : i - kCols + 256;
          if (by_box) {
            ep.template box<false>(o, c / 64, row_base, col0 + c, false, status, zeros);
          } else {
#pragma unroll 1
            for (int h = 0; h < 64; h += 32) {
              float v[32];
              zeros(0, v);
              ep.direct(o, row_base, col0 + c + h, v);
            }
          }
        }
        continue;
      }
      bool ok = true;
      if constexpr (WIDE) {
#pragma unroll 1
        for (int d = 0; d < 2 && ok; ++d) {
          ok = wait_bar(&tfull[d], round & 1u, status, limit_of(num_k));
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t acc = tmem + uint32_t(d * 256 + half * kCols) + (uint32_t(q * 32) << 16);
          const int gc0 = col0 + d * 256;
          if (by_box) {
#pragma unroll 1
            for (int b = 0; b < Epi::BOXES; ++b)
              ep.template box<false>(o, b, row_base, gc0 + b * 64, false, status,
                                     [&](int h, float (&v)[32]) {
                                       tmem_ld32(acc + uint32_t(b * 64 + h * 32), v);
                                     });
          } else if constexpr (!kC) {
#pragma unroll 1
            for (int c = 0; c < kCols; c += 32) {
              float v[32];
              tmem_ld32(acc + uint32_t(c), v);
              ep.direct(o, row_base, gc0 + c, v);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_leader_relaxed(leader_addr(&tempty[d]));
        }
        if (!ok) break;
        ++round;
        continue;
      }
      if (kC || SPLIT) ep.load_c(o, row_base, col0);
      if constexpr (SPLIT) {
        float sum[2][32];
        for (int ch = 0; ch < num_k; ++ch, ++round) {
          const uint32_t buf = round & 1u;
          ok = wait_bar(&tfull[buf], (round >> 1) & 1u, status);
          if (!ok) break;
          tc_fence_after();
          const uint32_t acc = tmem + buf * uint32_t(BN) + uint32_t(half * kCols) +
                               (uint32_t(q * 32) << 16);
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            float v[32];
            tmem_ld32(acc + uint32_t(cc * 32), v);
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[cc][j] = ch ? sum[cc][j] + v[j] : v[j];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_leader_relaxed(leader_addr(&tempty[buf]));
        }
        if (!__all_sync(0xffffffffu, ok)) break;
        ok = ep.add_c(o, sum, status);
        if constexpr (kC) {
          ep.planes(o, row_base, col0, mirror, sum);
        } else {
          ep.direct(o, row_base, col0, sum[0]);
          ep.direct(o, row_base, col0 + 32, sum[1]);
        }
        if (!ok) break;
      } else {
        const uint32_t buf = round & 1u;
        ok = wait_bar(&tfull[buf], (round >> 1) & 1u, status, limit_of(num_k));
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * uint32_t(BN) + uint32_t(half * kCols) +
                             (uint32_t(q * 32) << 16);
        if (by_box) {
#pragma unroll 1
          for (int b = 0; b < Epi::BOXES; ++b)
            ok = ep.template box<kC>(o, b, row_base, col0 + b * 64, mirror, status,
                                     [&](int h, float (&v)[32]) {
                                       tmem_ld32(acc + uint32_t(b * 64 + h * 32), v);
                                     }) && ok;
          if (!ok) break;
        } else if constexpr (!kC) {
#pragma unroll 1
          for (int c = 0; c < kCols; c += 32) {
            float v[32];
            tmem_ld32(acc + uint32_t(c), v);
            ep.direct(o, row_base, col0 + c, v);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader_relaxed(leader_addr(&tempty[buf]));
        ++round;
      }
    }
    if (lane == 0) boxes_written();  // they read this CTA's shared memory
  }
  // The other CTA's barriers and shared memory are used until both are done.
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(uint32_t(C::TMEM_COLS))
                 : "memory");
  }
}

// ------------------------------- host side --------------------------------------------
template <int BN, bool AMN, bool BMN, int MODE, int EPI, bool SPLIT>
cudaError_t set_smem() {
  return cudaFuncSetAttribute(product_kernel<BN, AMN, BMN, MODE, EPI, SPLIT>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              int(ProductCfg<BN, MODE, SPLIT>::SMEM));
}

template <int BN, bool AMN, bool BMN, int MODE, int EPI, bool SPLIT>
int launch(const Product& p, cudaStream_t q) {
  CUtensorMap ma, mb;
  if (!make_operand_map(&ma, p.a, p.bf16, 128) ||
      !make_operand_map(&mb, p.b, p.bf16, BN == 128 ? 64 : 128))
    return CHOL_ERR_UNSUPPORTED;
  Args g{};
  g.m = int(p.m), g.n = int(p.n), g.k = int(p.k), g.batch = int(p.batch);
  g.tiles_m = int((p.m + kTileM - 1) / kTileM);
  g.tiles_n = int((p.n + BN - 1) / BN);
  int64_t per = int64_t(g.tiles_m) * g.tiles_n;
  if (p.symmetric) {
    const int ratio = kTileM / BN;
    g.symmetric = ratio;
    per = 0;
    for (int tm = 0; tm < g.tiles_m; ++tm)
      per += ratio * (tm + 1) < g.tiles_n ? ratio * (tm + 1) : g.tiles_n;
  }
  int64_t total = per * p.batch;
  if (MODE == kRaggedM)  // an upper bound: every group may end in a partial tile
    total = ((p.total_rows + kTileM - 1) / kTileM + p.batch + 2) * g.tiles_n;
  // (tile numbers step by the grid's pairs past the last one)
  if (per > 0x7fffffffLL || total > 0x7fffffffLL - 1024) return CHOL_ERR_UNSUPPORTED;
  if (total == 0) return CHOL_OK;
  g.per_matrix = int(per);
  g.alpha = p.alpha, g.beta = p.beta, g.diag = p.diag;
  g.out = p.out;
  g.ldo = p.ldo, g.out_stride = p.out_stride, g.out_type = p.out_type;
  const int sector = p.out_type == LINALG_FP32 ? 8 : 16;
  g.out_vec = (reinterpret_cast<uintptr_t>(p.out) & 31) == 0 && p.ldo % sector == 0 &&
              p.out_stride % sector == 0;
  // the output's boxes, where its type and alignment allow: by group rows when these are ragged. A store
  // ends on a 16-byte chunk, not on the map's last column, and would put zeros into up to seven
  // elements behind it: the caller's rows have to be whole chunks (the workspace's are padded).
  CUtensorMap mo = ma, mm = ma, mc = ma;
  const int64_t planes = SPLIT ? 2 : 1;
  if (EPI == kPlanes ||
      (!SPLIT && EPI != kMuon && p.out_type != LINALG_FP32 && p.n % 8 == 0)) {
    const Operand out{p.out, MODE == kRaggedM ? p.total_rows : p.m, p.n, p.ldo,
                      MODE == kRaggedM ? 1 : p.batch * planes, p.out_stride, false};
    const bool b16 = EPI != kPlanes && p.out_type == LINALG_BF16;
    if (make_output_map(&mo, out, b16, false)) g.boxes = MODE == kRaggedM ? 1 : 2;
    if (EPI == kPlanes && (!g.boxes || !make_output_map(&mm, out, false, true)))
      return CHOL_ERR_UNSUPPORTED;
  }
  if ((EPI == kPlanes || SPLIT) && p.beta != 0.f &&
      !make_output_map(&mc, Operand{p.c, p.m, p.n, p.ldc, p.batch * planes, p.c_plane, false}, false,
                       false))
    return CHOL_ERR_UNSUPPORTED;
  g.decay = p.decay, g.rate = p.rate;
  g.offsets = p.offsets, g.offsets64 = p.offsets64;
  g.total_rows = int(p.total_rows), g.fill = p.fill;
  const uint32_t type = p.bf16 ? 1u : 0u;
  g.idesc = (1u << 4) | (type << 7) | (type << 10) | (uint32_t(AMN) << 15) |
            (uint32_t(BMN) << 16) | (uint32_t((BN < 256 ? BN : 256) >> 3) << 17) |
            (uint32_t(kTileM >> 4) << 24);
  int64_t pairs = sm_count() / 2;
  if (pairs > total) pairs = total;
  return chol::status_from(chol::launch_pdl(product_kernel<BN, AMN, BMN, MODE, EPI, SPLIT>,
                                            dim3(unsigned(2 * pairs)), dim3(kThreads),
                                            ProductCfg<BN, MODE, SPLIT>::SMEM, q, true, ma, mb, mo, mm,
                                            mc, g, chol::device_status_ptr()));
}

// BN = 256 wherever the tiles still fill the GPU: the wider tile moves a third less shared
// memory per product; narrower ones spread a small problem over more pairs.
bool narrow(const Product& p) {
  if (p.n <= 128) return true;
  const int64_t tm = p.mode == kRaggedM ? (p.total_rows + kTileM - 1) / kTileM + p.batch / 2
                                        : ((p.m + kTileM - 1) / kTileM) * p.batch;
  return tm * ((p.n + 255) / 256) < sm_count() / 2;
}

// BN = 512: a quarter less to load per product (48 KB per 1024 cycles of MMAs instead of 64 KB), for
// an epilogue that is only partly hidden: a tile takes 1.61 times a 256-wide one's time per block
// of K and 3 blocks more. Measured, 256 -> 512: 8192^3 842 -> 685 us, 4096^3 112 -> 96, 16384 rows
// in 16 groups, 2048 x 4096: 241 -> 219; the other way 5200 rows in 2 groups, 1100 x 2500: 68 and
// 86, 32768 in 8, 768 x 2048: 94 and 97. Ragged rows' tile counts are known only nearly, so their
// rounds count in fractions, with 0.65 for the last one. Symmetric results (and with C) stay at
// 256: G and B of 4096 x 4096 gained 3 % of a step, of 8192 x 8192 lost 2 %.
bool wide(const Product& p) {
  if (p.split || p.symmetric || p.beta != 0.f || p.n < 512) return false;
  if (p.mode != kBatch && p.batch > kWideGroups) return false;
  const int64_t pairs = sm_count() / 2, k = p.mode == kRaggedK ? p.total_rows / p.batch : p.k;
  const double blocks = double((k + kBlockK - 1) / kBlockK);
  auto rounds = [&](int64_t bn) {
    const int64_t tn = (p.n + bn - 1) / bn;
    if (p.mode == kRaggedM)
      return double(((p.total_rows + kTileM - 1) / kTileM + p.batch / 2) * tn) / pairs + 0.65;
    return double(((p.m + kTileM - 1) / kTileM * tn * p.batch + pairs - 1) / pairs);
  };
  return rounds(512) * (blocks * 1.61 + 3.0) < rounds(256) * blocks;
}

}  // namespace

#define LIN_FOR_EACH(F)                              \
  F(false, false, kBatch, kPlanes, false)            \
  F(true, true, kBatch, kPlanes, false)              \
  F(false, true, kBatch, kPlanes, false)             \
  F(false, false, kBatch, kFinal, false)             \
  F(false, true, kBatch, kFinal, false)              \
  F(false, false, kBatch, kMuon, false)              \
  F(false, true, kBatch, kMuon, false)               \
  F(false, false, kRaggedM, kStore16, false)         \
  F(false, true, kRaggedM, kStore16, false)          \
  F(true, true, kRaggedK, kStore16, false)
#define LIN_FOR_EACH_SPLIT(F)                        \
  F(false, false, kBatch, kPlanes, true)             \
  F(true, true, kBatch, kPlanes, true)               \
  F(false, true, kBatch, kPlanes, true)              \
  F(false, false, kBatch, kFinal, true)              \
  F(false, true, kBatch, kFinal, true)               \
  F(false, false, kBatch, kMuon, true)               \
  F(false, true, kBatch, kMuon, true)

// The widest tile of an instance. X^T X, the one batched product of two MN-major operands, is symmetric:
// wide() leaves it at 256.
template <bool AMN, bool BMN, int MODE, bool SPLIT>
constexpr int kWidest = SPLIT ? 128 : (AMN && BMN && MODE == kBatch ? 256 : 512);

int launch_product(const Product& p, cudaStream_t q) {
  if (!resolve_encode()) return CHOL_ERR_DEVICE;
  const int64_t lim = 0x7fffffffLL - 512;
  if (p.m > lim || p.n > lim || p.k > lim || p.batch > lim || p.total_rows > lim)
    return CHOL_ERR_UNSUPPORTED;
  const bool small = narrow(p), large = !small && wide(p);
#define LIN_CASE(AMN, BMN, MODE, EPI, SPLIT)                                                \
  if (p.a.mn_major == AMN && p.b.mn_major == BMN && p.mode == MODE && p.epilogue == EPI &&  \
      p.split == SPLIT) {                                                                   \
    if (SPLIT || small) return launch<128, AMN, BMN, MODE, EPI, SPLIT>(p, q);               \
    if (large) return launch<kWidest<AMN, BMN, MODE, SPLIT>, AMN, BMN, MODE, EPI, SPLIT>(p, q); \
    return launch<SPLIT ? 128 : 256, AMN, BMN, MODE, EPI, SPLIT>(p, q);                     \
  }
  LIN_FOR_EACH(LIN_CASE)
  LIN_FOR_EACH_SPLIT(LIN_CASE)
#undef LIN_CASE
  return CHOL_ERR_UNSUPPORTED;
}

cudaError_t prepare_products() {
  cudaError_t e;
#define LIN_SET(AMN, BMN, MODE, EPI, SPLIT)                                                   \
  if ((e = set_smem<128, AMN, BMN, MODE, EPI, SPLIT>()) != cudaSuccess) return e;             \
  if ((e = set_smem<SPLIT ? 128 : 256, AMN, BMN, MODE, EPI, SPLIT>()) != cudaSuccess) return e; \
  if ((e = set_smem<kWidest<AMN, BMN, MODE, SPLIT>, AMN, BMN, MODE, EPI, SPLIT>()) != cudaSuccess) \
    return e;
  LIN_FOR_EACH(LIN_SET)
  LIN_FOR_EACH_SPLIT(LIN_SET)
#undef LIN_SET
  return resolve_encode() ? cudaSuccess : cudaErrorNotSupported;
}

namespace {
thread_local int t_sms = 148;
}
int sm_count() { return t_sms; }
void use_sm_count(int sms) { t_sms = sms; }

}  // namespace lin
