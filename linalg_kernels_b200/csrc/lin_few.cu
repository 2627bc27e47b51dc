// lin_few.cu — grouped products with few rows per group (decoding, small batches): the weights are
// all there is to read.
//
// A 256-row tile (lin_gemm.cu) would load 256 rows of x per block of K, almost all of other groups,
// as many bytes as of weights. Here the weights stand on the MMA's M side and the rows on its N side:
//
//   D = W_e^T x^T:  128 columns of the output x NT rows (16, 32 or 64), sums in FP32
//
// so a stage is 16 KB of weights and 2 to 8 KB of rows, and each CTA keeps ~180 KB of copies in
// flight. Both orders of the weights are read as they lie (K-major or MN-major A operand).
// Bound by HBM: one read of the weights of the groups that have rows, at 5.75 TB/s and 5 to 8 us beside
// it (32, 64, 128 and 256 groups of 1024 x 2048: 31, 52, 98 and 192 us).
//
//   warp 0 TMA producer, warp 1 MMA issuer, warp 2 TMEM, warps 4..7 epilogue: TMEM lane = output
//   column, so a warp stores 32 neighbouring columns of a row at a time.
#include "lin_few.cuh"
#include "lin_tile.cuh"

namespace lin {

namespace {

using namespace tile;

constexpr int kFewThreads = 256;

template <int NT>
struct FewCfg {
  static constexpr int A_BYTES = 128 * kBlockK * 2;
  static constexpr int B_BYTES = NT * kBlockK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = NT == 64 ? 8 : 10;
  static constexpr size_t SMEM = size_t(STAGES) * STAGE + 512 + kTableBytes + 1024;
  static constexpr int TMEM_COLS = 2 * NT < 32 ? 32 : 2 * NT;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct FewArgs {
  int n, k, groups, total_rows, fill;
  int tiles_n;
  void* out;
  int64_t ldo;
  const void* offsets;
  int offsets64;
  uint32_t idesc;
};

__device__ __forceinline__ void mma_one(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int NT, bool AMN, typename T>
__global__ void __launch_bounds__(kFewThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
               const FewArgs g, int* status) {
  using C = FewCfg<NT>;
  constexpr int S = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + size_t(S) * C::STAGE);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;   // [2]
  uint64_t* tempty = tfull + 2;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  int* start = reinterpret_cast<int*>(smem + size_t(S) * C::STAGE + 512);
  int* first = start + kMaxGroups + 4;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&map_w);
    prefetch_map(&map_x);
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(uint32_t(C::TMEM_COLS))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  griddep_wait();
  if (warp == 0) {
    group_starts(start, g.offsets, g.offsets64, g.groups, g.total_rows);
    group_tiles(first, start, g.groups, g.fill, g.total_rows, NT, g.tiles_n);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch();
  const uint32_t tmem = *tmem_slot;
  const int all = g.groups + (g.fill ? 2 : 0);
  const int total = first[all];

  struct Spot {
    int group, row0, rows, col0;  // rows of this tile; first output column
  };
  int cursor = 0;
  auto at = [&](int t) {
    while (t >= first[cursor + 1]) ++cursor;
    Spot p;
    p.group = cursor;
    const int begin = cursor <= g.groups ? start[cursor] : 0;
    const int end = cursor < g.groups ? start[cursor + 1]
                                      : (cursor == g.groups ? g.total_rows : start[0]);
    const int tiles_r = (end - begin + NT - 1) / NT;
    const int r = t - first[cursor];
    const int tn = r / tiles_r, tr = r - tn * tiles_r;  // a block of weights serves its rows in turn
    p.row0 = begin + tr * NT;
    p.rows = end - p.row0 < NT ? end - p.row0 : NT;
    p.col0 = tn * 128;
    return p;
  };
  const int blocks_k = (g.k + kBlockK - 1) / kBlockK;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t kt = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const Spot p = at(t);
        const int num_k = p.group < g.groups ? blocks_k : 0;
        for (int kb = 0; kb < num_k; ++kb, ++kt) {
          const int s = int(kt % S);
          if (kt >= uint32_t(S) && !mbar_wait(&empty[s], ((kt / S) & 1u) ^ 1u, status)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + size_t(s) * C::STAGE;
          mbar_expect_tx(&full[s], C::STAGE);
          if (AMN) {
            tma_load_3d(sa, &map_w, p.col0, kb * kBlockK, p.group, &full[s]);
            tma_load_3d(sa + 8192, &map_w, p.col0 + 64, kb * kBlockK, p.group, &full[s]);
          } else {
            tma_load_3d(sa, &map_w, kb * kBlockK, p.col0, p.group, &full[s]);
          }
          tma_load_3d(sa + C::A_BYTES, &map_x, kb * kBlockK, p.row0, 0, &full[s]);
        }
      }
      if (!ok)  // copies still in flight write this CTA's shared memory
        for (uint32_t j = kt < uint32_t(S) ? 0 : kt - S; j < kt; ++j)
          mbar_wait(&full[j % S], (j / S) & 1u, status);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t kt = 0, round = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const Spot p = at(t);
        const int num_k = p.group < g.groups ? blocks_k : 0;
        if (num_k == 0) continue;
        const uint32_t buf = round & 1u;
        if (round >= 2 && !mbar_wait(&tempty[buf], ((round >> 1) & 1u) ^ 1u, status)) break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * uint32_t(NT);
        for (int kb = 0; kb < num_k; ++kb, ++kt) {
          const int s = int(kt % S);
          if (!mbar_wait(&full[s], (kt / S) & 1u, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint8_t* sa = smem + size_t(s) * C::STAGE;
          const uint64_t da = AMN ? sw128_desc_mn(sa) : sw128_desc(sa);
          const uint64_t db = sw128_desc(sa + C::A_BYTES);
          const int left = g.k - kb * kBlockK;
          const int slabs = left >= kBlockK ? kBlockK / 16 : (left + 15) / 16;
#pragma unroll
          for (int kk = 0; kk < kBlockK / 16; ++kk) {
            if (kk >= slabs) break;
            mma_one(acc, da + uint64_t(kk * (AMN ? 2048 : 32) / 16), db + uint64_t(kk * 2), g.idesc,
                    (kb | kk) ? 1u : 0u);
          }
          mma_commit(&empty[s]);
        }
        if (ok) mma_commit(&tfull[buf]);
        ++round;
      }
    }
  } else if (warp >= 4) {
    const int q = warp & 3;
    uint32_t round = 0;
    T* out = static_cast<T*>(g.out);
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const Spot p = at(t);
      const bool zeros = p.group >= g.groups;
      const uint32_t buf = round & 1u;
      if (!zeros) {
        const bool ok = mbar_wait(&tfull[buf], (round >> 1) & 1u, status, limit_of(blocks_k));
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
      }
      const int col = p.col0 + q * 32 + lane;
      T* o = out + int64_t(p.row0) * g.ldo + col;
#pragma unroll 1
      for (int c0 = 0; c0 < NT && c0 < p.rows; c0 += 16) {
        uint32_t v[16];
        if (zeros) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0;
        } else {
          asm volatile(
              "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
              "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
              : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
                "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
              : "r"(tmem + buf * uint32_t(NT) + uint32_t(c0) + (uint32_t(q * 32) << 16)));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        }
        if (col < g.n) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < p.rows) o[int64_t(c0 + j) * g.ldo] = from_float<T>(__uint_as_float(v[j]));
        }
      }
      if (!zeros) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[buf]);
        ++round;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(uint32_t(C::TMEM_COLS))
                 : "memory");
  }
}

template <int NT, bool AMN, typename T>
int launch(const Product& p, cudaStream_t q) {
  CUtensorMap mw, mx;
  if (!make_operand_map(&mw, p.b, p.bf16, 128) || !make_operand_map(&mx, p.a, p.bf16, NT))
    return CHOL_ERR_UNSUPPORTED;
  FewArgs g{};
  g.n = int(p.n), g.k = int(p.k), g.groups = int(p.batch), g.total_rows = int(p.total_rows);
  g.fill = p.fill;
  g.tiles_n = int((p.n + 127) / 128);
  g.out = p.out, g.ldo = p.ldo;
  g.offsets = p.offsets, g.offsets64 = p.offsets64;
  const uint32_t type = p.bf16 ? 1u : 0u;
  g.idesc = (1u << 4) | (type << 7) | (type << 10) | (uint32_t(AMN) << 15) |
            (uint32_t(NT >> 3) << 17) | (8u << 24);
  // an upper bound: every group may end in a partial tile
  const int64_t total = ((p.total_rows + NT - 1) / NT + p.batch + 2) * g.tiles_n;
  if (total > 0x7fffffffLL - 1024) return CHOL_ERR_UNSUPPORTED;  // tile numbers step past it
  const int64_t ctas = total < sm_count() ? total : sm_count();
  return chol::status_from(chol::launch_pdl(few_kernel<NT, AMN, T>, dim3(unsigned(ctas)),
                                            dim3(kFewThreads), FewCfg<NT>::SMEM, q, true, mw, mx, g,
                                            chol::device_status_ptr()));
}

template <int NT>
int launch_nt(const Product& p, cudaStream_t q) {
  if (p.b.mn_major)
    return p.bf16 ? launch<NT, true, __nv_bfloat16>(p, q) : launch<NT, true, __half>(p, q);
  return p.bf16 ? launch<NT, false, __nv_bfloat16>(p, q) : launch<NT, false, __half>(p, q);
}

template <int NT>
cudaError_t set_few() {
  const int bytes = int(FewCfg<NT>::SMEM);
  const cudaFuncAttribute a = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(few_kernel<NT, true, __nv_bfloat16>, a, bytes)) != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(few_kernel<NT, true, __half>, a, bytes)) != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(few_kernel<NT, false, __nv_bfloat16>, a, bytes)) != cudaSuccess) return e;
  return cudaFuncSetAttribute(few_kernel<NT, false, __half>, a, bytes);
}

}  // namespace

// The groups' sizes are on the device, so the rule goes by their mean. Measured in bf16, us, here /
// 256-row tiles, means of 1, 8, 24 and 32 rows, all groups alike:
//     8 groups, 2048 x 4096     30 / 40    30 / 32    32 / 33    31 / 33
//    32 groups, 1024 x 2048     32 / 40    32 / 35    34 / 35    34 / 35   (64 rows: 48 / 37)
//   128 groups, 2048 x 768      84 / 88    85 / 96    87 / 97    86 / 97
//   256 groups, 1024 x 1024    106 / 126  106 / 130  109 / 128  109 / 129
// Where it loses: rows that gather in few groups, whose weights are then read once per row tile (128
// groups, 2048 x 768, every row in one group: 43 / 21 at a mean of 8, 57 / 23 at 24; in half of the
// groups 49 / 52 at 8, 85 / 55 at 24).
bool few_better(const Product& p) {
  return p.mode == kRaggedM && p.total_rows <= 32 * p.batch;
}

// Row tiles a little above the average group.
int launch_few(const Product& p, cudaStream_t q) {
  if (p.total_rows <= 8 * p.batch) return launch_nt<16>(p, q);
  if (p.total_rows <= 24 * p.batch) return launch_nt<32>(p, q);
  return launch_nt<64>(p, q);
}

cudaError_t prepare_few() {
  cudaError_t e;
  if ((e = set_few<16>()) != cudaSuccess) return e;
  if ((e = set_few<32>()) != cudaSuccess) return e;
  return set_few<64>();
}

}  // namespace lin
