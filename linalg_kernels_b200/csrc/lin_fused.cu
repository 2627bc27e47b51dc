// lin_fused.cu — the Newton-Schulz iteration of a batch of middle-sized matrices (both sides > 128)
// in one launch: a CTA pair takes a matrix through all its steps.
//
// Launched product by product (lin_gemm.cu), a batch whose X, G and B together exceed L2 streams
// them through HBM three times a step (b640n512: 7 of 335 MB per step and array), and a small
// batch pays a launch and an idle GPU's ramp per product. Here a pair owns one X (two buffers),
// one G and one B, reused for each of its matrices, so they stay in L2, and the only work that
// passes HBM is the start value and the result. The tiles, the operands' orders and the epilogue
// are lin_gemm.cu's: 256 x 256 tiles, two accumulators, the epilogue of a tile beside the next
// tile's MMAs.
//
// A tile needs parts of the phase before it (G of X, B of G, X of B). The pair's epilogue warps
// count finished tiles in shared memory of both CTAs; the producers wait for the last tile that
// theirs reads, not for the phase: with two row blocks (n = 512) every phase starts while the last
// tile of the one before is in its epilogue. With one block (n = 256) the chain
// MMA -> epilogue -> TMA is exposed, 15 times per matrix; it is still shorter than a launch.
#include "lin_tile.cuh"
#include "lin_fused.cuh"

namespace lin {

namespace {

using namespace tile;

using C = Cfg<256, 2, 0>;
constexpr int S = C::STAGES;

struct FusedArgs {
  int m, n, s, batch;             // s: the smaller side
  int tiles_m, tiles_n, tiles_s;  // 256-wide blocks of rows, columns, smaller side
  int steps;
  __half* x;         // [pair][2]
  __half* sq;        // [pair][2]: G, B
  int64_t ldx, lds, x_plane, s_plane;
  float scale;
  void* out;
  int64_t ldo, out_stride;
  int out_type, out_vec, out_boxes;
  float decay, rate;
  uint32_t idesc;  // K-major operands
  float coef[3 * LINALG_MAX_STEPS];
};

// The tiles of one pair in order: per matrix and step G's lower tiles, B's, then X's.
template <bool TALL>
struct Sequence {
  const FusedArgs& g;
  int matrix, pairs, step, phase, index, count;  // count: tiles of the phase
  int number;                                    // of this tile among all the pair's
  int before;                                    // number of the first tile of the phase before
  int tm, tn;
  __device__ __forceinline__ Sequence(const FusedArgs& a, int pair, int p)
      : g(a), matrix(pair), pairs(p), step(0), phase(0), index(0), number(0), before(0), tm(0), tn(0) {
    count = lower();
  }
  __device__ __forceinline__ int lower() const { return g.tiles_s * (g.tiles_s + 1) / 2; }
  __device__ __forceinline__ bool valid() const { return matrix < g.batch; }
  __device__ __forceinline__ void next() {
    ++number;
    if (++index < count) {  // lower triangle by rows; X by rows, or by columns when tall (the first
                            // then need only B's first rows)
      if (TALL && phase == 2) {
        if (++tm == g.tiles_m) tm = 0, ++tn;
      } else if (++tn == (phase < 2 ? tm + 1 : g.tiles_n)) {
        tn = 0, ++tm;
      }
      return;
    }
    before = number - count;
    index = tm = tn = 0;
    if (++phase == 3) {
      phase = 0;
      if (++step == g.steps) {
        step = 0;
        matrix += pairs;
      }
    }
    count = phase < 2 ? lower() : g.tiles_m * g.tiles_n;
  }
  // Number of the last tile that this one reads from the phase before it; -1: none.
  __device__ __forceinline__ int needs() const {
    if (phase == 0) {
      if (step == 0) return -1;
      return TALL ? before + g.tiles_m * g.tiles_n - 1 : before + (tm + 1) * g.tiles_n - 1;
    }
    // rows r of a symmetric result: its lower tiles up to (last row, r) hold them or their mirror
    const int r = phase == 1 || !TALL ? tm : tn;
    return before + (g.tiles_s - 1) * g.tiles_s / 2 + r;
  }
  __device__ __forceinline__ int k_len() const {
    return phase == 0 ? (TALL ? g.m : g.n) : g.s;
  }
  __device__ __forceinline__ bool a_mn() const { return TALL && phase == 0; }
  __device__ __forceinline__ bool b_mn() const { return TALL ? phase == 0 : phase == 2; }
};

__device__ __forceinline__ uint32_t load_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.cluster.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}
__device__ __forceinline__ void add_relaxed(uint32_t cluster_addr) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(cluster_addr), "r"(1u)
               : "memory");
}
__device__ __forceinline__ uint32_t addr_in(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}

template <bool TALL, int LAST>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    fused_kernel(const __grid_constant__ CUtensorMap x0_rows,
                 const __grid_constant__ CUtensorMap x0_cols,
                 const __grid_constant__ CUtensorMap x_rows,
                 const __grid_constant__ CUtensorMap x_cols,
                 const __grid_constant__ CUtensorMap squares,
                 const __grid_constant__ CUtensorMap result, const FusedArgs g, int* status) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* epi = smem + size_t(S) * C::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + size_t(S) * C::STAGE + C::EPI);
  uint64_t* full = bars;           // [S] first CTA: a stage of both CTAs has landed
  uint64_t* empty = bars + S;      // [S] the MMAs have read the stage
  uint64_t* tfull = bars + 2 * S;  // [2] accumulator ready
  uint64_t* tempty = tfull + 2;    // [2] first CTA: accumulator drained by both CTAs
  uint64_t* c_bars = tempty + 2;   // [2 * kEpiWarps] C's boxes
  uint32_t* done = reinterpret_cast<uint32_t*>(c_bars + 2 * kEpiWarps);  // [4] finished tiles, by number mod 4
  uint32_t* tmem_slot = done + 4;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * kEpiWarps);
    }
    for (int b = 0; b < 2 * kEpiWarps; ++b) mbar_init(&c_bars[b], 1);
    for (int i = 0; i < 4; ++i) done[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&x0_rows);
    prefetch_map(&x0_cols);
    prefetch_map(&x_rows);
    prefetch_map(&x_cols);
    prefetch_map(&squares);
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(uint32_t(C::TMEM_COLS))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  griddep_wait();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  griddep_launch();
  const uint32_t tmem = *tmem_slot;
  const int pair = int(blockIdx.x >> 1), pairs = int(gridDim.x >> 1);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      uint32_t kt = 0;
      bool ok = true;
      for (Sequence<TALL> t(g, pair, pairs); t.valid() && ok; t.next()) {
        const int need = t.needs();
        if (need >= 0) {
          const uint32_t target = 2 * kEpiWarps * (uint32_t(need) / 4 + 1);
          const uint32_t* slot = &done[need & 3];
          if (load_acquire(slot) < target) {
            const uint64_t t0 = global_ns();
            while (load_acquire(slot) < target)
              if (global_ns() - t0 > kWaitLimitNs) {
                atomicExch(status, CHOL_ERR_WAIT_TIMEOUT);
                ok = false;
                break;
              }
            if (!ok) break;
          }
          asm volatile("fence.proxy.async;" ::: "memory");  // those stores before these copies
        }
        const bool first = t.step == 0;
        const int zx = first ? t.matrix : pair * 2 + ((t.step - 1) & 1);
        const CUtensorMap* rows = first ? &x0_rows : &x_rows;
        const CUtensorMap* cols = first ? &x0_cols : &x_cols;
        const CUtensorMap *ma, *mb;
        int za = zx, zb = zx;
        if (t.phase == 1) {
          ma = mb = &squares;
          za = zb = pair * 2;
        } else if (t.phase == 0) {
          ma = mb = TALL ? cols : rows;
        } else if (TALL) {
          ma = rows;
          mb = &squares;
          zb = pair * 2 + 1;
        } else {
          ma = &squares;
          za = pair * 2 + 1;
          mb = cols;
        }
        const int a_row = t.tm * kTileM + int(rank) * 128, b_row = t.tn * 256 + int(rank) * 128;
        const int num_k = (t.k_len() + kBlockK - 1) / kBlockK;
        const bool amn = t.a_mn(), bmn = t.b_mn();
        for (int kb = 0; kb < num_k; ++kb, ++kt) {
          const int s = int(kt % S);
          if (kt >= uint32_t(S) && !wait_bar(&empty[s], ((kt / S) & 1u) ^ 1u, status)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + size_t(s) * C::STAGE;
          uint8_t* sb = sa + C::A_BYTES;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * C::STAGE);
          const uint32_t bar = leader_addr(&full[s]);
          const int kx = kb * kBlockK;
          if (amn) {
            tma_load_pair(sa, ma, a_row, kx, za, bar);
            tma_load_pair(sa + 8192, ma, a_row + 64, kx, za, bar);
          } else {
            tma_load_pair(sa, ma, kx, a_row, za, bar);
          }
          if (bmn) {
            tma_load_pair(sb, mb, b_row, kx, zb, bar);
            tma_load_pair(sb + 8192, mb, b_row + 64, kx, zb, bar);
          } else {
            tma_load_pair(sb, mb, kx, b_row, zb, bar);
          }
        }
      }
      if (!ok && rank == 0)  // copies still in flight write this pair's shared memory
        for (uint32_t j = kt < uint32_t(S) ? 0 : kt - S; j < kt; ++j)
          wait_bar(&full[j % S], (j / S) & 1u, status);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (first CTA) ----------------
    if (rank == 0 && lane == 0) {
      uint32_t kt = 0, round = 0;
      bool ok = true;
      for (Sequence<TALL> t(g, pair, pairs); t.valid() && ok; t.next(), ++round) {
        const uint32_t buf = round & 1u;
        if (round >= 2 && !wait_bar(&tempty[buf], ((round >> 1) & 1u) ^ 1u, status)) break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * 256u;
        const int k_len = t.k_len(), num_k = (k_len + kBlockK - 1) / kBlockK;
        const bool amn = t.a_mn(), bmn = t.b_mn();
        const uint32_t idesc = g.idesc | (uint32_t(amn) << 15) | (uint32_t(bmn) << 16);
        const uint64_t stepa = amn ? 2048 / 16 : 32 / 16, stepb = bmn ? 2048 / 16 : 32 / 16;
        for (int kb = 0; kb < num_k; ++kb, ++kt) {
          const int s = int(kt % S);
          if (!wait_bar(&full[s], (kt / S) & 1u, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint8_t* sa = smem + size_t(s) * C::STAGE;
          const uint8_t* sb = sa + C::A_BYTES;
          const uint64_t da = amn ? sw128_desc_mn(sa) : sw128_desc(sa);
          const uint64_t db = bmn ? sw128_desc_mn(sb) : sw128_desc(sb);
          const int left = k_len - kb * kBlockK;
          const int slabs = left >= kBlockK ? kBlockK / 16 : (left + 15) / 16;
#pragma unroll
          for (int kk = 0; kk < kBlockK / 16; ++kk) {
            if (kk >= slabs) break;
            mma_pair(acc, da + uint64_t(kk) * stepa, db + uint64_t(kk) * stepb, idesc,
                     (kb | kk) ? 1u : 0u);
          }
          commit_pair(&empty[s]);
        }
        if (ok) commit_pair(&tfull[buf]);
      }
    }
  } else if (warp >= 4) {
    // ---------------- epilogue ----------------
    const int q = warp & 3, half = (warp - 4) >> 2;
    using Epi = WarpEpilogue<128, 2, false>;
    Epi ep{epi + (warp - 4) * 2 * kBoxBytes, c_bars + 2 * (warp - 4), 0u, lane};
    uint32_t round = 0;
    const float x_inv = 1.f / g.scale, g_inv = x_inv * x_inv;  // scales: X, G its square, B 1
    const uint32_t done0 = addr_in(done, 0), done1 = addr_in(done, 1);
    for (Sequence<TALL> t(g, pair, pairs); t.valid(); t.next(), ++round) {
      const int row_base = t.tm * kTileM + int(rank) * 128 + q * 32;
      const int col0 = t.tn * 256 + half * 128;
      const bool last = t.phase == 2 && t.step + 1 == g.steps;
      const bool mirror = t.phase < 2 && t.tm > t.tn;
      const float* cf = g.coef + 3 * t.step;
      Out o;
      o.alpha = 1.f, o.beta = 0.f, o.diag = 0.f;
      o.rows = o.n = g.s;
      o.map = &result;
      o.z = t.matrix;
      o.y = 0;
      o.boxes = LAST == kMuon ? 0 : g.out_boxes;
      o.type = LINALG_FP16;
      o.weights = 0;
      o.ldo = g.lds;
      __half* sq = g.sq + int64_t(pair) * 2 * g.s_plane;  // G, then B
      __half* to = sq;
      if (t.phase == 1) {
        o.alpha = cf[2] * g_inv * g_inv, o.beta = cf[1] * g_inv;
        o.diag = cf[0];
        to = sq + g.s_plane;
      } else if (t.phase == 2) {
        o.rows = g.m, o.n = g.n;
        o.ldo = g.ldx;
        to = g.x + (int64_t(pair) * 2 + (t.step & 1)) * g.x_plane;
        if (last) {
          o.alpha = x_inv;
          o.out = static_cast<char*>(g.out) +
                  int64_t(t.matrix) * g.out_stride * (g.out_type == LINALG_FP32 ? 4 : 2);
          o.ldo = g.ldo, o.type = g.out_type, o.vec = g.out_vec;
          o.weights = LAST == kMuon, o.decay = g.decay, o.rate = g.rate;
        }
      }
      const uint32_t buf = round & 1u;
      // C (G's tile) was written by this very warp, a phase ago
      uint4 cw[8];
      if (o.beta != 0.f) ep.fetch_c(o, sq, row_base, col0, cw);
      bool ok = wait_bar(&tfull[buf], (round >> 1) & 1u, status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * 256u + uint32_t(half * 128) + (uint32_t(q * 32) << 16);
      auto get = [&](int c, float (&v)[32]) { tmem_ld32(acc + uint32_t(c), v); };
      if (!last) {
        if (t.index == 0 && t.phase == 0 && t.step == 0) {  // the result's boxes of a matrix before
          if (lane == 0) boxes_read();
          __syncwarp();
        }
#pragma unroll 1
        for (int b = 0; b < Epi::BOXES; ++b) {
          ep.box_now(o, to, b, row_base, col0 + b * 64, mirror, cw,
                     [&](int h, float (&v)[32]) { get(b * 64 + h * 32, v); });
          if (b == 0 && o.beta != 0.f) ep.fetch_c(o, sq, row_base, col0 + 64, cw);
        }
      } else if (ep.by_box(o, row_base)) {
#pragma unroll 1
        for (int b = 0; b < Epi::BOXES; ++b)
          ep.template box<false>(o, b, row_base, col0 + b * 64, false, status,
                                 [&](int h, float (&v)[32]) { get(b * 64 + h * 32, v); });
      } else {
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          float v[32];
          get(c, v);
          ep.direct(o, row_base, col0 + c, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        arrive_leader_relaxed(leader_addr(&tempty[buf]));
        __threadfence();  // the warp's stores, before the report
        add_relaxed(done0 + (t.number & 3) * 4);
        add_relaxed(done1 + (t.number & 3) * 4);
      }
    }
    if (lane == 0) boxes_written();
  }
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

int64_t blocks(int64_t v) { return (v + 255) / 256; }

template <bool TALL, int LAST>
int launch(const CUtensorMap (&maps)[6], const FusedArgs& g, int pairs, cudaStream_t q) {
  return chol::status_from(chol::launch_pdl(
      fused_kernel<TALL, LAST>, dim3(unsigned(2 * pairs)), dim3(kThreads), C::SMEM, q, true,
      maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], g, chol::device_status_ptr()));
}

}  // namespace

int fused_pairs(int64_t batch) {
  const int64_t most = sm_count() / 2;
  return int(batch < most ? batch : most);
}

// Whether one pair per matrix is the shorter way, by a count of K blocks (512 cycles of MMAs):
// here every pair runs its matrices' tiles alone, with an exposed chain per phase when a phase is
// one tile; product by product the tiles of the batch spread over all pairs, at ~6 us (20 blocks)
// per launch for its start, first tile and last epilogue.
bool fused_better(int64_t batch, int64_t m, int64_t n) {
  const int64_t s = m < n ? m : n;
  if (s <= 128 || m > 4096 || n > 4096) return false;
  const int64_t pairs = sm_count() / 2;
  const int64_t bs = blocks(s), lower = bs * (bs + 1) / 2, all = blocks(m) * blocks(n);
  const int64_t ks = (s + 63) / 64, kl = ((m < n ? n : m) + 63) / 64;
  const int64_t chain = bs == 1 ? 30 : 8;  // blocks' worth of waiting per step
  const int64_t fused = ((batch + pairs - 1) / pairs) * (lower * kl + lower * ks + all * ks + chain);
  auto waves = [&](int64_t tiles) { return (tiles * batch + pairs - 1) / pairs; };
  int64_t apart = waves(lower) * kl + waves(lower) * ks + waves(all) * ks;
  // beyond L2 the products stream X four times, G and B twice each through HBM (~1.7 MB a block's time)
  const int64_t bytes = batch * 2 * (4 * m * n + 4 * s * s);
  if (batch * 2 * (2 * m * n + 2 * s * s) > (int64_t(100) << 20) && bytes / 1700000 > apart)
    apart = bytes / 1700000;
  return fused <= apart + 3 * 20;
}

int launch_fused(const FusedCall& f, cudaStream_t q) {
  FusedArgs g{};
  const bool tall = f.m > f.n;
  const int pairs = fused_pairs(f.batch);
  g.m = int(f.m), g.n = int(f.n), g.s = int(tall ? f.n : f.m), g.batch = int(f.batch);
  g.tiles_m = int(blocks(f.m)), g.tiles_n = int(blocks(f.n)), g.tiles_s = int(blocks(g.s));
  g.steps = f.steps;
  g.x = static_cast<__half*>(f.x);
  g.sq = static_cast<__half*>(f.squares);
  g.ldx = f.ldx, g.lds = f.lds, g.x_plane = f.x_plane, g.s_plane = f.s_plane;
  g.scale = f.scale;
  g.out = f.out, g.ldo = f.ldo, g.out_stride = f.out_stride, g.out_type = f.out_type;
  const int sector = f.out_type == LINALG_FP32 ? 8 : 16;
  g.out_vec = (reinterpret_cast<uintptr_t>(f.out) & 31) == 0 && f.ldo % sector == 0 &&
              f.out_stride % sector == 0;
  g.decay = f.decay, g.rate = f.rate;
  g.idesc = (1u << 4) | (32u << 17) | (16u << 24);  // fp16, FP32 sums, 256 x 256
  for (int i = 0; i < 3 * f.steps; ++i) g.coef[i] = f.coefficients[i];
  CUtensorMap maps[6];
  const int64_t two = 2 * pairs;
  const Operand x0{f.x0, f.m, f.n, f.ldx, f.batch, f.x_plane, false};
  const Operand x{f.x, f.m, f.n, f.ldx, two, f.x_plane, false};
  const Operand sq{f.squares, g.s, g.s, f.lds, two, f.s_plane, false};
  Operand x0_mn = x0, x_mn = x;
  x0_mn.mn_major = x_mn.mn_major = true;
  if (!make_operand_map(&maps[0], x0, false, 128) || !make_operand_map(&maps[1], x0_mn, false, 0) ||
      !make_operand_map(&maps[2], x, false, 128) || !make_operand_map(&maps[3], x_mn, false, 0) ||
      !make_operand_map(&maps[4], sq, false, 128))
    return CHOL_ERR_UNSUPPORTED;
  maps[5] = maps[0];
  if (!f.muon && f.out_type != LINALG_FP32 &&
      make_output_map(&maps[5], Operand{f.out, f.m, f.n, f.ldo, f.batch, f.out_stride, false},
                      f.out_type == LINALG_BF16, false))
    g.out_boxes = 2;
  if (f.muon)
    return tall ? launch<true, kMuon>(maps, g, pairs, q) : launch<false, kMuon>(maps, g, pairs, q);
  return tall ? launch<true, kFinal>(maps, g, pairs, q) : launch<false, kFinal>(maps, g, pairs, q);
}

template <bool TALL, int LAST>
cudaError_t set_fused() {
  return cudaFuncSetAttribute(fused_kernel<TALL, LAST>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              int(C::SMEM));
}

cudaError_t prepare_fused() {
  cudaError_t e;
  if ((e = set_fused<false, kFinal>()) != cudaSuccess) return e;
  if ((e = set_fused<true, kFinal>()) != cudaSuccess) return e;
  if ((e = set_fused<false, kMuon>()) != cudaSuccess) return e;
  return set_fused<true, kMuon>();
}

}  // namespace lin
