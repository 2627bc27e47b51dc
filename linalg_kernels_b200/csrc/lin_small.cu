// lin_small.cu — the whole Newton-Schulz iteration of small matrices (smaller side <= 128) in one
// launch, on chip.
//
// A matrix is held as s x L, s its smaller side (a tall matrix is transposed on the way in and
// out). p = floor(128 / s) matrices (s rounded up to 16) are stacked to the 128 rows of one tile: with the entries of
// G = X X^T between different matrices set to zero, G, G G and B = b G + c G G stay block
// diagonal and (a I + B) X acts on each matrix alone, so one set of M = 128 MMAs serves all of them.
//
// X lives in shared memory as 128-byte-swizzled K-major blocks of 64 columns; the same bytes are
// the MN-major B operand of B X (the summed index is then X's row). G and B share one buffer: an
// epilogue thread overwrites the elements it has read. Accumulators in TMEM, a thread per row
// and share of the columns.
//
//   per step:  G = X X^T -> mask, fp16   |   B = a I + b G + c G G -> fp16   |   X <- B X
//   (the diagonals of G and B stay in FP32, see below)
//
// A long matrix is split over a cluster of 2, 4 or 8 CTAs by columns. Only G needs all columns:
// each CTA writes its FP32 partials to the CTAs that own their columns, which sum them in rank
// order (the same bits every time) and write the rounded slice to all.
//
// `SPLIT`: two fp16 planes per operand and three products, as in lin_gemm.cu. One accumulator
// covers at most 192 columns of K, so it needs no drain.
//
// Bound by latency: per step three dependent chains MMA -> TMEM read -> convert -> shared memory,
// ~5500 cycles for a 128 x 128 tile (2000 of them MMAs), beside ~9000 for reading and the norm and
// ~5000 for writing. One 128 x 128 matrix takes 25 us (the products of lin_gemm.cu, 17 launches,
// took 86), an optimiser step on 512 x 128 in full precision over 4 CTAs 78 us (203 us). 1024 of
// 64 x 64 take 43 us, 0.39 TB/s (423 us): their 512 tiles are resident at once, four CTAs an SM, and
// share its issue slots for the conversions; the 64 registers that this leaves spill 156 bytes a
// thread (192 in the step). The diagonals in FP32 cost 3.5 us of the 25 and 8 us of the 43.
#include "lin_chip.cuh"
#include "lin_small.cuh"

namespace lin {

namespace {

using namespace chip;

struct SmallArgs {
  Matrix x, momentum, out;
  int s, len;        // smaller side, other side
  int pitch;         // rows of the tile per matrix: s rounded up to the MMA's 16-wide K slabs, so
                     // that a matrix's sums do not depend on its place in the tile
  int tall;
  int per_cta;       // matrices stacked in one tile
  int64_t batch;
  int cta_cols;      // columns per CTA of a cluster (multiple of 64)
  int ranks;         // CTAs per cluster
  int steps;
  int nesterov;
  int in_path, out_path;
  float beta, gain, decay, rate;
  float scale, eps;       // of X; G has scale^2, B 1
  float inv_gram, inv_x;  // their reciprocals
  float coef[3 * LINALG_MAX_STEPS];
};

struct Start {  // where read_start works
  uint8_t* xs;
  uint32_t x_plane;
  double *warp_sum, *mat_sum;
  float2* factor;
  int64_t tile;
  int c_first, cols;
};

// Norms, then X = scale * u / (norm + eps). Each matrix of the tile has its own warps, which walk
// its share of this CTA in the caller's order in chunks of eight columns, U in flight per
// thread. The last U stay in registers between the two passes: all of them up to 128 x 128.
// One instance per pair of types, and rolled loops: what runs once waits for its own
// instructions, so the path taken has to be short.
template <int T, bool SPLIT, bool MUON, bool CLUSTER, typename TX, typename TM>
__device__ __forceinline__ void read_start(const SmallArgs& g, const Start& st) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int team = (T / 32) / g.per_cta;  // warps per matrix (per_cta <= 8)
  const int mine = warp / team;           // matrix of the tile this warp reads
  const int64_t im = st.tile * g.per_cta + mine;
  const bool reads = mine < g.per_cta && im < g.batch;
  const int worker = tid - mine * team * 32, workers = team * 32;
  const int rows = g.tall ? st.cols : g.s, width = g.tall ? g.s : st.cols;
  // A wide matrix's row goes to one row of X: consecutive lanes take consecutive chunks. A tall
  // one's is scattered over X's rows, two bytes each: 8 rows x 4 chunks per warp, which trades
  // shorter reads for 4-way instead of 16-way bank conflicts.
  const int per_row = (width + 7) / 8;
  const int strips = g.tall ? (per_row + 3) / 4 : per_row;
  const uint32_t reciprocal = uint32_t(0xffffffffu / uint32_t(strips > 0 ? strips : 1)) + 1u;
  const int total = g.tall ? (rows + 7) / 8 * strips * 32 : rows * per_row;
  constexpr int U = T == 512 && !MUON ? 4 : 2;  // registers: 16 (32) per chunk and array
  const int batches = (total + U * workers - 1) / (U * workers);
  const int64_t x0 = im * g.x.stride + (g.tall ? int64_t(st.c_first) * g.x.ld : st.c_first);
  const int64_t m0 =
      im * g.momentum.stride + (g.tall ? int64_t(st.c_first) * g.momentum.ld : st.c_first);
  const int base = mine * g.pitch;
  float u[U][8];
  int rr[U], cc[U];
  double sum = 0.0;
  float2 f = make_float2(0.f, 0.f);
  bool finite = false;
#pragma unroll 1
  for (int it = 0; it < 2 * batches || it == 0; ++it) {
    const bool first = it < batches;
    if (it == batches) {
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) st.warp_sum[warp] = sum;
      __syncthreads();
      if (tid < g.per_cta) {
        double t = 0.0;
        for (int k = 0; k < team; ++k) t += st.warp_sum[tid * team + k];
        st.mat_sum[tid] = t;
      }
      if (CLUSTER) sync_cluster();
      if (tid < g.per_cta) {
        double t = st.mat_sum[tid];
        if (CLUSTER) {
          t = 0.0;
          for (int k = 0; k < g.ranks; ++k)
            t += ld_remote_f64(remote(smem_u32(st.mat_sum + tid), k));
        }
        // a matrix with a NaN or an infinity is worked on as zeros (its entries would reach the
        // others of the tile) and written as NaN: marked by a factor that is not finite
        st.factor[tid] = start_factor(t, g.scale, g.eps);
      }
      __syncthreads();
      if (batches == 0) break;
      if (reads) f = st.factor[mine];
      finite = isfinite(f.x);
    }
    if (!reads) continue;
    if (it != batches) {
      const int k0 = (first ? it : 2 * batches - 1 - it) * U * workers + worker;
      Eight<TX> x[U];
      Eight<TM> mo[MUON ? U : 1];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int k = k0 + q * workers;
        if (g.tall) {
          const int t = k >> 5, l = k & 31, block = div_by(t, reciprocal, strips);
          rr[q] = block * 8 + (l & 7);
          cc[q] = ((t - block * strips) * 4 + (l >> 3)) * 8;
        } else {
          rr[q] = div_by(k, reciprocal, strips);
          cc[q] = (k - rr[q] * per_row) * 8;
        }
        if (k >= total || rr[q] >= rows || cc[q] >= width) rr[q] = -1;
        if (rr[q] >= 0) {
          const int count = width - cc[q] < 8 ? width - cc[q] : 8;
          x[q].load(g.x, x0 + int64_t(rr[q]) * g.x.ld + cc[q], count);
          if (MUON) mo[MUON ? q : 0].load(g.momentum, m0 + int64_t(rr[q]) * g.momentum.ld + cc[q], count);
        }
      }
#pragma unroll
      for (int q = 0; q < U; ++q) {
        if (rr[q] < 0) continue;
        x[q].get(u[q]);
        if (MUON) {
          float m[8];
          mo[MUON ? q : 0].get(m);
          if (first) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = fmaf(g.beta, m[j], g.gain * u[q][j]);
            Eight<TM>::put(g.momentum, m0 + int64_t(rr[q]) * g.momentum.ld + cc[q], m,
                           width - cc[q] < 8 ? width - cc[q] : 8);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            u[q][j] = g.nesterov ? fmaf(g.beta, m[j], g.gain * u[q][j]) : m[j];
        }
      }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (rr[q] < 0) continue;
      const int count = width - cc[q] < 8 ? width - cc[q] : 8;
      if (first) {
        sum += squares8(u[q], count);
        continue;
      }
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = finite && j < count ? start_scaled(u[q][j], f) : 0.f;
      uint4 hi, lo;
      round8v<SPLIT>(y, hi, lo);
      if (!g.tall) {
        const uint32_t at = chunk_at(base + rr[q], cc[q]);
        *reinterpret_cast<uint4*>(st.xs + at) = hi;
        if (SPLIT) *reinterpret_cast<uint4*>(st.xs + st.x_plane + at) = lo;
      } else {
        const __half* h = reinterpret_cast<const __half*>(&hi);
        const __half* l = reinterpret_cast<const __half*>(&lo);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= count) break;
          const uint32_t at = chunk_at(base + cc[q] + j, rr[q]) + (rr[q] & 7) * 2;
          *reinterpret_cast<__half*>(st.xs + at) = h[j];
          if (SPLIT) *reinterpret_cast<__half*>(st.xs + st.x_plane + at) = l[j];
        }
      }
    }
  }
}

// Writes 64 columns of the result, staged as FP32, in the caller's order. Wide: [row][column],
// the 16-byte units of a row permuted by it; tall: [column][row].
template <int T, bool MUON, typename TO>
__device__ __forceinline__ void write_result(const SmallArgs& g, const Start& st,
                                             const float* stage, int n0) {
  const int left = st.cols - n0 < 64 ? st.cols - n0 : 64;  // columns of X in this piece
  const int per_row = g.tall ? g.pitch / 8 : 8;            // chunks of a caller's row
  const int lines = g.tall ? 64 * g.per_cta : 128;         // caller's rows
#pragma unroll 1
  for (int k = threadIdx.x; k < lines * per_row; k += T) {
    const int line = k / per_row, c = (k - line * per_row) * 8;
    int mt, er, ec, count;  // matrix of the tile; the caller's row, first column, columns
    const float* src;
    int flip = 0;
    if (g.tall) {
      mt = line >> 6;
      const int col = line & 63;
      er = st.c_first + n0 + col, ec = c;
      count = col < left ? g.s - c : 0;
      src = stage + col * 128 + mt * g.pitch + c;
    } else {
      mt = line / g.pitch;
      const int lr = line - mt * g.pitch;
      er = lr, ec = st.c_first + n0 + c;
      count = lr < g.s && mt < g.per_cta ? left - c : 0;
      flip = line & 15;
      src = stage + line * 64;
    }
    const int64_t im = st.tile * g.per_cta + mt;
    if (count <= 0 || im >= g.batch) continue;
    if (count > 8) count = 8;
    const int64_t at = im * g.out.stride + int64_t(er) * g.out.ld + ec;
    Eight<TO> w;
    if (MUON) w.load(g.out, at, count);
    float y[8];
    const float4 a = *reinterpret_cast<const float4*>(g.tall ? src : src + ((c / 4) ^ flip) * 4);
    const float4 b =
        *reinterpret_cast<const float4*>(g.tall ? src + 4 : src + ((c / 4 + 1) ^ flip) * 4);
    y[0] = a.x, y[1] = a.y, y[2] = a.z, y[3] = a.w;
    y[4] = b.x, y[5] = b.y, y[6] = b.z, y[7] = b.w;
    if (!isfinite(st.factor[mt].x)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __int_as_float(0x7fc00000);
    }
    if (MUON) {
      float old[8];
      w.get(old);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(-g.rate, y[e], g.decay * old[e]);
    }
    Eight<TO>::put(g.out, at, y, count);
  }
}

template <int T, bool SPLIT, bool MUON, bool CLUSTER>
__global__ void __launch_bounds__(T, T == 256 ? (MUON ? 3 : 4) : 1)
    small_kernel(const SmallArgs g, int* status) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  constexpr int P = SPLIT ? 2 : 1;
  constexpr int PARTS = T / 128;       // threads per row of the tile
  constexpr int GCOLS = 128 / PARTS;   // columns of G per thread
  const int blocks = g.cta_cols / 64;
  const uint32_t x_plane = uint32_t(blocks) * kBlockBytes;
  uint8_t* xs = smem;                            // [P] X: blocks of 64 columns
  uint8_t* gs = xs + P * x_plane;                // [P] G, then B: two blocks
  constexpr uint32_t g_plane = 2 * kBlockBytes;
  uint8_t* es = gs + P * g_plane;                // CLUSTER: FP32 partials of this CTA's slice of G
  double* warp_sum = reinterpret_cast<double*>(es);  // [T / 32] (CLUSTER: before es is used)
  double* mat_sum = reinterpret_cast<double*>(es + (CLUSTER ? 65536 : 128));  // [8] per matrix
  float2* factor = reinterpret_cast<float2*>(mat_sum + 8);  // [8]
  float* diag = reinterpret_cast<float*>(factor + 8);  // [128] half precision: G's diagonal
  float* own = diag + 128;                             // [128] and what a row of X is scaled with
  uint64_t* bar = reinterpret_cast<uint64_t*>(own + 128);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);

  const int tid = threadIdx.x, warp = tid >> 5;
  const int row = tid & 127, part = tid >> 7;  // this thread's TMEM lane and share of the columns
  const uint32_t rank = CLUSTER ? rank_in_cluster() : 0;
  const int64_t tile = CLUSTER ? blockIdx.x / g.ranks : blockIdx.x;
  const int in_tile = row / g.pitch;  // matrix of this row
  const int c_first = int(rank) * g.cta_cols;     // first column of this CTA
  const int cols = g.len - c_first < g.cta_cols ? (g.len - c_first > 0 ? g.len - c_first : 0)
                                                : g.cta_cols;
  const int tmem_cols = g.cta_cols <= 128 ? 128 : (g.cta_cols <= 256 ? 256 : 512);

  if (tid == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(uint32_t(tmem_cols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // zeros in X's padding: rows between and behind the matrices, columns behind the last
  if (g.per_cta * g.pitch < 128 || g.s < g.pitch || cols < g.cta_cols ||
      (tile + 1) * g.per_cta > g.batch)
    for (uint32_t k = tid * 16; k < P * x_plane; k += T * 16)
      *reinterpret_cast<uint4*>(xs + k) = make_uint4(0, 0, 0, 0);
  // and in G's: its entries between matrices stay as they are
  if (g.per_cta > 1)
    for (uint32_t k = tid * 16; k < P * g_plane; k += T * 16)
      *reinterpret_cast<uint4*>(gs + k) = make_uint4(0, 0, 0, 0);
  griddep_wait();
  griddep_launch();

  const Start st{xs, x_plane, warp_sum, mat_sum, factor, tile, c_first, cols};
  switch (g.in_path) {
    case 1:
      read_start<T, SPLIT, MUON, CLUSTER, __nv_bfloat16, float>(g, st);
      break;
    case 2:
      read_start<T, SPLIT, MUON, CLUSTER, float, float>(g, st);
      break;
    case 3:
      read_start<T, SPLIT, MUON, CLUSTER, __nv_bfloat16, __nv_bfloat16>(g, st);
      break;
    default:
      read_start<T, SPLIT, MUON, CLUSTER, Any, Any>(g, st);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
  uint32_t phase = 0;
  bool ok = true;
  auto wait = [&]() {  // for the MMAs committed last
    if (ok) ok = mbar_wait(bar, phase, status);
    phase ^= 1;
    tc_fence_after();
  };
  auto publish = [&]() {  // shared-memory writes before the next MMAs
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  const int k16 = (cols + 15) / 16;  // X's columns beyond `cols` are zero
  // the 32-column groups of G that hold entries of this warp's rows (lanes 32 q .. + 31)
  const int q32 = (warp & 3) * 32;
  const int last_col = ((q32 + 31) / g.pitch + 1) * g.pitch;
  const int win0 = g.per_cta == 1 ? 0 : q32 / g.pitch * g.pitch / 32;
  const int win1 = g.per_cta == 1 || last_col > 128 ? 4 : (last_col + 31) / 32;
  constexpr bool KEEP = T == 512 && !CLUSTER;  // G's FP32 values stay in registers until B
  constexpr int GROUPS = 4 / PARTS;            // 32-column groups of G per thread
  float gram[KEEP ? 32 : 1];

  for (int step = 0; step < g.steps; ++step) {
    const float ca = g.coef[3 * step], cb = g.coef[3 * step + 1], cc = g.coef[3 * step + 2];
    // ---- G = X X^T ----
    if (tid == 0 && ok) {
      const uint32_t id = idesc_half(128, 0);
      uint32_t any = 0;
#pragma unroll
      for (int t = SPLIT ? 0 : 2; t < 3; ++t) {  // lo hi, hi lo, hi hi
        const uint8_t* pa = xs + (t == 0 ? x_plane : 0);
        const uint8_t* pb = xs + (t == 1 ? x_plane : 0);
        const uint64_t da = sw128_desc(pa), db = sw128_desc(pb);
#pragma unroll 1
        for (int k = 0; k < k16; k += 4) {
          const uint64_t off = uint64_t((k >> 2) * kBlockBytes) >> 4;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (k + e >= k16) break;
            mma_half(tmem, da + off + e * 2, db + off + e * 2, id, any);
            any = 1;
          }
        }
      }
      if (!any)  // no columns here (a cluster longer than the matrix): zeros from zero columns
        mma_half(tmem, sw128_desc(xs), sw128_desc(xs), id, 0);
      mma_commit(bar);
    }
    wait();
    // (scale of G: X's squared, so the sums are stored as they are; entries between matrices are
    // dropped)
    if (!CLUSTER) {
#pragma unroll
      for (int n = 0; n < GROUPS; ++n) {
        const int q = win0 + part + n * PARTS;
        if (q >= win1) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[16];
          const int c0 = q * 32 + h * 16;
          tmem_ld16(tmem + lane_base + uint32_t(c0), v);
          // 16 columns are of one matrix: the pitch is a multiple of 16
          const bool mine = uint32_t(c0 - in_tile * g.pitch) < uint32_t(g.pitch);
          if (!SPLIT && q * 32 == q32) {  // the same for the whole warp (selects: no branches)
            float d = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const bool here = c0 + j == row;
              d = here ? v[j] : d;
              v[j] = here ? 0.f : v[j];
            }
            if (uint32_t(row - c0) < 16u) diag[row] = d;
          }
#pragma unroll
          for (int j = 0; j < 16; j += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              y[e] = mine ? v[j + e] : 0.f;
              if (KEEP) gram[KEEP ? h * 16 + j + e : 0] = y[e];
            }
            uint4 hi, lo;
            round8v<SPLIT>(y, hi, lo);
            const uint32_t at = chunk_at(row, c0 + j);
            *reinterpret_cast<uint4*>(gs + at) = hi;
            if (SPLIT) *reinterpret_cast<uint4*>(gs + g_plane + at) = lo;
          }
        }
      }
    } else {
      // FP32 partials to the CTA that owns their columns: [from][column / 4][row] x 4 floats. Only
      // writes cross the cluster, so nothing waits for a remote read.
      const int width = 128 / g.ranks;  // columns per owner: 64, 32 or 16
      const uint32_t slot = uint32_t(rank) * uint32_t(width) * 512;
#pragma unroll
      for (int q = 0; q < GCOLS / 32; ++q) {
        float v[32];
        const int c0 = part * GCOLS + q * 32;
        tmem_ld32(tmem + lane_base + uint32_t(c0), v);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const int owner = (c0 + j) / width, c = (c0 + j) - owner * width;
          const uint32_t at = smem_u32(es) + slot + (uint32_t(c >> 2) * 128 + row) * 16;
          st_remote16(remote(at, owner),
                      make_uint4(__float_as_uint(v[j]), __float_as_uint(v[j + 1]),
                                 __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3])));
        }
      }
      sync_cluster();
      // the slice this CTA owns: summed in rank order, rounded, written to every CTA
      for (int k = tid; k < 128 * (width / 8); k += T) {
        const int rr = k & 127, c = (k >> 7) * 8, c0 = int(rank) * width + c;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.f;
        const uint8_t* at = es + (uint32_t(c >> 2) * 128 + rr) * 16;
        for (int o = 0; o < g.ranks; ++o, at += width * 512) {
          const float4 a = *reinterpret_cast<const float4*>(at);
          const float4 b = *reinterpret_cast<const float4*>(at + 2048);
          y[0] += a.x, y[1] += a.y, y[2] += a.z, y[3] += a.w;
          y[4] += b.x, y[5] += b.y, y[6] += b.z, y[7] += b.w;
        }
        const int mt = rr / g.pitch;
        const bool mine = uint32_t(c0 - mt * g.pitch) < uint32_t(g.pitch);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = mine ? y[e] : 0.f;
        if (!SPLIT && uint32_t(rr - c0) < 8u) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            d = c0 + e == rr ? y[e] : d;
            y[e] = c0 + e == rr ? 0.f : y[e];
          }
          for (int o = 0; o < g.ranks; ++o) st_remote_f32(remote(smem_u32(diag + rr), o), d);
        }
        uint4 hi, lo;
        round8v<SPLIT>(y, hi, lo);
        const uint32_t to = smem_u32(gs) + chunk_at(rr, c0);
        for (int o = 0; o < g.ranks; ++o) {
          st_remote16(remote(to, o), hi);
          if (SPLIT) st_remote16(remote(to + g_plane, o), lo);
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");
      sync_cluster();
    }
    publish();
    // ---- B = b G + c G G ----
    if (tid == 0 && ok) {
      const uint32_t id = idesc_half(128, 0);
#pragma unroll
      for (int t = SPLIT ? 0 : 2; t < 3; ++t) {
        const uint8_t* pa = gs + (t == 0 ? g_plane : 0);
        const uint8_t* pb = gs + (t == 1 ? g_plane : 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t off = uint64_t((k >> 2) * kBlockBytes + (k & 3) * 32) >> 4;
          mma_half(tmem, sw128_desc(pa) + off, sw128_desc(pb) + off, id,
                   (k || t > (SPLIT ? 0 : 2)) ? 1u : 0u);
        }
      }
      mma_commit(bar);
    }
    wait();
    // Half precision: G and B in shared memory are without their diagonals D, whose rounding would
    // be the largest error by far (small matrices have few entries to average it, and X X^T of
    // a wide one is nearly a multiple of I: 32 x 4096 was 4.4e-3 off in bf16, now 1.7e-3). With G = D + O,
    //   (G G)_ij = (O O)_ij + (d_i + d_j) O_ij  off the diagonal,  (O O)_ii + d_i^2  on it,
    // and the diagonal of a I + b G + c G G scales the rows of X in FP32 at the end.
    // Full: a X is added in FP32 at the end, not summed by the tensor core, whose rounding towards
    // zero would weigh on the largest term; and B keeps 22 bits with a scale of 2048.
    constexpr float kPoly = b_scale(SPLIT);
    const float fb = cb * g.inv_gram * kPoly, fc = cc * g.inv_gram * g.inv_gram * kPoly;
#pragma unroll
    for (int n = 0; n < GROUPS; ++n) {
      const int q = win0 + part + n * PARTS;
      if (q >= win1) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[16];
        const int c0 = q * 32 + h * 16;
        tmem_ld16(tmem + lane_base + uint32_t(c0), v);
        if (!SPLIT && q * 32 == q32) {
          float oo = 0.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) oo = c0 + j == row ? v[j] : oo;
          if (uint32_t(row - c0) < 16u) {
            const float d = diag[row];
            own[row] = ca + fb * d + fc * (oo + d * d);
          }
        }
        const float di = SPLIT ? 0.f : fmaf(fc, diag[row], fb);
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
          float y[8];
          const uint32_t at = chunk_at(row, c0 + j);
          if (SPLIT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = v[j + e] * fc;
            add8(y, *reinterpret_cast<const uint4*>(gs + at), fb);
            add8(y, *reinterpret_cast<const uint4*>(gs + g_plane + at), fb);
          } else {
            const float4 d0 = *reinterpret_cast<const float4*>(diag + c0 + j);
            const float4 d1 = *reinterpret_cast<const float4*>(diag + c0 + j + 4);
            const float dj[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
            const uint4 w = KEEP ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(gs + at);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float2 o =
                  KEEP ? make_float2(gram[KEEP ? h * 16 + j + e : 0],
                                     gram[KEEP ? h * 16 + j + e + 1 : 0])
                       : __half22float2(*reinterpret_cast<const __half2*>(&ws[e / 2]));
              const float2 f = chol::ffma2(make_float2(fc, fc), make_float2(dj[e], dj[e + 1]),
                                           make_float2(di, di));  // fb + fc (d_i + d_j)
              const float2 t = chol::ffma2(f, o, make_float2(0.f, 0.f));
              const float2 r = chol::ffma2(make_float2(v[j + e], v[j + e + 1]), make_float2(fc, fc), t);
              y[e] = r.x;
              y[e + 1] = r.y;
            }
            if (q * 32 == q32) {
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = c0 + j + e == row ? 0.f : y[e];
            }
          }
          uint4 hi, lo;
          round8v<SPLIT>(y, hi, lo);
          *reinterpret_cast<uint4*>(gs + at) = hi;
          if (SPLIT) *reinterpret_cast<uint4*>(gs + g_plane + at) = lo;
        }
      }
    }
    publish();
    // ---- X <- B X ----
    if (tid == 0 && ok) {
      for (int n0 = 0; n0 < g.cta_cols; n0 += 256) {
        const int n = g.cta_cols - n0 < 256 ? g.cta_cols - n0 : 256;
        const uint32_t id = idesc_half(n, 1);
#pragma unroll
        for (int t = SPLIT ? 0 : 2; t < 3; ++t) {
          const uint8_t* pa = gs + (t == 0 ? g_plane : 0);
          const uint8_t* pb = xs + (t == 1 ? x_plane : 0) + (n0 >> 6) * kBlockBytes;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_half(tmem + uint32_t(n0),
                     sw128_desc(pa) + (uint64_t((k >> 2) * kBlockBytes + (k & 3) * 32) >> 4),
                     desc_cols(pb) + (uint64_t(k * 2048) >> 4), id,
                     (k || t > (SPLIT ? 0 : 2)) ? 1u : 0u);
        }
      }
      mma_commit(bar);
    }
    wait();
    const float row_factor = SPLIT ? ca : own[row];
    if (step + 1 < g.steps) {
      for (int c0 = part * 32; c0 < g.cta_cols; c0 += PARTS * 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[16];
          tmem_ld16(tmem + lane_base + uint32_t(c0 + h * 16), v);
#pragma unroll
          for (int j = 0; j < 16; j += 8) {
            float y[8];
            const uint32_t at = chunk_at(row, c0 + h * 16 + j);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = SPLIT ? v[j + e] * (1.f / kPoly) : v[j + e];
            add8(y, *reinterpret_cast<const uint4*>(xs + at), row_factor);
            if (SPLIT) add8(y, *reinterpret_cast<const uint4*>(xs + x_plane + at), ca);
            uint4 hi, lo;
            round8v<SPLIT>(y, hi, lo);
            *reinterpret_cast<uint4*>(xs + at) = hi;
            if (SPLIT) *reinterpret_cast<uint4*>(xs + x_plane + at) = lo;
          }
        }
      }
      publish();
      continue;
    }
    // ---- the result, 64 columns at a time through G's buffer (no MMA reads it any more), so that
    // the caller's rows are written in order ----
    float* stage = reinterpret_cast<float*>(gs);
#pragma unroll 1
    for (int n0 = 0; n0 < g.cta_cols; n0 += 64) {
      for (int h = part; h < 2; h += PARTS) {
        const int c0 = n0 + h * 32;
        float v[32];
        tmem_ld32(tmem + lane_base + uint32_t(c0), v);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = v[j + e] * (g.inv_x / kPoly);
          const uint32_t at = chunk_at(row, c0 + j);
          add8(y, *reinterpret_cast<const uint4*>(xs + at), row_factor * g.inv_x);
          if (SPLIT) add8(y, *reinterpret_cast<const uint4*>(xs + x_plane + at), ca * g.inv_x);
          if (g.tall) {
#pragma unroll
            for (int e = 0; e < 8; ++e) stage[(h * 32 + j + e) * 128 + row] = y[e];
          } else {
            const int unit = (h * 32 + j) / 4;
            *reinterpret_cast<float4*>(stage + row * 64 + ((unit ^ (row & 15)) * 4)) =
                make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(stage + row * 64 + (((unit + 1) ^ (row & 15)) * 4)) =
                make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      }
      __syncthreads();
      if (g.out_path == 1)
        write_result<T, MUON, __nv_bfloat16>(g, st, stage, n0);
      else if (g.out_path == 2)
        write_result<T, MUON, float>(g, st, stage, n0);
      else
        write_result<T, MUON, Any>(g, st, stage, n0);
      __syncthreads();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  if (CLUSTER) sync_cluster();  // no CTA leaves while another may read its shared memory
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(uint32_t(tmem_cols))
                 : "memory");
}

// Columns one CTA can hold: X and G (both planes) and, in a cluster, the FP32 partial of G fit
// the 227 KB of shared memory, and an accumulator of X the 512 columns of TMEM.
constexpr int kMaxCols = 512, kMaxColsSplit = 192;
constexpr int kMaxRanks = 8;
constexpr int kMaxSmem = 227 * 1024;

size_t smem_bytes(bool split, int ranks, int cta_cols) {
  size_t b = size_t(split ? 2 : 1) * (size_t(cta_cols / 64) + 2) * kBlockBytes;
  b += ranks > 1 ? 65536 : 128;
  b += 8 * 8 + 8 * 8 + 2 * 128 * 4 + 16 + 1008;  // 1008: to a 1024-byte boundary from a 16-byte one
  // CTAs of different clusters on one SM could wait for each other's TMEM: one CTA per SM
  if (ranks > 1 && b < 118 * 1024) b = 118 * 1024;
  return b;
}

template <int T, bool SPLIT, bool MUON, bool CLUSTER>
int launch(const SmallArgs& g, int64_t tiles, size_t smem, cudaStream_t q) {
  chol::note_launch(q);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tiles * g.ranks));
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = q;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(g.ranks);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  return chol::status_from(
      cudaLaunchKernelEx(&cfg, small_kernel<T, SPLIT, MUON, CLUSTER>, g, chol::device_status_ptr()));
}

}  // namespace

#define LIN_FOR_EACH_SMALL(F) \
  F(false, false, false)      \
  F(false, false, true)       \
  F(false, true, false)       \
  F(false, true, true)        \
  F(true, false, false)       \
  F(true, false, true)        \
  F(true, true, false)        \
  F(true, true, true)

bool small_supported(int64_t m, int64_t n, bool split) {
  const int64_t s = m < n ? m : n, len = m < n ? n : m;
  return s <= 128 && len <= int64_t(kMaxRanks) * (split ? kMaxColsSplit : kMaxCols);
}

int launch_small(const linalg_matrix* x, const linalg_matrix* momentum, const linalg_matrix* out,
                 int64_t batch, int64_t m, int64_t n, double beta, int nesterov, float decay,
                 float rate, int steps, const float* coefficients, float eps, bool split,
                 cudaStream_t q) {
  SmallArgs g{};
  g.x = device_matrix(x);
  if (momentum != nullptr) g.momentum = device_matrix(momentum);
  g.out = device_matrix(out);
  g.tall = m > n;
  g.s = int(g.tall ? n : m), g.len = int(g.tall ? m : n);
  g.pitch = (g.s + 15) / 16 * 16;
  g.per_cta = 128 / g.pitch;
  if (g.per_cta > batch) g.per_cta = int(batch);
  g.batch = batch;
  const int most = split ? kMaxColsSplit : kMaxCols;
  g.ranks = 1;
  while (int64_t(g.ranks) * most < g.len) g.ranks *= 2;
  const int64_t tiles = (batch + g.per_cta - 1) / g.per_cta;
  const int chunk = (g.len + g.ranks - 1) / g.ranks;
  g.cta_cols = (chunk + 63) / 64 * 64;
  g.steps = steps;
  g.in_path = input_path(g.x, momentum != nullptr ? &g.momentum : nullptr, n);
  g.out_path = output_path(g.out, n);
  g.beta = float(beta), g.gain = float(1.0 - beta), g.nesterov = nesterov;
  g.decay = decay, g.rate = rate;
  g.scale = x_scale(split), g.eps = eps;
  g.inv_x = 1.f / g.scale, g.inv_gram = g.inv_x * g.inv_x;
  for (int k = 0; k < 3 * steps; ++k) g.coef[k] = coefficients[k];
  const size_t smem = smem_bytes(split, g.ranks, g.cta_cols);
  if (tiles * g.ranks > 0x7fffffffLL) return CHOL_ERR_UNSUPPORTED;
  const bool muon = momentum != nullptr, cluster = g.ranks > 1;
  // 512 threads shorten the epilogues of a lone tile per SM; 256 leave registers for four tiles
  const bool wide = cluster || split || tiles <= sm_count();
#define LIN_SMALL(SPLIT, MUON, CLUSTER)                                      \
  if (split == SPLIT && muon == MUON && cluster == CLUSTER)                  \
    return wide ? launch<512, SPLIT, MUON, CLUSTER>(g, tiles, smem, q)       \
                : launch<SPLIT || CLUSTER ? 512 : 256, SPLIT, MUON, CLUSTER>(g, tiles, smem, q);
  LIN_FOR_EACH_SMALL(LIN_SMALL)
#undef LIN_SMALL
  return CHOL_ERR_UNSUPPORTED;
}

template <int T, bool SPLIT, bool MUON, bool CLUSTER>
cudaError_t set_small() {
  return cudaFuncSetAttribute(small_kernel<T, SPLIT, MUON, CLUSTER>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
}

cudaError_t prepare_small_ortho() {
  cudaError_t e;
#define LIN_SMALL(SPLIT, MUON, CLUSTER)                                                    \
  if ((e = set_small<512, SPLIT, MUON, CLUSTER>()) != cudaSuccess) return e;               \
  if ((e = set_small<SPLIT || CLUSTER ? 512 : 256, SPLIT, MUON, CLUSTER>()) != cudaSuccess) \
    return e;
  LIN_FOR_EACH_SMALL(LIN_SMALL)
#undef LIN_SMALL
  return cudaSuccess;
}

}  // namespace lin
