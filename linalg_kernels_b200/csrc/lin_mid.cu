// lin_mid.cu — the whole Newton-Schulz iteration of matrices with 128 < smaller side <= 256 and
// the other side <= 256, in one launch, on chip: a CTA pair per matrix.
//
// The matrix is held as s x len (a tall one transposed on the way in and out), padded with zeros to
// 256 x 256. A CTA of the pair keeps in shared memory
//   X   its 128 rows, K-major blocks of 64 columns   operands of G = X X^T
//   Xc  its 128 columns, all 256 rows                MN-major B operand of B X
//   G   its 128 rows of G, then of B                 operands of G G, A operand of B X
// G is symmetric, so the rows of a CTA are its half of the pair's B operand too; only X needs the
// second copy, of which half goes to the other CTA: 32 KB per step over distributed shared memory.
// Products are tcgen05.mma cta_group::2 (M256 x N256 x K16) on one FP32 accumulator of 256 TMEM
// columns; 512 threads drain it, a thread per row and 64 columns.
//
// Through global memory (a pair's tiles stored, loaded by TMA again) a phase of this chain took 11000
// cycles, 4000 of them for a CTA's 64 KB of stores at 16 bytes a cycle: 92 us for 64 matrices of
// 256 x 256. On chip the whole call takes 57 us.
#include "lin_chip.cuh"
#include "lin_mid.cuh"

namespace lin {

namespace {

using namespace chip;

constexpr int T = 512;
constexpr uint32_t kXcBlock = 2 * kBlockBytes;  // 256 rows x 64 columns

struct MidArgs {
  Matrix x, momentum, out;
  int s, len;  // smaller side, other side
  int tall, steps, nesterov;
  int in_path, out_path;
  float beta, gain, decay, rate;
  float scale, eps;       // of X; G has scale^2, B 1
  float inv_gram, inv_x;  // their reciprocals
  float coef[3 * LINALG_MAX_STEPS];
};

__device__ __forceinline__ void mma_two(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_two(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(uint16_t(3))
      : "memory");
}
// Xc as B operand: N = columns (contiguous), K = rows.
__device__ __forceinline__ uint64_t desc_xc(const void* tile) {
  const uint32_t addr = smem_u32(tile);
  uint64_t d = 0;
  d |= uint64_t((addr >> 4) & 0x3FFF);
  d |= uint64_t(kXcBlock >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
// Chunk of columns c .. c + 7 (of 128) of row r (of 256) in Xc.
__device__ __forceinline__ uint32_t xc_at(int r, int c) {
  return uint32_t(c >> 6) * kXcBlock + uint32_t(r) * 128 + ((uint32_t(c >> 3) & 7) ^ (r & 7)) * 16;
}

struct Place {
  uint8_t* xs;
  double *warp_sum, *cta_sum;
  float2* factor;
  int64_t matrix;
  int row0, rows;  // this CTA's rows of the s x len matrix
};

// This CTA's rows: their norm's share (with the momentum updated on the way), then
// X = scale * u / (norm + eps) into xs.
template <bool MUON, typename TX, typename TM>
__device__ __forceinline__ void read_rows(const MidArgs& g, const Place& p) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // in the caller's order: lines (rows, or columns of X when tall) of `width` elements
  const int lines = g.tall ? g.len : p.rows, width = g.tall ? p.rows : g.len;
  const int per_line = (width + 7) / 8;
  // tall: 8 lines x 4 chunks per warp against bank conflicts of the scattered stores
  const int strips = g.tall ? (per_line + 3) / 4 : per_line;
  const uint32_t reciprocal = uint32_t(0xffffffffu / uint32_t(strips > 0 ? strips : 1)) + 1u;
  const int total = g.tall ? (lines + 7) / 8 * strips * 32 : lines * per_line;
  constexpr int U = MUON ? 2 : 4;
  const int batches = (total + U * T - 1) / (U * T);
  const int64_t x0 = p.matrix * g.x.stride + (g.tall ? p.row0 : int64_t(p.row0) * g.x.ld);
  const int64_t m0 =
      p.matrix * g.momentum.stride + (g.tall ? p.row0 : int64_t(p.row0) * g.momentum.ld);
  float u[U][8];
  int rr[U], cc[U];
  double sum = 0.0;
  float2 f = make_float2(0.f, 0.f);
#pragma unroll 1
  for (int it = 0; it < 2 * batches || it == 0; ++it) {
    const bool first = it < batches;
    if (it == batches) {
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) p.warp_sum[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        double t = 0.0;
        for (int k = 0; k < T / 32; ++k) t += p.warp_sum[k];
        *p.cta_sum = t;
      }
      sync_cluster();
      if (tid == 0)
        *p.factor = start_factor(ld_remote_f64(remote(smem_u32(p.cta_sum), 0)) +
                                     ld_remote_f64(remote(smem_u32(p.cta_sum), 1)),
                                 g.scale, g.eps);
      __syncthreads();
      f = *p.factor;
      if (batches == 0) break;
    }
    if (it != batches) {
      const int k0 = (first ? it : 2 * batches - 1 - it) * U * T + tid;
      Eight<TX> x[U];
      Eight<TM> mo[MUON ? U : 1];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int k = k0 + q * T;
        if (g.tall) {
          const int t = k >> 5, l = k & 31, block = div_by(t, reciprocal, strips);
          rr[q] = block * 8 + (l & 7);
          cc[q] = ((t - block * strips) * 4 + (l >> 3)) * 8;
        } else {
          rr[q] = div_by(k, reciprocal, strips);
          cc[q] = (k - rr[q] * per_line) * 8;
        }
        if (k >= total || rr[q] >= lines || cc[q] >= width) rr[q] = -1;
        if (rr[q] >= 0) {
          const int count = width - cc[q] < 8 ? width - cc[q] : 8;
          x[q].load(g.x, x0 + int64_t(rr[q]) * g.x.ld + cc[q], count);
          if (MUON)
            mo[MUON ? q : 0].load(g.momentum, m0 + int64_t(rr[q]) * g.momentum.ld + cc[q], count);
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
      for (int j = 0; j < 8; ++j) y[j] = j < count ? start_scaled(u[q][j], f) : 0.f;
      uint4 hi, lo;
      round8v<false>(y, hi, lo);
      if (!g.tall) {
        *reinterpret_cast<uint4*>(p.xs + chunk_at(rr[q], cc[q])) = hi;
      } else {
        const __half* h = reinterpret_cast<const __half*>(&hi);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= count) break;
          *reinterpret_cast<__half*>(p.xs + chunk_at(cc[q] + j, rr[q]) + (rr[q] & 7) * 2) = h[j];
        }
      }
    }
  }
}

// 128 columns of the result from n0, staged as FP32 pieces of 64 columns: wide [row][column], the
// 16-byte units of a row permuted by it; tall [column][row].
template <bool MUON, typename TO>
__device__ __forceinline__ void write_rows(const MidArgs& g, const Place& p, const float* stage,
                                           int n0) {
  const int lines = g.tall ? 128 : 256, per_line = g.tall ? 16 : 8;  // two pieces
#pragma unroll 1
  for (int k = threadIdx.x; k < lines * per_line; k += T) {
    const int line = k / per_line, c = (k - line * per_line) * 8;
    int er, ec, count;
    const float *a, *b;
    if (g.tall) {  // line: a column of X, a row of the caller's
      er = n0 + line, ec = p.row0 + c;
      count = er < g.len ? p.rows - c : 0;
      a = stage + line * 128 + c;
      b = a + 4;
    } else {  // line: a row of one piece
      const int row = line & 127, piece = line >> 7;
      er = p.row0 + row, ec = n0 + piece * 64 + c;
      count = row < p.rows ? g.len - ec : 0;
      const float* src = stage + piece * 8192 + row * 64;
      a = src + (((c >> 2) ^ (row & 15)) << 2);
      b = src + ((((c >> 2) + 1) ^ (row & 15)) << 2);
    }
    if (count <= 0) continue;
    if (count > 8) count = 8;
    const int64_t at = p.matrix * g.out.stride + int64_t(er) * g.out.ld + ec;
    Eight<TO> w;
    if (MUON) w.load(g.out, at, count);
    const float4 lo = *reinterpret_cast<const float4*>(a), hi = *reinterpret_cast<const float4*>(b);
    float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (MUON) {
      float old[8];
      w.get(old);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(-g.rate, y[e], g.decay * old[e]);
    }
    Eight<TO>::put(g.out, at, y, count);
  }
}

template <bool MUON>
__global__ void __launch_bounds__(T, 1) __cluster_dims__(2, 1, 1)
    mid_kernel(const MidArgs g, int* status) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* xs = smem;                     // X: 4 blocks of 128 rows x 64 columns
  uint8_t* xc = xs + 4 * kBlockBytes;     // Xc: 2 blocks of 256 rows x 64 columns
  uint8_t* gs = xc + 2 * kXcBlock;        // G, then B: 4 blocks of 128 x 64
  double* warp_sum = reinterpret_cast<double*>(gs + 4 * kBlockBytes);  // [T / 32]
  double* cta_sum = warp_sum + T / 32;
  float2* factor = reinterpret_cast<float2*>(cta_sum + 1);
  uint64_t* bar = reinterpret_cast<uint64_t*>(factor + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);

  const int tid = threadIdx.x, warp = tid >> 5;
  const int row = tid & 127, part = tid >> 7;  // TMEM lane; columns 64 part .. + 63
  const uint32_t rank = rank_in_cluster();
  const int full_row = int(rank) * 128 + row;

  if (tid == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(256u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  Place p{xs, warp_sum, cta_sum, factor, int64_t(blockIdx.x >> 1), int(rank) * 128, 0};
  p.rows = g.s - p.row0 < 128 ? g.s - p.row0 : 128;
  if (p.rows < 128 || g.len < 256)  // X's padding
    for (uint32_t k = tid * 16; k < 4 * kBlockBytes; k += T * 16)
      *reinterpret_cast<uint4*>(xs + k) = make_uint4(0, 0, 0, 0);
  griddep_wait();
  griddep_launch();
  switch (g.in_path) {
    case 1:
      read_rows<MUON, __nv_bfloat16, float>(g, p);
      break;
    case 2:
      read_rows<MUON, float, float>(g, p);
      break;
    case 3:
      read_rows<MUON, __nv_bfloat16, __nv_bfloat16>(g, p);
      break;
    default:
      read_rows<MUON, Any, Any>(g, p);
  }
  __syncthreads();

  // columns 64 part .. + 63 of X belong to the Xc of CTA part / 2
  const uint32_t xc_to = remote(smem_u32(xc), uint32_t(part >> 1));
  const int xc_col = (part & 1) * 64;
  const uint32_t tmem = *tmem_slot;
  const uint32_t acc = tmem + uint32_t(part * 64) + (uint32_t((warp & 3) * 32) << 16);
  uint32_t phase = 0;
  bool ok = true;
  auto wait = [&]() {  // for the MMAs committed last
    if (ok) ok = mbar_wait(bar, phase, status);
    phase ^= 1;
    tc_fence_after();
  };
  auto publish = [&]() {  // both CTAs' shared-memory writes before the next MMAs
    asm volatile("fence.proxy.async;" ::: "memory");
    tc_fence_before();
    sync_cluster();
    tc_fence_after();
  };
#pragma unroll
  for (int c = 0; c < 64; c += 8)
    st_remote16(xc_to + xc_at(full_row, xc_col + c),
                *reinterpret_cast<const uint4*>(xs + chunk_at(row, part * 64 + c)));
  publish();

  const uint32_t id = (1u << 4) | (32u << 17) | (16u << 24);  // fp16, FP32 sums, 256 x 256
  const int k_len = (g.len + 15) / 16, k_s = (g.s + 15) / 16;
  const bool leader = rank == 0 && tid == 0;
  auto rows_product = [&](const uint8_t* t, int slabs) {  // t t^T, K-major
    const uint64_t d0 = sw128_desc(t);
#pragma unroll 1
    for (int k = 0; k < slabs; k += 4) {
      const uint64_t d = d0 + (uint64_t((k >> 2) * kBlockBytes) >> 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < slabs) mma_two(tmem, d + e * 2, d + e * 2, id, (k | e) ? 1u : 0u);
    }
    commit_two(bar);
  };

  for (int step = 0; step < g.steps; ++step) {
    const float ca = g.coef[3 * step], cb = g.coef[3 * step + 1], cc = g.coef[3 * step + 2];
    // ---- G = X X^T (stored as summed: X's scale squared) ----
    if (leader && ok) rows_product(xs, k_len);
    wait();
#pragma unroll
    for (int c0 = 0; c0 < 64; c0 += 16) {
      float v[16];
      tmem_ld16(acc + uint32_t(c0), v);
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        const float y[8] = {v[j], v[j + 1], v[j + 2], v[j + 3], v[j + 4], v[j + 5], v[j + 6], v[j + 7]};
        uint4 hi, lo;
        round8v<false>(y, hi, lo);
        *reinterpret_cast<uint4*>(gs + chunk_at(row, part * 64 + c0 + j)) = hi;
      }
    }
    publish();
    // ---- B = a I + b G + c G G ----
    if (leader && ok) rows_product(gs, k_s);
    wait();
    const float fb = cb * g.inv_gram, fc = cc * g.inv_gram * g.inv_gram;
    const int diag_warp = int(rank) * 128 + (warp & 3) * 32;  // first row of this warp
#pragma unroll
    for (int c0 = 0; c0 < 64; c0 += 16) {
      float v[16];
      tmem_ld16(acc + uint32_t(c0), v);
      const int col = part * 64 + c0;
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = v[j + e] * fc;
        uint4* at = reinterpret_cast<uint4*>(gs + chunk_at(row, col + j));
        add8(y, *at, fb);
        if ((col & ~31) == diag_warp) {  // the same for the whole warp
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] += col + j + e == full_row ? ca : 0.f;
        }
        uint4 hi, lo;
        round8v<false>(y, hi, lo);
        *at = hi;
      }
    }
    publish();
    // ---- X <- B X ----
    if (leader && ok) {
      const uint64_t da = sw128_desc(gs), db = desc_xc(xc);
#pragma unroll 1
      for (int k = 0; k < k_s; k += 4) {
        const uint64_t oa = uint64_t((k >> 2) * kBlockBytes) >> 4, ob = uint64_t(k * 2048) >> 4;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < k_s)
            mma_two(tmem, da + oa + e * 2, db + ob + e * 128, id | (1u << 16), (k | e) ? 1u : 0u);
      }
      commit_two(bar);
    }
    wait();
    if (step + 1 < g.steps) {
#pragma unroll
      for (int c0 = 0; c0 < 64; c0 += 16) {
        float v[16];
        tmem_ld16(acc + uint32_t(c0), v);
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
          const float y[8] = {v[j], v[j + 1], v[j + 2], v[j + 3],
                              v[j + 4], v[j + 5], v[j + 6], v[j + 7]};
          uint4 hi, lo;
          round8v<false>(y, hi, lo);
          *reinterpret_cast<uint4*>(xs + chunk_at(row, part * 64 + c0 + j)) = hi;
          st_remote16(xc_to + xc_at(full_row, xc_col + c0 + j), hi);
        }
      }
      publish();
    }
  }

  // ---- the result, 128 columns at a time through G's buffer (no MMA reads it any more) ----
  float* stage = reinterpret_cast<float*>(gs);
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    if (part >> 1 == h) {
      float* to = stage + (part & 1) * 8192;
#pragma unroll
      for (int c0 = 0; c0 < 64; c0 += 16) {
        float v[16];
        tmem_ld16(acc + uint32_t(c0), v);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] *= g.inv_x;
        if (g.tall) {
#pragma unroll
          for (int j = 0; j < 16; ++j) to[(c0 + j) * 128 + row] = v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 16; j += 4)
            *reinterpret_cast<float4*>(to + row * 64 + ((((c0 + j) >> 2) ^ (row & 15)) << 2)) =
                make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
      }
    }
    __syncthreads();
    if (g.out_path == 1)
      write_rows<MUON, __nv_bfloat16>(g, p, stage, h * 128);
    else if (g.out_path == 2)
      write_rows<MUON, float>(g, p, stage, h * 128);
    else
      write_rows<MUON, Any>(g, p, stage, h * 128);
    __syncthreads();
  }
  tc_fence_before();
  sync_cluster();  // no CTA leaves while the other may write its shared memory
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u)
                 : "memory");
  }
}

constexpr size_t kMidSmem = 8 * kBlockBytes + 2 * size_t(kXcBlock) + (T / 32 + 1) * 8 + 8 + 16 + 1024;
static_assert(kMidSmem <= 227 * 1024, "shared memory");

}  // namespace

bool mid_supported(int64_t m, int64_t n, bool split) {
  const int64_t s = m < n ? m : n, len = m < n ? n : m;
  return !split && s > 128 && len <= 256;
}

int launch_mid_ortho(const linalg_matrix* x, const linalg_matrix* momentum,
                     const linalg_matrix* out, int64_t batch, int64_t m, int64_t n, double beta,
                     int nesterov, float decay, float rate, int steps, const float* coefficients,
                     float eps, cudaStream_t q) {
  MidArgs g{};
  g.x = device_matrix(x);
  if (momentum != nullptr) g.momentum = device_matrix(momentum);
  g.out = device_matrix(out);
  g.tall = m > n;
  g.s = int(g.tall ? n : m), g.len = int(g.tall ? m : n);
  g.steps = steps, g.nesterov = nesterov;
  g.in_path = input_path(g.x, momentum != nullptr ? &g.momentum : nullptr, n);
  g.out_path = output_path(g.out, n);
  g.beta = float(beta), g.gain = float(1.0 - beta);
  g.decay = decay, g.rate = rate;
  g.scale = x_scale(false), g.eps = eps;
  g.inv_x = 1.f / g.scale, g.inv_gram = g.inv_x * g.inv_x;
  for (int k = 0; k < 3 * steps; ++k) g.coef[k] = coefficients[k];
  const dim3 grid(unsigned(2 * batch)), block(T);
  return chol::status_from(
      momentum != nullptr
          ? chol::launch_pdl(mid_kernel<true>, grid, block, kMidSmem, q, true, g, chol::device_status_ptr())
          : chol::launch_pdl(mid_kernel<false>, grid, block, kMidSmem, q, true, g,
                             chol::device_status_ptr()));
}

cudaError_t prepare_mid_ortho() {
  const cudaFuncAttribute a = cudaFuncAttributeMaxDynamicSharedMemorySize;
  const cudaError_t e = cudaFuncSetAttribute(mid_kernel<true>, a, int(kMidSmem));
  return e != cudaSuccess ? e : cudaFuncSetAttribute(mid_kernel<false>, a, int(kMidSmem));
}

}  // namespace lin
