// lin_ortho.cu — Newton-Schulz orthogonalisation of a batch of matrices, alone and inside the
// optimiser step around it.
//
//   X = u / (||u||_F + eps);  per step  G = X X^T,  B = a I + b G + c G G,  X <- B X
//
// (from the right, G = X^T X, X <- X B, when the matrices are taller than wide, so G is
// always the smaller square). One step is three products of lin_gemm.cu: G and B are
// symmetric, so only the tiles on and below the diagonal are computed and each is written twice.
// Per step 3 m^2 n + m^3 multiply-adds (m the smaller side) instead of the full products'
// 4 m^2 n + 2 m^3.
//
// In half precision a stands on B's diagonal, so that the third product reads no old X: one more
// rounding per row, of the size of X's own. In full precision a X is added in FP32.
//
// Number format: X, G and B are fp16, scaled by a power of two, and not bf16: with the default
// coefficients no entry of X passes 1.21, of G 1.46, of B 3.45, so fp16's range is enough, and its 11
// bits make each rounding 8 times smaller than bf16's at the same tensor rate. With bf16 results the
// error is then the last rounding to bf16 (on random matrices the iteration's own 5e-4 to 1.3e-3 of
// the norm, 2.6e-3 for 32 x 8192, against that rounding's 1.7e-3). The roundings are noise of full
// rank, and the iteration multiplies small singular values by up to 3.4 a step: a matrix of low rank
// (an expert's gradient from few rows) gets noise in the directions that it lacks, 2.4e-2 of the norm
// at rank 64 of 1024, 7e-2 at rank 4, 0.15 at rank 1 (with bf16 iterates 0.2, 0.5 and 1). Full precision
// (fp16 and fp32 results) keeps two planes, x = hi + lo: 8e-7 to 3.3e-6 on random matrices, 2e-4 at
// rank 1, about as FP32 products. The scale keeps the small entries of a large matrix (~1 / sqrt(m n)
// at the start, ~1 / (m sqrt n) in G) out of fp16's subnormals.
//
// The squares of the norm are summed in FP32 by eights, then in FP64 per block and over the blocks in a
// fixed order: the same input gives the same bits, whatever runs beside it.
#include <math.h>

#include <mutex>

#include "lin_chip.cuh"
#include "lin_few.cuh"
#include "lin_mid.cuh"
#include "lin_small.cuh"

namespace lin {

namespace {

constexpr int kPrepThreads = 256;

struct Prep {
  Matrix x, momentum;  // x: the input, or the gradient
  float beta, gain;  // gain: 1 - beta, rounded once
  int nesterov;
  int64_t rows;
  int n, chunks_row;  // chunks of 8 columns per row
  int64_t chunks;     // per matrix
  int parts;          // blocks per matrix
  double* sums;       // [batch][parts]
  __half* planes;     // X: [batch][P][rows][ldx]
  int64_t ldx;
  float scale, eps;
  int path;  // types: see walk_types
};

// The start value u of U chunks per thread, the loads of all of them in flight: the input itself, or
// the momentum average (updated on the way with UPDATE). body(chunk's row, column, count, u).
template <bool MUON, bool UPDATE, typename TX, typename TM, typename Body>
__device__ __forceinline__ void walk(const Prep& p, int64_t i, int part, const Body& body) {
  constexpr int U = MUON ? 2 : 4;
  const int64_t stride = int64_t(p.parts) * kPrepThreads;
  for (int64_t t0 = int64_t(part) * kPrepThreads + threadIdx.x; t0 < p.chunks; t0 += U * stride) {
    Eight<TX> x[U];
    Eight<TM> mo[MUON ? U : 1];
    int64_t r[U];
    int c[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int64_t t = t0 + q * stride;
      // (32-bit division where the chunks of a matrix allow it)
      r[q] = p.chunks <= 0x7fffffff ? int(t) / p.chunks_row : t / p.chunks_row;
      c[q] = int(t - r[q] * p.chunks_row) * 8;
      if (t >= p.chunks) {
        c[q] = -1;
        continue;
      }
      const int count = p.n - c[q] < 8 ? p.n - c[q] : 8;
      x[q].load(p.x, i * p.x.stride + r[q] * p.x.ld + c[q], count);
      if (MUON)
        mo[MUON ? q : 0].load(p.momentum, i * p.momentum.stride + r[q] * p.momentum.ld + c[q], count);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (c[q] < 0) continue;
      const int count = p.n - c[q] < 8 ? p.n - c[q] : 8;
      float u[8];
      x[q].get(u);
      if (MUON) {
        float m[8];
        mo[MUON ? q : 0].get(m);
        if (UPDATE) {
#pragma unroll
          for (int j = 0; j < 8; ++j) m[j] = fmaf(p.beta, m[j], p.gain * u[j]);
          // m: as stored
          Eight<TM>::put(p.momentum, i * p.momentum.stride + r[q] * p.momentum.ld + c[q], m, count);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = p.nesterov ? fmaf(p.beta, m[j], p.gain * u[j]) : m[j];
      }
      body(r[q], c[q], count, u);
    }
  }
}
// The same for the matrices' types: whole aligned chunks of the common ones, else any.
template <bool MUON, bool UPDATE, typename Body>
__device__ __forceinline__ void walk_types(const Prep& p, int64_t i, int part, const Body& body) {
  switch (p.path) {
    case 1:
      walk<MUON, UPDATE, __nv_bfloat16, float>(p, i, part, body);
      break;
    case 2:
      walk<MUON, UPDATE, float, float>(p, i, part, body);
      break;
    case 3:
      walk<MUON, UPDATE, __nv_bfloat16, __nv_bfloat16>(p, i, part, body);
      break;
    default:
      walk<MUON, UPDATE, Any, Any>(p, i, part, body);
  }
}

// Sum of squares of each block's share, with the momentum updated on the way. Bound by HBM: reads
// the input (and reads and writes the momentum) once.
template <bool MUON>
__global__ void __launch_bounds__(kPrepThreads) sum_kernel(const Prep p) {
  griddep_wait();
  griddep_launch();
  const int64_t i = blockIdx.x / p.parts;
  const int part = int(blockIdx.x - i * p.parts);
  double sum = 0.0;
  walk_types<MUON, true>(p, i, part, [&](int64_t, int, int count, const float (&u)[8]) {
    sum += chip::squares8(u, count);
  });
  __shared__ double warp_sum[kPrepThreads / 32];
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < kPrepThreads / 32; ++w) s += warp_sum[w];
    p.sums[blockIdx.x] = s;
  }
}

// X = scale * u / (||u||_F + eps) as fp16, or as hi + lo.
template <bool MUON, bool SPLIT>
__global__ void __launch_bounds__(kPrepThreads) scale_kernel(const Prep p) {
  griddep_wait();
  griddep_launch();
  const int64_t i = blockIdx.x / p.parts;
  const int part = int(blockIdx.x - i * p.parts);
  __shared__ float2 factor;
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int k = threadIdx.x; k < p.parts; k += 32) s += p.sums[i * p.parts + k];
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (threadIdx.x == 0) factor = start_factor(s, p.scale, p.eps);
  }
  __syncthreads();
  const float2 f = factor;
  constexpr int P = SPLIT ? 2 : 1;
  walk_types<MUON, false>(p, i, part, [&](int64_t r, int c, int count, const float (&u)[8]) {
    alignas(16) __half hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = j < count ? start_scaled(u[j], f) : 0.f;
      hi[j] = __float2half_rn(v);
      if (SPLIT) lo[j] = __float2half_rn(v - __half2float(hi[j]));
    }
    // rows of the workspace hold a multiple of 8 elements: whole chunks are written
    __half* o = p.planes + (i * P * p.rows + r) * p.ldx + c;
    *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(hi);
    if (SPLIT)
      *reinterpret_cast<uint4*>(o + p.rows * p.ldx) = *reinterpret_cast<const uint4*>(lo);
  });
}

// rows of the workspace start on 32-byte sectors
int64_t round16(int64_t v) { return (v + 15) & ~int64_t(15); }
size_t round256(size_t v) { return (v + 255) & ~size_t(255); }

struct Layout {
  int64_t planes, ldx, lds, side, x_plane, s_plane;
  size_t x_bytes, s_bytes, sums_bytes, total;
};

// Blocks per matrix of the first passes: about 4 chunks a thread, at most kPrepBlocks over the batch,
// 16 for each of a B200's 148 SMs. Fixed, because the workspace holds a sum per block: its size is
// asked for before any device is looked at, and callers keep it.
constexpr int64_t kPrepBlocks = 148 * 16;
int64_t prep_parts(int64_t batch, int64_t m, int64_t n) {
  const int64_t chunks = m * ((n + 7) / 8);
  int64_t parts = (chunks + kPrepThreads * 4 - 1) / (kPrepThreads * 4);
  const int64_t cap = (kPrepBlocks + batch - 1) / batch;
  if (parts > cap) parts = cap;
  return parts < 1 ? 1 : parts;
}

Layout layout(int64_t batch, int64_t m, int64_t n, bool split) {
  Layout l{};
  if (small_supported(m, n, split) || mid_supported(m, n, split)) return l;  // on chip
  l.planes = split ? 2 : 1;
  l.side = m < n ? m : n;
  l.ldx = round16(n);
  l.lds = round16(l.side);
  l.x_plane = m * l.ldx;
  l.s_plane = l.side * l.lds;
  l.x_bytes = round256(size_t(batch) * l.planes * l.x_plane * 2);
  l.s_bytes = round256(size_t(batch) * l.planes * l.s_plane * 2);
  l.sums_bytes = round256(size_t(batch) * prep_parts(batch, m, n) * sizeof(double));
  l.total = 2 * l.x_bytes + 2 * l.s_bytes + l.sums_bytes;
  return l;
}

bool valid_type(int t) { return t == LINALG_BF16 || t == LINALG_FP16 || t == LINALG_FP32; }
int type_bytes(int t) { return t == LINALG_FP32 ? 4 : 2; }

bool valid_matrix(const linalg_matrix* x, int64_t batch, int64_t m, int64_t n) {
  if (x == nullptr || x->data == nullptr || !valid_type(x->type)) return false;
  if (reinterpret_cast<uintptr_t>(x->data) % type_bytes(x->type)) return false;
  if (x->ld < n || (batch > 1 && x->stride < 0)) return false;
  // rows and matrices of one array must not overlap (the arrays are written)
  if (batch > 1 && x->stride < (m - 1) * x->ld + n && x->stride != 0) return false;
  return true;
}

// Bytes from the first to one past the last element.
void extent(const linalg_matrix* x, int64_t batch, int64_t m, int64_t n, uintptr_t* lo,
            uintptr_t* hi) {
  *lo = reinterpret_cast<uintptr_t>(x->data);
  *hi = *lo + uintptr_t((batch - 1) * x->stride + (m - 1) * x->ld + n) * type_bytes(x->type);
}
bool overlap(const linalg_matrix* x, const linalg_matrix* y, int64_t batch, int64_t m, int64_t n) {
  uintptr_t a, b, c, d;
  extent(x, batch, m, n, &a, &b);
  extent(y, batch, m, n, &c, &d);
  return a < d && c < b;
}

// Shared part of both entry points; momentum == nullptr: plain orthogonalisation.
int iterate(const linalg_matrix* x, const linalg_matrix* momentum, const linalg_matrix* out,
            int64_t batch, int64_t m, int64_t n, double beta, int nesterov, float decay, float rate,
            int steps, const float* coefficients, float eps, bool split, void* workspace,
            cudaStream_t q) {
  if (small_supported(m, n, split))
    return launch_small(x, momentum, out, batch, m, n, beta, nesterov, decay, rate, steps,
                        coefficients, eps, split, q);
  if (mid_supported(m, n, split))
    return launch_mid_ortho(x, momentum, out, batch, m, n, beta, nesterov, decay, rate, steps,
                            coefficients, eps, q);
  const Layout l = layout(batch, m, n, split);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  __half* xs[2] = {reinterpret_cast<__half*>(w), reinterpret_cast<__half*>(w + l.x_bytes)};
  __half* gram = reinterpret_cast<__half*>(w + 2 * l.x_bytes);
  __half* poly = reinterpret_cast<__half*>(w + 2 * l.x_bytes + l.s_bytes);
  const bool muon = momentum != nullptr;
  // Scales: X's is a power of two, G's its square (the sums are stored as they are), B's 1 in half
  // precision. Entries of G up to ~1.3 stay a factor 50 (half) or 12 (full) under fp16's
  // largest; X's small ones (1 / sqrt(m n) at the start) clear of its subnormals. B, with a
  // on its diagonal, needs no scale: what its subnormals lose, 3e-8 per entry, is small against
  // the rounding of its diagonal; the planes of full precision keep 22 bits with 2048.
  const float scale = x_scale(split), gram_scale = scale * scale;
  const float poly_scale = b_scale(split);

  Prep p{};
  p.x = device_matrix(x);
  if (muon) p.momentum = device_matrix(momentum);
  p.beta = float(beta), p.gain = float(1.0 - beta), p.nesterov = nesterov;
  p.rows = m, p.n = int(n);
  p.chunks_row = int((n + 7) / 8);
  p.chunks = m * p.chunks_row;
  p.path = input_path(p.x, muon ? &p.momentum : nullptr, n);
  p.parts = int(prep_parts(batch, m, n));
  p.sums = reinterpret_cast<double*>(w + l.total - l.sums_bytes);
  p.planes = xs[0];
  p.ldx = l.ldx;
  p.scale = scale, p.eps = eps;
  const dim3 grid(unsigned(p.parts * batch)), block(kPrepThreads);
  cudaError_t e;
  e = muon ? chol::launch_pdl(sum_kernel<true>, grid, block, 0, q, true, p)
           : chol::launch_pdl(sum_kernel<false>, grid, block, 0, q, true, p);
  if (e != cudaSuccess) return CHOL_ERR_LAUNCH;
  if (muon)
    e = split ? chol::launch_pdl(scale_kernel<true, true>, grid, block, 0, q, true, p)
              : chol::launch_pdl(scale_kernel<true, false>, grid, block, 0, q, true, p);
  else
    e = split ? chol::launch_pdl(scale_kernel<false, true>, grid, block, 0, q, true, p)
              : chol::launch_pdl(scale_kernel<false, false>, grid, block, 0, q, true, p);
  if (e != cudaSuccess) return CHOL_ERR_LAUNCH;

  const bool tall = m > n;
  const int64_t s = l.side, matrices = batch * l.planes;
  const Operand sq_gram{gram, s, s, l.lds, matrices, l.s_plane, false};
  const Operand sq_poly{poly, s, s, l.lds, matrices, l.s_plane, false};
  for (int k = 0; k < steps; ++k) {
    const float a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const __half* cur = xs[k & 1];
    const Operand rows_x{cur, m, n, l.ldx, matrices, l.x_plane, false};
    const Operand cols_x{cur, m, n, l.ldx, matrices, l.x_plane, true};
    Product g;  // G = X X^T or X^T X
    g.a = g.b = tall ? cols_x : rows_x;
    g.epilogue = kPlanes;
    g.split = split;
    g.symmetric = true;
    g.m = g.n = s, g.k = tall ? m : n, g.batch = batch;
    g.alpha = 1.f;
    g.out = gram, g.ldo = l.lds, g.out_stride = l.s_plane;
    int st = launch_product(g, q);
    if (st != CHOL_OK) return st;
    Product f;  // B = a I + b G + c G G
    f.a = f.b = sq_gram;
    f.epilogue = kPlanes;
    f.split = split;
    f.symmetric = true;
    f.m = f.n = f.k = s, f.batch = batch;
    f.alpha = c * (poly_scale / (gram_scale * gram_scale)), f.beta = b * (poly_scale / gram_scale);
    f.c = gram, f.ldc = l.lds, f.c_plane = l.s_plane;
    // half precision: a on B's diagonal (see above); full: a X is added in FP32 at the end, not summed
    // by the tensor core, whose rounding towards zero would weigh on the largest term
    f.diag = split ? 0.f : a * poly_scale;
    f.out = poly, f.ldo = l.lds, f.out_stride = l.s_plane;
    if ((st = launch_product(f, q)) != CHOL_OK) return st;
    Product u;  // X <- B X or X B
    u.a = tall ? rows_x : sq_poly;
    u.b = tall ? sq_poly : cols_x;
    u.split = split;
    u.m = m, u.n = n, u.k = s, u.batch = batch;
    u.alpha = 1.f / poly_scale;
    if (split) u.beta = a, u.c = cur, u.ldc = l.ldx, u.c_plane = l.x_plane;
    if (k + 1 < steps) {
      u.epilogue = kPlanes;
      u.out = xs[(k + 1) & 1], u.ldo = l.ldx, u.out_stride = l.x_plane;
    } else {
      u.epilogue = muon ? kMuon : kFinal;
      u.alpha /= scale, u.beta /= scale;
      u.out = out->data, u.ldo = out->ld, u.out_stride = out->stride, u.out_type = out->type;
      u.decay = decay, u.rate = rate;
    }
    if ((st = launch_product(u, q)) != CHOL_OK) return st;
  }
  return CHOL_OK;
}

int check_iteration(int64_t batch, int64_t m, int64_t n, int steps, const float* coefficients,
                    float eps, int precision) {
  if (batch < 0 || m < 0 || n < 0) return CHOL_ERR_INVALID_ARG;
  if (steps < 1 || steps > LINALG_MAX_STEPS || coefficients == nullptr) return CHOL_ERR_INVALID_ARG;
  if (precision < LINALG_PRECISION_AUTO || precision > LINALG_PRECISION_FULL)
    return CHOL_ERR_INVALID_ARG;
  for (int i = 0; i < 3 * steps; ++i)
    if (!isfinite(coefficients[i])) return CHOL_ERR_INVALID_ARG;
  if (!(eps >= 0.f) || !isfinite(eps)) return CHOL_ERR_INVALID_ARG;
  return CHOL_OK;
}

// Whether X, G and B stay within fp16's 65504 for every matrix under these coefficients. X's singular
// values start at 1 at most (the Frobenius norm's bound); with s the largest at a step and u = s^2, no
// entry of G passes u and none of B the largest |q| on [0, u], q(u) = b u + c u^2 (with a added where a
// stands on B's diagonal); the next s is the largest |t (a + b t^2 + c t^4)| for t up to s. Beyond the
// range the on-chip kernels would saturate and the products give infinities. Each s is taken
// 1/64 larger, for the roundings of X. (G's limit is the narrower one: X's own is implied.)
// And whether they stay clear of its smallest numbers: small singular values are multiplied by a in
// each step, and the product of the steps' a down to any step must not fall below 1/4. (With a = 0, B
// has no diagonal and X shrinks to its third power: (0, 2, -1) twice in half precision was 1e-2 off
// for 100 x 1500.)
bool in_range(int steps, const float* coefficients, bool split) {
  const double top = 65504.0, scale = x_scale(split);
  const double top_u = top / (scale * scale), top_b = top / b_scale(split);
  double s = 1.0, least = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const double u = s * s;
    if (!(u <= top_u)) return false;
    if (a == 0.0 && b == 0.0 && c == 0.0) return true;  // zeros from here on, exactly
    least *= fabs(a);
    if (!(least >= 0.25)) return false;
    auto q = [&](double x) { return fabs((split ? 0.0 : a) + (b + c * x) * x); };
    double most = fmax(q(0.0), q(u));
    if (c != 0.0 && -b / (2.0 * c) > 0.0 && -b / (2.0 * c) < u) most = fmax(most, q(-b / (2.0 * c)));
    if (!(most <= top_b)) return false;
    auto p = [&](double x) { return fabs(sqrt(x) * (a + (b + c * x) * x)); };
    s = p(u);
    // extrema: a + 3 b x + 5 c x^2 = 0, the roots without cancellation
    const double d = 9.0 * b * b - 20.0 * a * c;
    if (d >= 0.0) {
      const double h = -0.5 * (3.0 * b + copysign(sqrt(d), b));
      const double roots[2] = {c != 0.0 ? h / (5.0 * c) : -1.0, h != 0.0 ? a / h : -1.0};
      for (const double x : roots)
        if (x > 0.0 && x < u) s = fmax(s, p(x));
    }
    s *= 1.0 + 1.0 / 64;
  }
  return true;
}

bool too_large(int64_t batch, int64_t m, int64_t n) {
  const int64_t lim = 1 << 24;  // planes * batch and tile counts stay within 32 bits
  return batch > lim || m > lim || n > lim;
}

// Half precision sums all of G's K on the tensor core, which rounds towards zero after every 16 terms:
// the diagonal falls short by up to (K / 16) 2^-23 of itself. Up to 2^18 columns that hides behind the
// roundings to fp16; beyond (16 x 2^20 was 8e-3 off, 16 x 2^22 3e-2, 4 x 2^24 0.33) full
// precision, which drains every 64, takes over at three times the products (2^20: 4e-6).
constexpr int64_t kLongestHalf = int64_t(1) << 18;
bool works_split(bool full, int64_t m, int64_t n) {
  return full || m > kLongestHalf || n > kLongestHalf;
}
bool wants_split(int precision, int type, int64_t m, int64_t n) {
  const bool full = precision == LINALG_PRECISION_AUTO ? type != LINALG_BF16
                                                       : precision == LINALG_PRECISION_FULL;
  return works_split(full, m, n);
}

int check_workspace(int64_t batch, int64_t m, int64_t n, bool split, const void* ws, size_t bytes) {
  const size_t need = layout(batch, m, n, split).total;
  if (need == 0) return CHOL_OK;
  if (ws == nullptr || reinterpret_cast<uintptr_t>(ws) % 256) return CHOL_ERR_WORKSPACE;
  return bytes < need ? CHOL_ERR_WORKSPACE : CHOL_OK;
}

}  // namespace

namespace {
constexpr int kMaxDevices = 64;
struct {
  std::once_flag once;
  int status, sms;
} states[kMaxDevices];
}  // namespace

int prepare_device(int dev) {
  if (dev < 0 || dev >= kMaxDevices) return CHOL_ERR_DEVICE;
  std::call_once(states[dev].once, [dev]() {
    states[dev].status = chol::prepare_device_checked(dev);
    int prev = 0;
    if (states[dev].status != CHOL_OK) return;
    if (cudaGetDevice(&prev) != cudaSuccess || (prev != dev && cudaSetDevice(dev) != cudaSuccess)) {
      states[dev].status = CHOL_ERR_DEVICE;
      return;
    }
    if (cudaDeviceGetAttribute(&states[dev].sms, cudaDevAttrMultiProcessorCount, dev) !=
            cudaSuccess ||
        prepare_products() != cudaSuccess || prepare_small_ortho() != cudaSuccess ||
        prepare_few() != cudaSuccess || prepare_mid_ortho() != cudaSuccess)
      states[dev].status = CHOL_ERR_DEVICE;
    if (prev != dev) cudaSetDevice(prev);
  });
  return states[dev].status;
}

int prepare_current() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return CHOL_ERR_DEVICE;
  // A thread that has made no CUDA call yet (torch runs backward passes on threads of its own)
  // has no current context, and encoding a tensor map needs one: bind it once per thread.
  static thread_local int bound = -1;
  if (bound != dev) {
    if (cudaSetDevice(dev) != cudaSuccess) return CHOL_ERR_DEVICE;
    bound = dev;
  }
  const int st = prepare_device(dev);
  if (st == CHOL_OK) use_sm_count(states[dev].sms);
  return st;
}

}  // namespace lin

using namespace lin;

extern "C" {

int linalg_prepare(int device) { return prepare_device(device); }

size_t linalg_orthogonalize_workspace(int64_t batch, int64_t m, int64_t n, int precision) {
  if (batch <= 0 || m <= 0 || n <= 0 || too_large(batch, m, n)) return 0;
  return layout(batch, m, n, works_split(precision != LINALG_PRECISION_HALF, m, n)).total;
}

int linalg_orthogonalize(const linalg_matrix* x, const linalg_matrix* out, int64_t batch,
                         int64_t m, int64_t n, int steps, const float* coefficients, float eps,
                         int precision, void* workspace, size_t workspace_bytes, void* queue) {
  int st = check_iteration(batch, m, n, steps, coefficients, eps, precision);
  if (st != CHOL_OK) return st;
  if (batch == 0 || m == 0 || n == 0) return CHOL_OK;
  if (!valid_matrix(x, batch, m, n) || !valid_matrix(out, batch, m, n)) return CHOL_ERR_INVALID_ARG;
  if (batch > 1 && out->stride == 0) return CHOL_ERR_INVALID_ARG;
  if (too_large(batch, m, n)) return CHOL_ERR_UNSUPPORTED;
  const bool same = x->data == out->data && x->ld == out->ld && x->type == out->type &&
                    (batch == 1 || x->stride == out->stride);
  if (!same && overlap(x, out, batch, m, n)) return CHOL_ERR_INVALID_ARG;
  const bool split = wants_split(precision, out->type, m, n);
  if (!in_range(steps, coefficients, split)) return CHOL_ERR_UNSUPPORTED;
  if ((st = check_workspace(batch, m, n, split, workspace, workspace_bytes)) != CHOL_OK) return st;
  if ((st = prepare_current()) != CHOL_OK) return st;
  return iterate(x, nullptr, out, batch, m, n, 0.f, 0, 1.f, 0.f, steps, coefficients, eps, split,
                 workspace, static_cast<cudaStream_t>(queue));
}

int linalg_muon_update(const linalg_matrix* param, const linalg_matrix* grad,
                       const linalg_matrix* momentum, int64_t batch, int64_t m, int64_t n,
                       double beta, int nesterov, float decay, float rate, int steps,
                       const float* coefficients, float eps, int precision, void* workspace,
                       size_t workspace_bytes, void* queue) {
  int st = check_iteration(batch, m, n, steps, coefficients, eps, precision);
  if (st != CHOL_OK) return st;
  if (!isfinite(beta) || !isfinite(decay) || !isfinite(rate)) return CHOL_ERR_INVALID_ARG;
  if (batch == 0 || m == 0 || n == 0) return CHOL_OK;
  if (!valid_matrix(param, batch, m, n) || !valid_matrix(grad, batch, m, n) ||
      !valid_matrix(momentum, batch, m, n))
    return CHOL_ERR_INVALID_ARG;
  if (batch > 1 && (param->stride == 0 || momentum->stride == 0)) return CHOL_ERR_INVALID_ARG;
  if (too_large(batch, m, n)) return CHOL_ERR_UNSUPPORTED;
  if (overlap(param, grad, batch, m, n) || overlap(param, momentum, batch, m, n) ||
      overlap(grad, momentum, batch, m, n))
    return CHOL_ERR_INVALID_ARG;
  const bool split = wants_split(precision, param->type, m, n);
  if (!in_range(steps, coefficients, split)) return CHOL_ERR_UNSUPPORTED;
  if ((st = check_workspace(batch, m, n, split, workspace, workspace_bytes)) != CHOL_OK) return st;
  if ((st = prepare_current()) != CHOL_OK) return st;
  return iterate(grad, momentum, param, batch, m, n, beta, nesterov, decay, rate, steps,
                 coefficients, eps, split, workspace, static_cast<cudaStream_t>(queue));
}

}  // extern "C"
