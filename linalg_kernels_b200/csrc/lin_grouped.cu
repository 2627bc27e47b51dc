// lin_grouped.cu — C-ABI entry points of the products grouped by offsets (lin_gemm.cu).
#include "lin_few.cuh"

namespace lin {
namespace {

bool half_type(int t) { return t == LINALG_BF16 || t == LINALG_FP16; }

bool sizes_ok(int64_t groups, int64_t rows, int64_t k, int64_t n) {
  return groups >= 0 && rows >= 0 && k >= 0 && n >= 0;
}
bool too_large(int64_t groups, int64_t rows, int64_t k, int64_t n) {
  const int64_t lim = 0x7fffffffLL - 1024;
  return groups > LINALG_MAX_GROUPS || rows > lim || k > lim || n > lim;
}
bool aligned16(const linalg_matrix* x, int64_t count) {
  return reinterpret_cast<uintptr_t>(x->data) % 16 == 0 && x->ld % 8 == 0 &&
         (count <= 1 || x->stride % 8 == 0);
}

}  // namespace
}  // namespace lin

using namespace lin;

extern "C" {

int linalg_grouped_matmul(const linalg_matrix* x, const linalg_matrix* w, int w_rows_k,
                          const linalg_matrix* y, const void* offsets, int offsets64,
                          int64_t groups, int64_t rows, int64_t k, int64_t n, int fill,
                          void* queue) {
  if (!sizes_ok(groups, rows, k, n)) return CHOL_ERR_INVALID_ARG;
  if (rows == 0 || n == 0) return CHOL_OK;
  if (groups == 0 && !fill) return CHOL_OK;
  if (k == 0 || groups == 0) return CHOL_ERR_UNSUPPORTED;
  if (x == nullptr || w == nullptr || y == nullptr || offsets == nullptr ||
      x->data == nullptr || w->data == nullptr || y->data == nullptr)
    return CHOL_ERR_INVALID_ARG;
  if (!half_type(x->type) || w->type != x->type || y->type != x->type) return CHOL_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(offsets) % (offsets64 ? 8 : 4)) return CHOL_ERR_INVALID_ARG;
  const int64_t wr = w_rows_k ? k : n, wc = w_rows_k ? n : k;
  if (x->ld < k || w->ld < wc || y->ld < n || (groups > 1 && w->stride < 1))
    return CHOL_ERR_INVALID_ARG;
  if (too_large(groups, rows, k, n)) return CHOL_ERR_UNSUPPORTED;
  if (!aligned16(x, 1) || !aligned16(w, groups)) return CHOL_ERR_UNSUPPORTED;
  const int st = prepare_current();
  if (st != CHOL_OK) return st;
  Product p;
  p.a = Operand{x->data, rows, k, x->ld, 1, 0, false};
  p.b = Operand{w->data, wr, wc, w->ld, groups, w->stride, w_rows_k != 0};
  p.mode = kRaggedM;
  p.epilogue = kStore16;
  p.bf16 = x->type == LINALG_BF16;
  p.m = rows, p.n = n, p.k = k, p.batch = groups;
  p.out = y->data, p.ldo = y->ld, p.out_stride = 0, p.out_type = y->type;
  p.offsets = offsets, p.offsets64 = offsets64 != 0;
  p.total_rows = rows, p.fill = fill != 0;
  if (few_better(p)) return launch_few(p, static_cast<cudaStream_t>(queue));
  return launch_product(p, static_cast<cudaStream_t>(queue));
}

int linalg_grouped_outer(const linalg_matrix* a, const linalg_matrix* b, const linalg_matrix* dw,
                         const void* offsets, int offsets64, int64_t groups, int64_t rows,
                         int64_t k, int64_t n, void* queue) {
  if (!sizes_ok(groups, rows, k, n)) return CHOL_ERR_INVALID_ARG;
  if (groups == 0 || k == 0 || n == 0) return CHOL_OK;
  if (rows == 0) return CHOL_ERR_UNSUPPORTED;
  if (a == nullptr || b == nullptr || dw == nullptr || offsets == nullptr ||
      a->data == nullptr || b->data == nullptr || dw->data == nullptr)
    return CHOL_ERR_INVALID_ARG;
  if (!half_type(a->type) || b->type != a->type || dw->type != a->type) return CHOL_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(offsets) % (offsets64 ? 8 : 4)) return CHOL_ERR_INVALID_ARG;
  if (a->ld < k || b->ld < n || dw->ld < n) return CHOL_ERR_INVALID_ARG;
  if (groups > 1 && dw->stride < (k - 1) * dw->ld + n) return CHOL_ERR_INVALID_ARG;
  if (too_large(groups, rows, k, n)) return CHOL_ERR_UNSUPPORTED;
  if (!aligned16(a, 1) || !aligned16(b, 1)) return CHOL_ERR_UNSUPPORTED;
  const int st = prepare_current();
  if (st != CHOL_OK) return st;
  Product p;
  p.a = Operand{a->data, rows, k, a->ld, 1, 0, true};
  p.b = Operand{b->data, rows, n, b->ld, 1, 0, true};
  p.mode = kRaggedK;
  p.epilogue = kStore16;
  p.bf16 = a->type == LINALG_BF16;
  p.m = k, p.n = n, p.k = rows, p.batch = groups;
  p.out = dw->data, p.ldo = dw->ld, p.out_stride = dw->stride, p.out_type = dw->type;
  p.offsets = offsets, p.offsets64 = offsets64 != 0;
  p.total_rows = rows;
  return launch_product(p, static_cast<cudaStream_t>(queue));
}

}  // extern "C"
