/*
 * linalg_b200.h — C ABI of the orthogonalised optimiser update and the grouped matrix products
 * of the B200 (sm_100a) library. The conventions are chol_b200.h's: plain pointers, sizes and an
 * opaque queue handle (a cudaStream_t as void*, NULL = the legacy default queue) in, an integer
 * status out (CHOL_OK, CHOL_ERR_*; text from chol_strerror). All work is enqueued
 * asynchronously; nothing is allocated; no C++ exception crosses this boundary. Every call takes
 * its scratch from the caller, so calls on different queues do not interfere, and every call can
 * be captured into a CUDA graph (chol_prepare and linalg_prepare once before the capture).
 * The reference project has no counterpart to these entry points.
 */
#ifndef LINALG_B200_H
#define LINALG_B200_H

#include "chol_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define LINALG_BF16 0
#define LINALG_FP16 1
#define LINALG_FP32 2

/* Working precision of the Newton-Schulz iteration. */
#define LINALG_PRECISION_AUTO 0 /* HALF for bf16 results, FULL for fp16 and fp32 results */
#define LINALG_PRECISION_HALF 1 /* fp16 operands, FP32 accumulation: 0.5e-3 to 2.6e-3 of the result's
                                   norm on random matrices, more on those of low rank (2.4e-2 at rank
                                   64 of 1024, 0.15 at rank 1). With a side above 2^18 the work is
                                   FULL's all the same: sums that long fall short in HALF */
#define LINALG_PRECISION_FULL 2 /* operands split into two fp16 numbers (22 bits), three products
                                   per product: 1e-6 to 3.3e-6 of the result's norm, 2e-4 at rank 1,
                                   8e-5 with a side of 2^24 */

#define LINALG_MAX_STEPS 32   /* Newton-Schulz steps of one call */
#define LINALG_MAX_GROUPS 1024 /* groups of one grouped product */

/* Per-device set-up (idempotent, thread-safe; every entry point calls it for the current
   device). CHOL_ERR_DEVICE unless the device is sm_100. */
CHOL_API int linalg_prepare(int device);

/*
 * A batch of row-major matrices: element (i, r, c) at data + i * stride + r * ld + c.
 * ld >= cols; any alignment of the element type.
 */
typedef struct {
  void* data;
  int64_t ld, stride;
  int type; /* LINALG_* */
} linalg_matrix;

/* Bytes of device workspace (256-byte aligned) of linalg_orthogonalize and linalg_muon_update
   for `batch` m x n matrices at a working precision (HALF or FULL; AUTO counts as FULL). 0 where
   the iteration runs on chip (smaller side <= 128 and the other within a cluster's shared
   memory; in half precision also both sides <= 256). */
CHOL_API size_t linalg_orthogonalize_workspace(int64_t batch, int64_t m, int64_t n,
                                               int precision);

/*
 * Newton-Schulz approximation of the polar factor of each matrix of a batch:
 *   X = x / (||x||_F + eps), then `steps` times X <- a X + (b A + c A^2) X with A = X X^T
 * (from the right with A = X^T X when m > n), and out = X. coefficients: 3 * steps host floats
 * (a, b, c of each step). x and out may be the same array; partial overlap is not allowed.
 * The iterates are held in fp16, which gives the coefficients a range: with s_0 = 1 and
 * s_k+1 = 65/64 max |t (a + b t^2 + c t^4)| over t in [0, s_k], every step must keep s_k^2 <= 63.9
 * and |a + b t^2 + c t^4| <= 65504 (HALF), s_k^2 <= 15.9 and |b t^2 + c t^4| <= 31.9 (FULL), and
 * the product |a_0 ... a_k| must not fall below 1/4 (but for a step of three zeros). Coefficients
 * that may leave it for some matrix: CHOL_ERR_UNSUPPORTED, as for batch, m or n above 2^24.
 * A matrix with a NaN or an infinity yields NaN; the other matrices of the batch are not
 * affected. A zero matrix yields zeros (with eps > 0).
 */
CHOL_API int linalg_orthogonalize(const linalg_matrix* x, const linalg_matrix* out, int64_t batch,
                                  int64_t m, int64_t n, int steps, const float* coefficients,
                                  float eps, int precision, void* workspace,
                                  size_t workspace_bytes, void* queue);

/*
 * One optimiser step on a batch of weights, in place:
 *   momentum <- beta * momentum + (1 - beta) * grad
 *   u        =  nesterov ? beta * momentum + (1 - beta) * grad : momentum
 *   param    <- decay * param - rate * orthogonalize(u)
 * The three arrays must not overlap. precision AUTO goes by param's type.
 */
CHOL_API int linalg_muon_update(const linalg_matrix* param, const linalg_matrix* grad,
                                const linalg_matrix* momentum, int64_t batch, int64_t m,
                                int64_t n, double beta, int nesterov, float decay, float rate,
                                int steps, const float* coefficients, float eps, int precision,
                                void* workspace, size_t workspace_bytes, void* queue);

/*
 * Rows grouped by an index, each group times its own matrix:
 *   y[r] = x[r] W_e   for offsets[e] <= r < offsets[e + 1]
 * x: rows x k, y: rows x n (one matrix each; .stride unused). w: `groups` matrices; w_rows_k != 0:
 * k x n row-major, else n x k row-major (W_e transposed in memory). offsets: groups + 1 device
 * integers (32 bits, or 64 with offsets64), non-decreasing, within [0, rows]; values that are
 * not are clamped to the largest before them and to that range, so that no row outside the
 * arrays is touched. Rows of no group (before offsets[0], from offsets[groups] on): set to zero
 * with fill != 0, else left as they are. x, w, y share one type (bf16 or fp16); sums are FP32.
 * x and w: base 16-byte aligned, ld and stride multiples of 8 (CHOL_ERR_UNSUPPORTED otherwise);
 * y: any alignment, not overlapping the others. groups <= LINALG_MAX_GROUPS; sizes below 2^31 - 1024
 * (CHOL_ERR_UNSUPPORTED above). k = 0 or, with fill, groups = 0: CHOL_ERR_UNSUPPORTED.
 */
CHOL_API int linalg_grouped_matmul(const linalg_matrix* x, const linalg_matrix* w, int w_rows_k,
                                   const linalg_matrix* y, const void* offsets, int offsets64,
                                   int64_t groups, int64_t rows, int64_t k, int64_t n, int fill,
                                   void* queue);

/*
 * The matrix of each group's outer products, the weight gradient of linalg_grouped_matmul:
 *   dw_e = sum over offsets[e] <= r < offsets[e + 1] of a[r]^T b[r]     (k x n, row-major)
 * a: rows x k, b: rows x n, dw: `groups` matrices; zeros for a group without rows. Rows of no
 * group are not read. Types, alignment, limits and offsets as above; rows = 0: CHOL_ERR_UNSUPPORTED.
 */
CHOL_API int linalg_grouped_outer(const linalg_matrix* a, const linalg_matrix* b,
                                  const linalg_matrix* dw, const void* offsets, int offsets64,
                                  int64_t groups, int64_t rows, int64_t k, int64_t n, void* queue);

#ifdef __cplusplus
}
#endif

#endif /* LINALG_B200_H */
