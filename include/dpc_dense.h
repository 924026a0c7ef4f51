/* dpc_dense.h -- C ABI of the dense-layer operators (gfx950): the product of a layer with both sides held in 8 bits and a
 * scale for each block of 128, and the update of its weights by Newton-Schulz orthogonalisation (csrc/dense/libdpc_dense.so).
 * They serve the networks around the projector; the reference leaves both to stock TensorFlow (dpc/nets/pc_decoder.py:5-42,
 * dpc/nets/img_encoder.py:11-50, dpc/run/train.py:86-117).
 *
 * Conventions: as in dpc_hip.h -- device pointers, every call only ENQUEUES work on `stream`, no allocation, no
 * synchronisation, no global state; 0 = ok, <0 = invalid argument (DPC_DENSE_E_*), >0 = hipError_t.  The caller makes the
 * device that owns the pointers current.  Workspaces need no initial content and hold nothing between calls; two calls that
 * may run at the same time need two.
 */
#ifndef DPC_DENSE_H
#define DPC_DENSE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* dpc_dense_stream_t; /* hipStream_t */

#define DPC_DENSE_OK 0
#define DPC_DENSE_E_NULL (-1)      /* required pointer is null                         */
#define DPC_DENSE_E_SHAPE (-2)     /* negative or unsupported sizes                    */
#define DPC_DENSE_E_TYPE (-3)      /* unknown element type                             */
#define DPC_DENSE_E_WORKSPACE (-4) /* workspace too small or not 256-byte aligned      */
#define DPC_DENSE_E_VALUE (-5)     /* coefficients or steps outside what can be held   */

#define DPC_DENSE_F32 0
#define DPC_DENSE_BF16 1
#define DPC_DENSE_F16 2

#define DPC_DENSE_BLOCK 128       /* values that share a scale                         */
#define DPC_DENSE_MAX_MATRICES 40 /* of one dpc_dense_orthogonal call                  */
#define DPC_DENSE_MAX_STEPS 64

const char* dpc_dense_version(void);
size_t dpc_dense_abi_struct_bytes(int which); /* 0: DpcDenseMatrix, 1: DpcDenseSteps */

/* The 8-bit form of a matrix src [rows, cols] (element (r, c) at src + r * ld + c), along its columns and / or its rows:
 *   q  [rows, 128 * ceil(cols / 128)] e4m3, s  [ceil(cols / 128), rows]: blocks of 128 neighbours in a row share a scale
 *   qt [cols, 128 * ceil(rows / 128)] e4m3, st [ceil(rows / 128), cols]: the same of the transposed matrix
 * A value stands for q * 2^(s - 127); s is the smallest exponent (within 1 .. 254) for which the block's largest finite
 * magnitude is at most 448 * 2^(s - 127); values round to nearest even; what is not finite becomes NaN; the ends of the last
 * blocks are zeros.  q and s, or qt and st, may be null (not both pairs).  colsum (nullable, with qt only): float
 * [ceil(rows / 128), cols], the sums over each 128 rows, for dpc_dense_colsum. */
int dpc_dense_quantize(dpc_dense_stream_t stream, int rows, int cols, int dtype, const void* src, size_t ld, void* q, uint8_t* s,
                       void* qt, uint8_t* st, float* colsum);
/* out[c] (of type dtype) = sum over parts of colsum[part, c], in order */
int dpc_dense_colsum(dpc_dense_stream_t stream, int parts, int cols, const float* colsum, int dtype, void* out);

/* out [M, N] (row-major, of type dtype) = A B^T (+ bias [N], of type bias_dtype, nullable): A = (qa [M, 128 * blocks],
 * sa [blocks, M]), B = (qb [N, 128 * blocks], sb [blocks, N]) in the form that dpc_dense_quantize makes (q 16-byte aligned).  The
 * sums are held in 32 bits.  workspace: dpc_dense_product_workspace bytes (may be 0), 256-byte aligned. */
size_t dpc_dense_product_workspace(int M, int N, int blocks, int dtype);
int dpc_dense_product(dpc_dense_stream_t stream, int M, int N, int blocks, const void* qa, const uint8_t* sa, const void* qb,
                      const uint8_t* sb, const void* bias, int bias_dtype, void* out, int dtype, void* workspace,
                      size_t workspace_bytes);

/* A layer's passes in one call each: out [M, N] = Q(x) Q(w)^T (+ bias) of x [M, K], w [N, K], and its gradients, those of the held values'
 * product with dy held in 8 bits along the axis that each sums over: dx = Q(dy) Q(w^T)^T (of x_type), dw = Q(dy^T) Q(x^T)^T (of w_type),
 * db = the sums of dy's columns (of bias_type).  needs: 1 dx, 2 dw, 4 db, the same in all three calls (in the backward call: which of
 * dx, dw, db are not null).  sizes[3]: bytes of `saved` (what the forward call leaves for the backward one), of the forward and of the
 * backward workspace; all 256-byte aligned.  M, K, N: at most 128 * 65535. */
int dpc_dense_linear_sizes(int M, int K, int N, int x_type, int w_type, int needs, size_t* sizes);
int dpc_dense_linear_forward(dpc_dense_stream_t stream, int M, int K, int N, const void* x, size_t x_ld, int x_type, const void* w, size_t w_ld,
                             int w_type, const void* bias, int bias_type, void* out, int needs, void* saved, size_t saved_bytes,
                             void* workspace, size_t workspace_bytes);
int dpc_dense_linear_backward(dpc_dense_stream_t stream, int M, int K, int N, const void* dy, size_t dy_ld, int x_type, int w_type, int bias_type,
                              const void* saved, size_t saved_bytes, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes);
/* The same with a weight that was put into 8 bits before (q, s of dpc_dense_quantize).  Up to 16 rows take one launch that reads the weight
 * once. */
size_t dpc_dense_linear_serve_workspace(int M, int K, int N, int x_type);
int dpc_dense_linear_serve(dpc_dense_stream_t stream, int M, int K, int N, const void* x, size_t x_ld, int x_type, const void* q, const uint8_t* s,
                           const void* bias, int bias_type, void* out, void* workspace, size_t workspace_bytes);

/* One matrix of dpc_dense_orthogonal, row-major, [rows, cols], no gaps between rows. */
typedef struct DpcDenseMatrix {
  const void* grad; /* [rows, cols] of the call's dtype                                                   */
  float* momentum;  /* [rows, cols], read and written; null: the gradient itself is orthogonalised        */
  void* out;        /* momentum null: receives the result; else the weights, read and written             */
  int32_t rows, cols;
  float scale; /* weights <- (1 - lr * weight_decay) * weights - lr * scale * result                      */
  int32_t reserved;
} DpcDenseMatrix;

typedef struct DpcDenseSteps {
  int32_t steps;                           /* 1 .. DPC_DENSE_MAX_STEPS                                                        */
  int32_t nesterov;                        /* with momentum: orthogonalise (1 - mu) g + mu m instead of m                     */
  double momentum;                         /* mu: m <- mu m + (1 - mu) g                                                      */
  double lr, weight_decay;                 /* with momentum                                                                   */
  double eps;                              /* > 0, added to the Frobenius norm                                                */
  const float* lr_device;                  /* nullable: the learning rate is read from here when the work runs, not from lr   */
  float coefficients[DPC_DENSE_MAX_STEPS][3]; /* a, b, c of each step: X <- (a I + b X X^T + c (X X^T)^2) X                   */
} DpcDenseSteps;

/* X0 = U / (|U| + eps) (U the gradient, or what the momentum makes of it), then the steps' products, for all matrices at once.
 * dtype: of gradients and of out.  Coefficients for which a step's values could leave what 16 bits hold are refused
 * (DPC_DENSE_E_VALUE): the largest |x| that the scalar iteration reaches from [0, 1] must stay below 3.5. */
size_t dpc_dense_orthogonal_workspace(int count, const DpcDenseMatrix* matrices, int dtype);
int dpc_dense_orthogonal(dpc_dense_stream_t stream, int count, const DpcDenseMatrix* matrices, int dtype, const DpcDenseSteps* steps,
                         void* workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif
