/*
 * scao_train.h -- C ABI of the operators that run beside the optimizer's step
 * in a training or serving program, in the same library as scao_amd.h.
 *
 * The same rules: device pointers (but for the tables called HOST), sizes and
 * a hipStream_t passed as void*; every entry point launches on the stream it
 * is given, allocates no device memory, never synchronises the host, and
 * returns SCAO_OK or an error code with a message in scao_last_error().
 */
#ifndef SCAO_TRAIN_H
#define SCAO_TRAIN_H

#include "scao_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- gradient norm and clipping -------------------------------------------
 * Over the n tensors of a HOST table (it travels in the kernels' arguments;
 * empty tensors are skipped): N = scale * (sum |g|^p)^(1/p) with norm_type p =
 * 1 or 2, or scale * max |g| with norm_type 0, summed in double in a fixed
 * order, into *norm (device fp32).  scao_grad_clip then multiplies every
 * gradient by f = fp32(scale * min(1, max_norm / (N + 1e-6))), rounding once
 * to its type; with f = 1 nothing is written.  A NaN anywhere makes N and,
 * through f, every gradient NaN; an infinity makes N infinite and f zero, or
 * scale where max_norm is infinite (which clips nothing).
 * Tensors start at any multiple of their element size and must not overlap
 * when they are clipped (SCAO_ERR_INVALID).  workspace:
 * scao_grad_norm_workspace() bytes, aligned to 8. */
typedef struct scao_tensor_desc {
  void* data;               /* numel elements of dtype, contiguous               */
  int64_t numel;
  int32_t dtype;            /* enum scao_dtype                                   */
  int32_t pad0;
} scao_tensor_desc;
int64_t scao_grad_norm_workspace(const scao_tensor_desc* tensors, int n);
int scao_grad_norm(const scao_tensor_desc* tensors, int n, int norm_type, double scale,
                   float* norm, void* workspace, void* stream);
int scao_grad_clip(const scao_tensor_desc* tensors, int n, int norm_type, double scale,
                   double max_norm, float* norm, void* workspace, void* stream);

/* ---- gated feed-forward block ---------------------------------------------
 * a = x Wg^T, b = x Wu^T, h = f(a) * b, y = h Wd^T, all row-major: x tokens x d,
 * Wg and Wu f x d, Wd d x f, y tokens x d, with unit column stride and a row
 * stride of at least a row and less than 2^21 elements (that of a single row is
 * not looked at); fp32, bf16 or fp16, one type for all.  Sums are
 * fp32.  With `saved` (scao_ffn_saved_bytes() bytes) the forward pass keeps h, a
 * and b for scao_ffn_backward: dh = dy Wd, da = dh * b * f'(a), db = dh * f(a),
 * dx = da Wg + db Wu, dWg = da^T x, dWu = db^T x, dWd = dy^T h, each written
 * densely (row strides d, d, d, f) unless its pointer is null.  A NaN or an
 * infinity in a token's row of x or dy reaches that token's y and dx (as NaN also
 * where the exact result would be infinite) and the weights' gradients, and no
 * other token.  No atomics: the same call gives the same bits.  workspace: the
 * *_workspace() bytes for the same descriptor, aligned to 16, as is `saved`. */
enum scao_activation {
  SCAO_ACT_SILU = 0,        /* a / (1 + exp(-a))                                 */
  SCAO_ACT_GELU = 1,        /* a (1 + erf(a / sqrt 2)) / 2                       */
  SCAO_ACT_GELU_TANH = 2,   /* a (1 + tanh(sqrt(2/pi) (a + 0.044715 a^3))) / 2   */
  SCAO_ACT_RELU = 3,        /* a where a > 0 or a is NaN, else 0                  */
  SCAO_ACT_SIGMOID = 4      /* 1 / (1 + exp(-a))                                 */
};
typedef struct scao_ffn_desc {   /* HOST */
  const void* x;
  const void* w_gate;
  const void* w_up;
  const void* w_down;
  int64_t ldx, ld_gate, ld_up, ld_down;   /* row strides in elements             */
  int64_t tokens, d, f;                   /* all at least 1                      */
  int32_t dtype;            /* enum scao_dtype                                   */
  int32_t act;              /* enum scao_activation                              */
} scao_ffn_desc;
int64_t scao_ffn_saved_bytes(const scao_ffn_desc* desc);
int64_t scao_ffn_forward_workspace(const scao_ffn_desc* desc, int save);
int scao_ffn_forward(const scao_ffn_desc* desc, void* y, void* saved, void* workspace,
                     void* stream);
/* grads: which of them are wanted */
#define SCAO_FFN_DX 1
#define SCAO_FFN_DGATE 2
#define SCAO_FFN_DUP 4
#define SCAO_FFN_DDOWN 8
int64_t scao_ffn_backward_workspace(const scao_ffn_desc* desc, const void* dy, int64_t ld_dy,
                                    int grads);
int scao_ffn_backward(const scao_ffn_desc* desc, const void* dy, int64_t ld_dy, const void* saved,
                      void* dx, void* dw_gate, void* dw_up, void* dw_down, void* workspace,
                      void* stream);

/* ---- orthogonalised updates --------------------------------------------------
 * Newton-Schulz products: X = G / (|G|_F + eps), then `steps` times, with the
 * step's coefficients (a, b, c) = coefficients[3k .. 3k+2] (host doubles),
 *   A = X X^T,  X <- a X + (b A + c A A) X     (rows <= cols, else on X^T)
 * which sends every singular value s of G / (|G|_F + eps) through the odd
 * polynomials a s + b s^3 + c s^5.  The matrices of a HOST table may differ in
 * shape, type and precision; all of them share the launches.  Rows have unit column
 * stride and a row stride of at least a row; src and dst may differ in type.
 *   SCAO_ORTHO_FAST  products of fp16 words with fp32 sums, X, A and B (of some
 *                    matrices of up to 512 x 1024: X and A X) rounded to 11
 *                    significant bits once a step.  The published five steps:
 *                    results 0.6e-3 to 1.4e-3 off, a bf16's own rounding 1.7e-3.
 *                    With up to 128 rows or columns as SCAO_ORTHO_FP32;
 *   SCAO_ORTHO_FP32  words of 22 bits, three products each: fp32's accuracy.
 * A matrix with a NaN or an infinity (or with a sum of squares beyond double's
 * range) gives NaN throughout, and no other matrix; one of zeros gives zeros.
 * Coefficients that may take a singular value of [0, 1] beyond 1024 are refused.
 * eps, at least 1e-300, is meant to be small beside |G|: the first X is held to
 * 2^-39 absolutely in either precision.
 * The norm is summed in double, no atomics: the same call gives the same bits.
 *
 * scao_muon_step: with the momentum m (fp32) and the gradient g
 *   m <- mu m + (1 - mu) g,  G = nesterov ? mu m + (1 - mu) g : m,
 *   p <- decay p - rate orthogonalised(G)
 * p, g and m contiguous; p and g may have different types; p is rounded once.
 *
 * Written memory, from a matrix's first element to its last with the gaps between
 * rows, may not overlap with anything else of the table (SCAO_ERR_INVALID).  workspace: the *_workspace() bytes for the same table and
 * steps, aligned to 16, contents of no meaning. */
enum scao_ortho_precision { SCAO_ORTHO_FAST = 0, SCAO_ORTHO_FP32 = 1 };
typedef struct scao_ortho_desc {   /* HOST */
  const void* src;
  void* dst;
  int64_t rows, cols;              /* below 2^20, the smaller one up to 2^15     */
  int64_t ld_src, ld_dst;          /* row strides in elements                    */
  int32_t src_dtype, dst_dtype;    /* enum scao_dtype                            */
  int32_t precision, pad0;         /* enum scao_ortho_precision                  */
} scao_ortho_desc;
int64_t scao_orthogonalize_workspace(const scao_ortho_desc* matrices, int n, int steps);
int scao_orthogonalize(const scao_ortho_desc* matrices, int n, const double* coefficients, int steps,
                       double eps, void* workspace, void* stream);
typedef struct scao_muon_desc {    /* HOST */
  void* p;
  const void* g;
  float* m;
  int64_t rows, cols;
  int32_t dtype, grad_dtype;       /* of p, of g                                 */
  float rate, decay;
  int32_t precision, pad0;
} scao_muon_desc;
int64_t scao_muon_workspace(const scao_muon_desc* matrices, int n, int steps);
int scao_muon_step(const scao_muon_desc* matrices, int n, double momentum, int nesterov,
                   const double* coefficients, int steps, double eps, void* workspace,
                   void* stream);

/* ---- norms of queries and keys with their rotation ---------------------------
 * For every token and head of q ([0]) and k ([1]), of `dim` columns x with unit
 * stride:  y = x w / sqrt(mean x^2 + eps), and of y's first `rotary` columns the
 * pairs (i, i + rotary/2), or interleaved (2i, 2i + 1), turned by the token's angles:
 *   y'_i = y_i cos[p][i] - y_j sin[p][i],  y'_j = y_j cos[p][i] + y_i sin[p][i]
 * in fp32, rounded once to dtype.  p: positions[sequence][token], or null: the
 * token's place in its sequence; a p outside of the tables gives NaN in the rotated
 * columns.  w null: ones.  backward: dx (p null: not wanted) and dw (null: not
 * wanted), summed in a fixed order without atomics; the angles have no gradient.
 * Batch, token and head strides of any tensor are free; outputs may not overlap.
 * A call takes fewer than 2^32 lanes: up to 64 for four heads of q or k of a token.
 * workspace: scao_qk_rope_backward_workspace() bytes, aligned to 16; needed for
 * the weights' gradients. */
typedef struct scao_rope_tensor {  /* HOST; strides in elements                  */
  void* p;
  int64_t batch, token, head;
} scao_rope_tensor;
typedef struct scao_rope_desc {    /* HOST */
  scao_rope_tensor x[2];
  const void* w[2];
  const float* cos;                /* table_rows x rotary/2, ld_table apart      */
  const float* sin;
  const void* positions;           /* int64 (wide_positions) or int32            */
  int64_t position_strides[2];     /* of sequence and token                      */
  int64_t batch, seq, table_rows, ld_table;
  int32_t heads[2], w_dtype[2];
  int32_t dim, rotary;             /* 1 to 512; even, up to dim                  */
  int32_t dtype, wide_positions, interleaved;
  float eps;
} scao_rope_desc;
int scao_qk_rope_forward(const scao_rope_desc* desc, const scao_rope_tensor* y, void* stream);
int64_t scao_qk_rope_backward_workspace(const scao_rope_desc* desc);
int scao_qk_rope_backward(const scao_rope_desc* desc, const scao_rope_tensor* dy,
                          const scao_rope_tensor* dx, void* dw_q, void* dw_k, void* workspace,
                          void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SCAO_TRAIN_H */
