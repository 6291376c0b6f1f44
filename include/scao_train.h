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

#ifdef __cplusplus
}
#endif
#endif /* SCAO_TRAIN_H */
