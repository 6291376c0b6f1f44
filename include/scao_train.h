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
 * through f, every gradient NaN; an infinity makes N infinite and f zero.
 * Tensors start at any multiple of their element size and must not overlap
 * when they are clipped (SCAO_ERR_INVALID).  workspace:
 * scao_grad_norm_workspace() bytes. */
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

#ifdef __cplusplus
}
#endif
#endif /* SCAO_TRAIN_H */
