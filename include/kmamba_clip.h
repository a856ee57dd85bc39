/* kmamba_clip.h -- global norm of many gradient tensors, and clipping by it
 * (libkmamba_b200.so).  MBOptimConfig.clip_norm is not read by the AdamW step,
 * as in the reference; a training loop calls one of these between the backward
 * and the step.
 *
 *   norm = sqrt(sum over all tensors of g^2);  coefficient = max_norm / norm where
 *   norm is finite and above max_norm, else 1;  out = coefficient g
 *
 * The sum is kept in 64 bits, so it neither overflows nor underflows where an
 * fp32 square would, and is added in a fixed order.  A norm that is not finite
 * leaves the gradients as they are (the caller sees it in result[0]). */
#ifndef KMB200_CLIP_H
#define KMB200_CLIP_H
#include <stddef.h>
#include "kmamba.h"
#ifdef __cplusplus
extern "C" {
#endif

#ifndef KMB_DTYPE_F32
#define KMB_DTYPE_F32 0
#define KMB_DTYPE_BF16 1
#endif

typedef struct {
    const void *in;      /* device, n elements; aligned to its element */
    void *out;           /* device, n elements: in itself, a buffer that does not overlap any `in`, or NULL
                            (the tensor counts in the norm and is not scaled) */
    long long n;         /* >= 0 */
    int dtype;           /* of in and out */
} KMBGradTensor;

/* Floats of the workspace that a list of n_tensors takes. */
size_t kmb_grad_clip_workspace_floats(long n_tensors);
/* The list is host memory and is read before the call returns.  max_norm > 0;
 * INFINITY only measures (and copies where out is another buffer).  result[0] =
 * norm, result[1] = coefficient (device floats).  ws must be 8-byte aligned.
 * Enqueued on `stream`; allocates nothing. */
int kmb_grad_clip(const KMBGradTensor *tensors, long n_tensors, float max_norm, float *result, float *ws,
                  void *stream);
/* The model's gradient arena in place, between kmb_model_forward_backward and
 * kmb_model_optimizer_step.  max_norm <= 0 takes MBOptimConfig.clip_norm of
 * kmamba_enable_training; NaN is refused. */
int kmb_model_clip_gradients(KMamba *m, float max_norm, float *result, float *ws, void *stream);

#ifdef __cplusplus
}
#endif
#endif
