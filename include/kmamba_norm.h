/* kmamba_norm.h -- layer norm with its residual, forward and backward
 * (libkmamba_b200.so).  No counterpart in the reference, whose blocks feed each
 * other unnormalised.
 *
 *   s = x + residual          (rounded to the tensors' type; s = x without a residual)
 *   y = (s - mean) rstd w + b,  mean and rstd = 1 / sqrt(var + eps) over the D entries of a row
 *
 * Device pointers; rows are `ld` elements apart (0 = contiguous).  Statistics and
 * every sum are fp32.  0 on success, -1 with kmb_last_error() set otherwise;
 * calls only enqueue work on `stream` (NULL = default), allocate nothing and
 * keep nothing between calls.  Results do not depend on scheduling. */
#ifndef KMB200_NORM_H
#define KMB200_NORM_H
#include <stddef.h>
#ifdef __cplusplus
extern "C" {
#endif

#ifndef KMB_DTYPE_F32
#define KMB_DTYPE_F32 0
#define KMB_DTYPE_BF16 1
#endif
#define KMB_NORM_MAX_D 16384

typedef struct {
    long rows, D;               /* rows >= 0, 1 <= D <= KMB_NORM_MAX_D */
    int dtype;                  /* of x, residual, total, y and their gradients */
    float eps;                  /* >= 0 */
    const void *x;              /* [rows, D] */
    const void *residual;       /* [rows, D] or NULL */
    void *total;                /* [rows, D]: s, when there is a residual (NULL: not kept); may be x or residual */
    void *y;                    /* [rows, D]; may be x or residual */
    const float *w, *b;         /* [D], NULL = ones / zeros */
    float *mean, *rstd;         /* [rows], both or neither; the backward needs them */
    long ld_x, ld_residual, ld_total, ld_y;
} KMBNormParams;

typedef struct {
    const void *dy;             /* [rows, D] */
    const void *dtotal;         /* [rows, D] or NULL: gradient that reaches s past the norm; added to dx */
    void *dx;                   /* [rows, D]: gradient of s, hence of x and of the residual; may be dy or dtotal */
    float *dw, *db;             /* [D] or NULL */
    long ld_dy, ld_dtotal, ld_dx;
    int accumulate;             /* 1: dw, db += (dx is always assigned) */
} KMBNormGrads;

int kmb_layernorm_forward(const KMBNormParams *p, void *stream);
/* Floats of the workspace that the backward of this shape takes (0 when it needs none). */
size_t kmb_layernorm_workspace_floats(const KMBNormParams *p);
/* Reads s (total, or x where there is no residual), mean and rstd as the forward
 * left them; y, residual and b are not read.  ws: see above, NULL allowed when
 * neither dw nor db is wanted; its contents need not survive between calls. */
int kmb_layernorm_backward(const KMBNormParams *p, const KMBNormGrads *g, float *ws, void *stream);

#ifdef __cplusplus
}
#endif
#endif
