/* kmamba_delta.h -- the gated delta rule (libkmamba_b200.so): a recurrent mixer
 * with a matrix state per head, next to the scans.  No counterpart in the
 * reference.
 *
 * Per sequence and value head, S [dk, dv] in fp32:
 *   S' = exp(g_t) S_{t-1};   u_t = beta_t (v_t - S'^T k_t);   S_t = S' + k_t u_t^T
 *   o_t = scale S_t^T q_t
 * Layouts: q, k [batch, T, Hk, dk]; v, o [batch, T, Hv, dv]; g, beta [batch, T, Hv]
 * fp32; states [sequences, Hv, dk, dv] fp32.  Value head h reads key head
 * h / (Hv / Hk).  Tokens are `ld` elements apart (0 = contiguous), so q, k and v
 * may be slices of one projection's output; batch rows follow each other.
 *
 * Packed sequences: batch = 1, cu_seqlens (device, n_seq + 1 ints, from 0 to T,
 * not decreasing) gives the first token of each; empty sequences are allowed.
 * Offsets outside [0, T] are clamped to it and tokens that no sequence holds are
 * neither read nor written.
 *
 * Accuracy: bf16 inputs are exact, every product is good to 2^-22 and every sum
 * fp32; bf16 results are rounded once, and o has the same bits with keep = 0 and 1.
 * Factors are scaled by blocks of 16 tokens (or a quarter of dk) times 16 columns of
 * dv, keys and queries by rows: an entry below 2^-40 of its block's largest counts
 * as zero, and an infinity makes its block NaN.  A NaN at a token reaches the tokens
 * of its block of 16 before it as well as all behind; one in do reaches the tokens of
 * its block behind it as well as all before.  dg is a running sum over a chunk of 64
 * tokens: its error is relative to the chunk's largest, and a NaN in do makes the
 * chunk's dg NaN.  Scale keys so that beta |k|^2 <= 2 and g <= 0, as the rule itself
 * needs to stay bounded.
 *
 * Calls only enqueue work on `stream` (NULL = default), allocate nothing (but for
 * the device status word in a host thread's first call), keep nothing between
 * calls, and give the same bits every time.  0 on success, -1 with
 * kmb_last_error() set otherwise; a bounded wait that runs out is recorded in the
 * device status word (kmb_device_status). */
#ifndef KMB200_DELTA_H
#define KMB200_DELTA_H
#include <stddef.h>
#ifdef __cplusplus
extern "C" {
#endif

#ifndef KMB_DTYPE_F32
#define KMB_DTYPE_F32 0
#define KMB_DTYPE_BF16 1
#endif
#define KMB_DELTA_MAX_DIM 128

typedef struct {
    long batch, T;              /* >= 0 */
    long Hk, Hv;                /* Hv a multiple of Hk */
    long dk, dv;                /* 1 .. KMB_DELTA_MAX_DIM */
    int dtype;                  /* of q, k, v, o and their gradients */
    float scale;
    const int *cu_seqlens;      /* device [n_seq + 1], or NULL */
    long n_seq;                 /* with cu_seqlens */
    const void *q, *k, *v;
    const float *g;             /* log decay, NULL = 0; -INFINITY forgets the state; at a sequence's first token, and at
                                   any token of kmb_delta_step, also a state that holds infinities or NaN */
    const float *beta;          /* NULL = 1 */
    void *o;
    const float *h0;            /* initial states, NULL = 0 */
    float *hT;                  /* final states, or NULL; may be h0 */
    long ld_q, ld_k, ld_v, ld_o;
} KMBDeltaParams;

typedef struct {
    const void *do_;            /* [batch, T, Hv, dv] */
    const float *dhT;           /* gradient of the final states, or NULL */
    void *dq, *dk, *dv;         /* assigned; key heads receive the sum over their value heads */
    float *dg, *dbeta;          /* [batch, T, Hv] or NULL */
    float *dh0;                 /* or NULL */
    long ld_do, ld_dq, ld_dk, ld_dv;
} KMBDeltaGrads;

/* Floats of the workspace (16-byte aligned) of these sizes; train = 1 for a
 * forward whose backward follows. */
size_t kmb_delta_workspace_floats(const KMBDeltaParams *p, int train);
/* Chunked form.  keep = 1 leaves in ws what kmb_delta_backward reads. */
int kmb_delta_forward(const KMBDeltaParams *p, float *ws, int keep, void *stream);
/* Exact gradient of that forward: p as it was there, ws as it left it
 * (p->o and p->hT are not read). */
int kmb_delta_backward(const KMBDeltaParams *p, const KMBDeltaGrads *g, float *ws, void *stream);
/* Recurrent form, for serving: T new tokens (1 or a few) per batch row; the
 * states of the rows are entries of a pool, updated in place.  slots: device
 * [batch], the pool entry of each row (no entry twice), or NULL for row b at
 * entry b; a row whose slot is outside [0, n_slots) is idle: its o is zero.
 * p->h0, p->hT and p->cu_seqlens must be NULL. */
int kmb_delta_step(const KMBDeltaParams *p, float *pool, long n_slots, const int *slots, void *stream);

#ifdef __cplusplus
}
#endif
#endif
