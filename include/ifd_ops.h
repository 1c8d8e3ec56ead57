/* ifd operators of attention layers — C ABI beside include/ifd.h (sampling) and include/ifd_train.h (the UNet's
 * training step): attention with its log-sum-exp and a backward pass that recomputes the probabilities, the per-head
 * norm of queries and keys with the position rotation in the same pass, and AdamW over many tensors with 8-bit or
 * 32-bit states.
 *
 * Every tensor argument is a DEVICE pointer, every launch is asynchronous on `stream`, no call allocates, synchronises
 * or keeps anything: workspaces are the caller's (sizes from the *_ws_bytes queries) and may be reused once the work
 * enqueued before has finished on that stream. Reductions run in a fixed order (the same inputs give the same bits).
 * Status 0 = ok, else ifd_last_error() names the entry point and the reason (as in include/ifd.h).
 */
#ifndef IFD_OPS_H
#define IFD_OPS_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define IFD_F32 0
#define IFD_BF16 1
#define IFD_F16 2

/* Attention. q, out, dout, dq are [B][Tq][Hq][D], k, v, dk, dv [B][Tk][Hk][D] of one type; each has its own strides
 * {batch, token, head} in elements, the channel stride is 1. Hq is a multiple of Hk: query head h reads key-value head
 * h / (Hq / Hk). lse is fp32 [B][Hq][Tq], contiguous.
 * Row i of sequence b sees key j when j < kv_len[b] (NULL: Tk; values are clamped to [0, Tk]) and, with causal != 0,
 * j <= q_start[b] + i (NULL: q_start = Tk - Tq). A row that sees no key gets out 0, lse -inf and no gradient. Keys at
 * and past kv_len are not read; their dk, dv are written as zeros.
 * D <= 128 and a multiple of 8 (16-bit types) or 4 (fp32); pointers and strides in multiples of 16 bytes; scale > 0.
 * Scores, softmax statistics and every sum are fp32. The 16-bit types round P (and dS) once to the tensors' type as
 * operands of the second matrix products. */
typedef struct ifd_attention_args {
  int dtype, B, Tq, Tk, Hq, Hk, D, causal;
  float scale;
  int pad;
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t *kv_len, *q_start; /* [B] or NULL */
  int64_t q_s[3], k_s[3], v_s[3], out_s[3];
  /* backward only */
  const void* dout;
  void *dq, *dk, *dv;
  int64_t dout_s[3], dq_s[3], dk_s[3], dv_s[3];
} ifd_attention_args;

/* out and lse. Few query rows against many keys are split over the keys and joined (workspace). */
int64_t ifd_op_attention_ws_bytes(const ifd_attention_args* a);
int ifd_op_attention(const ifd_attention_args* a, void* ws, int64_t ws_bytes, void* stream);
/* dq, dk, dv from dout, q, k, v and the forward's out and lse (scratch linear in the tensors, no score matrix is kept). */
int64_t ifd_op_attention_bwd_ws_bytes(const ifd_attention_args* a);
int ifd_op_attention_bwd(const ifd_attention_args* a, void* ws, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
