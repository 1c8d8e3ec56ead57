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
 * j <= q_start[b] + i (NULL: q_start = Tk - Tq). A row that sees no key gets out 0, lse -inf and no gradient, whatever q
 * and dout hold there. Keys that no row of their sequence sees (at and past kv_len, or behind the last row's) are not
 * read; their dk, dv are written as zeros. A key that some rows see must be finite in v (backward: in k too), and in the
 * backward a row that sees some keys in q, out and dout: what is not finite there may spoil pairs that the mask leaves out
 * (0 times it is added), besides those that it is in.
 * D <= 128 and a multiple of 8 (16-bit types) or 4 (fp32); pointers and strides in multiples of 16 bytes; scale > 0.
 * Scores, softmax statistics and every sum are fp32. The 16-bit types round P (and dS) once to the tensors' type as
 * operands of the second matrix products (fp16: gradients much smaller than 1 need a loss scale, dS ends at 2^-24).
 * |scale q.k| up to 1e8: beyond 4e8 the exponent's fp32 reference point is too coarse and results are not finite. The
 * backward's probabilities are relatively off by up to |lse| 2^-22, the rounding of lse among it. */
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

/* Per-head RMS norm of queries and keys and the rotation by their positions, in one pass.
 *   n = x / sqrt(mean x^2 + eps) * w (norm != 0; w NULL: 1), else n = x
 *   the first `rot` channels in pairs (i, i + rot / 2), or (2i, 2i + 1) with interleaved != 0, turned by the angle
 *   2 pi pos turns[i] and scaled by mscale; the other channels are n.
 * q, k, their outputs and gradients: [B][T][Hq | Hk][D] of one type, strides {batch, token, head} in elements, channels
 * adjacent (on a multiple of an element; 16 bytes is fastest). Hq or Hk may be 0. An output may be its input (in place).
 * pos int64 with strides {batch, token} (0: shared); turns fp64 [rot / 2]: frequency / 2 pi. D <= 128, even. */
typedef struct ifd_qk_args {
  int dtype, B, T, Hq, Hk, D, rot, interleaved, norm;
  float eps, mscale;
  int pad;
  const void *q, *k;
  void *q_out, *k_out;
  const float *wq, *wk;
  const int64_t* pos;
  const double* turns;
  int64_t q_s[3], k_s[3], q_out_s[3], k_out_s[3], pos_s[2];
  /* backward only: gq, gk the gradients of the outputs; dq, dk, and dwq, dwk [D] fp32 (NULL: not wanted) are written */
  const void *gq, *gk;
  void *dq, *dk;
  float *dwq, *dwk;
  int64_t gq_s[3], gk_s[3], dq_s[3], dk_s[3];
} ifd_qk_args;
int ifd_op_qk_norm_rope(const ifd_qk_args* a, void* stream);
int64_t ifd_op_qk_norm_rope_bwd_ws_bytes(const ifd_qk_args* a);
int ifd_op_qk_norm_rope_bwd(const ifd_qk_args* a, void* ws, int64_t ws_bytes, void* stream);

/* The global norm of many gradients and its clip coefficient: norm_coef (device) = {norm, min(1, max_norm / (norm +
 * 1e-6))}, summed in fp64. g, n, gtype: HOST arrays of nt entries (addresses on the device, element counts, IFD_F32 ...);
 * a NULL gradient is skipped. */
int64_t ifd_op_grad_norm_ws_bytes(int nt, const int64_t* n);
int ifd_op_grad_norm(int nt, const void* const* g, const int64_t* n, const uint8_t* gtype, double max_norm,
                     double* norm_coef, void* ws, int64_t ws_bytes, void* stream);

/* One AdamW step over nt tensors (p, g, n, ptype, gtype: HOST arrays; a tensor with a NULL gradient is left alone).
 * Tensor i's states are blocks of 256 values, ceil(n[i] / 256) of them, after those of the tensors before it, from block
 * block0 on; what lies behind a tensor's end in its last block is 0.
 *   bits 32: m, v fp32 [blocks][256];  bits 8: m, v bytes [blocks][256] and m_scale, v_scale fp32 [blocks]
 *   (m: sign, 4 exponent, 3 fraction bits; v: 5 exponent, 3 fraction bits; largest value 1.875 scale; rounded up or down
 *   at random, from seed and step).
 * norm_coef (device, from ifd_op_grad_norm) or NULL: the gradients are scaled by norm_coef[1]; a norm that is not finite
 * leaves everything as it was. Without it a gradient that is not finite spoils its parameter and state, with 8-bit states
 * the states of the 256 values that share its scale (which is NaN or infinite from then on), and with the next step their
 * parameters. */
typedef struct ifd_adamw_args {
  int nt, bits, step;
  uint32_t seed;
  void* const* p;
  const void* const* g;
  const int64_t* n;
  const uint8_t *ptype, *gtype;
  void *m, *v;
  float *m_scale, *v_scale;
  int64_t block0;
  double lr, b1, b2, eps, wd;
  const double* norm_coef;
} ifd_adamw_args;
int ifd_op_adamw(const ifd_adamw_args* a, void* stream);
/* The fp32 values that 8-bit states stand for. */
int ifd_op_state_values(const void* m, const float* m_scale, const void* v, const float* v_scale, int64_t nblocks,
                        float* m_out, float* v_out, void* stream);

#ifdef __cplusplus
}
#endif
#endif
