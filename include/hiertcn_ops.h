/*
 * hiertcn_ops.h -- C-ABI of the sequence operators that stand beside the model handles of hiertcn.h: the gated linear recurrence, the
 * preference and policy losses on materialised logits with their gradients, and the AdamW step.  Exported by the same library.
 *
 * Conventions (those of hiertcn.h, and what follows from having no handle)
 *   - plain C, no exceptions, no torch types.  Pointers are DEVICE pointers owned by the caller unless the text says "host"; nothing is allocated
 *     or synchronised; all work is enqueued on `stream` (a hipStream_t), which must belong to the CURRENT device, as must the pointers.
 *   - every call may be captured into a graph unless it says otherwise (no memset nodes are recorded); calls share no state, so any number may run at
 *     once as long as each has its own workspace and outputs.
 *   - returns 0 on success, otherwise a negative hiertcn_status (hiertcn.h); hiertcn_ops_last_error() holds this thread's message.
 *   - sizes are int64_t: tensors of more than 2^32 elements are fine.  Element strides are given where a tensor need not be contiguous.
 *   - results do not depend on timing: every sum has a fixed order.  (The one atomic, in long recurrences, numbers workgroups as they start.)
 */
#ifndef HIERTCN_OPS_H_
#define HIERTCN_OPS_H_

#include "hiertcn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HIERTCN_OPS_VERSION 1
int hiertcn_ops_version(void);
const char* hiertcn_ops_last_error(void);
/* sizeof() of this header's structs as the library was compiled: hiertcn_glr_t, hiertcn_rows_t, hiertcn_preference_t, hiertcn_policy_t,
 * hiertcn_adamw_tensor_t, hiertcn_adamw_t */
#define HIERTCN_OPS_N_STRUCTS 6
int hiertcn_ops_struct_sizes(size_t out[HIERTCN_OPS_N_STRUCTS]);

enum hiertcn_dtype { HIERTCN_FP32 = 0, HIERTCN_BF16 = 1, HIERTCN_FP16 = 2 };

/* ---- gated linear recurrence ---------------------------------------------------------------------------------------------------------------
 * The update of a GRU cell (customed_gru_cell.py:309-337: new_h = u h + (1 - u) c) with gate and candidate that do not read the state, so that the
 * recurrence over a sequence is a scan:
 *   u = sigmoid(gate[b][t][d]);  c = cand or tanh(cand);  h_t = u * (mask[b][t] != 0 ? h_{t-1} : 0) + (1 - u) c        for t < lengths[b]
 * mask: the user-boundary reset of model_hier.py:93 (0 cuts the state whatever it holds, NaN included; anything else keeps it).  lengths: dynamic_rnn's
 * sequence_length (model_gru.py:47-53): behind it the output is 0 and the state is carried; gate, cand and dout are not read there.  Values below 0
 * and above T count as 0 and T.  States are fp32; out is rounded once to dtype.
 *   record   needed by the backward pass: the state before every 16th step (hiertcn_glr_record_floats floats), written by the forward pass when non-NULL
 *   backward lambda_t = dout_t + a_{t+1} lambda_{t+1} with a = u [mask != 0] and dstate_out entering behind the last step;
 *            dcand = lambda (1 - u) act'(cand), dgate = lambda (h_prev - c) u (1 - u), dstate_in = a_0 lambda_0; rows behind lengths[b] get 0
 * state_out may be state_in itself.  Other outputs overlap neither each other nor inputs (refused where it can be seen from pointers and strides).
 * B, T, D >= 0 (an empty call copies the state), B * ceil(D / 64) at most 2^26 - 1.  workspace: hiertcn_glr_workspace_bytes, 16-byte aligned; 0 where the shape needs none.  (Its workgroups wait for
 * one another through it.  A wait that cannot end -- two calls at once in one workspace -- gives up after some seconds, and what could not be learnt is NaN.) */
typedef struct {
  int64_t B, T, D;
  int32_t dtype;                       /* hiertcn_dtype of gate, cand, out, dout, dgate, dcand                                        */
  int32_t cand_act;                    /* 0: c = cand; 1: c = tanh(cand)                                                              */
  const void* gate; int64_t gate_sb, gate_st;     /* element strides of b and t; the last dimension is contiguous                     */
  const void* cand; int64_t cand_sb, cand_st;
  const float* mask; int64_t mask_sb, mask_st;    /* NULL: no resets                                                                  */
  const int32_t* lengths;              /* [B] or NULL: all T                                                                          */
  const float* state_in;               /* [B][D] or NULL: zeros (forward)                                                             */
  float* state_out;                    /* [B][D] or NULL: not wanted (forward)                                                        */
  float* record;                       /* forward: written when non-NULL; backward: read                                              */
  void* out; int64_t out_sb, out_st;   /* forward                                                                                     */
  const void* dout; int64_t dout_sb, dout_st;     /* backward                                                                         */
  const float* dstate_out;             /* [B][D] or NULL: zeros (backward)                                                            */
  void* dgate; int64_t dgate_sb, dgate_st;        /* backward                                                                         */
  void* dcand; int64_t dcand_sb, dcand_st;        /* backward                                                                         */
  float* dstate_in;                    /* [B][D] or NULL: not wanted (backward)                                                       */
  void* workspace; size_t workspace_bytes;
} hiertcn_glr_t;
size_t hiertcn_glr_record_floats(int64_t B, int64_t T, int64_t D);
size_t hiertcn_glr_workspace_bytes(int64_t B, int64_t T, int64_t D);
int hiertcn_glr_forward(const hiertcn_glr_t* a, void* stream);
int hiertcn_glr_backward(const hiertcn_glr_t* a, void* stream);

/* ---- losses on the log-probabilities of answers, with their gradients ----------------------------------------------------------------------
 * logits [n * T][V] of n sequences (row stride ld >= V elements), ids [n * T]: the item answered with at every step, 0 = none (padding).  A row whose id
 * lies outside 1 .. V-1 is not read, has log-probability 0 and gradient 0; so is a row of nothing but -inf (no distribution is left).  Column 0 takes part in
 * the soft-max, as in model_tcn.py:41.   logp = z[id] - log sum_j exp z_j.   V is at most 2^31 - 4097,
 * n T at most 2^24 - 1 rows of more than some hundred or thousand items (of their parts, where a row is cut into up to 64) and about 2^26 shorter ones: what goes into a launch.
 * dlogits (rows of stride dld, the logits' type) may be the logits' own buffer (ptr and stride equal): it is overwritten row by row. */
typedef struct {
  int64_t n, T, V;
  int32_t dtype; int32_t reserved;
  const void* logits; int64_t ld;
  const int32_t* ids;                  /* [n][T] contiguous                                                                           */
  float* logp;                         /* [n][T]: written                                                                             */
  void* dlogits; int64_t dld;          /* NULL: no gradient wanted                                                                    */
  float grad_scale;                    /* multiplies the gradient (loss scaling of 16-bit gradients, accumulation)                    */
  void* workspace; size_t workspace_bytes;        /* hiertcn_rows_workspace_bytes, 16-byte aligned                                    */
} hiertcn_rows_t;
size_t hiertcn_rows_workspace_bytes(int64_t n, int64_t T, int64_t V);
/* logp alone (the reference's and the behaviour policy's pass); dlogits is ignored */
int hiertcn_sequence_logp(const hiertcn_rows_t* r, void* stream);

/* Preference loss over P pairs (n = 2 P sequences, the preferred answers first: pair i = sequences i and P + i).  With s = the sum of logp over a
 * sequence (divided by its number of answers when `average`; 0 where there is none) and D = (s_i - ref_i) - (s_{P+i} - ref_{P+i}):
 *   kind 0  (1 - smoothing) softplus(-beta D) + smoothing softplus(beta D)
 *   kind 1  max(0, 1 - beta D)
 *   kind 2  (D - 1 / (2 beta))^2              (P is at most 2^22 - 1)
 * loss [1] = mean of pair_loss; the gradient is that of grad_scale * loss. */
typedef struct {
  int32_t kind, average;
  float beta, smoothing;
  const float* ref;                    /* [2 P]: the reference's s                                                                    */
  float* loss;                         /* [1]                                                                                         */
  float* pair_loss;                    /* [P]                                                                                         */
  float* margin;                       /* [P]: D                                                                                      */
  float* seq_logp;                     /* [2 P]: s                                                                                    */
} hiertcn_preference_t;
int hiertcn_preference_loss(const hiertcn_rows_t* r, const hiertcn_preference_t* p, void* stream);

/* Clipped policy loss with a penalty on the distance from a reference, per answer:
 *   ratio = exp(logp - old), l = -min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef k,  k = exp(ref - logp) - (ref - logp) - 1
 * (A = 0: the first term is 0.  kl_coef = 0: so is the penalty, though kl is reported, whatever it is: inf where an answer's logit is -inf).
 * loss [1] = mean over every sequence's answers, then over the sequences that have any (mean 0: the lane mean of model.py:111-117), or over all answers
 * (mean 1); 0 where there is none.  kl [1], clipped [1]: the same means of k and of [the clamp is the smaller branch].  The losses take logp before it
 * is rounded to fp32 (a ratio to an old that is this very logp is 1 to within that rounding).
 * old, ref [n][T]; advantage [n][T] with element strides (adv_sn, adv_st), 0 = broadcast. */
typedef struct {
  int32_t mean, reserved;
  float clip_low, clip_high, kl_coef;
  const float* old_logp;
  const float* ref_logp;               /* NULL: no penalty, kl = 0                                                                    */
  const float* advantage; int64_t adv_sn, adv_st;
  float* loss;                         /* [1]                                                                                         */
  float* kl;                           /* [1]                                                                                         */
  float* clipped;                      /* [1]                                                                                         */
} hiertcn_policy_t;
int hiertcn_policy_loss(const hiertcn_rows_t* r, const hiertcn_policy_t* p, void* stream);

/* ---- AdamW over many tensors at once ---------------------------------------------------------------------------------------------------------
 *   g = grad * grad_scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
 *   param = param (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps);   copy = param, rounded
 * state_bits 8: m and the ROOT of v are held as codes with one fp32 scale per 256 elements of a tensor (the largest of the block):
 *   m = sign(q) (q / 127)^2 m_scale, q int8;   sqrt(v) = (q / 255)^2 v_scale, q uint8
 * A code is rounded up or down at random such that the EXPECTED m (and v) is the value itself: with b2 = 0.999 a step moves v by a thousandth, far less
 * than half a code, so that rounding to nearest would hold v where it is.  The random bits are a function of (seed, t, index of the tensor, element).  A non-zero
 * v never gets the code of zero; a block whose largest value is below 2^-100 is stored as zeros.  A NaN or infinite gradient leaves its block's states not finite.
 * Tensors of a call do not overlap.  t and lr are arguments of the call: a captured call would replay the same step, so this call is REFUSED on a
 * capturing stream. */
typedef struct {
  int64_t numel;                       /* 0: skipped                                                                                  */
  float* param;
  const void* grad; int32_t grad_dtype;           /* grad NULL: the tensor is left as it is                                           */
  int32_t copy_dtype;                  /* of copy: HIERTCN_BF16 / HIERTCN_FP16                                                        */
  void* copy;                          /* NULL: none                                                                                  */
  void* m; void* v;                    /* float, or int8_t / uint8_t codes                                                            */
  float* m_scale; float* v_scale;      /* [ceil(numel / 256)], state_bits 8 only                                                      */
  float weight_decay; int32_t index;   /* index: names the tensor in the random rounding                                              */
} hiertcn_adamw_tensor_t;
typedef struct {
  double lr, beta1, beta2, eps, grad_scale;
  const float* grad_scale_dev;         /* optional device float [1]: a further factor of the gradient (clipping by the global norm)    */
  int64_t t;                           /* this step's number, from 1                                                                  */
  int64_t seed;                        /* of the 8-bit rounding                                                                       */
  int32_t state_bits;                  /* 32 or 8                                                                                     */
  int32_t reserved;
} hiertcn_adamw_t;
/* tensors: HOST array, read before the call returns.  The buffers of different tensors do not overlap (those of one are checked). */
int hiertcn_adamw_step(const hiertcn_adamw_tensor_t* tensors, int64_t n, const hiertcn_adamw_t* a, void* stream);
/* the values of 8-bit states: m_out[i], v_out[i] (HOST arrays of device float pointers, an entry may be NULL), which overlap neither one another nor anything of
 * the tensors (those of one tensor are checked against its states) */
int hiertcn_adamw_moments(const hiertcn_adamw_tensor_t* tensors, int64_t n, float* const* m_out, float* const* v_out, void* stream);
/* after another optimizer has changed a training handle's masters (hiertcn_train_arena 0): the 16-bit device copies, as hiertcn_adam_step refreshes them.
 * (A call on a handle: its message is in hiertcn_last_error().) */
int hiertcn_train_masters_changed(hiertcn_handle_t h, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* HIERTCN_OPS_H_ */
