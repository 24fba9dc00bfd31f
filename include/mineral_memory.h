/* mineral_memory.h — C ABI of the operators of a sequence memory (gfx950): linear attention with a decay per head, group norm
 * with an activation on channels-last data, and a linear layer with bias, activation and residual in its epilogue.
 *
 * Same conventions as mineral_ppo.h: device pointers, `stream` is a hipStream_t passed as void*, 0 / negative MRL_E* status with
 * mrl_last_error(), nothing allocates or synchronises, calls that share a workspace must not overlap, and the device that owns
 * the pointers is the current one.  Strides are in elements; the last dimension of every tensor is contiguous.  The reference
 * has no counterpart of these operators (its towers are mineral/nets/mlp.py, its rollout scans mineral/agents/ppo/experience.py).
 */
#ifndef MINERAL_MEMORY_H
#define MINERAL_MEMORY_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MRL_F32 0
#define MRL_BF16 1
#define MRL_F16 2

#define MRL_ATTENTION_MAX_DIM 128   /* largest dim_k and dim_v */

/* Linear attention with one decay per head:
 *     S_t = exp(log_decay[h]) * S_{t-1} + k_t v_t^T        (S_{t-1} = 0 where resets[b][t] != 0)
 *     o_t = scale * S_t^T q_t
 * for every batch row b and head h, with S of dim_k x dim_v in fp32.  A reset drops whatever the state held, NaN and infinity
 * included, and no token's output depends on a later token or on an earlier episode.  log_decay <= 0 is meant; -inf keeps nothing of a
 * finite state.  fp32 products are formed from three bf16 terms, exact for magnitudes from 2^-100 to 3.38e38 (a larger or infinite value
 * makes NaN of what it belongs to); the state and all sums are fp32.  batch x heads is below 2^23.
 *   q, k : [batch][steps][heads][dim_k], v : [batch][steps][heads][dim_v] of `dtype`; strides {batch, step, head}
 *   log_decay : [heads] fp32;  resets : [batch][steps] bytes or NULL;  initial_state : [batch][heads][dim_k][dim_v] fp32 or NULL (zero) */
typedef struct mrl_attention {
  int64_t batch, steps;
  int32_t heads, dim_k, dim_v, dtype;
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  const float* log_decay;
  const uint8_t* resets;
  const float* initial_state;
  float scale;
} mrl_attention;

/* Bytes of workspace of the forward call (backward = 0) or of the backward call (backward = 1); only the sizes are read. */
int64_t mrl_linear_attention_workspace_bytes(const mrl_attention* p, int32_t backward);

/* out : [batch][steps][heads][dim_v] of dtype, contiguous, on a 16-byte address; final_state : [batch][heads][dim_k][dim_v] fp32. */
int mrl_linear_attention(const mrl_attention* p, void* out, float* final_state, void* workspace, int64_t workspace_bytes, void* stream);

/* Gradients with respect to q, k, v (contiguous, of dtype, on 16-byte addresses) and the initial state (fp32); a NULL output is not computed
 * (d_initial_state comes with dv).
 *   d_out : [batch][steps][heads][dim_v], strides like the inputs;  d_final_state : fp32 or NULL (zero). */
int mrl_linear_attention_backward(const mrl_attention* p, const void* d_out, const int64_t* d_out_stride_host, const float* d_final_state, void* dq,
                                  void* dk, void* dv, float* d_initial_state, void* workspace, int64_t workspace_bytes, void* stream);

/* One token per batch row (p->steps == 1, the step strides are not read, p->initial_state is not read): `state` is updated in place. */
int mrl_linear_attention_step(const mrl_attention* p, float* state, void* out, void* stream);

#define MRL_ACT_NONE 0
#define MRL_ACT_SILU 1
#define MRL_ACT_ELU 2
#define MRL_ACT_RELU 3
#define MRL_ACT_TANH 4
#define MRL_ACT_GELU 5   /* z Phi(z), Phi from erf */

/* Group norm with an activation on channels-last data [batch][pixels][channels]: one mean and variance (divided by the count) for
 * the pixels x channels/groups values of a sample's group,
 *     y = act((x - mean) / sqrt(var + eps) * weight[c] + bias[c]).
 * x and y of `dtype`, contiguous; weight and bias [channels] of `param_dtype` (dtype or MRL_F32), NULL for one and zero.
 * Data on 16-byte addresses fits every width; sums are Welford's and pairwise joins of them, in fp32. */
typedef struct mrl_group_norm {
  int64_t batch, pixels;
  int32_t channels, groups, dtype, param_dtype, act;
  float eps;
} mrl_group_norm;

/* Bytes of workspace of the forward call (backward = 0) or of the backward call (backward = 1). */
int64_t mrl_group_norm_act_workspace_bytes(const mrl_group_norm* p, int32_t backward);

/* mean, rstd : [batch][groups] fp32, what the backward call reads (either both or neither may be NULL). */
int mrl_group_norm_act(const mrl_group_norm* p, const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* workspace,
                       int64_t workspace_bytes, void* stream);

/* dx like x; d_weight, d_bias [channels] of param_dtype, both or neither NULL.  Sums are formed in one order: equal calls give equal bits. */
int mrl_group_norm_act_backward(const mrl_group_norm* p, const void* x, const void* dy, const void* weight, const void* bias, const float* mean, const float* rstd,
                                void* dx, void* d_weight, void* d_bias, void* workspace, int64_t workspace_bytes, void* stream);

/* Linear layer: y = act(x W^T + bias) + residual.
 *   x : [rows][inputs], row stride x_stride; weight : [outputs][inputs]; bias : [outputs] or NULL; residual : [rows][outputs] or NULL;
 *   y : [rows][outputs]; all of `dtype`, contiguous but for x.  16-bit operands multiply as they are and fp32 ones as three exact
 *   bf16 terms (six products, error below an fp32 product's rounding, for magnitudes from 2^-100 to
 *   3.38e38; a larger or infinite operand gives NaN); everything accumulates in fp32 and is rounded once. */
typedef struct mrl_linear {
  int64_t rows, x_stride;
  int32_t inputs, outputs, dtype, act;
} mrl_linear;

/* slope : [rows][outputs] or NULL: act'(x W^T + bias), what the backward call reads where act is not MRL_ACT_NONE: fp32 beside MRL_F32,
 * otherwise 16 bits each, in a code of the library's own. */
int mrl_linear_act(const mrl_linear* p, const void* x, const void* weight, const void* bias, const void* residual, void* y, void* slope, void* stream);

int64_t mrl_linear_act_backward_workspace_bytes(const mrl_linear* p);

/* dx [rows][inputs], d_weight [outputs][inputs], d_bias [outputs], contiguous; a NULL output is not computed.  The residual's gradient
 * is dy itself.  dz = dy slope is rounded to dtype before the products (beside fp16 with room for every finite dy); d_bias sums it
 * unrounded.  Where MRL_ACT_RELU cuts, dy is dropped, whatever it is; beside the other activations a dy that is not finite makes a dz
 * that is not, saturated or not. */
int mrl_linear_act_backward(const mrl_linear* p, const void* x, const void* weight, const void* slope, const void* dy, void* dx, void* d_weight, void* d_bias,
                            void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MINERAL_MEMORY_H */
