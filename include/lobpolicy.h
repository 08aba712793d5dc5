/* lobpolicy.h - C-ABI of the operators a policy that remembers order flow needs next to the simulator of lobsim.h: decay attention
 * (a state per environment and head; one step of every environment, recorded segments, their gradients), a block's gated residual
 * with the norms before and after it, and the global gradient norm with clipping.
 *
 * Plain pointers and sizes, like lobsim.h; device pointers unless said otherwise.  Every call is asynchronous on `stream` (a hipStream_t;
 * 0 = the null stream) of the CURRENT device, allocates nothing, and may be captured into a graph: what it needs beyond its operands is
 * the caller's workspace, whose size the *_workspace function tells.  Calls are independent of one another: two threads or two
 * streams may run them at once, each with workspaces of its own.  0 on success, a negative lobpolicy_error otherwise (nothing was launched);
 * lobpolicy_last_error() has the calling thread's message.  rl4mm_amd/policy_ops.py is the binding.
 */
#ifndef LOBPOLICY_H
#define LOBPOLICY_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

#define LOBPOLICY_ABI_VERSION 1
#define LOBPOLICY_MAX_HEAD 128   /* largest dk, dv */
#define LOBPOLICY_MAX_WIDTH 8192 /* largest row of the block operators */

enum lobpolicy_error { LOBPOLICY_OK = 0, LOBPOLICY_ERR_ARG = -1, LOBPOLICY_ERR_HIP = -2 };
enum lobpolicy_dtype { LOBPOLICY_F32 = 0, LOBPOLICY_BF16 = 1 };

int lobpolicy_abi_version(void);
const char* lobpolicy_last_error(void);

/* An operand [steps][envs][heads][dk or dv]: strides in elements, the last dimension contiguous. */
typedef struct lobpolicy_operand {
    void* data;
    int64_t stride_t, stride_n, stride_h;
} lobpolicy_operand;

/* Decay attention.  Of every environment n and head h, with a state S [dk][dv] (float32):
 *     S = reset[t][n] ? 0 : S;   S = exp(log_decay[h]) S + k_t v_t^T;   out_t = scale q_t^T S          t = 0 .. min(lengths[n], steps) - 1
 * Rows t >= lengths[n] are not used; their rows of out, dq, dk and dv are set to 0.  A bfloat16 result is rounded once, as it is stored: sums and the
 * state are float32, scores and the state where they multiply a bfloat16 operand two bfloat16 each.  An infinite operand gives infinities and not-numbers as the
 * formula has them, however the steps are split. */
typedef struct lobpolicy_attention {
    int32_t dtype; /* of q, k, v, out and their gradients */
    int32_t heads, dk, dv;
    int64_t steps, envs;
    lobpolicy_operand q, k, v;
    lobpolicy_operand out;            /* forward, step: written; dout of the backward call: read */
    lobpolicy_operand grad_q, grad_k, grad_v;
    const float* log_decay;           /* [heads] */
    const uint8_t* reset;             /* [steps][envs] by the strides below, or NULL: no resets */
    int64_t reset_stride_t, reset_stride_n;
    const int32_t* lengths;           /* [envs], or NULL: all `steps`; values are clamped to 0 .. steps */
    const uint8_t* skip;              /* step only: [envs], or NULL; a skipped environment keeps its state, its row of out is 0 */
    const float* state_in;            /* [envs][heads][dk][dv] before the first token, or NULL: 0 */
    float* state_out;                 /* forward: after the last token, or NULL.  step: the state, updated in place */
    const float* grad_state_out;      /* backward: gradient of state_out, or NULL: 0 */
    float* grad_state_in;             /* backward: gradient of state_in, or NULL: not wanted */
    float scale;
    void* workspace;
    int64_t workspace_bytes;
    const void* forward_workspace;    /* backward: the workspace that the forward call left, unchanged (the states in front of each part) */
} lobpolicy_attention;

int64_t lobpolicy_attention_workspace(const lobpolicy_attention* a); /* bytes, of either call; negative: lobpolicy_error */
int lobpolicy_attention_forward(const lobpolicy_attention* a, void* stream);
int lobpolicy_attention_backward(const lobpolicy_attention* a, void* stream);
int lobpolicy_attention_step(const lobpolicy_attention* a, void* stream); /* one token of every environment: steps is 1 */

/* A block's end.  Of every row, elementwise but for the two means:
 *     y = x + res * sigmoid(gate) * post * b / rms(b);   z = pre * y / rms(y);   rms(a) = sqrt(mean(a^2) + eps)
 * Gradients: grad_x, grad_block, grad_gate by row; grad_post, grad_res, grad_pre [width], summed over the rows in a fixed order. */
typedef struct lobpolicy_block {
    int32_t stream_dtype; /* of x, y and their gradients */
    int32_t dtype;        /* of block, gate, z and their gradients */
    int64_t rows, width;
    const void *x, *block, *gate; /* gate NULL: no gate (its factor is 1) */
    int64_t x_stride, block_stride, gate_stride; /* elements from row to row */
    const float *post, *res, *pre;
    float eps;
    void *y, *z; /* forward: rows of `width`, without gaps */
    const void *grad_y, *grad_z; /* backward, NULL: 0 */
    int64_t grad_y_stride, grad_z_stride;
    void *grad_x, *grad_block, *grad_gate; /* rows of `width`, without gaps; grad_gate NULL without a gate */
    float *grad_post, *grad_res, *grad_pre;
    void* workspace;
    int64_t workspace_bytes;
} lobpolicy_block;

int64_t lobpolicy_block_workspace(const lobpolicy_block* b); /* of the backward call */
int lobpolicy_block_forward(const lobpolicy_block* b, void* stream);
int lobpolicy_block_backward(const lobpolicy_block* b, void* stream);

/* The norm over all tensors, and clipping by it, in place:
 *     norm = sqrt(sum x^2) (kind 2) or max |x| (kind 0);   x *= min(1, max_norm / (norm + 1e-6))
 * `tensors`, `counts` and `dtypes` are HOST arrays of n entries, read before the call returns; the tensors must not overlap.  norm: one
 * float.  A norm that is not a number reaches every element, an infinite one makes the finite elements 0. */
int64_t lobpolicy_clip_workspace(const int64_t* counts, const int32_t* dtypes, int64_t n);
int lobpolicy_clip(void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t n, int32_t kind, double max_norm, float* norm,
                   void* workspace, int64_t workspace_bytes, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif
#endif
