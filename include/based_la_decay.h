/*
 * based_la_decay.h -- further entry points of libbased_la.so (based_la.h): causal linear attention with
 * the identity feature map and a decay for each head, in chunks for prompts and training, with its
 * gradient, and one token at a time.  Conventions, status codes and argument rules are based_la.h's.
 * No reference counterparts (the reference's identity map has no decay,
 * benchmarks/chunked_attention_benchmark.py:81-93).
 *
 * With g_h = exp(log_decay[h]) and L tokens in sequence b,
 *   y_t = scale (sum_{u <= t} g^(t - u) (q_t . k_u) v_u + g^(t + 1) q_t S_in)         (t < L)
 *   S_out = g^L S_in + sum_{u < L} g^(L - 1 - u) k_u v_u^T
 * States are fp32 (B, H, d, dv).  log_decay: fp32 (H) in device memory, in general <= 0 (-inf: a decay of 0).
 * lengths: int32 (B) in device memory or NULL (L = N everywhere); values are taken between 0 and N.
 * Rows behind a sequence are not read, and their outputs and gradients are written as zeros.
 * A value that is not finite reaches, besides later outputs, those of its own 64 tokens (64 t .. 64 t + 63).
 * Limits: 1 <= d, dv <= 128 (LA_ERR_UNSUPPORTED_DIM), B H <= 2^21, N <= 2^30, scale positive, finite and not
 * subnormal.  With B, H or N of 0 nothing is launched and nothing written.
 */
#ifndef BASED_LA_DECAY_H
#define BASED_LA_DECAY_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Scratch of la_decay_fwd, or of la_decay_bwd (backward = 1; as much as la_decay_fwd's with its
 * fwd_workspace), 16-byte aligned; 0 for short sequences, for batches of many heads and for sizes outside the
 * limits: NULL is then accepted. */
size_t la_decay_workspace_bytes(int B, int H, int N, int d, int dv, int backward);

/*
 * y and, if state_out is given, the state after the last token.  state_in NULL: zero.  state_out must
 * not overlap state_in (LA_ERR_OVERLAP).  Element (b, h, t, i) of an operand x lies at
 * x + b x_strides[0] + h x_strides[1] + t x_strides[2] + i (in elements, >= 0, NULL: contiguous); out is
 * contiguous and 16-byte aligned, and so are states and workspace.  Operands whose start and strides are
 * multiples of 16 bytes and whose rows are whole 16-byte pieces are read 16 bytes at a time, those of which this
 * holds with 4 bytes by 4-byte words, others by element.
 */
int la_decay_fwd(const void* q, const void* k, const void* v, int in_dtype, void* out, int out_dtype, int B, int H,
                 int N, int d, int dv, const long long* q_strides, const long long* k_strides,
                 const long long* v_strides, const float* log_decay, const int* lengths, float scale,
                 const float* state_in, float* state_out, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Gradients of la_decay_fwd by q, k, v (contiguous, of the inputs' type) and state_in, from those of y (dout,
 * the inputs' type) and of state_out (NULL: zero).  dstate_in may be NULL; it must not overlap
 * dstate_out.  The decay is a constant: there is no gradient by it.  fwd_workspace: the workspace as
 * la_decay_fwd left it for the same q, k, v, sizes, decays, lengths and state_in, which holds states that are then not
 * computed again (NULL: they are); it is not written.
 */
int la_decay_bwd(const void* q, const void* k, const void* v, const void* dout, int in_dtype, void* dq, void* dk,
                 void* dv_out, int B, int H, int N, int d, int dv, const long long* q_strides,
                 const long long* k_strides, const long long* v_strides, const long long* dout_strides,
                 const float* log_decay, const int* lengths, float scale, const float* state_in,
                 const float* dstate_out, float* dstate_in, const void* fwd_workspace, void* workspace,
                 size_t workspace_bytes, void* hip_stream);

/*
 * One token: state <- g state + k v^T in place, out = scale q state.  q, k: (B, H, d), v, out: (B, H, dv),
 * contiguous; state (B, H, d, dv) fp32.
 */
int la_decay_step(const void* q, const void* k, const void* v, int in_dtype, const float* log_decay, float* state,
                  void* out, int out_dtype, int B, int H, int d, int dv, float scale, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* BASED_LA_DECAY_H */
