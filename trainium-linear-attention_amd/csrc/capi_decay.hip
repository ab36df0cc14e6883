// C-ABI entry points declared in include/based_la_decay.h: arguments are checked here, before any launch.
#include <float.h>
#include <math.h>

#include "../../include/based_la.h"
#include "../../include/based_la_decay.h"
#include "la_internal.hpp"

namespace {

bool al(const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }
bool dtype_ok(int t) { return t == LA_F32 || t == LA_BF16; }
bool overlap(const void* a, const void* b, size_t bytes) {
  const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
  return x != nullptr && y != nullptr && x < y + bytes && y < x + bytes;
}

int check_sizes(int B, int H, int N, int d, int dv, float scale) {
  if (B < 0 || H < 0 || N < 0 || d < 1 || dv < 1) return LA_ERR_BAD_SHAPE;
  if (d > 128 || dv > 128) return LA_ERR_UNSUPPORTED_DIM;
  // three sums of 512 threads a head are one launch, of fewer than 2^32 threads
  if ((long long)B * H > (1 << 21) || N > (1 << 30)) return LA_ERR_BAD_SHAPE;
  if (!isfinite(scale) || !(scale >= FLT_MIN)) return LA_ERR_BAD_SCALAR;
  return LA_OK;
}

// An operand's strides (contiguous if s is null) and its alignment.
int operand(const void* p, const long long* s, int H, int N, int w, int esz, long long* out) {
  if (p == nullptr) return LA_ERR_NULL_POINTER;
  if (!al(p, esz)) return LA_ERR_BAD_ALIGNMENT;
  const long long row = w, head = row * N, batch = head * H;
  out[0] = s ? s[0] : batch;
  out[1] = s ? s[1] : head;
  out[2] = s ? s[2] : row;
  return out[0] < 0 || out[1] < 0 || out[2] < 0 ? LA_ERR_BAD_SHAPE : LA_OK;
}

}  // namespace

extern "C" {

size_t la_decay_workspace_bytes(int B, int H, int N, int d, int dv, int backward) {
  if (B < 1 || H < 1 || N < 1 || check_sizes(B, H, N, d, dv, 1.f) != LA_OK) return 0;
  return backward < 0 || backward > 1 ? 0 : la::decay_workspace_bytes((long long)B * H, N, d, dv, backward);
}

int la_decay_fwd(const void* q, const void* k, const void* v, int in_dtype, void* out, int out_dtype, int B, int H,
                 int N, int d, int dv, const long long* q_strides, const long long* k_strides,
                 const long long* v_strides, const float* log_decay, const int* lengths, float scale,
                 const float* state_in, float* state_out, void* workspace, size_t workspace_bytes, void* hip_stream) {
  int rc = check_sizes(B, H, N, d, dv, scale);
  if (rc != LA_OK) return rc;
  if (!dtype_ok(in_dtype) || !dtype_ok(out_dtype)) return LA_ERR_BAD_DTYPE;
  if ((long long)B * H * N == 0) return LA_OK;
  la::DecayArgs a{};
  const int e = in_dtype == LA_F32 ? 4 : 2;
  if ((rc = operand(q, q_strides, H, N, d, e, a.q_strides)) != LA_OK) return rc;
  if ((rc = operand(k, k_strides, H, N, d, e, a.k_strides)) != LA_OK) return rc;
  if ((rc = operand(v, v_strides, H, N, dv, e, a.v_strides)) != LA_OK) return rc;
  if (out == nullptr || log_decay == nullptr) return LA_ERR_NULL_POINTER;
  if (!al(out, 16) || !al(log_decay, 4) || !al(lengths, 4) || !al(state_in, 16) || !al(state_out, 16))
    return LA_ERR_BAD_ALIGNMENT;
  if (overlap(state_in, state_out, (size_t)B * H * d * dv * 4)) return LA_ERR_OVERLAP;
  const size_t need = la::decay_workspace_bytes((long long)B * H, N, d, dv, 0);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return LA_ERR_WORKSPACE;
  if (need > 0 && !al(workspace, 16)) return LA_ERR_BAD_ALIGNMENT;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.state_in = state_in;
  a.state_out = state_out;
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.workspace = workspace;
  a.B = B;
  a.H = H;
  a.N = N;
  a.d = d;
  a.dv = dv;
  a.scale = scale;
  a.in_f32 = in_dtype == LA_F32;
  a.out_f32 = out_dtype == LA_F32;
  return la::launch_decay_fwd(a, static_cast<hipStream_t>(hip_stream));
}

int la_decay_bwd(const void* q, const void* k, const void* v, const void* dout, int in_dtype, void* dq, void* dk,
                 void* dv_out, int B, int H, int N, int d, int dv, const long long* q_strides,
                 const long long* k_strides, const long long* v_strides, const long long* dout_strides,
                 const float* log_decay, const int* lengths, float scale, const float* state_in,
                 const float* dstate_out, float* dstate_in, const void* fwd_workspace, void* workspace,
                 size_t workspace_bytes, void* hip_stream) {
  int rc = check_sizes(B, H, N, d, dv, scale);
  if (rc != LA_OK) return rc;
  if (!dtype_ok(in_dtype)) return LA_ERR_BAD_DTYPE;
  if ((long long)B * H * N == 0) return LA_OK;
  la::DecayArgs a{};
  const int e = in_dtype == LA_F32 ? 4 : 2;
  if ((rc = operand(q, q_strides, H, N, d, e, a.q_strides)) != LA_OK) return rc;
  if ((rc = operand(k, k_strides, H, N, d, e, a.k_strides)) != LA_OK) return rc;
  if ((rc = operand(v, v_strides, H, N, dv, e, a.v_strides)) != LA_OK) return rc;
  if ((rc = operand(dout, dout_strides, H, N, dv, e, a.dout_strides)) != LA_OK) return rc;
  if (dq == nullptr || dk == nullptr || dv_out == nullptr || log_decay == nullptr) return LA_ERR_NULL_POINTER;
  if (!al(dq, 16) || !al(dk, 16) || !al(dv_out, 16) || !al(log_decay, 4) || !al(lengths, 4) || !al(state_in, 16) ||
      !al(dstate_out, 16) || !al(dstate_in, 16))
    return LA_ERR_BAD_ALIGNMENT;
  if (overlap(dstate_in, dstate_out, (size_t)B * H * d * dv * 4)) return LA_ERR_OVERLAP;
  const size_t need = la::decay_workspace_bytes((long long)B * H, N, d, dv, fwd_workspace == nullptr);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return LA_ERR_WORKSPACE;
  if (need > 0 && (!al(workspace, 16) || !al(fwd_workspace, 16))) return LA_ERR_BAD_ALIGNMENT;
  if (need > 0 && overlap(fwd_workspace, workspace, need)) return LA_ERR_OVERLAP;
  a.fwd_states = static_cast<const float*>(fwd_workspace);
  a.q = q;
  a.k = k;
  a.v = v;
  a.dout = dout;
  a.dq = dq;
  a.dk = dk;
  a.dv_out = dv_out;
  a.state_in = state_in;
  a.dstate_out = dstate_out;
  a.dstate_in = dstate_in;
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.workspace = workspace;
  a.B = B;
  a.H = H;
  a.N = N;
  a.d = d;
  a.dv = dv;
  a.scale = scale;
  a.in_f32 = in_dtype == LA_F32;
  return la::launch_decay_bwd(a, static_cast<hipStream_t>(hip_stream));
}

int la_decay_step(const void* q, const void* k, const void* v, int in_dtype, const float* log_decay, float* state,
                  void* out, int out_dtype, int B, int H, int d, int dv, float scale, void* hip_stream) {
  const int rc = check_sizes(B, H, 1, d, dv, scale);
  if (rc != LA_OK) return rc;
  if (!dtype_ok(in_dtype) || !dtype_ok(out_dtype)) return LA_ERR_BAD_DTYPE;
  if ((long long)B * H == 0) return LA_OK;
  if (q == nullptr || k == nullptr || v == nullptr || log_decay == nullptr || state == nullptr || out == nullptr)
    return LA_ERR_NULL_POINTER;
  const uintptr_t e = in_dtype == LA_F32 ? 4 : 2;
  if (!al(q, e) || !al(k, e) || !al(v, e) || !al(out, out_dtype == LA_F32 ? 4 : 2) || !al(log_decay, 4) || !al(state, 16))
    return LA_ERR_BAD_ALIGNMENT;
  la::DecayStepArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.log_decay = log_decay;
  a.state = state;
  a.out = out;
  a.B = B;
  a.H = H;
  a.d = d;
  a.dv = dv;
  a.scale = scale;
  a.in_f32 = in_dtype == LA_F32;
  a.out_f32 = out_dtype == LA_F32;
  return la::launch_decay_step(a, static_cast<hipStream_t>(hip_stream));
}

}  // extern "C"
