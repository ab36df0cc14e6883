// C-ABI entry points declared in include/based_la_cache.h: arguments are checked here, before any launch.
#include <math.h>

#include "../../include/based_la.h"
#include "../../include/based_la_cache.h"
#include "la_internal.hpp"

namespace {

bool al(const void* ptr, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(ptr) & (bytes - 1)) == 0; }
bool dtype_ok(int t) { return t == LA_F32 || t == LA_BF16; }

int check_sizes(int B, int HK, int N, int d, int dv, int blocks) {
  if (B < 0 || HK < 0 || N < 0 || d < 1 || dv < 1 || blocks < 1 || blocks > (1 << 24)) return LA_ERR_BAD_SHAPE;
  if (d > 128 || dv > 128) return LA_ERR_UNSUPPORTED_DIM;
  // work-group indices and threads of the launches
  if (B > 0xffff || (long long)B * HK > 0xffff || N > (1 << 29)) return LA_ERR_BAD_SHAPE;
  return LA_OK;
}

int check_cache(const void* kc, const void* vc, const void* ks, const void* vs) {
  if (kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr) return LA_ERR_NULL_POINTER;
  return al(kc, 16) && al(vc, 16) && al(ks, 4) && al(vs, 4) ? LA_OK : LA_ERR_BAD_ALIGNMENT;
}

bool strides(const long long* s, int HK, int N, int w, long long* out) {
  out[0] = s ? s[0] : (long long)HK * N * w;
  out[1] = s ? s[1] : (long long)N * w;
  out[2] = s ? s[2] : w;
  return out[0] >= 0 && out[1] >= 0 && out[2] >= 0;
}

int check_step(int B, int H, int HK, int d, int dv, int blocks, int window) {
  const int rc = check_sizes(B, HK, 1, d, dv, blocks);
  if (rc != LA_OK) return rc;
  if (H < 0 || (HK > 0 && H % HK != 0) || (HK == 0 && H != 0)) return LA_ERR_BAD_SHAPE;
  if ((long long)B * H > 0xffffffLL || H > 0xffff) return LA_ERR_BAD_SHAPE;
  if (window < 0 || window > 64LL * (blocks - 1) + 1) return LA_ERR_BAD_SHAPE;
  return LA_OK;
}

}  // namespace

extern "C" {

int la_sliding_cache_dim(int d) { return la::sliding_cache_dim(d); }

int la_sliding_cache_append(const void* k, const void* v, int in_dtype, void* kc, void* vc, float* ks, float* vs,
                            const int* start, const int* lengths, int B, int HK, int N, int d, int dv, int blocks,
                            const long long* k_strides, const long long* v_strides, void* hip_stream) {
  int rc = check_sizes(B, HK, N, d, dv, blocks);
  if (rc != LA_OK) return rc;
  if (!dtype_ok(in_dtype)) return LA_ERR_BAD_DTYPE;
  if ((long long)B * HK * N == 0) return LA_OK;
  if (k == nullptr || v == nullptr) return LA_ERR_NULL_POINTER;
  if ((rc = check_cache(kc, vc, ks, vs)) != LA_OK) return rc;
  const uintptr_t e = in_dtype == LA_F32 ? 4 : 2;
  if (!al(k, e) || !al(v, e) || !al(start, 4) || !al(lengths, 4)) return LA_ERR_BAD_ALIGNMENT;
  la::SlidingCacheArgs a{};
  if (!strides(k_strides, HK, N, d, a.k_strides) || !strides(v_strides, HK, N, dv, a.v_strides)) return LA_ERR_BAD_SHAPE;
  a.k = k;
  a.v = v;
  a.kc = kc;
  a.vc = vc;
  a.ks = ks;
  a.vs = vs;
  a.start = start;
  a.lengths = lengths;
  a.B = B;
  a.HK = HK;
  a.N = N;
  a.d = d;
  a.dv = dv;
  a.blocks = blocks;
  a.in_f32 = in_dtype == LA_F32;
  return la::launch_sliding_append(a, static_cast<hipStream_t>(hip_stream));
}

size_t la_sliding_decode_workspace_bytes(int B, int H, int HK, int d, int dv, int blocks, int window) {
  if (B < 1 || HK < 1 || H < 1 || check_step(B, H, HK, d, dv, blocks, window) != LA_OK) return 0;
  return la::sliding_decode_workspace_bytes(B, H, HK, dv, blocks, window);
}

int la_sliding_decode_step(const void* q, const void* k, const void* v, int in_dtype, void* out, int out_dtype,
                           void* kc, void* vc, float* ks, float* vs, const int* lengths, int B, int H, int HK, int d,
                           int dv, int blocks, int window, float scale, void* workspace, size_t workspace_bytes,
                           void* hip_stream) {
  int rc = check_step(B, H, HK, d, dv, blocks, window);
  if (rc != LA_OK) return rc;
  if (!dtype_ok(in_dtype) || !dtype_ok(out_dtype)) return LA_ERR_BAD_DTYPE;
  if (!isfinite(scale) || !(scale > 0.f)) return LA_ERR_BAD_SCALAR;
  if ((long long)B * H == 0) return LA_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || lengths == nullptr) return LA_ERR_NULL_POINTER;
  if ((rc = check_cache(kc, vc, ks, vs)) != LA_OK) return rc;
  const uintptr_t e = in_dtype == LA_F32 ? 4 : 2;
  if (!al(q, e) || !al(k, e) || !al(v, e) || !al(out, out_dtype == LA_F32 ? 4 : 2) || !al(lengths, 4)) return LA_ERR_BAD_ALIGNMENT;
  const size_t need = la::sliding_decode_workspace_bytes(B, H, HK, dv, blocks, window);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return LA_ERR_WORKSPACE;
  if (need > 0 && !al(workspace, 16)) return LA_ERR_BAD_ALIGNMENT;
  la::SlidingCacheArgs a{};
  strides(nullptr, HK, 1, d, a.k_strides);
  strides(nullptr, HK, 1, dv, a.v_strides);
  a.q = q;
  a.out = out;
  a.k = k;
  a.v = v;
  a.kc = kc;
  a.vc = vc;
  a.ks = ks;
  a.vs = vs;
  a.lengths = lengths;
  a.last_of = true;
  a.workspace = workspace;
  a.B = B;
  a.H = H;
  a.HK = HK;
  a.N = 1;
  a.d = d;
  a.dv = dv;
  a.blocks = blocks;
  a.window = window;
  a.scale = scale;
  a.in_f32 = in_dtype == LA_F32;
  a.out_f32 = out_dtype == LA_F32;
  return la::launch_sliding_decode(a, static_cast<hipStream_t>(hip_stream));
}

}  // extern "C"
