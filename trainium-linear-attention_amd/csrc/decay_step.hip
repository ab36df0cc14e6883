// One token of linear attention with a decay per head, for gfx950: per head, with g = exp(log_decay),
//   S <- g S + k v^T (d x dv, fp32, in place),   y = s q^T S.
//
// A work-group has CW consecutive value columns of one head, so that no sum crosses work-groups; its
// threads take CW / 4 columns of four and, in between, rows of the state.  All of a thread's rows (at most
// kRows) are loaded before any is used.  HBM-bound in batches: the state is read and written once.
#include <math.h>

#include "la_common.hpp"
#include "la_internal.hpp"

namespace la {

namespace {

struct StepParams {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  float* state;
  void* out;
  int H, d, dv;
  float scale;
  int in_f32, out_f32;
};

constexpr int kStepThreads = 256;

__device__ __forceinline__ float elem(const void* base, size_t i, int f32) {
  return f32 ? static_cast<const float*>(base)[i] : bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
}

// VEC: rows of whole 16-byte pieces (dv % 4 == 0).
template <int CW, bool VEC>
__global__ __launch_bounds__(kStepThreads) void decay_step_kernel(const StepParams p) {
  constexpr int NT = kStepThreads, LPR = CW / 4, RPP = NT / LPR;      // lanes a row, rows a pass
  constexpr int PASSES = 128 / RPP > 0 ? 128 / RPP : 1;
  __shared__ float qs[128], ks[128];
  __shared__ __attribute__((aligned(16))) float red[4][CW];
  const int bh = blockIdx.x, tid = threadIdx.x, d = p.d, dv = p.dv;
  const int col = blockIdx.y * CW + 4 * (tid % LPR), row = tid / LPR;
  float* __restrict__ st = p.state + (size_t)bh * d * dv;
  f32x4 x[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row + RPP * i;
    x[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (r < d && col < dv) {
      const float* s = st + (size_t)r * dv + col;
      if (VEC) {
        x[i] = *reinterpret_cast<const f32x4*>(s);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < dv) x[i][e] = s[e];
      }
    }
  }
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = col + e < dv ? elem(p.v, (size_t)bh * dv + col + e, p.in_f32) : 0.f;
  if (tid < d) qs[tid] = elem(p.q, (size_t)bh * d + tid, p.in_f32);
  if (tid >= 128 && tid - 128 < d) ks[tid - 128] = elem(p.k, (size_t)bh * d + tid - 128, p.in_f32);
  const float g = expf(p.log_decay[bh % p.H]);
  __syncthreads();
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = row + RPP * i;
    if (r >= d) break;
    const float kr = ks[r], qr = qs[r];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[i][e] = __builtin_fmaf(kr, v[e], g * x[i][e]);
      y[e] = __builtin_fmaf(qr, x[i][e], y[e]);
    }
    if (col < dv) {
      float* s = st + (size_t)r * dv + col;
      if (VEC) {
        *reinterpret_cast<f32x4*>(s) = x[i];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < dv) s[e] = x[i][e];
      }
    }
  }
  // the rows of a wave, then the waves in order
#pragma unroll
  for (int m = LPR; m < 64; m <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], m);
  if ((tid & 63) < LPR) *reinterpret_cast<f32x4*>(&red[tid >> 6][4 * (tid % LPR)]) = y;
  __syncthreads();
  const int c = blockIdx.y * CW + tid;
  if (tid < CW && c < dv) {
    const float o = p.scale * (((red[0][tid] + red[1][tid]) + red[2][tid]) + red[3][tid]);
    const size_t at = (size_t)bh * dv + c;
    if (p.out_f32) static_cast<float*>(p.out)[at] = o;
    else static_cast<uint16_t*>(p.out)[at] = f32_to_bf16_bits(o);
  }
}

template <int CW>
int launch(const StepParams& p, int BH, hipStream_t stream) {
  const dim3 grid((unsigned)BH, (unsigned)((p.dv + CW - 1) / CW));
  if ((p.dv & 3) == 0)
    hipLaunchKernelGGL((decay_step_kernel<CW, true>), grid, dim3(kStepThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((decay_step_kernel<CW, false>), grid, dim3(kStepThreads), 0, stream, p);
  return (int)hipGetLastError();
}

}  // namespace

int launch_decay_step(const DecayStepArgs& a, hipStream_t stream) {
  const StepParams p{a.q, a.k, a.v, a.log_decay, a.state, a.out, a.H, a.d, a.dv, a.scale, a.in_f32, a.out_f32};
  const int BH = a.B * a.H;
  // narrow columns where heads are few, whole rows of up to 64 where they fill the chip
  if (a.dv <= 16 || (long long)BH * ((a.dv + 15) / 16) <= 4 * device_cu_count()) return launch<16>(p, BH, stream);
  return launch<64>(p, BH, stream);
}

}  // namespace la
