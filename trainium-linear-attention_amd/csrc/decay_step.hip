// One token of linear attention with a decay per head, for gfx950: per head, with g = exp(log_decay),
//   S <- g S + k v^T (d x dv, fp32, in place),   y = s q^T S.
//
// A work-group has CW consecutive value columns of one head, so that no sum crosses work-groups; its
// threads take CW / 4 columns of four and, in between, rows of the state.  All of a thread's rows are loaded
// before any is used.  Bound by memory in batches, where the state is read and written once: B64 H16, d = dv = 128 takes
// 20.3 us on the device (134 MB: 6.6 TB/s).  Small calls are a launch and two memory latencies: 3.4 us for B2 H16 at 64.
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

// VEC: rows of whole 16-byte pieces (dv % 4 == 0).  The state is read and written through a buffer over the head, so that
// rows from d on and columns from dv on need no branches, which would put a wait before every load.
template <int CW, bool VEC>
__global__ __launch_bounds__(kStepThreads) void decay_step_kernel(const StepParams p) {
  constexpr int NT = kStepThreads, LPR = CW / 4, RPP = NT / LPR, PASSES = 128 / RPP;      // lanes a row, rows a pass
  __shared__ float qs[128], ks[128];
  __shared__ __attribute__((aligned(16))) float red[4][CW];
  const int bh = blockIdx.x, tid = threadIdx.x, d = p.d, dv = p.dv;
  const int col = blockIdx.y * CW + 4 * (tid % LPR), row = tid / LPR;
  const auto rs = make_rsrc(p.state + (size_t)bh * d * dv, (u32)(d * dv * 4));
  int at[4];      // of the first row's columns, in bytes
#pragma unroll
  for (int e = 0; e < 4; ++e) at[e] = col + e < dv ? (row * dv + col + e) * 4 : kOffOutOfRange;
  const int step = RPP * dv * 4;
  f32x4 x[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (VEC) {
      x[i] = __builtin_bit_cast(f32x4, buf_load_b128(rs, at[0] + i * step));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at[e] + i * step, 0, 0));
    }
  }
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = col + e < dv ? elem(p.v, (size_t)bh * dv + col + e, p.in_f32) : 0.f;
  if (tid < 128) qs[tid] = tid < d ? elem(p.q, (size_t)bh * d + tid, p.in_f32) : 0.f;
  else ks[tid - 128] = tid - 128 < d ? elem(p.k, (size_t)bh * d + tid - 128, p.in_f32) : 0.f;
  const float g = expf(p.log_decay[bh % p.H]);
  __syncthreads();
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const float kr = ks[row + RPP * i], qr = qs[row + RPP * i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[i][e] = __builtin_fmaf(kr, v[e], g * x[i][e]);
      y[e] = __builtin_fmaf(qr, x[i][e], y[e]);
    }
    if (VEC) {
      buf_store_b128(__builtin_bit_cast(u32x4, x[i]), rs, at[0] + i * step);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = x[i][e];      // a bit cast of the vector's element itself compiles to element 0
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(u32, z), rs, at[e] + i * step, 0, 0);
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
    const size_t to = (size_t)bh * dv + c;
    if (p.out_f32) static_cast<float*>(p.out)[to] = o;
    else static_cast<uint16_t*>(p.out)[to] = f32_to_bf16_bits(o);
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
  // 16 columns where heads are few (BH 32, d = dv = 64: 2.8 us, 3.0 with 64), whole rows of 128 where they are many (BH
  // 1024, d = dv = 128: 21.6 us, 6.2 TB/s), else 64 (BH 512, d = dv = 64: 4.5 us, 5.7 with 16 and 5.2 with 128)
  if (a.dv <= 16 || BH * ((a.dv + 63) / 64) < 128) return launch<16>(p, BH, stream);
  if (a.dv > 64 && BH >= 2 * device_cu_count()) return launch<128>(p, BH, stream);
  return a.dv <= 32 ? launch<32>(p, BH, stream) : launch<64>(p, BH, stream);
}

}  // namespace la
