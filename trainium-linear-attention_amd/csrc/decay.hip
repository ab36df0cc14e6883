// Causal linear attention with a decay for each head, for gfx950.  With g = exp(log_decay) of the head
//   y_t = s (sum_{u <= t} g^(t - u) (q_t . k_u) v_u + g^(t + 1) q_t S_in),
//   S_out = g^L S_in + sum_{u < L} g^(L - 1 - u) k_u v_u^T        (L tokens, S (d x dv), fp32)
// and its gradients, which are sums of the same form: dq is the sum with (dy, v, k) for (q, k, v) and S^T
// for S; dk and dv are it from the sequence's end, with (v, dy, q) and (k, q, dy).
//
// Chunks of 64 tokens.  Inside a chunk the pairs are computed as such, P = mask(Q K^T) g^(i - j), O = P V;
// all earlier tokens enter through the state, O += g^(i + 1) Q S, and S <- g^64 S + K^T (g^(63 - j) V).  A
// sequence is cut into segments of whole chunks, one work-group each: a first pass computes each
// segment's own state, a scan joins them, and the last pass runs each segment from its first state.
//
// A wave owns 16 value columns of everything that has any: its part of the state stays in registers
// (accumulators of K^T V, which are already the A operand of S^T Q^T under a fixed permutation of d), the
// same transposed fragment of V serves V^T P^T and, weighted, the state's update.  The scores are computed
// once, their tiles dealt out to the waves, and go through LDS.
//
// Roundings for bf16 inputs: P and S enter bf16 products as two terms (16 bits), so that outputs are as
// far from 64 bits as their own rounding; the weighted values enter the update as three (24 bits), so that
// states, which are fp32, have fp32's accuracy.  fp32 inputs run on fp32 matrix instructions throughout.
#include <math.h>

#include <algorithm>

#include "la_decay.hpp"

namespace la {

namespace {

constexpr int C = kDecayC;

struct DecayParams {
  DecayTensor q, k, v;
  void* out;                   // contiguous (B, H, N, dv)
  const float* log_decay;      // (H)
  const int* lengths;          // (B) or null: N
  const float* state_in;       // (B, H, d, dv) or null; transposed: (B, H, dv, d)
  float* state_out;            // or null
  float* seg;                  // segment states (BH, nseg, DP * DVP) in accumulator order, or null: nseg = 1
  int H, N, d, dv, nseg, seg_chunks;
  float scale, in_mul, out_mul;   // state_in is taken times in_mul, state_out written times out_mul
  int in_trans, out_f32;
};

__device__ __forceinline__ int seq_len(const DecayParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.N) : p.N;
}

// log2 of the head's decay.  A decay of 0 has log -inf, for which 0 * log is no number: a large
// negative one gives g^0 = 1 and g^n = 0.
__device__ __forceinline__ float log2_decay(const DecayParams& p, int h) {
  return fmaxf(p.log_decay[h], -1e30f) * 1.44269504088896341f;
}

// g^n for a state: x + x (g^n - 1) where g^n is above a half, which keeps slow decays exact over many
// chunks (g^n itself rounds by 2^-24 each time), x g^n below, where g^n - 1 would cancel.
struct Fade {
  float f;
  bool slow;
  __device__ __forceinline__ Fade(float lg, int n) {
    const float e = lg * 0.693147180559945309f * (float)n;
    slow = e > -0.693f;
    f = slow ? expm1f(e) : expf(e);
  }
  __device__ __forceinline__ float operator()(float x) const { return __builtin_fmaf(x, f, slow ? x : 0.f); }
};

// Where entry (kd, vd) of the head's state lies in state_in.
__device__ __forceinline__ size_t state_at(int d, int dv, size_t bh, int kd, int vd, int trans) {
  return trans ? (bh * dv + vd) * d + kd : (bh * d + kd) * dv + vd;
}

// Rows r0 .. r0 + 63 of a sequence of len tokens into an LDS tile of W columns; token of row r: r, or
// len - 1 - r from the end.  Rows from len on and columns from w on are zero.
template <bool F32, int W, int NT, bool REV>
__device__ __forceinline__ void stage(const DecayTensor& x, size_t base, int w, int r0, int len,
                                      typename DecayOps<F32>::elem* tile, int tid) {
  typedef typename DecayOps<F32>::elem elem;
  constexpr int LD = W + DecayOps<F32>::kPad, E = 16 / sizeof(elem), PIECES = W / E;
  const elem* src = static_cast<const elem*>(x.p) + base;
#pragma unroll
  for (int i = 0; i < (C * PIECES + NT - 1) / NT; ++i) {
    const int at = tid + NT * i;
    if ((C * PIECES) % NT != 0 && at >= C * PIECES) break;
    const int row = at / PIECES, col = at % PIECES * E, r = r0 + row;
    u32x4 y = {0u, 0u, 0u, 0u};
    if (r < len && col < w) {
      const elem* s = src + (long long)(REV ? len - 1 - r : r) * x.s[2] + col;
      if (x.vec) {
        y = *reinterpret_cast<const u32x4*>(s);
      } else {
        elem e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = col + j < w ? s[j] : (elem)0;
        y = __builtin_bit_cast(u32x4, e);
      }
    }
    *reinterpret_cast<u32x4*>(tile + row * LD + col) = y;
  }
}

// One segment.  OUT: outputs (and, with one segment, the last state); else the segment's own state.
template <bool F32, int DP, int DVP, bool REV, bool OUT>
__global__ __launch_bounds__(4 * DVP) void decay_kernel(const DecayParams p) {
  typedef DecayOps<F32> Ops;
  typedef typename Ops::elem elem;
  typedef typename Ops::frag frag;
  constexpr int NW = DVP / 16, NT = 64 * NW, DT = DP / 16;
  constexpr int LDK = DP + Ops::kPad, LDV = DVP + Ops::kPad, LDP = C + Ops::kPad, NP = Ops::kPair, NF = Ops::kFine;
  __shared__ __attribute__((aligned(16))) elem Qs[OUT ? C * LDK : 1];
  __shared__ __attribute__((aligned(16))) elem Ks[C * LDK];
  __shared__ __attribute__((aligned(16))) elem Vs[C * LDV];
  __shared__ __attribute__((aligned(16))) elem Ps[OUT ? NP * C * LDP : 1];
  __shared__ float gq[C], gv[C];      // g^(i + 1) of the queries, g^(n - 1 - j) of a chunk's n keys

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x / p.nseg, seg = blockIdx.x - bh * p.nseg, b = bh / p.H, h = bh - b * p.H;
  const int len = seq_len(p, b), d = p.d, dv = p.dv, N = p.N;
  const int first = seg * p.seg_chunks * C, end = min(N, first + p.seg_chunks * C);
  const float lg = log2_decay(p, h);
  const size_t qb = (size_t)(b * p.q.s[0] + h * p.q.s[1]), kb = (size_t)(b * p.k.s[0] + h * p.k.s[1]),
               vb = (size_t)(b * p.v.s[0] + h * p.v.s[1]);

  // st[t][r] = S[16 t + 4 g + r][16 w + n16]
  f32x4 st[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    st[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (OUT) {
      if (p.seg != nullptr) {
        st[t] = *reinterpret_cast<const f32x4*>(p.seg + ((size_t)blockIdx.x * NW * DT + w * DT + t) * 256 + 4 * lane);
      } else if (p.state_in != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kd = 16 * t + 4 * g + r, vd = 16 * w + n16;
          if (kd < d && vd < dv) st[t][r] = p.state_in[state_at(d, dv, bh, kd, vd, p.in_trans)] * p.in_mul;
        }
      }
    }
  }
  const Fade whole(lg, C);
  if (tid < C) {
    gq[tid] = exp2_raw(lg * (float)(tid + (REV ? 0 : 1)));
    gv[tid] = exp2_raw(lg * (float)(C - 1 - tid + (REV ? 1 : 0)));
  }
  if (OUT)   // tiles above the diagonal that a step of 32 keys reads
    for (int i = tid; i < NP * 512; i += NT) {
      const int part = i >> 9, x = i & 511, tile = x >> 8, row = (x >> 4) & 15, col = x & 15;
      Ps[(part * C + 32 * tile + row) * LDP + 32 * tile + 16 + col] = (elem)0;
    }

  for (int r0 = first; r0 < end; r0 += C) {
    const int n = min(C, len - r0);      // tokens of this chunk
    if (n <= 0) {
      if (!OUT) break;
      for (int i = tid; i < C * dv; i += NT) {      // rows behind the sequence
        const int row = r0 + i / dv;
        if (row < N) {
          const size_t o = ((size_t)bh * N + row) * dv + i % dv;
          if (p.out_f32) static_cast<float*>(p.out)[o] = 0.f;
          else static_cast<uint16_t*>(p.out)[o] = 0;
        }
      }
      continue;
    }
    __syncthreads();
    if (OUT) stage<F32, DP, NT, REV>(p.q, qb, d, r0, len, Qs, tid);
    stage<F32, DP, NT, REV>(p.k, kb, d, r0, len, Ks, tid);
    stage<F32, DVP, NT, REV>(p.v, vb, dv, r0, len, Vs, tid);
    if (n < C && tid < C) gv[tid] = exp2_raw(lg * (float)max(n - 1 - tid + (REV ? 1 : 0), 0));
    __syncthreads();
    frag vf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) vf[s] = Ops::col(Vs, LDV, 32 * s, 16 * w, lane);
    if (OUT) {
      // scores: tiles (queries 16 qt.., keys 16 kt..), kt <= qt; a lane has one query and four keys
      for (int t = w; t < 10; t += NW) {
        const int qt = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, kt = t - qt * (qt + 1) / 2;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
          s = Ops::mma(Ops::row(Ks + (16 * kt + n16) * LDK + 32 * x + 8 * g), Ops::row(Qs + (16 * qt + n16) * LDK + 32 * x + 8 * g), s);
        const int gap = 16 * (qt - kt) + n16 - 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = gap - r >= 0 ? s[r] * exp2_raw(lg * (float)(gap - r)) : 0.f;
        elem* dst = Ps + (16 * qt + n16) * LDP + 16 * kt + 4 * g;
        if constexpr (F32) {
          *reinterpret_cast<f32x4*>(dst) = s;
        } else {
#pragma unroll
          for (int part = 0; part < NP; ++part) {
            const u32x2 y = {pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
            *reinterpret_cast<u32x2*>(dst + part * C * LDP) = y;
            s[0] -= bf16_lo_to_f32(y[0]);
            s[1] -= bf16_hi_to_f32(y[0]);
            s[2] -= bf16_lo_to_f32(y[1]);
            s[3] -= bf16_hi_to_f32(y[1]);
          }
        }
      }
      __syncthreads();
      frag sp[DP / 32][NP];
#pragma unroll
      for (int x = 0; x < DP / 32; ++x)
        Ops::template parts<NP>({{st[2 * x][0], st[2 * x][1], st[2 * x][2], st[2 * x][3], st[2 * x + 1][0],
                                  st[2 * x + 1][1], st[2 * x + 1][2], st[2 * x + 1][3]}}, sp[x]);
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        const elem* qrow = Qs + (16 * qt + n16) * LDK + 4 * g;
#pragma unroll
        for (int x = 0; x < DP / 32; ++x) {
          const frag qf = Ops::rows4(qrow + 32 * x, qrow + 32 * x + 16);
#pragma unroll
          for (int part = 0; part < NP; ++part) o = Ops::mma(sp[x][part], qf, o);
        }
        o *= gq[16 * qt + n16];
#pragma unroll
        for (int s = 0; s <= qt / 2; ++s)
#pragma unroll
          for (int part = 0; part < NP; ++part)
            o = Ops::mma(vf[s], Ops::row(Ps + (part * C + 16 * qt + n16) * LDP + 32 * s + 8 * g), o);
        o *= p.scale;
        const int r = r0 + 16 * qt + n16, vd = 16 * w + 4 * g;
        if (r < N && vd < dv) {
          const int t = r < len ? (REV ? len - 1 - r : r) : r;
          if (r >= len) o = (f32x4){0.f, 0.f, 0.f, 0.f};
          const size_t at = ((size_t)bh * N + t) * dv + vd;
          if ((dv & 3) == 0) {
            if (p.out_f32) *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + at) = o;
            else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + at) = (u32x2){pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (vd + e < dv) {
                if (p.out_f32) static_cast<float*>(p.out)[at + e] = o[e];
                else static_cast<uint16_t*>(p.out)[at + e] = f32_to_bf16_bits(o[e]);
              }
          }
        }
      }
      if (r0 + C >= end && (p.seg != nullptr || p.state_out == nullptr)) break;
    }
    // S <- g^n S + K^T (weighted V)
    const Fade fade = n == C ? whole : Fade(lg, n);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[t][r] = fade(st[t][r]);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 x = Ops::widen(vf[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x.v[e] *= gv[32 * s + 8 * g + e];
      frag vp[NF];
      Ops::template parts<NF>(x, vp);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const frag kf = Ops::col(Ks, LDK, 32 * s, 16 * t, lane);
#pragma unroll
        for (int part = NF - 1; part >= 0; --part) st[t] = Ops::mma(kf, vp[part], st[t]);
      }
    }
  }
  if (!OUT) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
      *reinterpret_cast<f32x4*>(p.seg + ((size_t)blockIdx.x * NW * DT + w * DT + t) * 256 + 4 * lane) = st[t];
  } else if (p.seg == nullptr && p.state_out != nullptr) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kd = 16 * t + 4 * g + r, vd = 16 * w + n16;
        if (kd < d && vd < dv) p.state_out[state_at(d, dv, bh, kd, vd, 0)] = st[t][r] * p.out_mul;
      }
  }
}

// Segments' own states to the states before them, in place, and the last state: one thread an entry of
// one head, eight segments' loads in flight.
template <int DP, int DVP>
__global__ __launch_bounds__(256) void decay_scan_kernel(const DecayParams p) {
  constexpr int REC = DP * DVP;
  const int per = REC / 256, bh = blockIdx.x / per, e = (blockIdx.x - bh * per) * 256 + threadIdx.x;
  const int b = bh / p.H, h = bh - b * p.H, len = seq_len(p, b);
  const int vec = e >> 8, lane = (e >> 2) & 63, kd = 16 * (vec % (DP / 16)) + 4 * (lane >> 4) + (e & 3),
            vd = 16 * (vec / (DP / 16)) + (lane & 15);
  const bool real = kd < p.d && vd < p.dv;
  const float lg = log2_decay(p, h);
  const int seg_tokens = p.seg_chunks * C;
  const Fade whole(lg, seg_tokens);
  float s = 0.f;
  if (p.state_in != nullptr && real) s = p.state_in[state_at(p.d, p.dv, bh, kd, vd, p.in_trans)] * p.in_mul;
  float* rec = p.seg + (size_t)bh * p.nseg * REC + e;
  for (int i0 = 0; i0 < p.nseg; i0 += 8) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i0 + j < p.nseg ? rec[(size_t)(i0 + j) * REC] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + j >= p.nseg) break;
      rec[(size_t)(i0 + j) * REC] = s;
      const int n = min(seg_tokens, max(0, len - (i0 + j) * seg_tokens));
      s = (n == seg_tokens ? whole : Fade(lg, n))(s) + x[j];
    }
  }
  if (p.state_out != nullptr && real) p.state_out[state_at(p.d, p.dv, bh, kd, vd, 0)] = s * p.out_mul;
}

int pad_dim(int x) { return x <= 32 ? 32 : x <= 64 ? 64 : 128; }

// Segments of a sequence: enough work-groups for the chip (four a CU), at least four chunks each.
int segments(long long BH, int N) {
  const int chunks = (N + C - 1) / C;
  const long long want = (4LL * device_cu_count() + BH - 1) / BH;
  return (int)std::max(1LL, std::min(want, (long long)(chunks / 4)));
}

template <bool F32, int DP, int DVP, bool REV>
int launch_pass(DecayParams p, int BH, hipStream_t stream) {
  const dim3 grid((unsigned)(BH * p.nseg)), block(4 * DVP);
  if (p.seg != nullptr) {
    hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, REV, false>), grid, block, 0, stream, p);
    hipLaunchKernelGGL((decay_scan_kernel<DP, DVP>), dim3((unsigned)(BH * (DP * DVP / 256))), dim3(256), 0, stream, p);
  }
  hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, REV, true>), grid, block, 0, stream, p);
  return (int)hipGetLastError();
}

template <bool F32, bool REV>
int launch_dims(const DecayParams& p, int BH, hipStream_t stream) {
  const int dp = pad_dim(p.d), dvp = pad_dim(p.dv);
#define LA_DECAY(DP, DVP) \
  if (dp == DP && dvp == DVP) return launch_pass<F32, DP, DVP, REV>(p, BH, stream);
  LA_DECAY(32, 32) LA_DECAY(32, 64) LA_DECAY(32, 128)
  LA_DECAY(64, 32) LA_DECAY(64, 64) LA_DECAY(64, 128)
  LA_DECAY(128, 32) LA_DECAY(128, 64) LA_DECAY(128, 128)
#undef LA_DECAY
  return (int)hipErrorInvalidValue;
}

DecayTensor operand(const void* ptr, const long long* s, int w, bool f32) {
  DecayTensor x{ptr, {s[0], s[1], s[2]}, 0};
  const int e = f32 ? 4 : 8;
  x.vec = (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && w % e == 0 && s[0] % e == 0 && s[1] % e == 0 && s[2] % e == 0;
  return x;
}

int run_pass(const DecayParams& base, bool in_f32, bool rev, int BH, void* workspace, hipStream_t stream) {
  DecayParams p = base;
  p.nseg = segments(BH, p.N);
  const int chunks = (p.N + C - 1) / C;
  p.seg_chunks = (chunks + p.nseg - 1) / p.nseg;
  p.nseg = (chunks + p.seg_chunks - 1) / p.seg_chunks;
  p.seg = p.nseg > 1 ? static_cast<float*>(workspace) : nullptr;
  if (in_f32) return rev ? launch_dims<true, true>(p, BH, stream) : launch_dims<true, false>(p, BH, stream);
  return rev ? launch_dims<false, true>(p, BH, stream) : launch_dims<false, false>(p, BH, stream);
}

}  // namespace

size_t decay_workspace_bytes(long long BH, int N, int d, int dv) {
  const int n = segments(BH, N);
  return n > 1 ? (size_t)BH * n * pad_dim(d) * pad_dim(dv) * sizeof(float) : 0;
}

int launch_decay_fwd(const DecayArgs& a, hipStream_t stream) {
  DecayParams p{};
  p.q = operand(a.q, a.q_strides, a.d, a.in_f32);
  p.k = operand(a.k, a.k_strides, a.d, a.in_f32);
  p.v = operand(a.v, a.v_strides, a.dv, a.in_f32);
  p.out = a.out;
  p.log_decay = a.log_decay;
  p.lengths = a.lengths;
  p.state_in = a.state_in;
  p.state_out = a.state_out;
  p.H = a.H;
  p.N = a.N;
  p.d = a.d;
  p.dv = a.dv;
  p.scale = a.scale;
  p.in_mul = p.out_mul = 1.f;
  p.out_f32 = a.out_f32;
  return run_pass(p, a.in_f32, false, a.B * a.H, a.workspace, stream);
}

int launch_decay_bwd(const DecayArgs& a, hipStream_t stream) {
  const DecayTensor q = operand(a.q, a.q_strides, a.d, a.in_f32), k = operand(a.k, a.k_strides, a.d, a.in_f32),
                    v = operand(a.v, a.v_strides, a.dv, a.in_f32), dy = operand(a.dout, a.dout_strides, a.dv, a.in_f32);
  DecayParams p{};
  p.log_decay = a.log_decay;
  p.lengths = a.lengths;
  p.H = a.H;
  p.N = a.N;
  p.scale = a.scale;
  p.out_f32 = a.in_f32;
  const int BH = a.B * a.H;
  // dq: (dy, v, k), from S^T
  p.q = dy, p.k = v, p.v = k, p.out = a.dq, p.d = a.dv, p.dv = a.d;
  p.state_in = a.state_in, p.in_trans = 1, p.in_mul = p.out_mul = 1.f;
  int rc = run_pass(p, a.in_f32, false, BH, a.workspace, stream);
  if (rc != 0) return rc;
  // dk: (v, dy, q) from the end, from dS^T (not scaled by s, so it enters divided by it)
  p.q = v, p.k = dy, p.v = q, p.out = a.dk;
  p.state_in = a.dstate_out, p.in_mul = 1.f / a.scale;
  rc = run_pass(p, a.in_f32, true, BH, a.workspace, stream);
  if (rc != 0) return rc;
  // dv: (k, q, dy) from the end, from dS; its last state is the first state's gradient over s
  p.q = k, p.k = q, p.v = dy, p.out = a.dv_out, p.d = a.d, p.dv = a.dv;
  p.in_trans = 0, p.state_out = a.dstate_in, p.out_mul = a.scale;
  return run_pass(p, a.in_f32, true, BH, a.workspace, stream);
}

}  // namespace la
