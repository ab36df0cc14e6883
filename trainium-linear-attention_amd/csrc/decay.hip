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
// far from 64 bits as their own rounding.  Weighted values enter the update as two as well, or as three (24 bits)
// where the state is an output, which is fp32 and has fp32's accuracy.  fp32 inputs run on fp32 matrix
// instructions throughout.
#include <math.h>

#include <algorithm>

#include "la_decay.hpp"

namespace la {

namespace {

constexpr int C = kDecayC;

// One sum of the form above: its operands (in their roles), its states and its output.
struct DecayJob {
  DecayTensor q, k, v;
  void* out;                   // contiguous (B, H, N, dv)
  const float* state_in;       // (B, H, d, dv) or null; in_trans: (B, H, dv, d)
  float* state_out;            // or null
  float* seg;                  // segment states, DP DVP each, in accumulator order; null: one segment
  float in_mul, out_mul;       // state_in is taken times in_mul, state_out written times out_mul
  int d, dv;
  int rev;                     // from the sequence's end
  int in_trans, seg_trans;     // state_in, the segments' states are of the transposed state
  int fine;                    // a state is an output: weighted values enter its updates in full
};

struct DecayParams {
  const float* log_decay;      // (H)
  const int* lengths;          // (B) or null: N
  int H, N, nseg, seg_chunks, units, njobs;   // units: (head, segment) pairs; work-groups: units njobs
  float scale;
  int out_f32;
  DecayJob job[3];
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

// A work-group's job and its (head, segment).  Work-groups go to the eight XCDs in turn: the jobs of one
// (head, segment), which read the same tensors, are given to one XCD one after another, and meet in its L2.
__device__ __forceinline__ int unit_of(const DecayParams& p, int& job) {
  const int id = blockIdx.x;
  if ((p.units & 7) == 0) {
    const int slot = id >> 3;
    job = slot % p.njobs;
    return slot / p.njobs * 8 + (id & 7);
  }
  job = id % p.njobs;
  return id / p.njobs;
}

// Chunks of a (b, h)'s rows on their way to an LDS tile of W columns, in registers: row r of the sequence
// is token r, or token len - 1 - r (rev).  VEC: rows are whole 16-byte pieces, read through a buffer over
// the chunk's rows, so that rows behind the sequence and columns behind the row read as zeros without a branch.
template <bool F32, int W, int NT, bool VEC>
struct RowLoader {
  typedef typename DecayOps<F32>::elem elem;
  static constexpr int LD = W + DecayOps<F32>::kPad, E = 16 / sizeof(elem), PIECES = W / E, ALL = C * PIECES, NL = (ALL + NT - 1) / NT;
  u32x4 x[NL];
  int off[NL];
  const elem* base;
  long long row;        // elements between tokens
  int w, rev;

  __device__ __forceinline__ void init(const DecayTensor& t, int b, int h, int width, int reversed, int tid) {
    base = static_cast<const elem*>(t.p) + b * t.s[0] + h * t.s[1];
    row = t.s[2];
    w = width;
    rev = reversed;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int at = tid + NT * i, r = at / PIECES, col = at % PIECES * E;
      off[i] = at < ALL && col < w ? (rev ? C - 1 - r : r) * (int)(row * sizeof(elem)) + col * (int)sizeof(elem) : kOffOutOfRange;
    }
  }
  // rows r0 .. r0 + n - 1 (n <= 64) of len; the others zeros
  __device__ __forceinline__ void load(int r0, int n, int len, int tid) {
    if (VEC) {
      // n >= 1: a last load past the end is of the last chunk again, and not used
      const int rb = (int)(row * sizeof(elem));
      const auto rs = make_rsrc(base + (rev ? len - r0 - n : r0) * row, (u32)((n - 1) * rb + w * (int)sizeof(elem)));
      const int back = rev ? (C - n) * rb : 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) x[i] = buf_load_b128(rs, off[i] - back);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int at = tid + NT * i, r = at / PIECES, col = at % PIECES * E;
        elem e[E];
        const elem* s = base + (long long)(rev ? len - 1 - r0 - r : r0 + r) * row + col;
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = at < ALL && r < n && col + j < w ? s[j] : (elem)0;
        x[i] = __builtin_bit_cast(u32x4, e);
      }
    }
  }
  __device__ __forceinline__ void store(elem* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int at = tid + NT * i;
      if (ALL % NT == 0 || at < ALL) *reinterpret_cast<u32x4*>(tile + at / PIECES * LD + at % PIECES * E) = x[i];
    }
  }
};

// One segment.  OUT: outputs (and, with one segment, the last state); else the segment's own state.
template <bool F32, int DP, int DVP, bool OUT, bool VEC>
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
  __shared__ __attribute__((aligned(16))) float gq[C], gv[C];      // g^(i + 1) of the queries, g^(n - 1 - j) of a chunk's n keys

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  int jn;
  const int unit = unit_of(p, jn), bh = unit / p.nseg, seg = unit - bh * p.nseg, b = bh / p.H, h = bh - b * p.H;
  const DecayJob& job = p.job[jn];
  const int len = seq_len(p, b), d = job.d, dv = job.dv, N = p.N, rev = job.rev;
  const int first = seg * p.seg_chunks * C, end = min(N, first + p.seg_chunks * C), stop = min(end, len);
  const float lg = log2_decay(p, h);
  const int esz = p.out_f32 ? 4 : 2;

  // st[t][r] = S[16 t + 4 g + r][16 w + n16]
  f32x4 st[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    st[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (OUT) {
      if (job.seg != nullptr) {
        const float* rec = job.seg + (size_t)unit * (DP * DVP);
        if (job.seg_trans) {      // the record is of the transposed state
#pragma unroll
          for (int r = 0; r < 4; ++r) st[t][r] = rec[(t * NW + w) * 256 + (n16 >> 2) * 64 + (4 * g + r) * 4 + (n16 & 3)];
        } else {
          st[t] = *reinterpret_cast<const f32x4*>(rec + (w * DT + t) * 256 + 4 * lane);
        }
      } else if (job.state_in != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kd = 16 * t + 4 * g + r, vd = 16 * w + n16;
          if (kd < d && vd < dv) st[t][r] = job.state_in[state_at(d, dv, bh, kd, vd, job.in_trans)] * job.in_mul;
        }
      }
    }
  }
  if (OUT) {      // rows behind the sequence
    const size_t o = (size_t)bh * N * dv;
    for (size_t i = (size_t)max(first, len) * dv + tid; i < (size_t)end * dv; i += NT) {
      if (p.out_f32) static_cast<float*>(job.out)[o + i] = 0.f;
      else static_cast<uint16_t*>(job.out)[o + i] = 0;
    }
  }
  const Fade whole(lg, C);
  if (tid < C) {
    gq[tid] = exp2_raw(lg * (float)(tid + 1 - rev));
    gv[tid] = exp2_raw(lg * (float)(C - 1 - tid + rev));
  }
  if (OUT)   // tiles above the diagonal that a step of 32 keys reads
    for (int i = tid; i < NP * 512; i += NT) {
      const int part = i >> 9, x = i & 511, tile = x >> 8, row = (x >> 4) & 15, col = x & 15;
      Ps[(part * C + 32 * tile + row) * LDP + 32 * tile + 16 + col] = (elem)0;
    }
  const bool fine = NF > 1 && job.fine;

  RowLoader<F32, DP, NT, VEC> ql, kl;
  RowLoader<F32, DVP, NT, VEC> vl;
  if (OUT) ql.init(job.q, b, h, d, rev, tid);
  kl.init(job.k, b, h, d, rev, tid);
  vl.init(job.v, b, h, dv, rev, tid);
  if (first < stop) {
    const int n = min(C, stop - first);
    if (OUT) ql.load(first, n, len, tid);
    kl.load(first, n, len, tid);
    vl.load(first, n, len, tid);
  }
  const bool keep = !OUT || (job.seg == nullptr && job.state_out != nullptr);      // the last chunk's update counts

  for (int r0 = first; r0 < stop; r0 += C) {
    const int n = min(C, stop - r0);      // tokens of this chunk
    __syncthreads();
    if (OUT) ql.store(Qs, tid);
    kl.store(Ks, tid);
    vl.store(Vs, tid);
    if (n < C && tid < C) gv[tid] = exp2_raw(lg * (float)max(n - 1 - tid + rev, 0));
    {      // the next chunk's rows, in flight while this one is computed
      const int next = r0 + C < stop ? r0 + C : r0, m = min(C, stop - next);
      if (OUT) ql.load(next, m, len, tid);
      kl.load(next, m, len, tid);
      vl.load(next, m, len, tid);
    }
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
      // rows of the chunk in the output, from token r0 or, from the end, len - r0 - n
      const auto orow = make_rsrc(static_cast<char*>(job.out) + ((size_t)bh * N + (rev ? len - r0 - n : r0)) * (dv * esz), (u32)(n * dv * esz));
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
        const int r = 16 * qt + n16, vd = 16 * w + 4 * g, at = ((rev ? n - 1 - r : r) * dv + vd) * esz;
        if ((dv & 3) == 0) {      // rows from n on are out of the buffer's range on either side
          const int to = vd < dv ? at : kOffOutOfRange;
          if (p.out_f32) buf_store_b128(__builtin_bit_cast(u32x4, o), orow, to);
          else buf_store_b64((u32x2){pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])}, orow, to);
        } else if (r < n) {
          const size_t to = ((size_t)bh * N + (rev ? len - 1 - r0 - r : r0 + r)) * dv + vd;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (vd + e < dv) {
              if (p.out_f32) static_cast<float*>(job.out)[to + e] = o[e];
              else static_cast<uint16_t*>(job.out)[to + e] = f32_to_bf16_bits(o[e]);
            }
        }
      }
      if (r0 + C >= stop && !keep) break;
    }
    // S <- g^n S + K^T (weighted V)
    const Fade fade = n == C ? whole : Fade(lg, n);
    if (fade.slow) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[t][r] = __builtin_fmaf(st[t][r], fade.f, st[t][r]);
    } else {
#pragma unroll
      for (int t = 0; t < DT; ++t) st[t] *= fade.f;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x8 x = Ops::widen(vf[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x.v[e] *= gv[32 * s + 8 * g + e];
      frag vp[NF];
      Ops::template parts<NF>(x, vp);
      frag kf[DT];
#pragma unroll
      for (int t = 0; t < DT; ++t) kf[t] = Ops::col(Ks, LDK, 32 * s, 16 * t, lane);
      if (fine) {
#pragma unroll
        for (int t = 0; t < DT; ++t) st[t] = Ops::mma(kf[t], vp[NF - 1], st[t]);
      }
#pragma unroll
      for (int part = NF > 1 ? NF - 2 : 0; part >= 0; --part)
#pragma unroll
        for (int t = 0; t < DT; ++t) st[t] = Ops::mma(kf[t], vp[part], st[t]);
    }
  }
  if (!OUT) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
      *reinterpret_cast<f32x4*>(job.seg + ((size_t)unit * NW * DT + w * DT + t) * 256 + 4 * lane) = st[t];
  } else if (job.seg == nullptr && job.state_out != nullptr) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kd = 16 * t + 4 * g + r, vd = 16 * w + n16;
        if (kd < d && vd < dv) job.state_out[state_at(d, dv, bh, kd, vd, 0)] = st[t][r] * job.out_mul;
      }
  }
}

// Segments' own states to the states before them, in place, and the last state: a thread has one entry of one
// head, 16 segments' loads in flight.
constexpr int kScanThreads = 64, kScanLoads = 16;
template <int DP, int DVP>
__global__ __launch_bounds__(kScanThreads) void decay_scan_kernel(const DecayParams p) {
  constexpr int REC = DP * DVP, per = REC / kScanThreads;
  const DecayJob& job = p.job[blockIdx.y];
  const int bh = blockIdx.x / per, e = (blockIdx.x - bh * per) * kScanThreads + threadIdx.x;
  const int b = bh / p.H, h = bh - b * p.H, len = seq_len(p, b), d = job.d, dv = job.dv;
  const int vec = e >> 8, lane = (e >> 2) & 63, kd = 16 * (vec % (DP / 16)) + 4 * (lane >> 4) + (e & 3),
            vd = 16 * (vec / (DP / 16)) + (lane & 15);
  const bool real = kd < d && vd < dv;
  const float lg = log2_decay(p, h);
  const int seg_tokens = p.seg_chunks * C;
  const Fade whole(lg, seg_tokens);
  float s = 0.f;
  if (job.state_in != nullptr && real) s = job.state_in[state_at(d, dv, bh, kd, vd, job.in_trans)] * job.in_mul;
  float* rec = job.seg + (size_t)bh * p.nseg * REC + e;
  for (int i0 = 0; i0 < p.nseg; i0 += kScanLoads) {
    float x[kScanLoads];
#pragma unroll
    for (int j = 0; j < kScanLoads; ++j) x[j] = i0 + j < p.nseg ? rec[(size_t)(i0 + j) * REC] : 0.f;
#pragma unroll
    for (int j = 0; j < kScanLoads; ++j) {
      if (i0 + j >= p.nseg) break;
      rec[(size_t)(i0 + j) * REC] = s;
      const int n = min(seg_tokens, max(0, len - (i0 + j) * seg_tokens));
      s = (n == seg_tokens ? whole : Fade(lg, n))(s) + x[j];
    }
  }
  if (job.state_out != nullptr && real) job.state_out[state_at(d, dv, bh, kd, vd, 0)] = s * job.out_mul;
}

int pad_dim(int x) { return x <= 32 ? 32 : x <= 64 ? 64 : 128; }

#ifndef LA_DECAY_WGS
#define LA_DECAY_WGS 4      // work-groups a CU that sequences are cut for
#endif

// Segments of a sequence: enough work-groups for the chip, at least four chunks each.
int segments(long long BH, int N) {
  const int chunks = (N + C - 1) / C;
  const long long want = ((long long)LA_DECAY_WGS * device_cu_count() + BH - 1) / BH;
  return (int)std::max(1LL, std::min(want, (long long)(chunks / 4)));
}

enum Pass { kStates, kScan, kOutputs };

template <bool F32, int DP, int DVP>
void launch_dims(const DecayParams& p, Pass pass, hipStream_t stream) {
  const dim3 grid((unsigned)(p.units * p.njobs)), block(4 * DVP);
  bool vec = true;
  for (int j = 0; j < p.njobs; ++j) vec = vec && p.job[j].k.vec && p.job[j].v.vec && (pass != kOutputs || p.job[j].q.vec);
  if (pass == kScan)
    hipLaunchKernelGGL((decay_scan_kernel<DP, DVP>), dim3((unsigned)(p.units / p.nseg * (DP * DVP / kScanThreads)), (unsigned)p.njobs),
                       dim3(kScanThreads), 0, stream, p);
  else if (pass == kStates && vec)
    hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, false, true>), grid, block, 0, stream, p);
  else if (pass == kStates)
    hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, false, false>), grid, block, 0, stream, p);
  else if (vec)
    hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, true, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, true, false>), grid, block, 0, stream, p);
}

// One pass over the first n of p's jobs, which have the same widths.
template <bool F32>
void launch_pass(DecayParams p, int n, Pass pass, hipStream_t stream) {
  const int dp = pad_dim(p.job[0].d), dvp = pad_dim(p.job[0].dv);
  p.njobs = n;
#define LA_DECAY(DP, DVP) \
  if (dp == DP && dvp == DVP) return launch_dims<F32, DP, DVP>(p, pass, stream);
  LA_DECAY(32, 32) LA_DECAY(32, 64) LA_DECAY(32, 128)
  LA_DECAY(64, 32) LA_DECAY(64, 64) LA_DECAY(64, 128)
  LA_DECAY(128, 32) LA_DECAY(128, 64) LA_DECAY(128, 128)
#undef LA_DECAY
}

DecayTensor operand(const void* ptr, const long long* s, int w, bool f32) {
  DecayTensor x{ptr, {s[0], s[1], s[2]}, 0};
  const int e = f32 ? 4 : 8;
  // 64 rows stay within 2^29 bytes, a buffer's offsets
  x.vec = (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && w % e == 0 && s[0] % e == 0 && s[1] % e == 0 && s[2] % e == 0 &&
          s[2] * (f32 ? 4 : 2) <= (1 << 23);
  return x;
}

DecayParams common(const DecayArgs& a) {
  DecayParams p{};
  p.log_decay = a.log_decay;
  p.lengths = a.lengths;
  p.H = a.H;
  p.N = a.N;
  const int chunks = (a.N + C - 1) / C, nseg = segments((long long)a.B * a.H, a.N);
  p.seg_chunks = (chunks + nseg - 1) / nseg;
  p.nseg = (chunks + p.seg_chunks - 1) / p.seg_chunks;
  p.units = a.B * a.H * p.nseg;
  p.scale = a.scale;
  return p;
}

}  // namespace

size_t decay_workspace_bytes(long long BH, int N, int d, int dv, bool backward) {
  const int n = segments(BH, N);
  return n > 1 ? (size_t)BH * n * pad_dim(d) * pad_dim(dv) * sizeof(float) * (backward ? 2 : 1) : 0;
}

int launch_decay_fwd(const DecayArgs& a, hipStream_t stream) {
  DecayParams p = common(a);
  p.out_f32 = a.out_f32;
  DecayJob& j = p.job[0];
  j.q = operand(a.q, a.q_strides, a.d, a.in_f32);
  j.k = operand(a.k, a.k_strides, a.d, a.in_f32);
  j.v = operand(a.v, a.v_strides, a.dv, a.in_f32);
  j.out = a.out;
  j.state_in = a.state_in;
  j.state_out = a.state_out;
  j.seg = p.nseg > 1 ? static_cast<float*>(a.workspace) : nullptr;
  j.in_mul = j.out_mul = 1.f;
  j.d = a.d;
  j.dv = a.dv;
  j.fine = a.state_out != nullptr;
  auto pass = a.in_f32 ? launch_pass<true> : launch_pass<false>;
  if (j.seg != nullptr) {
    pass(p, 1, kStates, stream);
    pass(p, 1, kScan, stream);
  }
  pass(p, 1, kOutputs, stream);
  return (int)hipGetLastError();
}

// dq is the forward sum of (dy, v, k) from S^T; dk and dv are sums from the sequence's end, of (v, dy, q) from
// dS^T and of (k, q, dy) from dS, where dS (not scaled by s) enters divided by s.  Two passes compute the
// states of the segments, S of (k, v) and dS of (q, dy), which the three outputs' pass shares.
int launch_decay_bwd(const DecayArgs& a, hipStream_t stream) {
  const DecayTensor q = operand(a.q, a.q_strides, a.d, a.in_f32), k = operand(a.k, a.k_strides, a.d, a.in_f32),
                    v = operand(a.v, a.v_strides, a.dv, a.in_f32), dy = operand(a.dout, a.dout_strides, a.dv, a.in_f32);
  DecayParams p = common(a);
  p.out_f32 = a.in_f32;
  auto pass = a.in_f32 ? launch_pass<true> : launch_pass<false>;
  float *s = nullptr, *ds = nullptr;
  if (p.nseg > 1) {
    s = static_cast<float*>(a.workspace);
    ds = s + (size_t)p.units * pad_dim(a.d) * pad_dim(a.dv);
  }
  DecayJob js{}, jd{};      // S, from the beginning, and dS, from the end
  js.k = k, js.v = v, js.seg = s, js.state_in = a.state_in, js.in_mul = js.out_mul = 1.f, js.d = a.d, js.dv = a.dv;
  jd.q = k, jd.k = q, jd.v = dy, jd.out = a.dv_out, jd.seg = ds, jd.state_in = a.dstate_out, jd.state_out = a.dstate_in;
  jd.in_mul = 1.f / a.scale, jd.out_mul = a.scale, jd.d = a.d, jd.dv = a.dv, jd.rev = 1, jd.fine = a.dstate_in != nullptr;
  if (p.nseg > 1) {
    p.job[0] = js;
    p.job[1] = jd;
    pass(p, 2, kStates, stream);
    pass(p, 2, kScan, stream);
  }
  DecayJob jq = js, jk = jd;
  jq.q = dy, jq.k = v, jq.v = k, jq.out = a.dq, jq.d = a.dv, jq.dv = a.d, jq.seg_trans = jq.in_trans = 1;
  jk.q = v, jk.k = dy, jk.v = q, jk.out = a.dk, jk.d = a.dv, jk.dv = a.d, jk.seg_trans = jk.in_trans = 1;
  jk.state_out = nullptr, jk.fine = 0;
  p.job[0] = jq;
  p.job[1] = jk;
  p.job[2] = jd;
  if (pad_dim(a.d) == pad_dim(a.dv)) {
    pass(p, 3, kOutputs, stream);
  } else {
    pass(p, 2, kOutputs, stream);
    p.job[0] = jd;
    pass(p, 1, kOutputs, stream);
  }
  return (int)hipGetLastError();
}

}  // namespace la
