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
//
// What bounds it, measured on the device.  d = dv = 64 in bf16 is bound by memory: B1 H16 N65536 takes 185 us, of which the
// segments' pass 68 (reads 268 MB: 3.9 TB/s), the scan 9, the outputs' pass 106 (536 MB read and written: 5.1 TB/s).  Two
// chunks on their way instead of one left both passes as they were.  d = dv = 128 is bound by a chunk's chain of
// LDS reads and matrix products in the one work-group of eight waves that the registers leave a CU: B4 H8 N3001 takes 58 us
// (16 + 8 + 33); four waves of 32 columns read half as much LDS, but take 370 registers and 15 % longer.  Small calls
// are two or three launches' latencies: B1 H4 N1024 in fp32 15 us.  The gradients of B2 H16 N8192 at d = dv = 64 take 97 us
// (17 + 6 + 74) with the states that the forward pass left.
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
  int join;                    // no scan: a segment adds up the states of those before it
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
  const float x = p.log_decay[h];
  return (x < -1e30f ? -1e30f : x) * 1.44269504088896341f;
}

// g^n for a state: x + x (g^n - 1) where g^n is between a half and two, which keeps slow decays exact over many
// chunks (g^n itself rounds by 2^-24 each time), x g^n elsewhere (below, g^n - 1 would cancel).
struct Fade {
  float f;
  bool slow;
  __device__ __forceinline__ Fade(float lg, int n) {
    const float e = lg * (float)n, x = e * 0.693147180559945309f;
    slow = fabsf(e) < 1.f;
    // e^x - 1 by its series, whose tenth term is below 2^-27 of the first for |x| <= ln 2
    float s = 1.f / 362880.f;
    const float c[8] = {1.f / 40320.f, 1.f / 5040.f, 1.f / 720.f, 1.f / 120.f, 1.f / 24.f, 1.f / 6.f, 0.5f, 1.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(s, x, c[i]);
    f = slow ? s * x : exp2_raw(e);
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

// Chunks of a (b, h)'s rows on their way to an LDS tile of W columns, in registers, one chunk of 64 rows after
// another: row r of the sequence is token r, or token len - 1 - r (rev).  Rows of whole 16-byte pieces (kPieces) or whole
// words (kWords) are read through a buffer over the chunk's rows, so that rows behind the sequence and columns behind the row read
// as zeros without a branch; others by element (bf16, B2 H16 N4096, d = dv = 100: 129 us by words, 210 by element; d = dv = 128: 102).
template <bool F32, int W, int NT, Rows ROWS>
struct RowLoader {
  typedef typename DecayOps<F32>::elem elem;
  static constexpr int E = 16 / sizeof(elem), PIECES = W / E, ALL = C * PIECES, NL = (ALL + NT - 1) / NT;
  static constexpr int RPP = NT / PIECES;      // rows between a thread's pieces, which have one column
  static_assert(NT % PIECES == 0, "a column per thread");
  u32x4 x[NL];
  static constexpr int LOADS = ROWS == kPieces ? 1 : 4;      // of a piece
  int off[LOADS];       // of the first piece, in bytes
  int rb;               // bytes between tokens (kPieces, kWords)
  const elem* p;        // the next chunk's first row in memory, as if it had 64
  long long row;        // elements between tokens
  int w, move;          // move: tokens in memory from one chunk to the next

  // from the chunk at row `first` on, forwards (step 1) or backwards (step -1)
  __device__ __forceinline__ void init(const DecayTensor& t, int b, int h, int width, int rev, int first, int step, int len, int tid) {
    move = rev ? -C * step : C * step;
    row = t.s[2];
    w = width;
    rb = (int)(row * sizeof(elem));
    p = static_cast<const elem*>(t.p) + b * t.s[0] + h * t.s[1] + (rev ? len - first - C : first) * row;
    const int r = tid / PIECES, col = tid % PIECES * E;
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      off[j] = r < C && col + j * (E / 4) < w ? (rev ? C - 1 - r : r) * rb + col * (int)sizeof(elem) + 4 * j : kOffOutOfRange;
  }
  // the next chunk, of n >= 1 rows; the others zeros
  __device__ __forceinline__ void load(int n, int rev, int tid) {
    if constexpr (ROWS != kElements) {
      // from the end, the n rows are the last of the 64: the buffer starts at them, and earlier ones have negative
      // offsets, which are out of range too, as kOffOutOfRange stays with any of these steps
      const int back = rev ? (C - n) * rb : 0, step = rev ? -RPP * rb : RPP * rb;
      const auto rs = make_rsrc(reinterpret_cast<const char*>(p) + back, (u32)((n - 1) * rb + w * (int)sizeof(elem)));
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if constexpr (ROWS == kPieces) {
          x[i] = buf_load_b128(rs, off[0] + (i * step - back));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i][j] = (u32)__builtin_amdgcn_raw_buffer_load_b32(rs, off[j] + (i * step - back), 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int r = tid / PIECES + RPP * i, col = tid % PIECES * E;
        elem e[E];
        const elem* s = p + (long long)(rev ? C - 1 - r : r) * row + col;
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = r < n && col + j < w ? s[j] : (elem)0;
        x[i] = __builtin_bit_cast(u32x4, e);
      }
    }
    p += move * row;
  }
  __device__ __forceinline__ void store(elem* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = tid / PIECES + RPP * i;
      if (ALL % NT == 0 || r < C) *reinterpret_cast<u32x4*>(tile + DecayOps<F32>::template at<W>(r, tid % PIECES * E)) = x[i];
    }
  }
};

// Row of a state's accumulators: entry r of tile t in lane group g is feature 32 (t / 2) + 8 g + 4 (t % 2) + r, so that
// tiles 2 x and 2 x + 1 together are a fragment of the features 32 x + 8 g .. + 7, the order of Q's and K's rows.
__device__ __forceinline__ int state_row(int t, int g, int r) { return 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r; }

// One segment.  OUT: outputs (and, with one segment, the last state); else the segment's own state.
template <bool F32, int DP, int DVP, bool OUT, Rows ROWS>
__global__ __launch_bounds__(4 * DVP) __attribute__((amdgpu_waves_per_eu(DP <= 64 && DVP <= 64 && ROWS == kPieces ? 3 : 1))) void decay_kernel(const DecayParams p) {
  typedef DecayOps<F32> Ops;
  typedef typename Ops::elem elem;
  typedef typename Ops::frag frag;
  constexpr int NW = DVP / 16, NT = 64 * NW, DT = DP / 16, KS = DP / 32, NP = Ops::kPair, NF = Ops::kFine;
  constexpr int KR = Ops::row_elems(DP), VR = Ops::row_elems(DVP), PR = Ops::row_elems(C), KT = C * KR, VT = C * VR, PT = C * PR;
  constexpr int NB = OUT ? 1 : 2;      // tiles of K and V: without outputs there is one barrier a chunk, and two of each
  constexpr int TPW = (10 + NW - 1) / NW;      // score tiles a wave
  // one array, so that addresses in different tiles differ by constants: K, V, Q, P
  constexpr int VS = NB * KT, QS = VS + NB * VT, PS = QS + (OUT ? KT : 0);
  __shared__ __attribute__((aligned(16))) elem lds[PS + (OUT ? NP * PT : 0)];
  __shared__ __attribute__((aligned(16))) float gv[NB][C];      // g^(n - 1 - j) of a chunk's n keys

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, g = lane >> 4;
  int jn;
  const int unit = unit_of(p, jn), bh = unit / p.nseg, seg = unit - bh * p.nseg, b = bh / p.H, h = bh - b * p.H;
  const DecayJob& job = p.job[jn];
  const int len = seq_len(p, b), d = job.d, dv = job.dv, N = p.N, rev = job.rev;
  const int first = seg * p.seg_chunks * C, end = min(N, first + p.seg_chunks * C), stop = min(end, len);
  const int esz = p.out_f32 ? 4 : 2;

  // A segment's own state is a sum in any order: it is taken from the segment's end, so that what this pass read last, the
  // segments' beginnings, is what the outputs' pass reads first, while the memory-side cache still holds it.
  const int begin = OUT || stop <= first ? first : first + (stop - 1 - first) / C * C, step = OUT ? C : -C;
  RowLoader<F32, DP, NT, ROWS> ql, kl;
  RowLoader<F32, DVP, NT, ROWS> vl;
  if (OUT) ql.init(job.q, b, h, d, rev, begin, OUT ? 1 : -1, len, tid);
  kl.init(job.k, b, h, d, rev, begin, OUT ? 1 : -1, len, tid);
  vl.init(job.v, b, h, dv, rev, begin, OUT ? 1 : -1, len, tid);
  auto inside = [&](int r0) { return r0 >= first && r0 < stop; };
  // the rows of the chunk at r0 on their way
  auto load = [&](int r0) {
    if (!inside(r0)) return;
    const int n = min(C, stop - r0);
    if (OUT) ql.load(n, rev, tid);
    kl.load(n, rev, tid);
    vl.load(n, rev, tid);
  };
  load(begin);
  const float lg = log2_decay(p, h);
  // .. and in the tiles, with the weights of its keys: powers to the chunk's end, or the segment's
  auto put = [&](int r0, int buf) {
    if (OUT) ql.store(lds + QS, tid);
    kl.store(lds + buf * KT, tid);
    vl.store(lds + VS + buf * VT, tid);
    if (tid < C) gv[buf][tid] = exp2_raw(lg * (float)max((OUT ? min(C, stop - r0) : stop - r0) - 1 - tid + rev, 0));
  };

  // st[t][r] = S[state_row(t, g, r)][16 w + n16]
  f32x4 st[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) st[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int vd = 16 * w + n16;
  if (OUT && job.state_in != nullptr && (job.seg == nullptr || p.join)) {
    const auto rs = make_rsrc(job.state_in + (size_t)bh * d * dv, (u32)(d * dv * 4));
    const int kstep = (job.in_trans ? 1 : dv) * 4, vat = vd < dv ? vd * (job.in_trans ? d : 1) * 4 : kOffOutOfRange;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kd = state_row(t, g, r);
        st[t][r] = job.in_mul * __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, kd < d ? vat + kd * kstep : kOffOutOfRange, 0, 0));
      }
  }
  if (OUT && job.seg != nullptr) {
    // The record of a segment, or of its transposed state: that one's wave and lane of our row r = 0
    const int rt = state_row(0, g, 0), ttv = 2 * (vd >> 5) + (vd >> 2 & 1), gtv = vd >> 3 & 3;
    const int at0 = job.seg_trans ? ((rt >> 4) * NW + ttv) * 256 + (16 * gtv + (rt & 15)) * 4 + (vd & 3) : w * DT * 256 + 4 * lane;
    auto record = [&](const float* rec, f32x4 (&x)[DT]) {
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        if (job.seg_trans) {
#pragma unroll
          for (int r = 0; r < 4; ++r) x[t][r] = rec[at0 + (t >> 1) * 2 * NW * 256 + (4 * (t & 1) + r) * 4];
        } else {
          x[t] = *reinterpret_cast<const f32x4*>(rec + at0 + t * 256);
        }
      }
    };
    if (!p.join) {
      record(job.seg + (size_t)unit * (DP * DVP), st);
    } else {
      // the states of the segments before this one (whole ones, or this one is empty), a few in flight
      constexpr int FLY = DT <= 2 ? 8 : DT <= 4 ? 4 : 1;
      const Fade skip(lg, p.seg_chunks * C);
      const float* rec = job.seg + (size_t)bh * p.nseg * (DP * DVP);
      for (int i = 0; i < seg; i += FLY) {
        f32x4 x[FLY][DT];
#pragma unroll
        for (int j = 0; j < FLY; ++j)
          if (i + j < seg) record(rec + (size_t)(i + j) * (DP * DVP), x[j]);
#pragma unroll
        for (int j = 0; j < FLY; ++j)
          if (i + j < seg) {
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) st[t][r] = skip(st[t][r]) + x[j][t][r];
          }
      }
    }
  }
  if (OUT && len < end) {      // rows behind the sequence
    const size_t o = (size_t)bh * N * dv;
#pragma unroll 1
    for (size_t i = (size_t)max(first, len) * dv + tid; i < (size_t)end * dv; i += NT) {
      if (p.out_f32) static_cast<float*>(job.out)[o + i] = 0.f;
      else static_cast<uint16_t*>(job.out)[o + i] = 0;
    }
  }
  // Score tiles (queries 16 qt.., keys 16 kt..), kt <= qt, are dealt out to the waves; a wave too many repeats the last
  // one.  sd: s g^(i - j) of this lane's places (one query, four keys), 0 above the diagonal.
  auto tile_q = [](int t) { return t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3; };
  f32x4 sd[TPW];
  float gq[4];      // s g^(i + 1) of this lane's query of each tile
#pragma unroll
  for (int i = 0; i < TPW; ++i) {
    const int t = min(w + NW * i, 9), qt = tile_q(t), kt = t - qt * (qt + 1) / 2, gap = 16 * (qt - kt) + n16 - 4 * g;
#pragma unroll
    for (int r = 0; r < 4; ++r) sd[i][r] = gap - r >= 0 ? p.scale * exp2_raw(lg * (float)(gap - r)) : 0.f;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) gq[t] = p.scale * exp2_raw(lg * (float)(16 * t + n16 + 1 - rev));
  if (OUT)   // tiles above the diagonal that a step of 32 keys reads
    for (int i = tid; i < NP * 512; i += NT) {
      const int part = i >> 9, x = i & 511, tile = x >> 8, row = (x >> 4) & 15, col = x & 15;
      lds[PS + part * PT + Ops::template at<C>(32 * tile + row, 32 * tile + 16 + col)] = (elem)0;
    }
  // this lane's places in a tile: row n16 of Q, K and of P, columns of K and of V
  int krow[KS], prow[2], kcol[KS][2], vcol[2];
#pragma unroll
  for (int x = 0; x < KS; ++x) {
    krow[x] = Ops::template at<DP>(n16, 32 * x + 8 * g);
#pragma unroll
    for (int i = 0; i < 2; ++i) kcol[x][i] = Ops::template col_at<DP, 8>(i, 32 * x, lane);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    prow[i] = PS + Ops::template at<C>(n16, 32 * i + 8 * g);
    vcol[i] = VS + Ops::template col_at<DVP, 4>(i, 16 * w, lane);
  }
  // and in the output's rows of a chunk, in bytes, of its first tile
  const int ob = dv * esz, vd0 = 16 * w + 4 * g;
  const int oat = vd0 < dv ? (rev ? C - 1 - n16 : n16) * ob + vd0 * esz : kOffOutOfRange;
  const bool fine = NF > 2 && job.fine;
  // with one segment, or no scan, the last state is that of the last segment's work-group
  const bool last = OUT && job.state_out != nullptr && (job.seg == nullptr || (p.join && (stop == len && (first < stop || seg == 0))));
  const bool keep = !OUT || last;      // the last chunk's update counts
  const Fade whole(lg, C);

  if (first < stop) {
    put(begin, 0);
    load(begin + step);
  }
  int buf = 0;
  for (int r0 = begin; inside(r0); r0 += step) {
    const int n = min(C, stop - r0);      // tokens of this chunk
    int w0 = w;
    asm volatile("" : "+s"(w0));      // addresses of score tiles are computed anew: their registers would cost a work-group a CU
    lds_barrier();      // tiles are whole, and the last chunk's P has been read
    const elem *kt_ = lds + buf * KT, *vt_ = lds + buf * VT;
    if (!OUT && inside(r0 - C)) {      // the other tiles have been read
      put(r0 - C, buf ^ 1);
      load(r0 - 2 * C);
    }
    frag vf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) vf[s] = Ops::template col<DVP>(vt_ + vcol[0] + 32 * s * VR, vt_ + vcol[1] + 32 * s * VR);
    f32x4 o[4];
    if (OUT) {
      f32x4 sc[TPW];
#pragma unroll
      for (int i = 0; i < TPW; ++i) {
        const int t = min(w0 + NW * i, 9), qt = tile_q(t), kt = t - qt * (qt + 1) / 2;
        sc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < KS; ++x)
          sc[i] = Ops::mma(Ops::row(kt_ + 16 * kt * KR + krow[x]), Ops::row(lds + QS + 16 * qt * KR + krow[x]), sc[i]);
      }
#pragma unroll
      for (int i = 0; i < TPW; ++i) {
        const int t = min(w0 + NW * i, 9), qt = tile_q(t), kt = t - qt * (qt + 1) / 2;
        f32x4 s;      // a score above the diagonal may be infinite
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = sd[i][r] != 0.f ? sc[i][r] * sd[i][r] : 0.f;
        elem* dst = lds + PS + 16 * qt * PR + Ops::template at<C>(n16, 16 * kt + 4 * g);
        if constexpr (F32) {
          *reinterpret_cast<f32x4*>(dst) = s;
        } else {
#pragma unroll
          for (int part = 0; part < NP; ++part) {
            const u32x2 y = {pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
            *reinterpret_cast<u32x2*>(dst + part * PT) = y;
            s[0] -= bf16_lo_to_f32(y[0]);
            s[1] -= bf16_hi_to_f32(y[0]);
            s[2] -= bf16_lo_to_f32(y[1]);
            s[3] -= bf16_hi_to_f32(y[1]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);      // phases kept apart: their operands together would not fit the registers
      // earlier tokens
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) o[qt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const f32x4 a = st[2 * x], e = st[2 * x + 1];
        frag sp[NP];
        Ops::template parts<NP>({{a[0], a[1], a[2], a[3], e[0], e[1], e[2], e[3]}}, sp);
#pragma unroll
        for (int qt = 0; qt < 4; ++qt) {
          const frag qf = Ops::row(lds + QS + 16 * qt * KR + krow[x]);
#pragma unroll
          for (int part = 0; part < NP; ++part) o[qt] = Ops::mma(sp[part], qf, o[qt]);
        }
      }
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) o[qt] *= gq[qt];
      __builtin_amdgcn_sched_barrier(0);
    }
    if (keep || r0 + C < stop) {      // S <- g^n S + K^T (weighted V)
      if (OUT) {
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
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f32x8 x = Ops::widen(vf[s]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x.v[e] *= gv[buf][32 * s + 8 * g + e];
        auto kfrag = [&](int t) {
          const int at = 4 * (t & 1) + 32 * s * KR;
          return Ops::template col<DP>(kt_ + kcol[t / 2][0] + at, kt_ + kcol[t / 2][1] + at);
        };
        if (fine) {      // all parts, the least first
          frag vp[NF];
          Ops::template parts<NF>(x, vp);
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            const frag kf = kfrag(t);
#pragma unroll
            for (int part = NF - 1; part >= 0; --part) st[t] = Ops::mma(kf, vp[part], st[t]);
          }
        } else {
          frag vp[NP];
          Ops::template parts<NP>(x, vp);
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            const frag kf = kfrag(t);
#pragma unroll
            for (int part = NP - 1; part >= 0; --part) st[t] = Ops::mma(kf, vp[part], st[t]);
          }
        }
      }
    }
    if (OUT) {
      lds_barrier();      // P is whole, and the tiles have been read
      if (r0 + C < stop) {
        put(r0 + C, 0);
        load(r0 + 2 * C);
      }
#pragma unroll
      for (int qt = 0; qt < 4; ++qt)
#pragma unroll
        for (int s = 0; s <= qt / 2; ++s)
#pragma unroll
          for (int part = 0; part < NP; ++part) o[qt] = Ops::mma(vf[s], Ops::row(lds + prow[s] + part * PT + 16 * qt * PR), o[qt]);
      // Rows of the chunk in the output, from token r0 or, from the end, len - r0 - n; the others are out of the buffer's
      // range on either side.
      char* out = static_cast<char*>(job.out) + ((size_t)bh * N + (rev ? len - r0 - n : r0)) * ob;
      if ((dv & 3) == 0) {
        const auto orow = make_rsrc(out, (u32)(n * ob));
        const int back = rev ? (C - n) * ob : 0, step = rev ? -16 * ob : 16 * ob;
#pragma unroll
        for (int qt = 0; qt < 4; ++qt) {
          const int to = oat + (qt * step - back);
          if (p.out_f32) buf_store_b128(__builtin_bit_cast(u32x4, o[qt]), orow, to);
          else buf_store_b64((u32x2){pack_bf16x2(o[qt][0], o[qt][1]), pack_bf16x2(o[qt][2], o[qt][3])}, orow, to);
        }
      } else {
#pragma unroll
        for (int qt = 0; qt < 4; ++qt) {
          const int r = 16 * qt + n16, at = (rev ? n - 1 - r : r) * dv + vd0;
          if (r >= n) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (vd0 + e < dv) {
              if (p.out_f32) reinterpret_cast<float*>(out)[at + e] = o[qt][e];
              else reinterpret_cast<uint16_t*>(out)[at + e] = f32_to_bf16_bits(o[qt][e]);
            }
        }
      }
    } else {
      buf ^= 1;
    }
  }
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    if (!OUT) {
      *reinterpret_cast<f32x4*>(job.seg + ((size_t)unit * NW * DT + w * DT + t) * 256 + 4 * lane) = st[t];
    } else if (last) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kd = state_row(t, g, r);
        if (kd < d && vd < dv) job.state_out[state_at(d, dv, bh, kd, vd, 0)] = st[t][r] * job.out_mul;
      }
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
  const int vec = e >> 8, lane = (e >> 2) & 63, kd = state_row(vec % (DP / 16), lane >> 4, e & 3),
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

// Work-groups a CU that sequences are cut for: as many as run at once at d = dv = 64 (2 to 8 measure alike but for what is
// left over in the last round).
constexpr int kWgsPerCu = 3;
// Bytes of a head's segments' states up to which each segment adds up those before it, without a scan: B1 H4 N1024 in fp32 takes
// 15 us so, 28 with the scan; at B2 H16 N2048, at the limit, the two are equal.
constexpr int kJoinBytes = 1 << 17;

// Segments of a sequence: enough work-groups for the chip, of at least four chunks, six where a state has more bytes than eight
// chunks' keys (B4 H8 N3001 at 128 x 128: 61 us, 66 with four and 75 with eight); but of two as long as there is not one for
// every CU (bf16 H8 N2048 at 128 x 128: 28 us, 46 with more; fp32 47 and 123), and of one for half of the CUs, if the scan stays
// short (H8 N1000 at 64 x 64: 13.6 us, 15.7 with two, fp32 16 and 22; three chunks, H16 N192: 10.0 and 9.3, fp32 12.5 and 16.5;
// one for every CU, B2 H16 N512: 17.7 and 14.6; 128 of one, H2 N8192: 26.5 and 21).
struct Segments {
  int n, chunks;
  bool join;
};
Segments segments(long long BH, int N, int d, int dv) {
  const int chunks = (N + C - 1) / C, few = kJoinBytes / (pad_dim(d) * pad_dim(dv) * (int)sizeof(float));
  const long long want = (long long)kWgsPerCu * device_cu_count() / BH;
  const int least = pad_dim(d) * pad_dim(dv) > 8192 ? 6 : 4;
  const bool single = chunks > 2 && chunks <= 64 && BH * chunks <= device_cu_count() / 2;
  const long long most = single ? chunks : chunks / 2;
  long long n = std::max(std::min(want, (long long)(chunks / least)), std::min(most, device_cu_count() / BH));
  if (n < few) n = std::min({want, most, (long long)few});
  n = std::max(1LL, n);
  Segments s{};
  s.chunks = (int)((chunks + n - 1) / n);
  s.n = (chunks + s.chunks - 1) / s.chunks;
  s.join = s.n > 1 && s.n <= few;
  return s;
}

enum Pass { kStates, kScan, kOutputs };

template <bool F32, int DP, int DVP>
void launch_dims(const DecayParams& p, Pass pass, hipStream_t stream) {
  const dim3 grid((unsigned)(p.units * p.njobs)), block(4 * DVP);
  if (pass == kScan) {
    hipLaunchKernelGGL((decay_scan_kernel<DP, DVP>), dim3((unsigned)(p.units / p.nseg * (DP * DVP / kScanThreads)), (unsigned)p.njobs),
                       dim3(kScanThreads), 0, stream, p);
    return;
  }
  Rows rows = kPieces;
  for (int j = 0; j < p.njobs; ++j) {
    rows = std::min({rows, p.job[j].k.rows, p.job[j].v.rows});
    if (pass == kOutputs) rows = std::min(rows, p.job[j].q.rows);
  }
#define LA_ROWS(R)                                                                                   \
  if (rows == R) {                                                                                   \
    if (pass == kStates)                                                                             \
      hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, false, R>), grid, block, 0, stream, p);         \
    else                                                                                             \
      hipLaunchKernelGGL((decay_kernel<F32, DP, DVP, true, R>), grid, block, 0, stream, p);          \
  }
  LA_ROWS(kPieces) LA_ROWS(kWords) LA_ROWS(kElements)
#undef LA_ROWS
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

DecayParams common(const DecayArgs& a) {
  DecayParams p{};
  p.log_decay = a.log_decay;
  p.lengths = a.lengths;
  p.H = a.H;
  p.N = a.N;
  const Segments s = segments((long long)a.B * a.H, a.N, a.d, a.dv);
  p.seg_chunks = s.chunks;
  p.nseg = s.n;
  p.join = s.join;
  p.units = a.B * a.H * p.nseg;
  p.scale = a.scale;
  return p;
}

}  // namespace

size_t decay_workspace_bytes(long long BH, int N, int d, int dv, int backward) {
  const int n = segments(BH, N, d, dv).n;
  return n > 1 ? (size_t)BH * n * pad_dim(d) * pad_dim(dv) * sizeof(float) * (backward + 1) : 0;
}

int launch_decay_fwd(const DecayArgs& a, hipStream_t stream) {
  DecayParams p = common(a);
  p.out_f32 = a.out_f32;
  DecayJob& j = p.job[0];
  j.q = strided_operand(a.q, a.q_strides, a.d, a.in_f32);
  j.k = strided_operand(a.k, a.k_strides, a.d, a.in_f32);
  j.v = strided_operand(a.v, a.v_strides, a.dv, a.in_f32);
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
    if (!p.join) pass(p, 1, kScan, stream);
  }
  pass(p, 1, kOutputs, stream);
  return (int)hipGetLastError();
}

// dq is the forward sum of (dy, v, k) from S^T; dk and dv are sums from the sequence's end, of (v, dy, q) from
// dS^T and of (k, q, dy) from dS, where dS (not scaled by s) enters divided by s.  Two passes compute the
// states of the segments, S of (k, v), if the forward pass's are not given, and dS of (q, dy), which the three outputs'
// pass shares.
int launch_decay_bwd(const DecayArgs& a, hipStream_t stream) {
  const DecayTensor q = strided_operand(a.q, a.q_strides, a.d, a.in_f32), k = strided_operand(a.k, a.k_strides, a.d, a.in_f32),
                    v = strided_operand(a.v, a.v_strides, a.dv, a.in_f32), dy = strided_operand(a.dout, a.dout_strides, a.dv, a.in_f32);
  DecayParams p = common(a);
  p.out_f32 = a.in_f32;
  auto pass = a.in_f32 ? launch_pass<true> : launch_pass<false>;
  float *s = nullptr, *ds = nullptr;
  if (p.nseg > 1) {
    ds = static_cast<float*>(a.workspace);
    s = a.fwd_states != nullptr ? const_cast<float*>(a.fwd_states) : ds + (size_t)p.units * pad_dim(a.d) * pad_dim(a.dv);
  }
  DecayJob js{}, jd{};      // S, from the beginning, and dS, from the end
  js.k = k, js.v = v, js.seg = s, js.state_in = a.state_in, js.in_mul = js.out_mul = 1.f, js.d = a.d, js.dv = a.dv;
  jd.q = k, jd.k = q, jd.v = dy, jd.out = a.dv_out, jd.seg = ds, jd.state_in = a.dstate_out, jd.state_out = a.dstate_in;
  jd.in_mul = 1.f / a.scale, jd.out_mul = a.scale, jd.d = a.d, jd.dv = a.dv, jd.rev = 1, jd.fine = a.dstate_in != nullptr;
  if (p.nseg > 1) {
    const int jobs = a.fwd_states != nullptr ? 1 : 2;      // the forward pass left S as it is needed
    p.job[0] = jd;
    p.job[1] = js;
    pass(p, jobs, kStates, stream);
    if (!p.join) pass(p, jobs, kScan, stream);
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
