// An 8-bit cache of keys and values and one-token softmax attention over it, for gfx950.  The layout is
// based_la_cache.h's: blocks of 64 tokens, e4m3 codes with a power-of-two scale for each block and head, the
// values of a block transposed.
//
// Why this layout: a wave takes a block at a time, and every operand of its products is a 16-byte load of
// consecutive codes.  S^T = K Q^T has the block's keys as rows and up to 16 query heads as columns; of its four
// tiles of 16 keys, row 4 g + r of tile m is key 16 g + 4 m + r, so that lane group g ends up with the scores of
// keys 16 g .. + 15, which is the order in which it holds V^T's codes (16 consecutive keys of a value column)
// for O^T = V^T P^T.  Nothing is transposed or passed through LDS before the waves' results are joined.
// Power-of-two scales make x / scale exact, so that a code is rounded once, and codes that move to a larger
// scale only round where they fall below e4m3's normal range.
#include <math.h>

#include <algorithm>

#include "la_common.hpp"
#include "la_decay.hpp"
#include "la_internal.hpp"

namespace la {

namespace {

constexpr int CB = 64;       // tokens of a block

// Exponent of the smallest power of two, 2^-100 at the least, that brings a magnitude (as bits) to 448 = 1.75 2^8
// or below.
__device__ __forceinline__ int scale_exp(u32 bits) {
  return max((int)(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -100);
}
__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (u32)(e + 127) << 23); }
// 1 / s for a power of two within 2^-126 .. 2^126
__device__ __forceinline__ float inv_pow2(float s) { return __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(u32, s)); }
__device__ __forceinline__ u32 finite_mag(float x) {
  const u32 m = __builtin_bit_cast(u32, x) & 0x7fffffffu;
  return m < 0x7f800000u ? m : 0u;
}

// Four values to four codes; what no code stands for (infinities) becomes NaN.
__device__ __forceinline__ u32 encode4(float a, float b, float c, float d) {
  const float nan = __builtin_nanf("");
  a = fabsf(a) > 448.f ? nan : a;
  b = fabsf(b) > 448.f ? nan : b;
  c = fabsf(c) > 448.f ? nan : c;
  d = fabsf(d) > 448.f ? nan : d;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ u32 rescale4(u32 w, float f) {
  return encode4(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * f,
                 __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * f, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * f);
}

// Bytes t .. t + 3 of a mask of valid places lo .. hi - 1.
__device__ __forceinline__ u32 byte_mask(int t, int lo, int hi) {
  u32 m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) m |= t + j >= lo && t + j < hi ? 0xffu << (8 * j) : 0u;
  return m;
}

struct CacheParams {
  DecayTensor k, v;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const int* start;
  const int* lengths;
  int last_of;       // lengths are whole sequences', of which the last token is appended
  int HK, N, d, dv, blocks, in_f32;
};

// Columns col .. col + E - 1 of row r of a block's new rows from .. to - 1 (x: row `from`), zeros in other rows and behind
// a row of w.  Rows of whole pieces or words are read through a buffer over these rows, so that no load waits
// for a branch (bf16, B8 H16 N4096, d = dv = 100: 71 us by words, 152 by element).
template <bool F32, Rows ROWS, int E>
__device__ __forceinline__ void load_row(const void* x, long long stride, int r, int from, int to, int col, int w, float (&y)[E]) {
  constexpr int Z = F32 ? 4 : 2;
  if constexpr (ROWS != kElements) {
    const auto rs = make_rsrc(x, (u32)((to - from - 1) * (int)stride + w) * Z);
    const int at = ((r - from) * (int)stride + col) * Z;
    u32x4 a[E * Z / 16];
#pragma unroll
    for (int i = 0; i < E * Z / 16; ++i) {
      if constexpr (ROWS == kPieces) {
        a[i] = buf_load_b128(rs, col + i * 16 / Z < w ? at + 16 * i : kOffOutOfRange);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[i][j] = (u32)__builtin_amdgcn_raw_buffer_load_b32(rs, col + (4 * i + j) * 4 / Z < w ? at + 16 * i + 4 * j : kOffOutOfRange, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < E * Z / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32 z = a[i][j];
        if constexpr (F32) y[4 * i + j] = __builtin_bit_cast(float, z);
        else y[8 * i + 2 * j] = bf16_lo_to_f32(z), y[8 * i + 2 * j + 1] = bf16_hi_to_f32(z);
      }
  } else {
    const bool there = r >= from && r < to;
    const long long at = (r - from) * stride + col;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      y[j] = 0.f;
      if (there && col + j < w) y[j] = F32 ? static_cast<const float*>(x)[at + j] : bf16_bits_to_f32(static_cast<const uint16_t*>(x)[at + j]);
    }
  }
}

// One block of one (sequence, cached head): blockIdx.x the block among those the call touches.  A thread has E columns
// of a token: 16-byte stores of codes (8 at the narrowest rows, so that every thread has some).  Bound by memory: B8, 8
// heads of 128, 8200 tokens in bf16 take 74 us (403 MB read and written: 5.4 TB/s), B2, 16 heads of 64, 4096 tokens 11 us.
template <bool F32, int DP, int DVP, Rows ROWS>
__global__ __launch_bounds__(256) void cache_append_kernel(const CacheParams p) {
  constexpr int KE = DP >= 64 ? 16 : 8, VE = DVP >= 64 ? 16 : 8, KI = CB * DP / KE / 256, VI = CB * DVP / VE / 256;
  constexpr int KP = DP / KE, VP = DVP / VE, VROW = CB + 4, Z = F32 ? 4 : 2;
  __shared__ u32 top[2][4];
  __shared__ __attribute__((aligned(16))) uint8_t vt[DVP * VROW];
  const int tid = threadIdx.x, bh = blockIdx.y, b = bh / p.HK, hk = bh - b * p.HK;
  int from = p.start ? p.start[b] : 0, n = p.lengths ? min(max(p.lengths[b], 0), p.N) : p.N;
  if (p.last_of) {
    from = p.lengths[b] - 1;
    n = from >= 0 ? 1 : 0;
  }
  const int lb = from / CB + blockIdx.x, end = from + n;      // tokens from .. end - 1
  if (n <= 0 || from < 0 || lb * CB >= end) return;
  if (lb + p.blocks <= (end - 1) / CB) return;                // taken over later in this call
  const int kept = max(from - lb * CB, 0), stop = min(end - lb * CB, CB);
  const size_t rec = (size_t)bh * p.blocks + lb % p.blocks;
  const long long t0 = lb * CB + kept - from;                 // the block's first new token
  const char* kg = static_cast<const char*>(p.k.p) + (b * p.k.s[0] + hk * p.k.s[1] + t0 * p.k.s[2]) * Z;
  const char* vg = static_cast<const char*>(p.v.p) + (b * p.v.s[0] + hk * p.v.s[1] + t0 * p.v.s[2]) * Z;
  uint8_t* kc = p.kc + rec * (CB * DP);
  uint8_t* vc = p.vc + rec * (CB * DVP);

  float kx[KI][KE], vx[VI][VE];
  u32 km = 0, vm = 0;
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int at = tid + 256 * i;
    load_row<F32, ROWS, KE>(kg, p.k.s[2], at / KP, kept, stop, at % KP * KE, p.d, kx[i]);
  }
#pragma unroll
  for (int i = 0; i < VI; ++i) {
    const int at = tid + 256 * i;
    load_row<F32, ROWS, VE>(vg, p.v.s[2], at / VP, kept, stop, at % VP * VE, p.dv, vx[i]);
  }
#pragma unroll
  for (int i = 0; i < KI; ++i)
#pragma unroll
    for (int j = 0; j < KE; ++j) km = max(km, finite_mag(kx[i][j]));
#pragma unroll
  for (int i = 0; i < VI; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) vm = max(vm, finite_mag(vx[i][j]));
  km = wave_max_u32(km);
  vm = wave_max_u32(vm);
  if ((tid & 63) == 0) {
    top[0][tid >> 6] = km;
    top[1][tid >> 6] = vm;
  }
  const float old_k = kept ? p.ks[rec] : 0.f, old_v = kept ? p.vs[rec] : 0.f;
  __syncthreads();
  km = max(max(top[0][0], top[0][1]), max(top[0][2], top[0][3]));
  vm = max(max(top[1][0], top[1][1]), max(top[1][2], top[1][3]));
  const float sk = fmaxf(pow2f(scale_exp(km)), old_k), sv = fmaxf(pow2f(scale_exp(vm)), old_v);
  const float ik = inv_pow2(sk), iv = inv_pow2(sv);
  if (tid == 0) {
    p.ks[rec] = sk;
    p.vs[rec] = sv;
  }
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int at = tid + 256 * i, row = at / KP;
    u32* dst = reinterpret_cast<u32*>(kc + KE * at);
    u32 w[KE / 4];
#pragma unroll
    for (int j = 0; j < KE / 4; ++j)
      w[j] = row < kept ? rescale4(dst[j], old_k * ik)
                        : encode4(kx[i][4 * j] * ik, kx[i][4 * j + 1] * ik, kx[i][4 * j + 2] * ik, kx[i][4 * j + 3] * ik);
    if constexpr (KE == 16) *reinterpret_cast<u32x4*>(dst) = (u32x4){w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<u32x2*>(dst) = (u32x2){w[0], w[1]};
  }
#pragma unroll
  for (int i = 0; i < VI; ++i) {
    const int at = tid + 256 * i, row = at / VP, col = at % VP * VE;
#pragma unroll
    for (int j = 0; j < VE; j += 4) {
      const u32 w = encode4(vx[i][j] * iv, vx[i][j + 1] * iv, vx[i][j + 2] * iv, vx[i][j + 3] * iv);
#pragma unroll
      for (int k = 0; k < 4; ++k) vt[(col + j + k) * VROW + row] = (uint8_t)(w >> (8 * k));
    }
  }
  __syncthreads();
  for (int i = tid; i < DVP * CB / 16; i += 256) {
    const int col = i / (CB / 16), t = i % (CB / 16) * 16;
    u32x4* dst = reinterpret_cast<u32x4*>(vc + col * CB + t);
    const u32* src = reinterpret_cast<const u32*>(vt + col * VROW + t);
    u32x4 w = {src[0], src[1], src[2], src[3]};
    if (t < kept) {
      const u32x4 old = *dst;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32 m = byte_mask(t + 4 * j, 0, kept);
        w[j] = (w[j] & ~m) | (rescale4(old[j], old_v * iv) & m);
      }
    }
    *dst = w;
  }
}

// ---- attention

struct StepParams {
  const void* q;
  const void* k;     // the new tokens (B, HK, d), (B, HK, dv), contiguous; null: they are in the cache already
  const void* v;
  void* out;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  const int* lengths;
  float* part;       // (B H, splits, DVP + 2): O, maximum, sum; or null: one split
  int H, HK, G, d, dv, blocks, window, splits, per;      // per: blocks of a split
  float scale;
  int in_f32, out_f32, q_vec;      // q_vec: rows of q are whole 16-byte pieces (bf16)
};

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf2;

// Eight codes as eight bf16 values (exact)
__device__ __forceinline__ u32x4 codes_bf16(u32 a, u32 b) {
  return (u32x4){__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                 __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true))};
}

__device__ __forceinline__ float load_one(const void* p, size_t i, int f32) {
  return f32 ? static_cast<const float*>(p)[i] : bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// One row of w elements (lane l: elements l, l + 64) as the codes at base + STEP times the element, by one wave, into place
// `at` of a block of BYTES codes; its first place clears the block, and a larger scale than before moves the block's codes
// to it (zeros stay zeros).
template <int W, int STEP, int BYTES>
__device__ __forceinline__ void put_token(const void* row, size_t first, int w, int f32, uint8_t* block, uint8_t* base, float* scale, int at, int lane) {
  float x[(W + 63) / 64];
  u32 m = 0;
#pragma unroll
  for (int i = 0; i < (W + 63) / 64; ++i) {
    x[i] = lane + 64 * i < w ? load_one(row, first + lane + 64 * i, f32) : 0.f;
    m = max(m, finite_mag(x[i]));
  }
  const float old = at ? *scale : 0.f, s = fmaxf(pow2f(scale_exp(wave_max_u32(m))), old), inv = inv_pow2(s);
  if (at == 0 || s != old) {
#pragma unroll
    for (int i = 0; i < BYTES / 1024; ++i) {
      u32x4* dst = reinterpret_cast<u32x4*>(block + 16 * (lane + 64 * i));
      u32x4 y = {0u, 0u, 0u, 0u};
      if (at) {
        y = *dst;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = rescale4(y[j], old * inv);
      }
      *dst = y;
    }
    if (lane == 0) *scale = s;
    // other lanes' bytes of these pieces are written next
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }
#pragma unroll
  for (int i = 0; i < (W + 63) / 64; ++i)
    if (lane + 64 * i < W) base[(size_t)STEP * (lane + 64 * i)] = (uint8_t)encode4(x[i] * inv, 0.f, 0.f, 0.f);
}

// Work-group: up to 16 query heads of one cached head of one sequence, one split of its blocks, which the four
// waves take in turn.  F32: q as three bf16 terms and P as three; bf16 q is itself, P two (16 bits).
// Bound by memory where sequences are long: B8, 32 query and 8 cached heads of 128 over 16384 to 32768 tokens read about
// 400 MB in 82 us (4.9 TB/s).  A window of 64 over 2 x 16 heads of 64 takes 5 us: a launch and three memory latencies.
template <bool F32, int DP, int DVP>
__global__ __launch_bounds__(256) void cache_attn_kernel(const StepParams p) {
  constexpr int NQ = F32 ? 3 : 1, NP = F32 ? 3 : 2, KS = DP / 32, MT = DVP / 16;
  constexpr int KL = DP >= 64 ? DP / 64 : 1;       // loads of a key row per lane, of 16 (DP = 32: 8) bytes
  __shared__ float ms[4][16], ls[4][16];
  __shared__ float os[4][DVP][17];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, ng = (p.G + 15) / 16, hk = blockIdx.y / ng, hg = blockIdx.y - hk * ng, b = blockIdx.z;
  const int h0 = hk * p.G + 16 * hg, nh = min(16, p.G - 16 * hg);      // query heads h0 .. h0 + nh - 1
  const int len = p.lengths[b], last = len - 1;
  // positions p0 .. last, in blocks b0 .. b1 - 1; this split's of them
  int p0 = max(0, (last / CB + 1 - p.blocks) * CB);
  if (p.window > 0) p0 = max(p0, len - p.window);
  const int b0 = p0 / CB, nb = len > 0 ? last / CB + 1 - b0 : 0, per = p.per;
  const int s0 = b0 + split * per, s1 = min(b0 + nb, s0 + per);

  // Q^T: head n16, dims in the order of the key loads; heads behind the last and dims behind d are zeros
  const size_t qat = ((size_t)b * p.H + h0) * p.d;
  constexpr int Z = F32 ? 4 : 2;
  const auto qr = make_rsrc(static_cast<const char*>(p.q) + qat * Z, (u32)(nh * p.d * Z));
  u32x4 qf[KS][NQ];
#pragma unroll
  for (int x = 0; x < KS; ++x) {
    const int c = DP >= 64 ? 64 * (x / 2) + 16 * g + 8 * (x & 1) : 8 * g, at = (n16 * p.d + c) * Z;
    if constexpr (F32) {
      f32x8 y;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y.v[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(qr, c + j < p.d ? at + 4 * j : kOffOutOfRange, 0, 0));
      DecayOps<false>::parts<NQ>(y, qf[x]);
    } else if (p.q_vec) {
      qf[x][0] = buf_load_b128(qr, c < p.d ? at : kOffOutOfRange);
    } else {
      uint16_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(qr, c + j < p.d ? at + 2 * j : kOffOutOfRange, 0, 0);
      qf[x][0] = __builtin_bit_cast(u32x4, e);
    }
  }

  // the new token, by the wave that takes its block, which is that wave's last
  if (p.k != nullptr && s1 == b0 + nb && s1 > s0 && w == ((s1 - 1 - s0) & 3)) {
    const int bhk = b * p.HK + hk, at = last % CB;
    const size_t rec = (size_t)bhk * p.blocks + last / CB % p.blocks;
    uint8_t *kb = p.kc + rec * (CB * DP), *vb = p.vc + rec * (CB * DVP);
    put_token<DP, 1, CB * DP>(p.k, (size_t)bhk * p.d, p.d, p.in_f32, kb, kb + at * DP, p.ks + rec, at, lane);
    put_token<DVP, CB, CB * DVP>(p.v, (size_t)bhk * p.dv, p.dv, p.in_f32, vb, vb + at, p.vs + rec, at, lane);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }

  float m = -INFINITY, l = 0.f;
  f32x4 o[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const float c2 = p.scale * 1.44269504088896341f;
  // A block's keys are loaded while the block before it takes its softmax and its values' product, and its values while its
  // scores are computed: the registers are the same, and a wave has half a block on its way all the time.
  u32x4 kx[4][KL], vx[MT];
  float ks0 = 0.f, vs0 = 0.f;
  auto record = [&](int blk) { return ((size_t)b * p.HK + hk) * p.blocks + blk % p.blocks; };
  auto load_keys = [&](int blk) {
    const size_t rec = record(blk);
    const uint8_t* kc = p.kc + rec * (CB * DP);
    ks0 = p.ks[rec] * c2;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t* row = kc + ((n16 >> 2) * 16 + 4 * t + (n16 & 3)) * DP;
#pragma unroll
      for (int c = 0; c < KL; ++c) {
        if constexpr (DP >= 64) {
          kx[t][c] = *reinterpret_cast<const u32x4*>(row + 64 * c + 16 * g);
        } else {
          const u32x2 y = *reinterpret_cast<const u32x2*>(row + 8 * g);
          kx[t][c] = (u32x4){y[0], y[1], 0u, 0u};
        }
      }
    }
  };
  auto load_values = [&](int blk) {
    const size_t rec = record(blk);
    const uint8_t* vc = p.vc + rec * (CB * DVP);
    vs0 = p.vs[rec];
#pragma unroll
    for (int t = 0; t < MT; ++t) vx[t] = *reinterpret_cast<const u32x4*>(vc + (16 * t + n16) * CB + 16 * g);
  };
  if (s0 + w < s1) {
    load_keys(s0 + w);
    load_values(s0 + w);
  }
  for (int blk = s0 + w; blk < s1; blk += 4) {
    const float ksc = ks0, vsc = vs0;
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const u32x4 kf = codes_bf16(kx[t][x / 2][2 * (x & 1)], kx[t][x / 2][2 * (x & 1) + 1]);
#pragma unroll
        for (int j = NQ - 1; j >= 0; --j) s[t] = mfma16x16x32(kf, qf[x][j], s[t]);
      }
    }
    if (blk + 4 < s1) load_keys(blk + 4);
    const int lo = p0 - blk * CB, hi = len - blk * CB;     // valid places of the block
    const bool edge = lo > 0 || hi < CB;
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][r] *= ksc;
        if (edge) {
          const int key = 16 * g + 4 * t + r;
          if (key < lo || key >= hi) s[t][r] = -INFINITY;
        }
        mx = fmaxf(mx, s[t][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn, fade = exp2_raw(m - ref);
    m = mn;
    l *= fade;
#pragma unroll
    for (int t = 0; t < MT; ++t) o[t] *= fade;
    u32x4 pf[2][NP];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x8 y;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = exp2_raw(s[2 * x + j / 4][j % 4] - ref);
        l += e;
        y.v[j] = e * vsc;
      }
      DecayOps<false>::parts<NP>(y, pf[x]);
    }
    if (edge) {      // places that hold no token of the window may hold anything
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32 mask = byte_mask(16 * g + 4 * j, lo, hi);
#pragma unroll
        for (int t = 0; t < MT; ++t) vx[t][j] &= mask;
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const u32x4 vf = codes_bf16(vx[t][2 * x], vx[t][2 * x + 1]);
#pragma unroll
        for (int j = NP - 1; j >= 0; --j) o[t] = mfma16x16x32(vf, pf[x][j], o[t]);
      }
    if (blk + 4 < s1) load_values(blk + 4);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // join the waves
  if (g == 0) {
    ms[w][n16] = m;
    ls[w][n16] = l;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) os[w][16 * t + 4 * g + r][n16] = o[t][r];
  __syncthreads();
  for (int i = tid; i < nh * DVP; i += 256) {
    const int h = i / DVP, c = i % DVP;
    const float mm = fmaxf(fmaxf(ms[0][h], ms[1][h]), fmaxf(ms[2][h], ms[3][h])), ref = mm == -INFINITY ? 0.f : mm;
    float sum = 0.f, y = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = exp2_raw(ms[x][h] - ref);
      sum = __builtin_fmaf(ls[x][h], f, sum);
      y = __builtin_fmaf(os[x][c][h], f, y);
    }
    const size_t head = (size_t)b * p.H + h0 + h;
    if (p.part != nullptr) {
      float* dst = p.part + (head * p.splits + split) * (DVP + 2);
      dst[c] = y;
      if (c == 0) {
        dst[DVP] = mm;
        dst[DVP + 1] = sum;
      }
    } else if (c < p.dv) {
      y = nb > 0 ? y / sum : 0.f;
      if (p.out_f32) static_cast<float*>(p.out)[head * p.dv + c] = y;
      else static_cast<uint16_t*>(p.out)[head * p.dv + c] = f32_to_bf16_bits(y);
    }
  }
}

// A head's splits: group j of kJoinGroups takes eight at a time, the 8 j-th and on, all in flight; then the groups in order
// (one cached head of 128, 131072 tokens, 410 splits: 20.5 us a step, 43 with one group; eight splits are equal).
constexpr int kJoinGroups = 4;
constexpr int join_columns(int dvp) { return dvp < 64 ? 64 : dvp; }
template <int DVP>
__global__ __launch_bounds__(kJoinGroups * join_columns(DVP)) void cache_combine_kernel(const StepParams p) {
  constexpr int T = join_columns(DVP);
  __shared__ float gm[kJoinGroups], gl[kJoinGroups], gy[kJoinGroups][T];
  const size_t head = blockIdx.x;
  const int t = threadIdx.x % T, group = threadIdx.x / T, c = min(t, DVP - 1);
  const float* src = p.part + head * p.splits * (DVP + 2);
  float m = -INFINITY, sum = 0.f, y = 0.f;
  for (int s0 = 8 * group; s0 < p.splits; s0 += 8 * kJoinGroups) {
    float ms[8], ls[8], os[8], mx = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* part = src + (size_t)min(s0 + i, p.splits - 1) * (DVP + 2);
      ms[i] = part[DVP];
      ls[i] = part[DVP + 1];
      os[i] = part[c];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s0 + i >= p.splits) ms[i] = -INFINITY;
      mx = fmaxf(mx, ms[i]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx, fade = exp2_raw(m - ref);
    sum *= fade;
    y *= fade;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = exp2_raw(ms[i] - ref);
      sum = __builtin_fmaf(ls[i], f, sum);
      y = __builtin_fmaf(os[i], f, y);
    }
    m = mx;
  }
  if (t == 0) {
    gm[group] = m;
    gl[group] = sum;
  }
  gy[group][t] = y;
  __syncthreads();
  if ((int)threadIdx.x >= p.dv) return;
  m = gm[0];
#pragma unroll
  for (int j = 1; j < kJoinGroups; ++j) m = fmaxf(m, gm[j]);
  const float ref = m == -INFINITY ? 0.f : m;
  sum = y = 0.f;
#pragma unroll
  for (int j = 0; j < kJoinGroups; ++j) {
    const float f = exp2_raw(gm[j] - ref);
    sum = __builtin_fmaf(gl[j], f, sum);
    y = __builtin_fmaf(gy[j][t], f, y);
  }
  y = p.lengths[head / p.H] > 0 ? y / sum : 0.f;
  if (p.out_f32) static_cast<float*>(p.out)[head * p.dv + t] = y;
  else static_cast<uint16_t*>(p.out)[head * p.dv + t] = f32_to_bf16_bits(y);
}

template <int DP, int DVP>
int launch_append(const CacheParams& p, int BHK, hipStream_t stream) {
  const dim3 grid((unsigned)((p.N + 2 * CB - 2) / CB), (unsigned)BHK);      // blocks that N tokens may touch
  const Rows rows = std::min(p.k.rows, p.v.rows);
#define LA_ROWS(F32, R) \
  if (p.in_f32 == F32 && rows == R) hipLaunchKernelGGL((cache_append_kernel<F32, DP, DVP, R>), grid, dim3(256), 0, stream, p);
  LA_ROWS(true, kPieces) LA_ROWS(true, kWords) LA_ROWS(true, kElements)
  LA_ROWS(false, kPieces) LA_ROWS(false, kWords) LA_ROWS(false, kElements)
#undef LA_ROWS
  return (int)hipGetLastError();
}

template <bool F32, int DP, int DVP>
int launch_attn(const StepParams& p, int B, hipStream_t stream) {
  const dim3 grid((unsigned)p.splits, (unsigned)(p.HK * ((p.G + 15) / 16)), (unsigned)B);
  hipLaunchKernelGGL((cache_attn_kernel<F32, DP, DVP>), grid, dim3(256), 0, stream, p);
  if (p.part != nullptr)
    hipLaunchKernelGGL((cache_combine_kernel<DVP>), dim3((unsigned)(B * p.H)), dim3(kJoinGroups * join_columns(DVP)), 0, stream, p);
  return (int)hipGetLastError();
}

#define LA_CACHE_DIMS(CALL)                                   \
  if (dp == 32 && dvp == 32) return CALL(32, 32);             \
  if (dp == 32 && dvp == 64) return CALL(32, 64);             \
  if (dp == 32 && dvp == 128) return CALL(32, 128);           \
  if (dp == 64 && dvp == 32) return CALL(64, 32);             \
  if (dp == 64 && dvp == 64) return CALL(64, 64);             \
  if (dp == 64 && dvp == 128) return CALL(64, 128);           \
  if (dp == 128 && dvp == 32) return CALL(128, 32);           \
  if (dp == 128 && dvp == 64) return CALL(128, 64);           \
  return CALL(128, 128);

int append_dims(const CacheParams& p, int BHK, hipStream_t stream) {
  const int dp = sliding_cache_dim(p.d), dvp = sliding_cache_dim(p.dv);
#define LA_CALL(A, B) launch_append<A, B>(p, BHK, stream)
  LA_CACHE_DIMS(LA_CALL)
#undef LA_CALL
}

template <bool F32>
int attn_dims(const StepParams& p, int B, hipStream_t stream) {
  const int dp = sliding_cache_dim(p.d), dvp = sliding_cache_dim(p.dv);
#define LA_CALL(A, C) launch_attn<F32, A, C>(p, B, stream)
  LA_CACHE_DIMS(LA_CALL)
#undef LA_CALL
}

// Splits of a sequence's blocks: as many work-groups as run at once, two a CU, where the longest window is that long (B8, 32 query
// and 8 cached heads of 128 over up to 32768 tokens: 82 us, 96 with three and 85 with four), of four blocks (one a wave) at
// least.  A split has the same number of blocks in every sequence, so that short ones end in fewer work-groups and
// the chip's dispatch evens out a batch of unlike lengths.
int decode_splits(int B, int H, int HK, int blocks, int window, int* per) {
  const long long groups = (long long)B * HK * ((H / HK + 15) / 16);
  const long long most = window > 0 ? std::min<long long>(blocks, (window + 2 * CB - 2) / CB) : blocks;
  const long long want = std::max(1LL, 2LL * device_cu_count() / groups);
  *per = (int)std::max(4LL, (most + want - 1) / want);
  return (int)((most + *per - 1) / *per);
}

}  // namespace

int sliding_cache_dim(int d) { return d < 1 || d > 128 ? 0 : d <= 32 ? 32 : d <= 64 ? 64 : 128; }

size_t sliding_decode_workspace_bytes(int B, int H, int HK, int dv, int blocks, int window) {
  int per;
  const int s = decode_splits(B, H, HK, blocks, window, &per);
  return s > 1 ? (size_t)B * H * s * (sliding_cache_dim(dv) + 2) * sizeof(float) : 0;
}

int launch_sliding_append(const SlidingCacheArgs& a, hipStream_t stream) {
  const CacheParams p{strided_operand(a.k, a.k_strides, a.d, a.in_f32), strided_operand(a.v, a.v_strides, a.dv, a.in_f32), static_cast<uint8_t*>(a.kc),
                      static_cast<uint8_t*>(a.vc), a.ks, a.vs, a.start, a.lengths, a.last_of ? 1 : 0, a.HK, a.N, a.d, a.dv,
                      a.blocks, a.in_f32 ? 1 : 0};
  return append_dims(p, a.B * a.HK, stream);
}

int launch_sliding_decode(const SlidingCacheArgs& a, hipStream_t stream) {
  StepParams p{};
  p.q = a.q;
  p.out = a.out;
  p.kc = static_cast<uint8_t*>(a.kc);
  p.vc = static_cast<uint8_t*>(a.vc);
  p.ks = a.ks;
  p.vs = a.vs;
  if (a.H / a.HK <= 16) {      // one work-group reads the last block, and writes the token to it first
    p.k = a.k;
    p.v = a.v;
  } else {
    const int rc = launch_sliding_append(a, stream);
    if (rc != 0) return rc;
  }
  p.lengths = a.lengths;
  p.H = a.H;
  p.HK = a.HK;
  p.G = a.H / a.HK;
  p.d = a.d;
  p.dv = a.dv;
  p.blocks = a.blocks;
  p.window = a.window;
  p.splits = decode_splits(a.B, a.H, a.HK, a.blocks, a.window, &p.per);
  p.part = p.splits > 1 ? static_cast<float*>(a.workspace) : nullptr;
  p.scale = a.scale;
  p.in_f32 = a.in_f32 ? 1 : 0;
  p.out_f32 = a.out_f32 ? 1 : 0;
  p.q_vec = a.d % 8 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
  return a.in_f32 ? attn_dims<true>(p, a.B, stream) : attn_dims<false>(p, a.B, stream);
}

}  // namespace la
