// Pieces shared by the kernels of linear attention with a decay per head (decay.hip): launch
// descriptors, operand fragments for bf16 and fp32, LDS tiles and their staging.
//
// Fragments.  A 16x16 product over 32 contraction indices takes eight of them per lane: lane l holds
// row (A) or column (B) l % 16 and the indices of group g = l / 16.  bf16: one v_mfma_f32_16x16x32_bf16.
// fp32: eight v_mfma_f32_16x16x4_f32, the e-th over element e of the four groups; any assignment of
// indices to (g, e) will do as long as A and B agree, so both types share one layout.
#pragma once

#include "la_common.hpp"
#include "la_internal.hpp"

namespace la {

constexpr int kDecayC = 64;        // tokens per chunk

struct f32x8 {
  float v[8];
};

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

template <bool F32>
struct DecayOps;

template <>
struct DecayOps<false> {
  typedef uint16_t elem;
  typedef u32x4 frag;
  // Rows of an LDS tile are W elements; the 16-byte unit c of row r lies at c ^ swizzle(r), under which no access here
  // has more bank conflicts than its shape forces: 16-byte reads take the lanes of equal lane / 32 and equal parity of
  // lane bits 2..4 in one pass over 64 banks, transposed ones 32 consecutive lanes.
  template <int W>
  static __device__ __forceinline__ int swizzle(int r) {
    const int r2 = (r >> 2) & 1, r23 = ((r >> 2) ^ (r >> 3)) & 1;
    if constexpr (W == 32) return r2 | r23 << 1;
    if constexpr (W == 64) return r2 | (r & 2) | r23 << 2;
    return r2 | (r & 3) << 1 | r23 << 3;
  }
  static constexpr int row_elems(int W) { return W; }
  template <int W>
  static __device__ __forceinline__ int at(int r, int c) { return r * W + ((c >> 3 ^ swizzle<W>(r)) << 3) + (c & 7); }
  static constexpr int kPair = 2;        // parts of a score or state entry in a bf16 product
  static constexpr int kFine = 3;        // parts of a weighted value in the state's update
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b, f32x4 c) { return mfma16x16x32(a, b, c); }
  // Columns 8 c .. + 7 of row r; at(r, 8 c) + the elements of 16 whole rows more, or of another tile
  static __device__ __forceinline__ frag row(const elem* p) { return *reinterpret_cast<const u32x4*>(p); }
  // Rows 8 g .. + 7 of one column for each lane of a 16-lane group: columns c0 + STEP j .. + 3 for lanes 4 j .. 4 j + 3.  Two
  // transposed reads of four rows, in each of which lane i of the group addresses four columns of row i / 4.
  template <int W, int STEP>
  static __device__ __forceinline__ int col_at(int half, int c0, int lane) {
    return at<W>(8 * (lane >> 4 & 3) + (lane >> 2 & 3) + 4 * half, c0 + STEP * (lane & 3));
  }
  template <int W>
  static __device__ __forceinline__ frag col(const elem* p0, const elem* p1) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p0));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p1));
    return (u32x4){a[0], a[1], b[0], b[1]};
  }
  static __device__ __forceinline__ f32x8 widen(const frag& a) {
    f32x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.v[2 * i] = bf16_lo_to_f32(a[i]);
      r.v[2 * i + 1] = bf16_hi_to_f32(a[i]);
    }
    return r;
  }
  // x as P bf16 terms, x = p[0] + p[1] + .. : 8, 16 or 24 significant bits
  template <int P>
  static __device__ __forceinline__ void parts(f32x8 x, frag (&p)[P]) {
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[j][i] = pack_bf16x2(x.v[2 * i], x.v[2 * i + 1]);
        if (j + 1 < P) {
          x.v[2 * i] -= bf16_lo_to_f32(p[j][i]);
          x.v[2 * i + 1] -= bf16_hi_to_f32(p[j][i]);
        }
      }
  }
};

template <>
struct DecayOps<true> {
  typedef float elem;
  typedef f32x8 frag;
  static constexpr int row_elems(int W) { return W + 4; }
  template <int W>
  static __device__ __forceinline__ int at(int r, int c) { return r * (W + 4) + c; }
  static constexpr int kPair = 1;
  static constexpr int kFine = 1;
  static __device__ __forceinline__ f32x4 mma(const frag& a, const frag& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag row(const elem* p) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
    return {{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
  template <int W, int STEP>
  static __device__ __forceinline__ int col_at(int half, int c0, int lane) {
    return at<W>(8 * (lane >> 4 & 3) + 4 * half, c0 + STEP * (lane >> 2 & 3) + (lane & 3));
  }
  template <int W>
  static __device__ __forceinline__ frag col(const elem* p0, const elem* p1) {
    frag r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = p0[e * (W + 4)], r.v[4 + e] = p1[e * (W + 4)];
    return r;
  }
  static __device__ __forceinline__ f32x8 widen(const frag& a) { return a; }
  template <int P>
  static __device__ __forceinline__ void parts(const f32x8& x, frag (&p)[P]) {
    static_assert(P == 1, "fp32 operands are exact");
    p[0] = x;
  }
};

// A barrier for LDS alone: a work-group's global loads and stores stay in flight (__syncthreads() waits for them).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// How an operand's rows are read, by what start, strides and width are multiples of: 16 bytes, 4 bytes, an element.
enum Rows { kElements, kWords, kPieces };

// A (B, H, N, w) operand: element (b, h, t, i) at p + b s[0] + h s[1] + t s[2] + i.
struct DecayTensor {
  const void* p;
  long long s[3];
  Rows rows;
};

inline DecayTensor strided_operand(const void* p, const long long* s, int w, bool f32) {
  auto whole = [&](int bytes) {
    const int e = bytes / (f32 ? 4 : 2);
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && w % e == 0 && s[0] % e == 0 && s[1] % e == 0 && s[2] % e == 0;
  };
  // rows that do not overlap, 64 of them within 2^29 bytes: a buffer's offsets tell rows behind a sequence by their size
  const bool buffer = s[2] >= w && s[2] * (f32 ? 4 : 2) <= (1 << 23);
  return {p, {s[0], s[1], s[2]}, !buffer ? kElements : whole(16) ? kPieces : whole(4) ? kWords : kElements};
}

}  // namespace la
