/*
 * based_la_cache.h -- further entry points of libbased_la.so (based_la.h): an 8-bit cache of keys and values for
 * sliding-window softmax attention, and that attention for one token of each sequence, the companion of
 * la_sliding_window_fwd for decoding.  Conventions, status codes and argument rules are based_la.h's.
 * No reference counterparts (the reference has no decode path).
 *
 * The cache.  A sequence's position p lies in block (p / 64) % blocks at place p % 64: with enough blocks for
 * the longest sequence a plain cache, with fewer a ring of the last ones.  All arrays are the caller's, in
 * device memory, contiguous and 16-byte aligned; a new cache is all zeros:
 *   kc  (B, HK, blocks, 64, dp)    e4m3 codes of the keys, dp = 32, 64 or 128, the least that holds d
 *   vc  (B, HK, blocks, dvp, 64)   e4m3 codes of the values, each block transposed, dvp for dv likewise
 *   ks, vs  (B, HK, blocks)        fp32 scales, powers of two: an entry is its code times its block's scale
 * A block's scale is the smallest power of two, 2^-100 at the least, that brings its largest finite magnitude to
 * 448 or below; codes are rounded to nearest even, and infinities become NaN.  Where later tokens of a block
 * raise its scale, its earlier codes are rounded again under the new one.  Places behind a sequence's last
 * token are not read; an append writes zeros to those of its last block.  A token at the first place of a
 * block takes the block over: the one of `blocks` blocks ago is gone.
 *
 * Limits: 1 <= d, dv <= 128 (LA_ERR_UNSUPPORTED_DIM), 1 <= blocks <= 2^24, B HK <= 65535, N <= 2^29; of a step H <= 65535,
 * B H < 2^24.
 */
#ifndef BASED_LA_CACHE_H
#define BASED_LA_CACHE_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LA_CACHE_BLOCK 64

/* dp (or dvp) for d (or dv): 32, 64 or 128; 0 outside the limits. */
int la_sliding_cache_dim(int d);

/*
 * Tokens into the cache: row t < lengths[b] of sequence b at position start[b] + t.  k: (B, HK, N, d),
 * v: (B, HK, N, dv), strides as in based_la_decay.h (NULL: contiguous).  start (NULL: 0; >= 0) and lengths
 * (NULL: N; taken between 0 and N) are int32 (B) in device memory; positions before start must have been
 * appended before (of the block that start lies in), positions stay below 2^31 - 64.  Rows behind a
 * sequence are not read.
 */
int la_sliding_cache_append(const void* k, const void* v, int in_dtype, void* kc, void* vc, float* ks, float* vs,
                            const int* start, const int* lengths, int B, int HK, int N, int d, int dv, int blocks,
                            const long long* k_strides, const long long* v_strides, void* hip_stream);

/*
 * One token of each sequence: k (B, HK, d) and v (B, HK, dv) go to position lengths[b] - 1, then
 *   out (B, H, dv) = softmax over the last `window` positions up to it of scale q.k, times v,
 * q: (B, H, d), contiguous; query head h reads cached head h / (H / HK).  window 0: every position that the
 * cache holds whole blocks of; else window <= 64 (blocks - 1) + 1 (LA_ERR_BAD_SHAPE), so that no block that it
 * needs has been taken over.  lengths: int32 (B) in device memory, the sequences' tokens with this one; a
 * sequence of lengths[b] <= 0 takes no part: nothing is written to its cache, its output is zero.
 * workspace: la_sliding_decode_workspace_bytes bytes, 16-byte aligned (NULL if 0): partial results where a
 * sequence's blocks are split over work-groups.
 */
size_t la_sliding_decode_workspace_bytes(int B, int H, int HK, int d, int dv, int blocks, int window);
int la_sliding_decode_step(const void* q, const void* k, const void* v, int in_dtype, void* out, int out_dtype,
                           void* kc, void* vc, float* ks, float* vs, const int* lengths, int B, int H, int HK, int d,
                           int dv, int blocks, int window, float scale, void* workspace, size_t workspace_bytes,
                           void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* BASED_LA_CACHE_H */
