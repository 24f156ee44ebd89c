/*
 * gdn_attn.h -- C ABI of what stands around a hybrid model's attention layers,
 * for MI355X (gfx950): root-mean-square norm with the residual's addition (in
 * its own type or 8 bits, and its gradients), rotary positions, a paged
 * key-value cache that is quantised as it is written, and attention of the
 * newest tokens over it.  Same conventions as gdn.h: caller-owned device
 * pointers, nothing allocated or synchronised, work enqueued on `stream` of
 * the current device, 0 / < 0 (argument error, nothing enqueued) / > 0
 * (hipError_t), gdn_last_error().  Element types are GDN_DTYPE_* codes
 * (gdn_layer.h) or, for 8 bits, those below.
 * The reference (848267592/avelang) has no counterpart.
 */
#ifndef AVELANG_AMD_GDN_ATTN_H
#define AVELANG_AMD_GDN_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "gdn_layer.h"

#define GDN_DTYPE_E4M3 3 /* 8-bit float of 4 exponent and 3 mantissa bits, largest value 448 */
#define GDN_DTYPE_I8 4   /* 8-bit integers, -127 .. 127 */

#ifdef __cplusplus
extern "C" {
#endif

/*
 * `rows` rows of D elements (contiguous):
 *     h = x + residual, rounded to the residual's type (without one h = x)
 *     y = h rstd (weight + offset),   rstd = 1 / sqrt(mean(h^2) + eps)
 * in fp32.  dtype: x's type; r_dtype: the residual's and h's, x's or fp32;
 * weight [D] (w_dtype; nullable: y = h rstd).  h is written with a residual
 * (it may be x of the same type, or residual).  out_dtype is dtype, or an 8-bit type:
 *     scale[row] = max |y| / M,  y's codes are y / scale rounded (M = 448, 127)
 * A row of zeros has scale 0 and codes 0; one under 2^-100 has the scale of
 * 2^-100; one that is not finite (or whose squares overflow fp32) has a scale
 * of NaN.  y may be x where the types are the same; neither overlaps the weight (y of
 * a single row may be it, of its type).  (h of 2^64 or more: its square
 * overflows fp32, and y is 0 or NaN.)
 */
int gdn_rms_norm_fwd(const void* x, const void* residual, const void* weight, void* y, void* h,
                     float* scale, long long rows, int D, float eps, float offset, int dtype,
                     int r_dtype, int w_dtype, int out_dtype, void* stream);

/*
 * Its gradients, from h (h_dtype: dtype, or fp32 where the residual was), dy
 * (dtype) and, nullable, dh (h_dtype; dL/dh from what else reads h):
 *     dx = rstd (e - hh mean(e hh)) + dh,  e = dy (weight + offset), hh = h rstd
 * in x's type, dr (nullable) the same in h_dtype, dweight (w_dtype; nullable)
 * summed over the rows in a fixed order.  workspace: as many bytes where dweight
 * is wanted (0 for few rows).
 */
size_t gdn_rms_norm_bwd_workspace_bytes(long long rows, int D, int dtype);
int gdn_rms_norm_bwd(const void* h, const void* weight, const void* dy, const void* dh, void* dx,
                     void* dr, void* dweight, long long rows, int D, float eps, float offset,
                     int dtype, int h_dtype, int w_dtype, void* workspace, size_t workspace_bytes,
                     void* stream);

/*
 * Rotary positions of the first R (even) of D elements of every head: pair j at
 * position p turns by the angle p inv_freq[j] (fp64 [R / 2]; formed and reduced
 * to a turn in 64 bits), in fp32:
 *     (a, b) -> magnitude (a cos - b sin, b cos + a sin)
 * pairs (j, j + R / 2), or with `interleaved` (2 j, 2 j + 1); elements R .. D - 1
 * are copied.  `inverse` turns the other way (the gradient).
 * q, k (nullable) [B, T, Hq | Hk, D] into q_out, k_out, elements contiguous:
 * strides holds the elements from one batch, token and head to the next, of q,
 * k, q_out and k_out (3 each).  q_out may be q and k_out k (the same strides: in
 * place, both or none), else they overlap neither; q_out and k_out share no element.
 * positions [B, T]: int32, or int64 with pos_int64; pos_batch: from one batch's
 * to the next's (0: the same positions).
 */
int gdn_rotary(const void* q, const void* k, void* q_out, void* k_out, const long long* strides,
               int B, int T, int Hq, int Hk, int D, const void* positions, int pos_int64,
               long long pos_batch, const double* inv_freq, int R, float magnitude,
               int interleaved, int inverse, int dtype, void* stream);

/*
 * A paged cache: k_cache, v_cache [num_pages, H, page_size, D] of cache_dtype,
 * with 8-bit types k_scale, v_scale [num_pages, H, page_size] fp32 (else NULL).
 * Slot s is row s % page_size of page s / page_size.  D in {64, 128, 256}; the
 * caches 16-byte aligned.
 *
 * write: token t's rows (k, v: strides in elements of token and head, elements
 * contiguous) go to slots[t] (int32, or int64 with slots_int64) as they are
 * (cache_dtype == dtype) or as codes round(x M / max |x|), ties to even, with
 * scale max |x| / M (gdn_rms_norm_fwd's M and limits).  A slot outside the cache
 * is a padding token's: skipped.  What a slot that two tokens name holds
 * afterwards is not defined.  The caches overlap neither each other nor k, v.
 * read: the rows of `slots`, codes times their scales in fp32, rounded to
 * dtype, into k, v [T, H, D] contiguous; a slot outside the cache gives zeros.
 */
int gdn_paged_write(const void* k, const void* v, long long k_token, long long k_head,
                    long long v_token, long long v_head, const void* slots, int slots_int64,
                    void* k_cache, void* v_cache, float* k_scale, float* v_scale, int T, int H,
                    int D, int num_pages, int page_size, int dtype, int cache_dtype,
                    void* stream);
int gdn_paged_read(const void* k_cache, const void* v_cache, const float* k_scale,
                   const float* v_scale, const void* slots, int slots_int64, void* k, void* v,
                   int T, int H, int D, int num_pages, int page_size, int dtype, int cache_dtype,
                   void* stream);

/*
 * Attention of every sequence's newest L tokens over the cache (page_size a
 * multiple of 16): q, o [N, L, Hq, D] of dtype (bf16, f16; q_seq, q_token,
 * q_head: q's strides in elements, multiples of 8, elements contiguous; o
 * contiguous, overlapping neither q nor the caches), lengths [N] int32: tokens that sequence n has cached, the
 * newest L among them; token t of it is row t % page_size of page
 * block_table[n * table_row + t / page_size] (int32).  q-head h reads kv-head
 * h / (Hq / Hkv); row i stands at position p = lengths[n] - L + i and sees the
 * tokens t <= p, with window > 0 those of t > p - window:
 *     o = sum_t e^{s_t} v_t / sum_t e^{s_t},   s_t = scale q . k_t
 *     lse (nullable, fp32 [N, L, Hq]) = log sum_t e^{s_t}
 * A row that sees nothing (a length under L, 0 or negative) is 0, its lse
 * -inf.  Lengths count up to max_length only, for which a table's row must have
 * entries; what a table holds behind a sequence's last page is not looked at, and
 * a page outside the cache makes the rows that see it NaN.  Values that are not
 * finite reach the rows that see their token alone.  cache_dtype is dtype or
 * an 8-bit type (scales then).  Deterministic.
 * workspace (16-byte aligned): gdn_paged_attn_workspace_bytes bytes.
 */
size_t gdn_paged_attn_workspace_bytes(int N, int L, int Hq, int Hkv, int D, int max_length);
int gdn_paged_attn_fwd(const void* q, long long q_seq, long long q_token, long long q_head,
                       const void* k_cache, const void* v_cache, const float* k_scale,
                       const float* v_scale, const int32_t* block_table, long long table_row,
                       const int32_t* lengths, void* o, float* lse, int N, int L, int Hq, int Hkv,
                       int D, int num_pages, int page_size, int max_length, int window,
                       float scale, int dtype, int cache_dtype, void* workspace,
                       size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AVELANG_AMD_GDN_ATTN_H */
