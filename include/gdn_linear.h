/*
 * gdn_linear.h -- C ABI of linear attention with a decay for each head and of
 * layer norm, for MI355X (gfx950).  Same conventions as gdn.h: caller-owned
 * device pointers, nothing allocated or synchronised, work enqueued on
 * `stream`, 0 / < 0 (argument error, nothing enqueued) / > 0 (hipError_t),
 * gdn_last_error().  Element types are GDN_DTYPE_* codes (gdn_layer.h).
 *
 * Linear attention, one state [K, V] per v-head (v-head h reads qk-head
 * h / (Hv / Hqk)):
 *     S_t = e^{g_t} S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t
 *   q, k [B, T, Hqk, K], v, o [B, T, Hv, V]  bf16, K and V in {64, 128}
 *   g    [B, T, Hv], or (g_per_head) [Hv], the same decay at every token; a
 *        decay under -150 (-inf: a reset) counts as -150, e^-150 = 0 in fp32
 *   h0, ht [N, Hv, K, V] fp32 (nullable: zeros, not written; ht may be h0)
 *   q_row, k_row, v_row: elements from one token's rows to the next's (a
 *   token's heads contiguous): a multiple of 8, at least the heads' width and
 *   under 2^23.  o is contiguous.  All tensors but g and cu_seqlens are
 *   16-byte aligned.  Under 2^15 v-heads; chunked, segments (a sequence is one
 *   at least) times v-heads times lanes (4 V, backward 2 (K + V)) under 2^32.
 *   cu_seqlens [N + 1] int32 (B == 1) or NULL (N == B), under gdn.h's
 *   contract; a violation found on the device empties every sequence: o (or
 *   the gradients) is zero and ht is h0.
 * The reference (848267592/avelang) has no counterpart.
 */
#ifndef AVELANG_AMD_GDN_LINEAR_H
#define AVELANG_AMD_GDN_LINEAR_H

#include <stddef.h>
#include <stdint.h>

#include "gdn_layer.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Chunked form (prompts, training).  workspace: gdn_linear_chunk_workspace_bytes
 * bytes, for these sizes or for others of the same heads with B, T and N no
 * smaller.  states (nullable): gdn_linear_states_bytes bytes that receive what
 * gdn_linear_chunk_bwd reads of this forward (the state at every chunk's
 * start, 16 bits per value: nine after the leading one); o may then be NULL
 * (states only).
 */
size_t gdn_linear_chunk_workspace_bytes(int B, int T, int Hqk, int Hv, int K, int V, int N,
                                        int has_cu_seqlens);
size_t gdn_linear_states_bytes(int B, int T, int Hv, int K, int V, int N, int has_cu_seqlens);
int gdn_linear_chunk_fwd(const void* q, const void* k, const void* v,
                         long long q_row, long long k_row, long long v_row,
                         const void* g, int g_dtype, int g_per_head,
                         const float* h0, float* ht, void* o, const int32_t* cu_seqlens,
                         int B, int T, int Hqk, int Hv, int K, int V, int N, float scale,
                         void* states, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Its gradients: dO [B, T, Hv, V] bf16 contiguous, dht nullable; dq, dk, dv
 * bf16 contiguous (q's, k's, v's shapes), dg (g's shape and type), dh0 (nullable).
 * None of them may overlap an input or another (dh0 may be dht).
 * dg is formed in fp32, of whatever type, but from these states: up to 2^-9 of
 * its terms each, a few 10^-4 of it over many heads and tokens, more of a single
 * number whose terms cancel.
 * With g_per_head dg is the sum over all tokens, in fp32 and in a fixed order.
 * states: what gdn_linear_chunk_fwd left for these same inputs.
 * Deterministic; workspace: gdn_linear_chunk_bwd_workspace_bytes bytes, likewise.
 */
size_t gdn_linear_chunk_bwd_workspace_bytes(int B, int T, int Hqk, int Hv, int K, int V, int N,
                                            int has_cu_seqlens);
int gdn_linear_chunk_bwd(const void* q, const void* k, const void* v,
                         long long q_row, long long k_row, long long v_row,
                         const void* g, int g_dtype, int g_per_head,
                         const void* dO, const float* dht, const void* states,
                         void* dq, void* dk, void* dv, void* dg, float* dh0,
                         const int32_t* cu_seqlens,
                         int B, int T, int Hqk, int Hv, int K, int V, int N, float scale,
                         void* workspace, size_t workspace_bytes, void* stream);

/*
 * Token by token (decode).  state_indices (nullable, int32 [N]): h0 / ht are a
 * pool [num_slots, Hv, K, V] and sequence n uses slot state_indices[n]; a slot
 * outside the pool marks a padding sequence (state untouched, output rows
 * unwritten).  Sequences that name the same slot leave it untouched and get
 * NaN output rows.  Without state_indices num_slots is N.
 */
int gdn_linear_recurrent_fwd(const void* q, const void* k, const void* v,
                             long long q_row, long long k_row, long long v_row,
                             const void* g, int g_dtype, int g_per_head,
                             const float* h0, float* ht, void* o, const int32_t* cu_seqlens,
                             const int32_t* state_indices,
                             int B, int T, int Hqk, int Hv, int K, int V, int N, int num_slots,
                             float scale, void* stream);

/*
 * Layer norm of `rows` rows of D elements (contiguous):
 *     y = (x - mean) / sqrt(var + eps) * weight + bias
 * with the biased variance, in fp32.  Row r uses row r % heads of weight and
 * bias [heads, D] (w_dtype; each nullable).  stats (nullable, fp32 [rows, 2])
 * receives the mean and 1 / sqrt(var + eps) for gdn_layer_norm_bwd.  Rows times
 * the lanes of one (16 to 64 for rows of up to 2048 16-bit or 1024 32-bit
 * elements, else 256) under 2^32.
 */
int gdn_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats,
                       long long rows, int heads, int D, float eps, int dtype, int w_dtype,
                       void* stream);

/*
 * Its gradients: dx (x's type) and, each nullable, dweight / dbias [heads, D]
 * (w_dtype), summed over the rows in a fixed order; heads * D under 2^28 with
 * either of these.
 */
size_t gdn_layer_norm_bwd_workspace_bytes(long long rows, int heads, int D, int dtype);
int gdn_layer_norm_bwd(const void* x, const void* weight, const void* dy, const float* stats,
                       void* dx, void* dweight, void* dbias, long long rows, int heads, int D,
                       int dtype, int w_dtype, void* workspace, size_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AVELANG_AMD_GDN_LINEAR_H */
