/*
 * gfx950_fmha.h -- C ABI of the MI355X (gfx950) attention forward passes, built
 * into the same library as gfx950_gemm.h (whose status codes and element types
 * it uses): g9_fmha_fwd (below) over equal lengths, g9_varlen_fwd over packed
 * prompts, g9_tree_fwd over a paged cache, and the cache's bookkeeping.
 *
 * g9_fmha_fwd:
 * O = softmax(Q K^T * sm_scale) V for every (batch, query head), non-causal,
 * with grouped K/V heads: query head h reads K/V head h * HK / HQ (HQ a
 * multiple of HK; HK == HQ is plain multi-head, HK == 1 multi-query).  Q, K, V
 * and O hold 16-bit elements (`dtype` G9_F16 or G9_BF16) with head dim 128
 * or 64; scores, softmax and the output accumulator are fp32.
 */
#ifndef GFX950_FMHA_H
#define GFX950_FMHA_H

#include <stddef.h>
#include <stdint.h>

#include "gfx950_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Replaces the launch in run_gluon_attention
 * (kernels/attention/fmha_v4.py:761-790; same interface as
 * kernels/attention/fmha_v3.py:522-549), including its kernel arguments
 * (q, k, v, sm_scale, L, o, the four stride tuples, HQ, HK, N_CTX, SCALE_ON_Q).
 *
 * q, o: B x HQ x S x D; k, v: B x HK x S x D, addressed through strides in
 * ELEMENTS given as (batch, head, seq, dim) -- the order of
 * get_strides_from_layout (kernels/attention/common.py:84-92), so both the
 * bhsd and the bshd layouts (and any other with a unit dim stride) are
 * accepted.  Requirements: D == 128 or D == 64 (the reference's powers of
 * two; its layouts are written for 128), S a multiple of 64, unit dim stride,
 * 16-byte aligned base pointers and batch / head / seq strides, and
 * (S + 256) * seq_stride * 2 < 2^31 bytes for each tensor.
 *
 * lse: optional (NULL to skip) fp32 B x HQ x S, contiguous: the natural-log
 * log-sum-exp of each query's scaled scores (the reference's L / M buffer).
 * scale_on_q != 0 multiplies Q by sm_scale * log2(e) and rounds it to the
 * input type before the loop (SCALE_ON_Q=True, the reference default); 0
 * applies the scale to the fp32 scores.  sm_scale must be positive.
 * variant selects the softmax rescale of the reference kernel of that number:
 * 3 rescales the output accumulator whenever a row's running max grows
 * (kernels/attention/fmha_v3.py:96-152), 4 advances a row's max only when a
 * tile exceeds it by more than 8 (log2 units) and skips the rescale when no
 * row of a wave moved (kernels/attention/fmha_v4.py:143-210, 247-270).  Both
 * give the same softmax up to fp32 rounding; another value -> G9_ERR_SCHEDULE.
 *
 * Launches one kernel on `stream`; allocates nothing.
 */
int g9_fmha_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int64_t B, int64_t HQ,
                int64_t HK, int64_t S, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                const int64_t* v_strides, const int64_t* o_strides, float sm_scale, int dtype, int scale_on_q,
                int variant, void* stream);

/*
 * Packed and paged attention (no reference counterpart: its attention is
 * non-causal over equal lengths).  Common to the entries below:
 *
 * - 16-bit elements (`dtype` G9_F16 or G9_BF16; g9_write_cache moves either),
 *   head dim D 64 or 128; query head h reads K/V head h * HK / HQ.  Scores, the
 *   softmax's maxima and sums, and the accumulation are fp32; each weight is rounded
 *   to the input type before its product with V, as in g9_fmha_fwd (the matrix unit
 *   takes both alike): up to half a step, 2^-8 (bf16) or 2^-11 (fp16), of the average
 *   of |V|.
 * - Strides are in ELEMENTS with a unit head-dim stride left out: (token, head)
 *   for packed tensors, (block, token, head) for caches.  They are multiples of
 *   8 and not negative; base pointers are 16-byte aligned.  What is written (o,
 *   the caches) must not overlap itself; what is only read may (expanded tensors),
 *   but for g9_tree_fwd's caches.  Offsets are 64-bit throughout.
 * - Lengths, tables and offsets are device data, read when the kernel runs.
 *   Whatever they hold, nothing outside the tensors is touched: negative lengths
 *   count as 0, cu_seqlens are held inside the packed tensor, a table entry
 *   outside [0, num_blocks) reads as zeros, and keys behind the table's width are
 *   left out.
 * - cu_seqlens: B + 1 ascending row offsets; rows before cu_seqlens[0] and from
 *   cu_seqlens[B] on belong to no sequence and their outputs stay as they were.
 * - A query with no key it may read gives zeros, and -inf in lse.
 * - Keys that no query may read (cache rows behind a request, unused blocks,
 *   other sequences) have no effect, whatever they hold, NaN included.
 * - Each call enqueues its kernels on `stream`, allocates nothing, synchronises
 *   nothing and can be captured into a graph.
 */

/* Most requests of one g9_assign_slots call, of one g9_tree_fwd call. */
#define G9_SLOTS_MAX_REQUESTS 4096
#define G9_TREE_MAX_REQUESTS 8192

/*
 * Where the next counts[b] tokens of each request go in a paged cache of blocks
 * of block_size tokens.  lengths[b] tokens of request b are in the cache, their
 * blocks in the first ceil(lengths[b] / block_size) entries of its table row.
 *
 * New blocks come from free_blocks[start], free_blocks[start + 1], ... in the
 * order of the requests and of their positions (start = free_start[0], or 0
 * where free_start is NULL) and are entered into the table; taken[0] is their
 * number, also where it is more than the list holds.  cu_seqlens[B + 1] are the
 * offsets of the requests' tokens in the packed batch.  For token t < T,
 * positions[t] is its position in its request and slots[t] = block * block_size
 * + offset, or -1 where the free list or the table's width does not reach (the
 * table entry then becomes -1).  Rows behind the last token get position 0 and
 * slot -1.  Nothing but new table entries depends on earlier results: the same
 * call twice gives the same outputs.  B <= G9_SLOTS_MAX_REQUESTS.
 */
int g9_assign_slots(const int32_t* lengths, const int32_t* counts, int64_t B, int32_t* block_table,
                    int64_t table_stride, int64_t width, const int32_t* free_blocks, int64_t num_free,
                    const int32_t* free_start, int64_t block_size, int64_t T, int32_t* cu_seqlens, int64_t* slots,
                    int64_t* positions, int32_t* taken, void* stream);

/*
 * k and v (T x HK x D) into the caches (num_blocks x block_size x HK x D) at
 * their slots; rows whose slot lies outside the cache are skipped.  Slots must
 * be distinct.  block_size: a power of two, 16 to 1024.
 */
int g9_write_cache(const void* k, const void* v, void* k_cache, void* v_cache, const int64_t* slots, int64_t T,
                   int64_t HK, int64_t D, int64_t num_blocks, int64_t block_size, const int64_t* k_strides,
                   const int64_t* v_strides, const int64_t* kc_strides, const int64_t* vc_strides, void* stream);

/*
 * Attention over packed sequences: q, o T x HQ x D; k, v TK x HK x D; sequence b
 * holds the queries [cu_q[b], cu_q[b+1]) and the keys [cu_k[b], cu_k[b+1]).
 * causal != 0 lets query i of Lq read the keys j <= i + Lk - Lq, so that a prompt
 * whose first part is cached passes its new queries only.  lse: optional fp32
 * HQ x T, contiguous: the natural-log log-sum-exp of each query's scaled scores.
 * (T / 256 + min(B, T)) x HQ below 2^23; token strides below 2^22 elements (of one
 * row, any).
 */
int g9_varlen_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* cu_q,
                  const int32_t* cu_k, int64_t B, int64_t T, int64_t TK, int64_t HQ, int64_t HK, int64_t D,
                  const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                  const int64_t* o_strides, float sm_scale, int dtype, int causal, void* stream);

/*
 * Attention of drafted tokens over a paged cache: request b brings the queries
 * [cu_q[b], cu_q[b+1]), its nodes; its table row (B x width, int32) names the
 * blocks of its lengths[b] context tokens and, at the positions behind them, of
 * its nodes (whose K and V rows are in the cache already).  Node i reads every
 * context token and the nodes j whose bit j % 64 is set in word j / 64 of row
 * cu_q[b] + i of tree_mask (T x words, int64); without a mask the nodes j <= i.
 * One node per request without a mask is plain decoding.  lse as g9_varlen_fwd.
 *
 * B <= G9_TREE_MAX_REQUESTS; width * block_size <= 2^30; the caches' tokens at
 * least D elements apart.
 *
 * workspace: g9_tree_workspace_size bytes, 32-byte aligned, contents arbitrary;
 * it holds partial results between the call's kernels, so calls that can run
 * at the same time need one each.
 */
int g9_tree_fwd(const void* q, const void* k_cache, const void* v_cache, void* o, float* lse,
                const int32_t* block_table, int64_t table_stride, int64_t width, const int32_t* lengths,
                const int32_t* cu_q, const int64_t* tree_mask, int64_t words, int64_t B, int64_t T, int64_t HQ,
                int64_t HK, int64_t D, int64_t num_blocks, int64_t block_size, const int64_t* q_strides,
                const int64_t* kc_strides, const int64_t* vc_strides, const int64_t* o_strides, float sm_scale,
                int dtype, void* workspace, size_t workspace_bytes, void* stream);
size_t g9_tree_workspace_size(int64_t B, int64_t T, int64_t HQ, int64_t HK, int64_t D);

#ifdef __cplusplus
}
#endif

#endif /* GFX950_FMHA_H */
