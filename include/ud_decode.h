/*
 * ud_decode.h -- C ABI of the gfx950 decoder attention: grouped-query attention over a paged
 * K/V cache for one new token per sequence, the rotate-half RoPE and the paged cache append.
 *
 * This is the decode-step attention of DictatorEngine's Voxtral decoder (one token per sequence,
 * or up to 8 positions per sequence, Sources/DictatorEngine/Models/Voxtral.swift:347-397), batched
 * over independent sequences whose
 * K/V caches live in fixed-size pages instead of the reference's per-session sliding window
 * (SlidingKV, Voxtral.swift:206-250).  Conventions are those of ud_encoder.h: 0 or a negative
 * ud_status, message in ud_last_error(), device pointers *_dev, asynchronous on hip_stream.
 *
 * Paged cache layout (this library's): k_pages / v_pages hold `num_blocks` pages of
 * [kv_heads][block_size][head_dim] elements (one kv head's rows of a page are contiguous).
 * block_table [n][max_blocks] int32 maps logical block b of sequence i (keys b*block_size ..
 * b*block_size + block_size - 1) to a page.  Entries are read only for blocks that hold a key of
 * the sequence's range; other entries may be anything.
 */
#ifndef UD_DECODE_H
#define UD_DECODE_H

#include <stddef.h>
#include <stdint.h>

#include "ud_encoder.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Replaces Step.attention (Sources/DictatorEngine/Core/Ops.swift:136-169) and its kernels
 * attention_gqa / attention_mq_split + attention_combine
 * (Sources/DictatorEngine/Metal/30_voxtral.metal:45-101, 240-338) for one query token per
 * sequence, reading keys through the page table:
 *   out[i, h] = sum_j softmax_j(q[i, h] . k[i, j, h / (Hq/Hkv)] / sqrt(head_dim)) v[i, j, kvh]
 *   over logical keys j in [ranges[i].x, ranges[i].y) (0 if empty).
 *   q_dev        fp32 [n, q_heads * head_dim] (already rotated)
 *   k/v_pages    kv_dtype (UD_BF16 or UD_F16), layout above
 *   block_table  int32 [n, max_blocks]
 *   ranges_dev   int32 [n, 2] logical key range per sequence; ranges[i].y <= max_blocks*block_size
 *   out_dev      fp32 [n, q_heads * head_dim]
 *   max_keys     an upper bound of ranges[i].y over the batch (sizes the grid)
 *   workspace    device scratch of ud_gqa_workspace_bytes(n, q_heads, head_dim, max_keys) bytes
 * Supported: head_dim in {64, 128}, q_heads % kv_heads == 0, q_heads / kv_heads in {1, 2, 4, 8},
 * block_size 16, n <= 65535, max_keys <= 65535 * 128 (UD_ERR_SHAPE otherwise).
 * Precision: f16 pages are widened and used in fp32 arithmetic, as the reference kernel does.
 * bf16 pages use packed bf16 dot products: q and the softmax probabilities are rounded once to
 * bf16 (products exact, sums in fp32), within the bf16 activation bar (max abs 2e-2, cosine
 * 0.9995).  Each split of the keys rounds its probabilities against its own maximum; at head_dim 128
 * its size (128 or 256 keys) follows n, the query count, kv_heads and max_keys, so the last bits of a
 * sequence's output may differ between calls that differ in these. */
UD_API size_t ud_gqa_workspace_bytes(int32_t n, int32_t q_heads, int32_t head_dim, int32_t max_keys);
UD_API int ud_gqa_attention_paged(int32_t kv_dtype, const float* q_dev, const void* k_pages, const void* v_pages,
                                  const int32_t* block_table, int32_t max_blocks, const int32_t* ranges_dev,
                                  float* out_dev, int32_t n, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                  int32_t block_size, int32_t max_keys, void* workspace, size_t workspace_bytes,
                                  void* hip_stream);

/* Replaces Step.attention with 2 .. 8 queries (Ops.swift:141-162 -> attention_mq_split_f16 +
 * attention_combine, 30_voxtral.metal:240-338; the M positions VoxtralSession.decode passes per
 * call, Voxtral.swift:347-371): n_queries (1 .. 8) query rows per sequence, each with its own key
 * range, over the sequence's pages; every K/V page is read once for all of them.
 *   q_dev        fp32 [n, n_queries, q_heads * head_dim]
 *   ranges_dev   int32 [n, n_queries, 2]: query m of sequence i attends to keys
 *                [ranges[i][m].x, ranges[i][m].y) (0 if empty)
 *   out_dev      fp32 [n, n_queries, q_heads * head_dim]
 *   workspace    ud_gqa_workspace_bytes(n * n_queries, q_heads, head_dim, max_keys) bytes
 * Block-table entries are read for the blocks between the lowest start and the highest end of a
 * sequence's non-empty query ranges.  Otherwise as ud_gqa_attention_paged (formula, formats,
 * precision, limits; n * n_queries <= 65535), which is this call with n_queries = 1. */
UD_API int ud_gqa_attention_paged_mq(int32_t kv_dtype, const float* q_dev, const void* k_pages, const void* v_pages,
                                     const int32_t* block_table, int32_t max_blocks, const int32_t* ranges_dev,
                                     float* out_dev, int32_t n, int32_t n_queries, int32_t q_heads, int32_t kv_heads,
                                     int32_t head_dim, int32_t block_size, int32_t max_keys, void* workspace,
                                     size_t workspace_bytes, void* hip_stream);

/* Allocation-free variant of ud_gqa_attention_paged.  It has no counterpart in the reference: it
 * is for callers that cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  Same arguments, kernels and results as
 * ud_gqa_attention_paged, minus the workspace: the split partials go to a static device array of
 * UD_GQA_NOALLOC_SCRATCH_BYTES per device, held until the process ends (its address is looked up
 * on the first call on each device).  The call allocates and frees nothing.
 * Limit: ud_gqa_workspace_bytes(n, q_heads, head_dim, max_keys) <= UD_GQA_NOALLOC_SCRATCH_BYTES
 * (e.g. 64 sequences x 32 query heads x 4096 keys at head_dim 128 use 32.5 MiB); larger calls
 * return UD_ERR_SHAPE before anything is launched.  Every call on one device shares that device's
 * array: calls that overlap on one device (on different HIP streams, or from several threads)
 * race and must be serialised by the caller.  Nothing in the array needs to start at zero. */
#define UD_GQA_NOALLOC_SCRATCH_BYTES (40u << 20)
UD_API int ud_gqa_attention_paged_noalloc(int32_t kv_dtype, const float* q_dev, const void* k_pages,
                                          const void* v_pages, const int32_t* block_table, int32_t max_blocks,
                                          const int32_t* ranges_dev, float* out_dev, int32_t n, int32_t q_heads,
                                          int32_t kv_heads, int32_t head_dim, int32_t block_size, int32_t max_keys,
                                          void* hip_stream);

/* Replaces Step.rope (Ops.swift rope) / rope_rotate_half (30_voxtral.metal:20-36): in place on
 * x [rows, ld] (dtype UD_F32, UD_BF16 or UD_F16), heads H of head_dim d starting at column 0:
 *   angle = pos(t) * inv_freq[i];  x_i' = x_i cos - x_{i+d/2} sin;  x_{i+d/2}' = x_{i+d/2} cos + x_i sin
 * pos(t) = positions_dev[t] when positions_dev is non-null, else pos0 + t.  inv_freq_dev fp32
 * [d/2] (the reference builds it as 1 / theta^(2i/d), Voxtral.swift:176-179). */
UD_API int ud_rope_rotate_half(int32_t dtype, void* x_dev, int32_t rows, int32_t heads, int32_t head_dim, int32_t ld,
                               const int32_t* positions_dev, int32_t pos0, const float* inv_freq_dev, void* hip_stream);

/* Replaces the K/V writes into the session cache (the projections write rows of SlidingKV,
 * Voxtral.swift:371-376): copies row i of k_new / v_new ([n, kv_heads*head_dim], kv_dtype) to
 * logical position positions_dev[i] of sequence i in the paged cache. */
UD_API int ud_paged_kv_append(int32_t kv_dtype, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                              const int32_t* block_table, int32_t max_blocks, const int32_t* positions_dev, int32_t n,
                              int32_t kv_heads, int32_t head_dim, int32_t block_size, void* hip_stream);

/* ---------------------------------------------------------------- windows, sinks, prompts, 4-bit pages
 * The calls below take the same pages and block tables, and besides bf16 and half pages (kv_format UD_BF16 / UD_F16)
 * pages of 4 bits:
 *   UD_MXFP4   per page and kv head block_size rows of head_dim / 2 bytes, channel 2b in the low nibble of byte b, then
 *              block_size rows of head_dim / 32 bytes: the exponent + 127 of each block of 32 channels.  A nibble is a
 *              sign bit and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (codes 0 .. 7), times 2^exponent: 4.25 bits a value.
 *              Exponent byte 255: the block held a NaN or an infinity and reads as NaN.  Else the byte is 27 .. 252, what
 *              ud_qk_norm_rope_append writes: a page that a row sees has no other.
 * k_pages / v_pages are ud_kv_page_bytes(..) bytes a page, 16-byte aligned, num_blocks pages each.  A block-table entry
 * outside [0, num_blocks) is a page that is not held: nothing of it is read or written, and its keys are not there.
 * They have no counterpart in the reference beyond the ones named; limits: head_dim 64 or 128, block_size 16. */
#define UD_MXFP4 16

/* Bytes of one page of keys (or of values); 0 for a format or size that is not supported. */
UD_API size_t ud_kv_page_bytes(int32_t kv_format, int32_t kv_heads, int32_t head_dim, int32_t block_size);

/* The heads of one attention layer's projected rows, made ready in one pass (Step.rope and the K/V writes of
 * VoxtralSession.decode, Voxtral.swift:364-376, with the per-head norm that decoders put before the rotation):
 *   y = x / sqrt(mean_c x_c^2 + eps) * weight     per head of q and k, where its weight is given
 *   (y_i, y_{i+d/2}) -> (y_i cos a - y_{i+d/2} sin a, y_{i+d/2} cos a + y_i sin a),  a = position * inv_freq[i]
 * Row t belongs to sequence seqs_dev[t] (null: t) at position positions_dev[t].  q goes to q_out, k and v (as it is) to
 * the pages.
 *   q, k, v      dtype (UD_F32, UD_BF16, UD_F16), rows q_ld / k_ld / v_ld elements apart (pieces of one fused row, or
 *                buffers of their own); q_heads 0: no q.  dtype is fp32 or the pages' own; any for UD_MXFP4
 *   q_out        dtype, rows q_out_ld apart; may be q where q_out_ld is q_ld, and shares no memory with q, k and v otherwise
 *   q_weight, k_weight   fp32 [head_dim] or null (no norm);  inv_freq fp32 [head_dim / 2] or null (no rotation)
 * A row whose sequence is outside [0, n), whose position is negative or not below max_blocks * block_size, or whose page
 * is not held, is padding: nothing is written for it, q_out included.  Rows of one call name different keys.
 * Precision: angles in 64 bits, the rest in fp32 and one rounding at the end (half saturates); k for UD_MXFP4 pages
 * in 64 bits up to its codes.  MXFP4: a block's exponent is the smallest with max |x| <= 7 * 2^exponent (but
 * -100 .. 125), values go to the nearest code, ties to the even one, beyond the largest to that. */
UD_API int ud_qk_norm_rope_append(int32_t dtype, int32_t kv_format, const void* q_dev, int32_t q_ld, const void* k_dev,
                                  int32_t k_ld, const void* v_dev, int32_t v_ld, void* q_out_dev, int32_t q_out_ld,
                                  const float* q_weight_dev, const float* k_weight_dev, float eps, const float* inv_freq_dev,
                                  const int32_t* positions_dev, const int32_t* seqs_dev, void* k_pages, void* v_pages,
                                  int32_t num_blocks, const int32_t* block_table, int32_t n, int32_t max_blocks,
                                  int32_t rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t block_size,
                                  void* hip_stream);

/* Rows of the cache read back: row t is the key / value of position positions_dev[t] of sequence seqs_dev[t] (null: t),
 * [rows, kv_heads * head_dim] of dtype UD_F32, the pages' own type, or UD_BF16 from UD_MXFP4 pages (exact).  A row that
 * ud_qk_norm_rope_append would take as padding is 0. */
UD_API int ud_paged_kv_read(int32_t kv_format, int32_t dtype, const void* k_pages, const void* v_pages, int32_t num_blocks,
                            const int32_t* block_table, int32_t n, int32_t max_blocks, const int32_t* positions_dev,
                            const int32_t* seqs_dev, void* k_out, void* v_out, int32_t rows, int32_t kv_heads,
                            int32_t head_dim, int32_t block_size, void* hip_stream);

/* ud_gqa_attention_paged_mq with sinks, for any group of heads and page format, at a cost that follows the window:
 *   out[i, m, h] = sum_j softmax_j(q[i, m, h] . k[i, j, h / (Hq/Hkv)] / sqrt(head_dim)) v[i, j, kvh]
 *   over keys j in [lo, hi) = ranges[i][m] and the sinks j in [0, min(n_sinks, lo)); 0 where lo >= hi (then without the
 *   sinks too).  Ranges are cut to [0, max_blocks * block_size).
 *   q_dev, out_dev  [n, n_queries, q_heads * head_dim] of dtype UD_F32, or the pages' own type, or any 16-bit type on
 *                   UD_MXFP4 pages
 *   max_span        upper bound of a sequence's keys from its lowest lo to its highest hi (sizes the grid; a longer
 *                   sequence is slower, not wrong).  A sequence's keys are shared out among workgroups only as far as n *
 *                   kv_heads leaves the chip room, so one that is far longer than the others is better called by itself
 *   workspace       ud_gqa_window_workspace_bytes(..) bytes (0: may be null); its contents need not be kept
 * Only entries of the block table whose pages hold a sink or a key between a sequence's lowest lo and highest hi are
 * read: the pages between may have been given back.  n_queries 1 .. 8, n_queries * q_heads / kv_heads <= 64.
 * A call repeated gives the same bits; the keys are split over workgroups by n and max_span, so that the last bits of a
 * row may differ between calls that differ in these.
 * Precision: fp32 queries and outputs are as good as fp32 arithmetic; 16-bit ones: exact products, sums in fp32, the
 * probabilities rounded once to the pages' type (bf16 for UD_MXFP4, twice that for half queries); a value past 2^90
 * may pass fp32's range in the sums, which are divided at the end.  A NaN or infinity in a key or value reaches only the
 * rows that see it: a NaN in a key makes them NaN, an infinity in a key may; a channel with an infinity among the values is
 * that infinity, however small its probability (half outputs: 65504), with one of both signs or a NaN it is NaN; a
 * call that meets one takes up to twelve times as long.
 * For fp32 queries over bf16 or half pages, without sinks and with 1, 2, 4 or 8 query heads to a kv head,
 * ud_gqa_attention_paged(_mq) computes the same.  Take this call where accuracy counts on bf16 pages (the other rounds
 * queries and probabilities to bf16), for batches and from some 2,000 keys on, the other for one short sequence and, a little,
 * for several queries over bf16 pages.  us, this call / the other, 32/8 heads of 128: one sequence of 1,000 keys 12 / 9.5, of
 * 8,192 half 13.5 / 16.2, bf16 13.3 / 15.0; 64 of 1,000 half 50 / 74, bf16 50 / 56; 64 of 4,096 184 / 251, 183 / 199; 12 of
 * 300 .. 8,192 with 4 queries each 61 / 130, 61 / 56. */
UD_API size_t ud_gqa_window_workspace_bytes(int32_t n, int32_t n_queries, int32_t q_heads, int32_t kv_heads,
                                            int32_t head_dim, int32_t n_sinks, int32_t max_span);
UD_API int ud_gqa_window_attention_paged(int32_t kv_format, int32_t dtype, const void* q_dev, const void* k_pages,
                                         const void* v_pages, int32_t num_blocks, const int32_t* block_table,
                                         int32_t max_blocks, const int32_t* ranges_dev, int32_t n_sinks, void* out_dev,
                                         int32_t n, int32_t n_queries, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                         int32_t block_size, int32_t max_span, void* workspace, size_t workspace_bytes,
                                         void* hip_stream);

/* The same attention for prompts and pieces of prompts: any number of query rows per sequence (Step.attention with the
 * whole prompt's rows, Ops.swift:136-169; VoxtralSession's first decode, Voxtral.swift:425-465).
 *   q_dev, out_dev  [rows, q_heads * head_dim] of dtype UD_BF16 or UD_F16 (the pages' own, or either on UD_MXFP4 pages)
 *   q_start_dev     int32 [n + 1], ascending: rows q_start[i] .. q_start[i + 1] - 1 belong to sequence i, at most
 *                   max_rows each; out rows of no sequence are left as they were
 *   ranges_dev      int32 [rows, 2]: row r sees [lo, hi) and the sinks below lo, as above (a causal prompt: hi = its
 *                   position + 1).  The keys are read from the pages: append before the call
 *   max_span        upper bound of a sequence's keys from its lowest lo to its highest hi (a plan, as above; n and
 *                   max_rows count in it too)
 *   workspace       ud_gqa_prefill_workspace_bytes(..) bytes (0: may be null)
 * Precision: exact products, sums and softmax in fp32, probabilities rounded once to dtype, one rounding at the end; NaN and
 * infinities as above.  UD_MXFP4 pages under half queries: keys and values become halves.  Blocks of exponents -23 .. 13
 * stay as they are; above, values past 65504 saturate to it, and below, values are rounded to a multiple of 2^-24, 2^-25 and
 * less to 0 (ud_gqa_window_attention_paged takes all of them as they are). */
UD_API size_t ud_gqa_prefill_workspace_bytes(int32_t n, int32_t rows, int32_t max_rows, int32_t q_heads, int32_t kv_heads,
                                             int32_t head_dim, int32_t n_sinks, int32_t max_span);
UD_API int ud_gqa_prefill_paged(int32_t kv_format, int32_t dtype, const void* q_dev, const void* k_pages,
                                const void* v_pages, int32_t num_blocks, const int32_t* block_table, int32_t max_blocks,
                                const int32_t* q_start_dev, const int32_t* ranges_dev, int32_t n_sinks, void* out_dev,
                                int32_t n, int32_t rows, int32_t max_rows, int32_t q_heads, int32_t kv_heads,
                                int32_t head_dim, int32_t block_size, int32_t max_span, void* workspace,
                                size_t workspace_bytes, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif
