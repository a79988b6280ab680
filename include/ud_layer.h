/*
 * ud_layer.h -- C ABI of what a decoder does between two attentions and after the last one, with its products in 8 bits:
 * the norm with the residual's addition, rows in 8 bits (plain or gated), the int8 matrix product, and the choice of the
 * next token from penalised, biased and masked logits.
 *
 * The decoder's attention and its cache are in ud_decode.h; one layer is
 *   ud_rms_norm (8 bits) -> ud_i8_linear (q|k|v) -> ud_qk_norm_rope_append -> an attention -> ud_i8_quantize ->
 *   ud_i8_linear -> ud_rms_norm (8 bits, adding that to the residual) -> ud_i8_linear (gate|up) -> ud_i8_quantize (gated) ->
 *   ud_i8_linear (down, adding the residual)
 * and behind the last one ud_rms_norm -> ud_i8_linear (fp32 logits) -> ud_logits_process.
 *
 * Conventions are those of ud_encoder.h: 0 or a negative ud_status, message in ud_last_error(), device pointers,
 * asynchronous on hip_stream, nothing allocated, nothing synchronised (every call may be captured into a graph).  *_ld: elements
 * from one row to the next.  Types are UD_F32, UD_BF16, UD_F16; a half output saturates.
 *
 * Rows in 8 bits: codes int8 [rows, dim] and one fp32 scale per row (a token of activations, an output channel of weights),
 * value = code * scale.  Of a row y: scale = max(max|y| / 127, 2^-126), code = y / scale rounded to the nearest whole number
 * (even one of two), so -127 .. 127; a row with an infinity or a NaN has the scale NaN and codes 0.  fp32 arithmetic: a y within
 * 2^-12 scale of the border between two codes may get either.
 */
#ifndef UD_LAYER_H
#define UD_LAYER_H

#include <stddef.h>
#include <stdint.h>

#include "ud_encoder.h"

#ifdef __cplusplus
extern "C" {
#endif

#define UD_I8 32

/* rms_norm (Step.rmsNorm, Sources/DictatorEngine/Core/Ops.swift:40, Metal/20_conformer.metal:51-69) behind the residual's
 * addition, one pass over the rows:
 *   s = x + residual            rounded to sum_dtype and stored to sum_out (residual null: s = x, sum_out is null too)
 *   y = s * weight / sqrt(mean(s^2) + eps)
 *   x            dtype, rows x_ld apart
 *   residual     sum_dtype (dtype, or UD_F32), rows sum_ld apart; sum_out: the same, may be residual itself
 *   weight       fp32 [dim] or null (1)
 *   out          out_dtype: dtype, or UD_I8 with scales fp32 [rows] (otherwise null)
 * dim a multiple of 8, 8 .. 32768; rows below 2^22; lds multiples of 8, pointers 16-byte aligned (codes 8, scales 4).  eps 1e-30 .. 1e30.
 * The norm is that of the sums as they are stored.  An output may be an input of the same type and ld (in place); any
 * other overlap is refused.  Precision: squares summed in 64 bits, the rest in fp32, one rounding at the end. */
UD_API int ud_rms_norm(int32_t dtype, const void* x_dev, int32_t x_ld, int32_t sum_dtype, const void* residual_dev,
                       void* sum_out_dev, int32_t sum_ld, const float* weight_dev, float eps, int32_t out_dtype, void* out_dev,
                       int32_t out_ld, float* scales_dev, int32_t rows, int32_t dim, void* hip_stream);

/* Rows to 8 bits (Quant.quantizeRowsInt8, Sources/DictatorEngine/Core/Quant.swift:7-21, on the device), plain or gated
 * (swiglu, Metal/30_voxtral.metal:105-148):
 *   y = x, or x * gate / (1 + exp(-gate)) where gate_dev is given
 *   x, gate      dtype, rows ld apart both (two pieces of one fused row, or buffers of their own)
 *   codes        int8, rows codes_ld apart;  scales fp32 [rows]
 * dim a multiple of 8, 8 .. 32768; rows below 2^22; lds multiples of 8, x and gate 16-byte aligned, codes 8.  An output that overlaps
 * an input is refused.  exp(-gate) near fp32's largest or past it (gates below -87) makes y 0. */
UD_API int ud_i8_quantize(int32_t dtype, const void* x_dev, const void* gate_dev, int32_t ld, int8_t* codes_dev, int32_t codes_ld,
                          float* scales_dev, int32_t rows, int32_t dim, void* hip_stream);

/* The product of rows in 8 bits with weights in 8 bits (Step.gemm with int8 weights, whose activations the reference keeps in
 * 16 bits; here both are int8 and the sum over k is exact):
 *   out[m, n] = (sum_k codes[m, k] w[n, k]) * scales[m] * w_scales[n] + bias[n] + residual[m, n]
 *   codes        int8 [M, K], rows codes_ld apart;  scales fp32 [M]
 *   w            int8 [N, K], rows w_ld apart;      w_scales fp32 [N]        (any int8, -128 too)
 *   bias         fp32 [N] or null
 *   residual     dtype [M, N], rows res_ld apart, or null; may be out itself where res_ld is out_ld
 *   out          dtype [M, N], rows out_ld apart
 * K a multiple of 16, 16 .. 131056 (the sum stays in 32 bits); codes and w 16-byte aligned, their lds multiples of 16, at most
 * 2^22; N 1 .. 2^24, M below 2^22, M N at most 2^38.  out and residual need the alignment of their elements only.  Other overlaps
 * of out are refused.  Rows of codes and w that start at multiples of 128 bytes are read fastest (others cost up to half the
 * time again: pad the lds).  Precision: the sum exact, then fp32 in the order written (the second scale and the bias in one
 * operation), one rounding at the end: a row's result is the same in a batch of any size (of a NaN,
 * that it is one: its sign and its other bits may differ). */
UD_API int ud_i8_linear(int32_t dtype, const int8_t* codes_dev, int32_t codes_ld, const float* scales_dev, const int8_t* w_dev,
                        int32_t w_ld, const float* w_scales_dev, const float* bias_dev, const void* residual_dev, int32_t res_ld,
                        void* out_dev, int32_t out_ld, int32_t M, int32_t N, int32_t K, void* hip_stream);

/* Logits made ready for the choice of a token, and the greedy one (argmax_rows, Metal/30_voxtral.metal:105-148).  Row i, token t:
 *   l = logits[i, t]
 *   t in the history:            l = l > 0 ? l / repetition : l * repetition
 *   t generated c > 0 times:     l = l - (frequency * c + presence)
 *   t in the list of biases:     l = l + value         (listed twice: the last one counts)
 *   t forbidden by the mask:     l = -inf              (whatever l is, a NaN too)
 *   out[i, t] = l;   token[i] = the lowest t of the largest l that is neither NaN nor -inf, -1 if there is none
 *   logits       dtype [n, vocab], rows ld apart;  out fp32 [n, vocab], rows out_ld apart, may be logits itself (UD_F32, ld ==
 *                out_ld)
 *   token        int32 [n] or null
 *   tokens       int32 [n_tokens]: the rows' histories;  ranges int32 [n, 3], (a, b, c) = ranges[i]: row i's history is
 *                tokens[a .. c), cut to [0, n_tokens); what of it lies in front of place b is its prompt, the rest it has
 *                generated (where b <= a all of it, where b >= c nothing).  An id outside [0, vocab) is padding.  Rows may share tokens.
 *                null: no histories
 *   penalties    fp32 [n, 3]: repetition (> 0), presence, frequency; null: 1, 0, 0
 *   bias_ids, bias_values   int32 / fp32 [n_biases];  bias_ranges int32 [n, 2]: row i's are [lo, hi), cut to [0, n_biases); rows may
 *                share them.  An id outside [0, vocab) is padding.  null: none
 *   mask         uint32 [n_masks, mask_ld], bit t % 32 of word t / 32: token t is allowed;  mask_rows int32 [n]: row i's mask,
 *                outside [0, n_masks): none (everything is allowed); null: mask i (n_masks >= n).  mask null: none
 *   workspace    ud_logits_workspace_bytes(n, vocab) bytes, 8-byte aligned, where token is given (else may be null); its contents
 *                need not be kept, and calls that may run at the same time need one each.  More rows or a larger vocabulary never
 *                need less: one for the largest batch serves the smaller ones
 * vocab 1 .. 2^24, n 0 .. 65535.  Pointers need the alignment of their elements only.  An out that overlaps an input in any other
 * way is refused.  fp32 arithmetic. */
UD_API size_t ud_logits_workspace_bytes(int32_t n, int32_t vocab);
UD_API int ud_logits_process(int32_t dtype, const void* logits_dev, int32_t ld, float* out_dev, int32_t out_ld, int32_t* token_dev,
                             int32_t n, int32_t vocab, const int32_t* tokens_dev, int32_t n_tokens, const int32_t* ranges_dev,
                             const float* penalties_dev, const int32_t* bias_ids_dev, const float* bias_values_dev, int32_t n_biases,
                             const int32_t* bias_ranges_dev, const uint32_t* mask_dev, int32_t mask_ld, int32_t n_masks,
                             const int32_t* mask_rows_dev, void* workspace, size_t workspace_bytes, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif
