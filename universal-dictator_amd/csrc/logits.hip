// Logits made ready for the choice of a token, and the greedy one (include/ud_layer.h): penalties for what a row's history
// holds, biases, a grammar's mask, the largest of what is left.
//
// A workgroup takes one row's segment of the vocabulary: its logits stay in registers, and what the history says about its tokens
// is counted in LDS, for which the whole history is read by every workgroup of the row (from L2 after the first).  No table
// over the vocabulary is kept between calls, and whole numbers are all that is added up atomically, so no order counts.
#include "layer.hpp"

namespace ud {

struct LogitArgs {
    const void* logits; float* out; uint64_t* best;
    int64_t ld, out_ld;
    const int32_t* tokens; const int32_t* ranges; const float* penalties;
    const int32_t* bias_ids; const float* bias_values; const int32_t* bias_ranges;
    const uint32_t* mask; const int32_t* mask_rows; int64_t mask_ld;
    int vocab, n_tokens, n_biases, n_masks;
};

constexpr uint32_t kInPrompt = 1u << 31;           // a token's word: in the prompt, and how often it was generated

// Larger for a larger logit, and for the lower token of equal ones; 0 for one that may not be chosen.
__device__ __forceinline__ uint64_t choice_key(float l, int t) {
    if (!(l > -__builtin_inff())) return 0;        // -inf, NaN
    const uint32_t u = __float_as_uint(l + 0.0f);  // -0 as 0
    return (uint64_t)(u & kInPrompt ? ~u : u | kInPrompt) << 32 | (uint32_t)~t;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, d));
    return v;
}

// Eight logits from p, `left` of them there (the others -inf); p need not be aligned to more than an element.
template <typename T> __device__ __forceinline__ void load_logits(const T* p, int left, float (&f)[8]) {
    if (left >= 8) {
        Raw8<T> r;
        __builtin_memcpy(&r, p, sizeof r);
        widen8<T>(r, f);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = e < left ? to_f<T>(p[e]) : -__builtin_inff();
    }
}

// 256 threads; a thread's E pieces of eight tokens are 2,048 apart.
template <typename T, int E> __global__ __launch_bounds__(256) void logits_kernel(LogitArgs a) {
    constexpr int SEG = 2048 * E;
    __shared__ __attribute__((aligned(16))) uint32_t word[SEG];
    __shared__ uint64_t top[4];
    const int tid = threadIdx.x, row = blockIdx.y, t0 = blockIdx.x * SEG, len = min(SEG, a.vocab - t0);
    const T* in = static_cast<const T*>(a.logits) + row * a.ld + t0;
    float l[E][8];
#pragma unroll
    for (int i = 0; i < E; i++) load_logits<T>(in + (i * 256 + tid) * 8, len - (i * 256 + tid) * 8, l[i]);
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < SEG / 1024; i++) *reinterpret_cast<uint4*>(&word[(i * 256 + tid) * 4]) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    };
    // what(token's place in the segment, index) for entries lo .. hi - 1 of `ids`
    auto scan = [&](const int32_t* ids, int lo, int hi, auto what) {
        for (int64_t i = lo + 4 * tid; i < hi; i += 1024) {
            int32_t v[4];
            if (i + 4 <= hi) {
                __builtin_memcpy(v, ids + i, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = i + e < hi ? ids[i + e] : -1;
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (v[e] >= t0 && v[e] - t0 < len) what(v[e] - t0, (int)i + e);
        }
        __syncthreads();
    };
    if (a.tokens) {
        const int lo = max(a.ranges[3 * row], 0), hi = min(a.ranges[3 * row + 2], a.n_tokens), fresh = a.ranges[3 * row + 1];
        if (lo < hi) {
            clear();
            scan(a.tokens, lo, hi, [&](int at, int i) {
                if (i < fresh) atomicOr(&word[at], kInPrompt);
                else atomicAdd(&word[at], 1u);
            });
            const float rep = a.penalties[3 * row], pres = a.penalties[3 * row + 1], freq = a.penalties[3 * row + 2];
#pragma unroll
            for (int i = 0; i < E; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t w = word[(i * 256 + tid) * 8 + e];
                    if (!w) continue;
                    float x = l[i][e];
                    x = x > 0.0f ? x / rep : x * rep;
                    const uint32_t c = w & ~kInPrompt;
                    l[i][e] = c ? x - (freq * (float)c + pres) : x;
                }
        }
    }
    if (a.bias_ids) {
        const int lo = max(a.bias_ranges[2 * row], 0), hi = min(a.bias_ranges[2 * row + 1], a.n_biases);
        if (lo < hi) {
            __syncthreads();
            clear();
            scan(a.bias_ids, lo, hi, [&](int at, int i) { atomicMax(&word[at], (uint32_t)(i - lo) + 1); });
#pragma unroll
            for (int i = 0; i < E; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t w = word[(i * 256 + tid) * 8 + e];
                    if (w) l[i][e] += a.bias_values[lo + (int64_t)w - 1];
                }
        }
    }
    const int m = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
    const bool masked = m >= 0 && m < a.n_masks;
    const uint8_t* mask = masked ? reinterpret_cast<const uint8_t*>(a.mask + m * a.mask_ld) + t0 / 8 : nullptr;
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int c = (i * 256 + tid) * 8, left = len - c;
        if (left <= 0) continue;
        if (masked) {
            const uint32_t bits = mask[c / 8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (!(bits >> e & 1)) l[i][e] = -__builtin_inff();
        }
        float* o = a.out + row * a.out_ld + t0 + c;
        if (left >= 8) {
            __builtin_memcpy(o, l[i], 32);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < left) o[e] = l[i][e];
        }
        if (a.best)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < left) best = max(best, choice_key(l[i][e], t0 + c + e));
    }
    if (!a.best) return;
    best = wave_max_key(best);
    if (tid % 64 == 0) top[tid / 64] = best;
    __syncthreads();
    if (tid == 0) a.best[(int64_t)row * gridDim.x + blockIdx.x] = max(max(top[0], top[1]), max(top[2], top[3]));
}

// The largest of a row's segments.
__global__ __launch_bounds__(64) void choose_kernel(const uint64_t* best, int segments, int32_t* token) {
    uint64_t v = 0;
    for (int i = threadIdx.x; i < segments; i += 64) v = max(v, best[(int64_t)blockIdx.x * segments + i]);
    v = wave_max_key(v);
    if (threadIdx.x == 0) token[blockIdx.x] = v ? (int32_t)~(uint32_t)v : -1;
}

// Pieces of eight tokens per thread: as many as leave the chip two workgroups per CU, since each reads the row's history.
static int logit_pieces(int64_t n, int64_t vocab) {
    for (int e = 4; e > 1; e /= 2)
        if (n * ((vocab + 2048 * e - 1) / (2048 * e)) >= 512) return e;
    return 1;
}

template <typename T> static void launch_logits(const LogitArgs& a, int n, int e, int segments, hipStream_t st) {
    const dim3 grid(segments, n);
    if (e == 4) hipLaunchKernelGGL((logits_kernel<T, 4>), grid, dim3(256), 0, st, a);
    else if (e == 2) hipLaunchKernelGGL((logits_kernel<T, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((logits_kernel<T, 1>), grid, dim3(256), 0, st, a);
}

}  // namespace ud

using namespace ud;

extern "C" UD_API size_t ud_logits_workspace_bytes(int32_t n, int32_t vocab) {
    if (n < 1 || n > 65535 || vocab < 1 || vocab > (1 << 24)) return 0;
    const int seg = 2048 * logit_pieces(n, vocab);
    return (size_t)n * ((vocab + seg - 1) / seg) * sizeof(uint64_t);
}

extern "C" UD_API int ud_logits_process(int32_t dtype, const void* logits_dev, int32_t ld, float* out_dev, int32_t out_ld,
                                        int32_t* token_dev, int32_t n, int32_t vocab, const int32_t* tokens_dev, int32_t n_tokens,
                                        const int32_t* ranges_dev, const float* penalties_dev, const int32_t* bias_ids_dev,
                                        const float* bias_values_dev, int32_t n_biases, const int32_t* bias_ranges_dev,
                                        const uint32_t* mask_dev, int32_t mask_ld, int32_t n_masks, const int32_t* mask_rows_dev,
                                        void* workspace, size_t workspace_bytes, void* hip_stream) {
    static const char* who = "ud_logits_process";
    const int64_t size = type_bytes(dtype);
    if (!size) return layer_fail(UD_ERR_INVALID, "%s: dtype %d", who, dtype);
    if (n < 0 || n > 65535 || vocab < 1 || vocab > (1 << 24))
        return layer_fail(UD_ERR_SHAPE, "%s: %d rows (0 .. 65535) of %d tokens (1 .. 2^24)", who, n, vocab);
    if (ld < vocab || out_ld < vocab) return layer_fail(UD_ERR_SHAPE, "%s: rows %d/%d elements apart for %d tokens", who, ld, out_ld, vocab);
    if (n_tokens < 0 || n_biases < 0) return layer_fail(UD_ERR_SHAPE, "%s: %d tokens of history, %d biases", who, n_tokens, n_biases);
    if (mask_dev && (mask_ld < (vocab + 31) / 32 || n_masks < 0 || (!mask_rows_dev && n_masks < n)))
        return layer_fail(UD_ERR_SHAPE, "%s: %d masks of %d words for %d rows of %d tokens", who, n_masks, mask_ld, n, vocab);
    if (n == 0) return UD_OK;
    if (!logits_dev || !out_dev || (tokens_dev && !ranges_dev) || (bias_ids_dev && (!bias_values_dev || !bias_ranges_dev)))
        return layer_fail(UD_ERR_INVALID, "%s: null pointer", who);
    const size_t need = ud_logits_workspace_bytes(n, vocab);
    if (token_dev && (!workspace || workspace_bytes < need))
        return layer_fail(UD_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : 0, need);
    uintptr_t at = (uintptr_t)out_dev | (uintptr_t)token_dev | (uintptr_t)tokens_dev | (uintptr_t)ranges_dev | (uintptr_t)penalties_dev |
                   (uintptr_t)bias_ids_dev | (uintptr_t)bias_values_dev | (uintptr_t)bias_ranges_dev | (uintptr_t)mask_dev |
                   (uintptr_t)mask_rows_dev;
    if ((at & 3) || ((uintptr_t)logits_dev & (size - 1)) || (token_dev && ((uintptr_t)workspace & 7)))
        return layer_fail(UD_ERR_INVALID, "%s: pointers must be aligned to their elements (the workspace to 8 bytes)", who);
    auto flat = [](const void* p, int64_t elements) { return Block{p, 0, 4 * elements, 1}; };
    const Block out{out_dev, out_ld * (int64_t)4, vocab * (int64_t)4, n}, in{logits_dev, ld * size, vocab * size, n};
    const Block token = flat(token_dev, n), ws{token_dev ? workspace : nullptr, 0, (int64_t)need, 1};
    const Block inputs[] = {flat(tokens_dev, n_tokens), flat(ranges_dev, tokens_dev ? 3 * (int64_t)n : 0), flat(penalties_dev, 3 * (int64_t)n),
                            flat(bias_ids_dev, n_biases), flat(bias_values_dev, n_biases), flat(bias_ranges_dev, bias_ids_dev ? 2 * (int64_t)n : 0),
                            flat(mask_dev, (int64_t)n_masks * mask_ld), flat(mask_rows_dev, n)};
    bool clash = (blocks_meet(out, in) && !(size == 4 && blocks_same(out, in))) || blocks_meet(token, in) || blocks_meet(ws, in) ||
                 blocks_meet(out, token) || blocks_meet(out, ws) || blocks_meet(token, ws);
    for (const Block& b : inputs) clash = clash || (b.width && (blocks_meet(out, b) || blocks_meet(token, b) || blocks_meet(ws, b)));
    if (clash) return layer_fail(UD_ERR_INVALID, "%s: an output overlaps an input or another output (out may be fp32 logits, at the same ld)", who);
    LogitArgs a{};
    a.logits = logits_dev; a.out = out_dev; a.best = token_dev ? static_cast<uint64_t*>(workspace) : nullptr;
    a.ld = ld; a.out_ld = out_ld;
    if (tokens_dev && penalties_dev && n_tokens) { a.tokens = tokens_dev; a.ranges = ranges_dev; a.penalties = penalties_dev; }
    if (bias_ids_dev && n_biases) { a.bias_ids = bias_ids_dev; a.bias_values = bias_values_dev; a.bias_ranges = bias_ranges_dev; }
    if (mask_dev) { a.mask = mask_dev; a.mask_rows = mask_rows_dev; a.mask_ld = mask_ld; }
    a.vocab = vocab; a.n_tokens = n_tokens; a.n_biases = n_biases; a.n_masks = n_masks;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int e = logit_pieces(n, vocab), segments = (vocab + 2048 * e - 1) / (2048 * e);
    if (dtype == UD_F32) launch_logits<float>(a, n, e, segments, st);
    else if (dtype == UD_BF16) launch_logits<bf16>(a, n, e, segments, st);
    else launch_logits<f16>(a, n, e, segments, st);
    if (token_dev) hipLaunchKernelGGL(choose_kernel, dim3(n), dim3(64), 0, st, a.best, segments, token_dev);
    return layer_launched(who);
}
