// Logits made ready for the choice of a token, and the greedy one (include/ud_layer.h): penalties for what a row's history
// holds, biases, a grammar's mask, the largest of what is left.
//
// A workgroup takes one row's segment of the vocabulary: its logits stay in registers, and what the history says about its tokens
// is counted in LDS, for which the whole history is read by every workgroup of the row (from L2 after the first).  No table
// over the vocabulary is kept between calls, and whole numbers are all that is added up atomically, so no order counts.
#include "layer.hpp"

namespace ud {

struct LogitArgs {
    const void* logits; float* out; uint64_t* best; int32_t* token;
    int64_t ld, out_ld;
    const int32_t* tokens; const int32_t* ranges; const float* penalties;
    const int32_t* bias_ids; const float* bias_values; const int32_t* bias_ranges;
    const uint32_t* mask; const int32_t* mask_rows; int64_t mask_ld;
    int vocab, n_tokens, n_biases, n_masks;
};

// A token's word: whether it is in the prompt, and how often it was generated; of a row whose lists are not longer than that, the place of
// its last bias + 1 in the bits between.
constexpr uint32_t kInPrompt = 1u << 31, kCounts = 0xffff, kSlots = 0x7fff;

// Larger for a larger logit, and for the lower token of equal ones; 0 for one that may not be chosen.
__device__ __forceinline__ uint64_t choice_key(float l, int t) {
    if (!(l > -__builtin_inff())) return 0;        // -inf, NaN
    const uint32_t u = __float_as_uint(l + 0.0f);  // -0 as 0
    return (uint64_t)(u & kInPrompt ? ~u : u | kInPrompt) << 32 | (uint32_t)~t;
}
__device__ __forceinline__ int32_t chosen(uint64_t key) { return key ? (int32_t)~(uint32_t)key : -1; }
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, d));
    return v;
}

// Four logits as they lie in memory, and as floats.
template <typename T> struct Raw4 { T v[4]; };
// From p, `left` of them there (the others -inf); p need not be aligned to more than an element.
template <typename T> __device__ __forceinline__ Raw4<T> load_logits(const T* p, int left) {
    Raw4<T> r;
    if (left >= 4) {
        __builtin_memcpy(&r, p, sizeof r);
    } else {
        const float none = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (e < left) r.v[e] = p[e];
            else if constexpr (std::is_same<T, bf16>::value) r.v[e] = (bf16)(__float_as_uint(none) >> 16);
            else r.v[e] = (T)none;
        }
    }
    return r;
}

// Entries at .. of a list of ids that ends at `hi`, D loads of four of them a thread, 4 THREADS apart; -1 behind the end.
template <int THREADS, int D> __device__ __forceinline__ void load_ids(const int32_t* ids, int64_t at, int hi, int32_t (&v)[D][4]) {
#pragma unroll
    for (int d = 0; d < D; d++) {
        const int64_t i = at + 4 * (d * THREADS + (int)threadIdx.x);
        if (i + 4 <= hi) {
            __builtin_memcpy(v[d], ids + i, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[d][e] = i + e < hi ? ids[i + e] : -1;
        }
    }
}

// 16 waves, SEG tokens: a thread's E pieces of four are 4,096 apart, so that a wave reads and writes whole lines (pieces of eight: 22.9 -> 21.0 us
// at 64 rows).  A small segment leaves threads that only read the lists (one row of 131,072 with a history of 100,000 38 -> 15 us).  What the row's lists say is asked for at once, at the start: one after
// the other their latencies would be most of a short call.
template <typename T, int SEG> __global__ __launch_bounds__(1024) void logits_kernel(LogitArgs a) {
    constexpr int W = 16, THREADS = 64 * W, E = (SEG + 4 * THREADS - 1) / (4 * THREADS);
    __shared__ __attribute__((aligned(16))) uint32_t word[SEG];
    __shared__ float top[W];
    __shared__ int first;
    const int tid = threadIdx.x, row = blockIdx.y, t0 = blockIdx.x * SEG, len = min(SEG, a.vocab - t0);
    // (used behind the last of these branches only, so that all of a row's numbers are on their way together)
    int from = 0, fresh = 0, to = 0, bias_from = 0, bias_to = 0, mask_row = row;
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if (a.tokens) {
        const int32_t* range = a.ranges + 3 * row;
        const float* pen = a.penalties + 3 * row;
        from = range[0], fresh = range[1], to = range[2];
        rep = pen[0], pres = pen[1], freq = pen[2];
    }
    if (a.bias_ids) bias_from = a.bias_ranges[2 * row], bias_to = a.bias_ranges[2 * row + 1];
    if (a.mask_rows) mask_row = a.mask_rows[row];
    const int lo = max(from, 0), hi = min(to, a.n_tokens), blo = max(bias_from, 0), bhi = min(bias_to, a.n_biases);
    const int m = a.mask ? mask_row : -1;
    const bool masked = m >= 0 && m < a.n_masks;
    const T* in = static_cast<const T*>(a.logits) + row * a.ld + t0;
    Raw4<T> raw[E];
    uint32_t allowed = 0;                          // four bits of the mask a piece
    int32_t ids[4][4], bias_ids[1][4];             // the first of each list
#pragma unroll
    for (int i = 0; i < E; i++) {
        const int c = (i * THREADS + tid) * 4;
        raw[i] = load_logits<T>(in + c, len - c);
    }
    if (lo < hi) load_ids<THREADS>(a.tokens, lo, hi, ids);
    if (blo < bhi) load_ids<THREADS>(a.bias_ids, blo, bhi, bias_ids);
    if (masked) {
        const uint8_t* mask = reinterpret_cast<const uint8_t*>(a.mask + m * a.mask_ld) + t0 / 8;
#pragma unroll
        for (int i = 0; i < E; i++)
            if ((i * THREADS + tid) * 4 < len) allowed |= (uint32_t)(mask[(i * THREADS + tid) / 2] >> (tid % 2 * 4) & 15) << (4 * i);
    }
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < E; i++)
            if (SEG >= 4 * THREADS || tid * 4 < SEG) *reinterpret_cast<uint4*>(&word[(i * THREADS + tid) * 4]) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    };
    auto words = [&](int i, uint32_t (&w)[4]) __attribute__((always_inline)) {
        const uint4 u = ld16(&word[SEG >= 4 * THREADS ? (i * THREADS + tid) * 4 : min(tid * 4, SEG - 4)]);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    };
    // what(token's word, index) for entries from .. to - 1 of a list, the first of which are in v
    auto scan = [&](const int32_t* list, int from, int to, auto& v, auto what) __attribute__((always_inline)) {
        constexpr int D = sizeof(v) / 16;
        for (int64_t at = from; at < to; at += 4 * THREADS * D) {
            if (at != from) load_ids<THREADS>(list, at, to, v);
#pragma unroll
            for (int d = 0; d < D; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t p = (uint32_t)v[d][e] - (uint32_t)t0;   // (an id below t0 is past len, too)
                    if (p < (uint32_t)len) what(word[p], (int)at + 4 * (d * THREADS + tid) + e);
                }
        }
        __syncthreads();
    };
    auto count = [&](uint32_t& w, int i) __attribute__((always_inline)) {
        if (i < fresh) atomicOr(&w, kInPrompt);
        else atomicAdd(&w, 1u);
    };
    const float r = 1.0f / rep;
    auto repeated = [&](float x) __attribute__((always_inline)) { return x * (x > 0.0f ? r : rep); };
    // A token in the prompt, generated c times; y: its logit under the repetition's penalty.
    auto penalize = [&](float x, float y, bool seen, uint32_t c) __attribute__((always_inline)) {
        const float z = c ? y - fmaf(freq, (float)c, pres) : y;
        return seen ? z : x;
    };
    float most = -__builtin_inff();
    int at = 0;                                    // the first place that holds it
    auto widen = [&](int i, float (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = to_f<T>(raw[i].v[e]);
    };
    // A piece whose lists are done with: masked, written, its largest kept (a NaN is passed over).
    auto finish = [&](int i, float (&x)[4]) __attribute__((always_inline)) {
        const int c = (i * THREADS + tid) * 4, left = len - c;
        if (left <= 0) return;
        if (masked)
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = allowed >> (4 * i + e) & 1 ? x[e] : -__builtin_inff();
        float* o = a.out + row * a.out_ld + t0 + c;
        if (left >= 4) {
            // (past the caches: 64 rows of 131,072 29.5 -> 25.1 us, much of it the next kernel's wait for what the caches write back)
            typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
            __builtin_nontemporal_store(f4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f4*>(o));
        } else {
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (e < left) o[e] = x[e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (x[e] > most && e < left) {
                most = x[e];
                at = c + e;
            }
    };
    // Lists that are short enough: both in one pass over the words, the last bias of a token and the number of times it was generated
    // side by side.  A repetition whose reciprocal would be infinite or short of bits goes the other way, where it divides (a division for all
    // rows: 64 rows of 131,072 21.4 -> 23.6 us).
    const bool lists = lo < hi || blo < bhi, far = !(rep >= 0x1p-100f && rep <= 0x1p100f);
    if (!lists || (hi - (int64_t)lo <= kCounts && bhi - (int64_t)blo <= kSlots && !far)) {
        if (lists) {
            clear();
            if (blo < bhi)
                scan(a.bias_ids, blo, bhi, bias_ids,
                     [&](uint32_t& w, int i) __attribute__((always_inline)) { atomicMax(&w, (uint32_t)(i - blo + 1) << 16); });
            if (lo < hi) scan(a.tokens, lo, hi, ids, count);
        }
#pragma unroll
        for (int i = 0; i < E; i++) {
            float x[4];
            widen(i, x);
            if (lists) {
                uint32_t w[4], any = 0;
                words(i, w);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    any |= w[e];
                    x[e] = penalize(x[e], repeated(x[e]), w[e] & (kInPrompt | kCounts), w[e] & kCounts);
                }
                if (any & kSlots << 16)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (const uint32_t s = w[e] >> 16 & kSlots) x[e] += a.bias_values[blo + (int64_t)s - 1];
            }
            finish(i, x);
            __builtin_amdgcn_sched_barrier(0);     // piece by piece: all at once they would not fit the registers (nor do they all below)
        }
    } else {
        float l[E][4];
        clear();
        scan(a.tokens, lo, hi, ids, count);
#pragma unroll
        for (int i = 0; i < E; i++) {
            uint32_t w[4];
            words(i, w);
            widen(i, l[i]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = l[i][e];
                l[i][e] = penalize(x, far && x > 0.0f ? x / rep : repeated(x), w[e], w[e] & ~kInPrompt);
            }
        }
        __syncthreads();
        clear();
        scan(a.bias_ids, blo, bhi, bias_ids, [&](uint32_t& w, int i) __attribute__((always_inline)) { atomicMax(&w, (uint32_t)(i - blo) + 1); });
#pragma unroll
        for (int i = 0; i < E; i++) {
            uint32_t w[4];
            words(i, w);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (w[e]) l[i][e] += a.bias_values[blo + (int64_t)w[e] - 1];
            finish(i, l[i]);
        }
    }
    if (!a.best && !a.token) return;
    // The segment's largest, and the first of the places that hold it.
    const float wave_most = wave_max(most);
    if (tid % 64 == 0) top[tid / 64] = wave_most;
    if (tid == 0) first = INT32_MAX;
    __syncthreads();
    const float largest = wave_max(top[tid % W]);
    if (most == largest && largest > -__builtin_inff()) atomicMin(&first, at);
    __syncthreads();
    if (tid) return;
    const uint64_t best = choice_key(largest, t0 + first);
    if (a.best) a.best[(int64_t)row * gridDim.x + blockIdx.x] = best;
    else a.token[row] = chosen(best);
}

// The largest of a row's segments: a wave a row.
__global__ __launch_bounds__(256) void choose_kernel(const uint64_t* best, int segments, int32_t* token, int n) {
    const int row = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
    if (row >= n) return;
    uint64_t v = 0;
    for (int i = lane; i < segments; i += 64) v = max(v, best[(int64_t)row * segments + i]);
    v = wave_max_key(v);
    if (lane == 0) token[row] = chosen(v);
}

// Tokens of a workgroup, 2,048 to 32,768: as many as the row has and leave the chip a workgroup per CU, since each reads the row's history.
static int logit_segment(int64_t n, int64_t vocab) {
    for (int s = 32768; s > 2048; s /= 2)
        if (s / 2 < vocab && n * ((vocab + s - 1) / s) >= 256) return s;
    return 2048;
}

template <typename T> static void launch_logits(const LogitArgs& a, int n, int seg, hipStream_t st) {
    const dim3 grid((a.vocab + seg - 1) / seg, n);
    if (seg == 32768) hipLaunchKernelGGL((logits_kernel<T, 32768>), grid, dim3(1024), 0, st, a);
    else if (seg == 16384) hipLaunchKernelGGL((logits_kernel<T, 16384>), grid, dim3(1024), 0, st, a);
    else if (seg == 8192) hipLaunchKernelGGL((logits_kernel<T, 8192>), grid, dim3(1024), 0, st, a);
    else if (seg == 4096) hipLaunchKernelGGL((logits_kernel<T, 4096>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((logits_kernel<T, 2048>), grid, dim3(1024), 0, st, a);
}

}  // namespace ud

using namespace ud;

extern "C" UD_API size_t ud_logits_workspace_bytes(int32_t n, int32_t vocab) {
    if (n < 1 || n > 65535 || vocab < 1 || vocab > (1 << 24)) return 0;
    // A key for each of the row's segments at least, and never less for more rows or more tokens.  (Segments between the smallest and the
    // largest are taken where twice as large ones would be fewer than 256, or a row is one: there are fewer than 512 of them, or as many as rows.)
    const size_t most = (size_t)n * ((vocab + 2047) / 2048), least = (size_t)n * ((vocab + 32767) / 32768);
    return sizeof(uint64_t) * (most < 512 ? most : least < 512 ? 512 : least);
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
                            Block{mask_dev, 4 * (int64_t)mask_ld, (vocab + 31) / 32 * (int64_t)4, n_masks}, flat(mask_rows_dev, n)};
    bool clash = (blocks_meet(out, in) && !(size == 4 && blocks_same(out, in))) || blocks_meet(token, in) || blocks_meet(ws, in) ||
                 blocks_meet(out, token) || blocks_meet(out, ws) || blocks_meet(token, ws);
    for (const Block& b : inputs) clash = clash || (b.width && (blocks_meet(out, b) || blocks_meet(token, b) || blocks_meet(ws, b)));
    if (clash) return layer_fail(UD_ERR_INVALID, "%s: an output overlaps an input or another output (out may be fp32 logits, at the same ld)", who);
    LogitArgs a{};
    a.logits = logits_dev; a.out = out_dev;
    a.ld = ld; a.out_ld = out_ld;
    if (tokens_dev && penalties_dev && n_tokens) { a.tokens = tokens_dev; a.ranges = ranges_dev; a.penalties = penalties_dev; }
    if (bias_ids_dev && n_biases) { a.bias_ids = bias_ids_dev; a.bias_values = bias_values_dev; a.bias_ranges = bias_ranges_dev; }
    if (mask_dev) { a.mask = mask_dev; a.mask_rows = mask_rows_dev; a.mask_ld = mask_ld; }
    a.vocab = vocab; a.n_tokens = n_tokens; a.n_biases = n_biases; a.n_masks = n_masks;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const int seg = logit_segment(n, vocab), segments = (vocab + seg - 1) / seg;
    // one segment a row: the token is written at once
    if (token_dev && segments > 1) a.best = static_cast<uint64_t*>(workspace);
    else a.token = token_dev;
    if (dtype == UD_F32) launch_logits<float>(a, n, seg, st);
    else if (dtype == UD_BF16) launch_logits<bf16>(a, n, seg, st);
    else launch_logits<f16>(a, n, seg, st);
    if (a.best) hipLaunchKernelGGL(choose_kernel, dim3((n + 3) / 4), dim3(256), 0, st, a.best, segments, token_dev, n);
    return layer_launched(who);
}
