// Attention of prompts: a ragged batch of query rows over the paged caches of their sequences, each row with its own key
// range (causal, windowed) and the sinks before it; pages of bf16, half or MXFP4 (include/ud_decode.h).
//
//   out[r] = sum_j softmax_j(q[r] . k[j] / sqrt(D)) v[j]   over j in [0, min(sinks, lo_r)) and [lo_r, hi_r)
//
// Bound: the matrix cores, 4 D operations per (query head, visible key).  One workgroup = 128 query rows of a kv head (a
// row is a position and one of the G query heads that share it, so the rows of a workgroup are 128 / G positions and its
// mask wastes little), a share of the page list that these rows see, 64 keys at a time through LDS.
//  - S^T = K . Q^T and O^T = V^T . P^T on v_mfma_f32_32x32x16, a wave's 32 rows in the lanes: a lane has 32 scores of its
//    row (the other half of the wave has the row's other 32), so that the running maximum and sum are in-lane but for one
//    swap of the halves, and its probabilities are the B operand of the second product as they stand.
//  - K and V rows lie in LDS permuted piecewise against bank conflicts; V^T is read by ds_read_b64_tr_b16.
#include "paged_attention.hpp"

namespace ud {

struct PrefillArgs {
    const void* q;                 // [rows][Hq][D]
    const char* kp; const char* vp;
    const int32_t* bt;
    const int32_t* q_start;        // [n + 1]
    const int32_t* ranges;         // [rows][2]
    void* out;                     // [rows][Hq][D]
    float* part;                   // [rows][Hq][splits][D], then (maximum, sum) [rows][Hq][splits][2]
    float* stat;
    int rows, max_rows, G, Hq, Hkv;
    int max_blocks, num_blocks;
    int sinks, splits, q_blocks;
    float scale;                   // log2(e) / sqrt(D)
};

typedef float f32x16_t __attribute__((ext_vector_type(16)));
template <bool H> __device__ __forceinline__ f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
    if constexpr (H) return __builtin_amdgcn_mfma_f32_32x32x16_f16(as_f16x8(a), as_f16x8(b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// Eight codes of a block as pairs of the products' type.  As halves, a block whose scale is past 2^13 saturates.
template <bool H> __device__ __forceinline__ uint4 fp4_to_16(uint32_t w, uint32_t byte) {
    const float scale = fp4_scale(byte);
    if constexpr (!H) {
        return fp4_to_bf16(w, scale);
    } else {
        uint32_t x[4] = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3))};
        if (byte > 140 && byte < 255) {
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = (uint32_t)f2h(half_lo(x[e])) | (uint32_t)f2h(half_hi(x[e])) << 16;
        }
        return make_uint4(x[0], x[1], x[2], x[3]);
    }
}

template <int N, typename F> __device__ __forceinline__ int wave_fold(int v, F f) {
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
    return v;
}

template <typename E, int FMT, int D>
__global__ __launch_bounds__(256, 2) void prefill_kernel(PrefillArgs a) {
    typedef typename E::S S;
    constexpr bool H = std::is_same<E, ElH>::value;
    constexpr int KS = D / 16, CT = D / 32;        // products over the channels; channel tiles
    constexpr int HEAD = Page<FMT, D>::BYTES;
    constexpr int VR = FMT == FMT_FP4 ? 1 : D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, seq = blockIdx.z;
    const int split = blockIdx.y % a.splits, qb = a.q_blocks - 1 - (int)(blockIdx.y / a.splits);   // the longest first
    const int s0 = min(max(a.q_start[seq], 0), a.rows), s1 = min(min(max(a.q_start[seq + 1], s0), a.rows), s0 + a.max_rows);
    const int64_t total = (int64_t)(s1 - s0) * a.G;
    if ((int64_t)qb * 128 >= total) return;
    __shared__ __align__(16) char kt[2][64 * 2 * D], vt[2][64 * 2 * D];
    __shared__ int fold[4][4];
    __shared__ int page_of[2][4];                  // logical page, or -1 where there is none
    __shared__ int odd;                            // a value that is no number has been left out

    // ---- this lane's row, and what the workgroup's rows see
    const int64_t rho = (int64_t)qb * 128 + 32 * wave + col;
    const bool real = rho < total;
    const int64_t tok = s0 + (real ? rho : total - 1) / a.G;
    const int64_t at = tok * a.Hq + (int64_t)kvh * a.G + (real ? rho : total - 1) % a.G;
    const int kmax = a.max_blocks * KPAGE;
    const int rlo = max(a.ranges[2 * tok], 0), rhi = min(a.ranges[2 * tok + 1], kmax);
    const bool some_key = real && rlo < rhi;
    const int rsk = some_key ? min(a.sinks, rlo) : 0;
    auto least = [](int x, int y) { return min(x, y); };
    auto most = [](int x, int y) { return max(x, y); };
    const int wlo = wave_fold<32>(some_key ? rlo : kmax, least), whi = wave_fold<32>(some_key ? rhi : 0, most);
    const int wlo_most = __builtin_amdgcn_readfirstlane(wave_fold<32>(some_key ? rlo : 0, most));
    const int whi_least = __builtin_amdgcn_readfirstlane(wave_fold<32>(some_key ? rhi : kmax, least));
    if (lane == 0) { fold[wave][0] = wlo; fold[wave][1] = whi; fold[wave][2] = wlo_most; fold[wave][3] = whi_least; }
    if (tid == 0) odd = 0;
    __syncthreads();
    int lo = fold[0][0], hi = fold[0][1], lo_most = fold[0][2], hi_least = fold[0][3];
#pragma unroll
    for (int w = 1; w < 4; w++) {
        lo = min(lo, fold[w][0]); hi = max(hi, fold[w][1]);
        lo_most = max(lo_most, fold[w][2]); hi_least = min(hi_least, fold[w][3]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo_most = __builtin_amdgcn_readfirstlane(lo_most);
    hi_least = __builtin_amdgcn_readfirstlane(hi_least);
    const PageList list = page_list(lo, hi, a.sinks);
    const int tiles = (list.count + 3) / 4;
    const int t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);

    // ---- q: B operand, lane (row, h): channels 16 s + 8 h .. + 7
    uint4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) qf[s] = ld16(static_cast<const S*>(a.q) + at * D + 16 * s + 8 * h);

    f32x16_t o[CT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[c][i] = 0.0f;
    // probabilities are 2^(score - base): base follows the running maximum, but not before that is BASE_LAG ahead, so that
    // the sums are hardly ever rescaled (a probability is then at most 2^BASE_LAG, far inside half's range)
    constexpr float BASE_LAG = 8.0f;
    float base = -INFINITY, rsum = 0.0f;

    // ---- wave w brings page 4 tile + w: into registers two tiles ahead, into LDS one tile ahead
    const int32_t* bt = a.bt + (int64_t)seq * a.max_blocks;
    uint4 kr[VR], vr[VR];
    uint32_t ks = 0, vs = 0;
    int myblk = 0;
    bool myheld = false;
    auto load = [&](int tile) {
        const int u = 4 * tile + wave;
        const bool in = u < list.count;
        myblk = page_at(list, in ? u : 0);
        int page = bt[myblk];
        myheld = in && page >= 0 && page < a.num_blocks;
        page = myheld ? page : 0;
        const int64_t at = ((int64_t)page * a.Hkv + kvh) * HEAD;
        const char* k = a.kp + at;
        const char* v = a.vp + at;
        if constexpr (FMT == FMT_FP4) {
            if constexpr (D == 128) {
                kr[0] = ld16(k + lane * 16);
                vr[0] = ld16(v + lane * 16);
                ks = *reinterpret_cast<const uint8_t*>(k + Page<FMT, D>::CODES + lane);
                vs = *reinterpret_cast<const uint8_t*>(v + Page<FMT, D>::CODES + lane);
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(k + lane * 8), y = *reinterpret_cast<const uint2*>(v + lane * 8);
                kr[0] = make_uint4(x.x, x.y, 0, 0);
                vr[0] = make_uint4(y.x, y.y, 0, 0);
                ks = *reinterpret_cast<const uint8_t*>(k + Page<FMT, D>::CODES + (lane >> 1));
                vs = *reinterpret_cast<const uint8_t*>(v + Page<FMT, D>::CODES + (lane >> 1));
            }
        } else {
#pragma unroll
            for (int i = 0; i < VR; i++) {
                kr[i] = ld16(k + i * 1024 + lane * 16);
                vr[i] = ld16(v + i * 1024 + lane * 16);
            }
        }
    };
    auto sees = [&](int l, int e, int sk, int j) { return (j >= l && j < e) || j < sk; };
    // a page that some row of the workgroup does not see whole
    auto partial = [&](int blk) { return blk * KPAGE < lo_most || blk * KPAGE + KPAGE > hi_least; };
    auto store = [&](int buf) {
        // In such a page the values of rows that no query row sees become 0, and so does every value that is no number
        // (0 x NaN is NaN): the rows that do see it are given it at the end.
        const bool part = !myheld || partial(myblk);
        auto keep = [&](uint4 x, int key) {
            if (!part) return x;
            const int j = myblk * KPAGE + key;
            if (!myheld || !((j >= lo && j < hi) || (j < a.sinks && j < lo_most))) return make_uint4(0, 0, 0, 0);
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                constexpr uint32_t EX = H ? 0x7c00u : 0x7f80u;
                if ((w[e] & EX) == EX) { w[e] &= 0xffff0000u; odd = 1; }
                if ((w[e] >> 16 & EX) == EX) { w[e] &= 0xffffu; odd = 1; }
            }
            return make_uint4(w[0], w[1], w[2], w[3]);
        };
        if constexpr (FMT == FMT_FP4) {
            const int key = lane >> 2;
            const uint32_t kw[4] = {kr[0].x, kr[0].y, kr[0].z, kr[0].w}, vw[4] = {vr[0].x, vr[0].y, vr[0].z, vr[0].w};
#pragma unroll
            for (int e = 0; e < D / 32; e++) {
                const int p = v_at<D>(16 * wave + key, (lane & 3) * (D / 32) + e);
                *reinterpret_cast<uint4*>(kt[buf] + p) = fp4_to_16<H>(kw[e], ks);
                *reinterpret_cast<uint4*>(vt[buf] + p) = keep(fp4_to_16<H>(vw[e], vs), key);
            }
        } else {
            constexpr int PPR = D / 8;
#pragma unroll
            for (int i = 0; i < VR; i++) {
                const int key = (64 * i + lane) / PPR, p = v_at<D>(16 * wave + key, lane % PPR);
                *reinterpret_cast<uint4*>(kt[buf] + p) = kr[i];
                *reinterpret_cast<uint4*>(vt[buf] + p) = keep(vr[i], key);
            }
        }
        if (lane == 0) page_of[buf][wave] = myheld ? myblk : -1;
    };
    if (t0 < t1) {
        load(t0);
        store(0);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
    }
    for (int tile = t0; tile < t1; tile++) {
        const int buf = (tile - t0) & 1;
        if (tile + 1 < t1) {
            store(buf ^ 1);                        // read by all before the last barrier
            if (tile + 2 < t1) load(tile + 2);
        }
        int b[4];
        bool some = false;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            b[t] = __builtin_amdgcn_readfirstlane(page_of[buf][t]);
            some = some || b[t] < 0 || b[t] * KPAGE < wlo_most || b[t] * KPAGE + KPAGE > whi_least;
        }

        // ---- scores, keys 32 c + 8 (i / 4) + 4 h + i % 4 of the tile
        f32x16_t p[2];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) p[c][i] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int c = 0; c < 2; c++)
                p[c] = mfma32<H>(*reinterpret_cast<const uint4*>(kt[buf] + v_at<D>(32 * c + col, 2 * s + h)), qf[s], p[c]);
        if (some) {
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = 2 * c + (i >> 3), j = b[t] * KPAGE + 8 * ((i >> 2) & 1) + 4 * h + (i & 3);
                    p[c][i] = b[t] >= 0 && sees(rlo, rhi, rsk, j) ? p[c][i] : -INFINITY;
                }
        }
        float m = p[0][0];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int i = c == 0; i < 16; i++) m = fmaxf(m, p[c][i]);
        m = xmax32(m) * a.scale;
        if (__any(m > base + BASE_LAG)) {          // the row's first key too: base is -inf
            const float to = fmaxf(base, m), keep = to == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(base - to);
            rsum *= keep;
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[c][i] *= keep;
            base = to;
        }
        const float off = base == -INFINITY ? 0.0f : base;
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                p[c][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[c][i], a.scale, -off));
                sum += p[c][i];
            }
        rsum += sum;

        // ---- O^T += V^T . P^T, 16 keys at a time: 16 kk + 4 h .. + 3 and 8 on
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            const int x = 8 * (kk & 1);
            const f32x16_t& pp = p[kk >> 1];
            const uint4 pf = make_uint4(pack16<H>(pp[x], pp[x + 1]), pack16<H>(pp[x + 2], pp[x + 3]), pack16<H>(pp[x + 4], pp[x + 5]),
                                        pack16<H>(pp[x + 6], pp[x + 7]));
            const int r = 16 * kk + 4 * h + ((lane & 15) >> 2);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const int pc = 4 * c + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), hb = (lane & 1) * 8;
                const uint2 y = lds_tr16(vt[buf] + v_at<D>(r, pc) + hb), z = lds_tr16(vt[buf] + v_at<D>(r + 8, pc) + hb);
                o[c] = mfma32<H>(make_uint4(y.x, y.y, z.x, z.y), pf, o[c]);
            }
        }
        __syncthreads();
    }

    if (odd) {
        // values that are no numbers, in pages that the workgroup's rows see in part: to the rows that see them
        for (int u = 4 * t0; u < min(4 * t1, list.count); u++) {
            const int blk = page_at(list, u), page = bt[blk];
            if (!partial(blk) || page < 0 || page >= a.num_blocks) continue;
            const char* v = a.vp + ((int64_t)page * a.Hkv + kvh) * HEAD;
            for (int key = 0; key < KPAGE; key++) {
                const bool mine = sees(rlo, rhi, rsk, blk * KPAGE + key);
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int ch = 32 * c + 8 * (i >> 2) + 4 * h + (i & 3);
                        float x;
                        if constexpr (FMT == FMT_FP4) {
                            const uint8_t e = *reinterpret_cast<const uint8_t*>(v + Page<FMT, D>::CODES + key * (D / FP4_BLOCK) + ch / FP4_BLOCK);
                            x = e == 255 ? NAN : 0.0f;
                        } else {
                            const uint16_t w = *reinterpret_cast<const uint16_t*>(v + (key * D + ch) * 2);
                            x = H ? h2f(w) : bf2f(w);
                        }
                        o[c][i] += mine && !__builtin_isfinite(x) ? x : 0.0f;
                    }
            }
        }
    }

    if (!real) return;
    const float l = some_key ? xadd32(rsum) : 0.0f;
    // a row without a key: 0.  l is NaN where a score is (base may still be -inf then).
    const float inv = l == 0.0f ? 0.0f : a.splits > 1 ? 1.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = inv == 0.0f ? 0.0f : o[c][4 * i + e] * inv;
            const int ch = 32 * c + 8 * i + 4 * h;
            if (a.splits > 1) *reinterpret_cast<float4*>(a.part + (at * a.splits + split) * D + ch) = make_float4(y[0], y[1], y[2], y[3]);
            else store4<E>(static_cast<S*>(a.out) + at * D + ch, y);
        }
    if (a.splits > 1 && h == 0)
        *reinterpret_cast<float2*>(a.stat + (at * a.splits + split) * 2) = make_float2(some_key ? base : -INFINITY, l);
}

template <typename E, int FMT>
static void launch_prefill(const PrefillArgs& a, int n, int D, hipStream_t st) {
    const dim3 grid(a.Hkv, a.q_blocks * a.splits, n);
    const JoinRows rows{(int64_t)a.max_rows * a.Hq, a.Hq, a.rows, a.q_start, n};
    if (D == 128) {
        hipLaunchKernelGGL((prefill_kernel<E, FMT, 128>), grid, dim3(256), 0, st, a);
        if (a.splits > 1) launch_join<E, 128>(a.part, a.stat, a.out, rows, a.splits, st);
    } else {
        hipLaunchKernelGGL((prefill_kernel<E, FMT, 64>), grid, dim3(256), 0, st, a);
        if (a.splits > 1) launch_join<E, 64>(a.part, a.stat, a.out, rows, a.splits, st);
    }
}

// Blocks of 128 query rows of the longest sequence, and splits of their keys: wanted where the blocks leave CUs idle, and
// not below 8 tiles of 64 keys each.
constexpr int64_t PREFILL_TARGET = 256;
static int64_t prefill_blocks(int64_t max_rows, int64_t group) { return (max_rows * group + 127) / 128; }
static int prefill_splits(int64_t n, int64_t kv_heads, int64_t blocks, int64_t n_sinks, int64_t max_span) {
    return split_plan(n * kv_heads * blocks, (max_pages(max_span, n_sinks) + 3) / 4, PREFILL_TARGET, 1, 8).splits;
}

}  // namespace ud

using namespace ud;

extern "C" UD_API size_t ud_gqa_prefill_workspace_bytes(int32_t n, int32_t rows, int32_t max_rows, int32_t q_heads, int32_t kv_heads,
                                                        int32_t head_dim, int32_t n_sinks, int32_t max_span) {
    if (n <= 0 || rows <= 0 || max_rows <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads < kv_heads || head_dim <= 0 || n_sinks < 0 || max_span < 0) return 0;
    const int s = prefill_splits(n, kv_heads, prefill_blocks(max_rows, q_heads / kv_heads), n_sinks, max_span);
    return s == 1 ? 0 : (size_t)rows * q_heads * s * (head_dim + 2) * sizeof(float);
}

extern "C" UD_API int ud_gqa_prefill_paged(int32_t kv_format, int32_t dtype, const void* q_dev, const void* k_pages, const void* v_pages,
                                           int32_t num_blocks, const int32_t* block_table, int32_t max_blocks, const int32_t* q_start_dev,
                                           const int32_t* ranges_dev, int32_t n_sinks, void* out_dev, int32_t n, int32_t rows,
                                           int32_t max_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t block_size,
                                           int32_t max_span, void* workspace, size_t workspace_bytes, void* hip_stream) {
    static const char* who = "ud_gqa_prefill_paged";
    int rc = paged_check(who, kv_format, k_pages, v_pages, num_blocks, block_table, n, max_blocks, kv_heads, head_dim, block_size);
    if (rc != UD_OK) return rc;
    if (rows < 0 || rows > 1 << 30 || max_rows < 0 || max_rows > rows) return paged_fail(UD_ERR_SHAPE, "%s: rows %d, at most %d per sequence", who, rows, max_rows);
    if (rows == 0 || max_rows == 0) return UD_OK;
    if (!q_dev || !q_start_dev || !ranges_dev || !out_dev) return paged_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if (dtype != UD_BF16 && dtype != UD_F16) return paged_fail(UD_ERR_INVALID, "%s: dtype %d (bf16 or half)", who, dtype);
    if (kv_format != UD_MXFP4 && dtype != kv_format)
        return paged_fail(UD_ERR_INVALID, "%s: queries of dtype %d for pages of format %d (the same, or MXFP4 pages)", who, dtype, kv_format);
    if (q_heads < 1 || q_heads % kv_heads || q_heads / kv_heads > 128)
        return paged_fail(UD_ERR_SHAPE, "%s: heads %d/%d (groups of 1 .. 128)", who, q_heads, kv_heads);
    if (n_sinks < 0 || max_span < 0) return paged_fail(UD_ERR_SHAPE, "%s: %d sinks, span %d", who, n_sinks, max_span);
    const int G = q_heads / kv_heads;
    const int64_t blocks = prefill_blocks(max_rows, G);
    const int splits = prefill_splits(n, kv_heads, blocks, n_sinks, max_span);
    if (blocks * splits > 65535 || (splits > 1 && (int64_t)max_rows * q_heads > 1 << 25))
        return paged_fail(UD_ERR_SHAPE, "%s: %d rows of a sequence beyond the grid (65535 x 128 rows of a kv head)", who, max_rows);
    if (((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) return paged_fail(UD_ERR_INVALID, "%s: buffers must be 16-byte aligned", who);
    const size_t need = splits == 1 ? 0 : (size_t)rows * q_heads * splits * (head_dim + 2) * sizeof(float);
    if (need && !workspace) return paged_fail(UD_ERR_INVALID, "%s: null workspace", who);
    if (workspace_bytes < need) return paged_fail(UD_ERR_SHAPE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
    if ((uintptr_t)workspace & 15) return paged_fail(UD_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    PrefillArgs a{};
    a.q = q_dev; a.kp = static_cast<const char*>(k_pages); a.vp = static_cast<const char*>(v_pages); a.bt = block_table;
    a.q_start = q_start_dev; a.ranges = ranges_dev; a.out = out_dev;
    a.part = static_cast<float*>(workspace);
    a.stat = a.part + (size_t)rows * q_heads * splits * head_dim;
    a.rows = rows; a.max_rows = max_rows; a.G = G; a.Hq = q_heads; a.Hkv = kv_heads;
    a.max_blocks = max_blocks; a.num_blocks = num_blocks; a.sinks = n_sinks; a.splits = splits; a.q_blocks = (int)blocks;
    a.scale = (float)(1.4426950408889634 / sqrt((double)head_dim));
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (kv_format == UD_BF16) launch_prefill<ElBf, FMT_BF16>(a, n, head_dim, st);
    else if (kv_format == UD_F16) launch_prefill<ElH, FMT_F16>(a, n, head_dim, st);
    else if (dtype == UD_BF16) launch_prefill<ElBf, FMT_FP4>(a, n, head_dim, st);
    else launch_prefill<ElH, FMT_FP4>(a, n, head_dim, st);
    return paged_launched(who);
}
