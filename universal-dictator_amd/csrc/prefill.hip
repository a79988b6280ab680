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
// Measured, 32/8 heads of 128, causal: 8,192 rows of bf16 429 .. 490 us a call, 0.84 .. 0.96 PFLOP/s (the library's 8192^3
// product on the same card: 1.21); 6 x 37 .. 563 rows behind 4,000 .. 12,000 MXFP4 keys 300 .. 311 us, 0.80 .. 0.83 PFLOP/s with its
// join (half queries 329).  The chip holds 1.9 GHz there; matrix cores and vector units are busy 48 % and 47 % of the time, one
// after the other within a wave, side by side between the two of a SIMD.  Without bank conflicts.  One row group more per wave (64 rows) is slower, 515 us for 482:
// its registers leave one wave per SIMD.
//  - K and V rows lie in LDS at padded distances against bank conflicts; V^T is read by ds_read_b64_tr_b16.

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

// Eight codes of a block as pairs of the products' type.  As halves, a block whose scale is past 2^13 saturates and one below
// 2^-23 is rounded: bf16 products of two terms of q and of the probabilities would be exact, but twice as many, and q's second
// term does not fit the registers of two waves a SIMD.
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

// Keeps the instructions that make v where they are written.
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// f over 32 lanes (each half of the wave has the same values), in every lane.
template <int CTRL> __device__ __forceinline__ int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false); }
template <typename F> __device__ __forceinline__ int fold32(int v, F f) {
    v = f(v, dpp_int<DPP_QUAD_1032>(v));
    v = f(v, dpp_int<DPP_QUAD_2301>(v));
    v = f(v, dpp_int<DPP_ROW_HALF_MIRROR>(v));
    v = f(v, dpp_int<DPP_ROW_MIRROR>(v));
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    return f((int)r[0], (int)r[1]);
}

template <typename E, int FMT, int D>
__global__ __launch_bounds__(256, 2) void prefill_kernel(PrefillArgs a) {
    typedef typename E::S S;
    constexpr bool H = std::is_same<E, ElH>::value;
    constexpr int KS = D / 16, CT = D / 32;        // products over the channels; channel tiles
    constexpr int HEAD = Page<FMT, D>::BYTES;
    // Bytes between rows in LDS.  A lane's products read at fixed distances from one address each for K and V: no address
    // arithmetic between them (a permutation of the pieces would need some, and the loop is short of VALU slots).  K: 16
    // rows' pieces on distinct banks; V: 4 rows' 64 bytes on distinct banks.
    constexpr int KROW = 2 * D + 16, VROW = 2 * D + 64;
    constexpr int VR = FMT == FMT_FP4 ? 1 : D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, seq = blockIdx.z;
    const int split = blockIdx.y % a.splits, qb = a.q_blocks - 1 - (int)(blockIdx.y / a.splits);   // the longest first
    const int s0 = min(max(a.q_start[seq], 0), a.rows), s1 = min(min(max(a.q_start[seq + 1], s0), a.rows), s0 + a.max_rows);
    const int total = (s1 - s0) * a.G;             // at most 65535 x 128, the grid's limit
    if (qb * 128 >= total) return;
    __shared__ __align__(16) char kt[2][64 * KROW], vt[2][64 * VROW];
    __shared__ int fold[4][4];
    __shared__ int odd;                            // a value that is no number has been left out

    // ---- this lane's row, and what the workgroup's rows see
    const int rho = qb * 128 + 32 * wave + col, rr = min(rho, total - 1), tk = rr / a.G;
    const bool real = rho < total;
    const int64_t tok = s0 + tk, at = tok * a.Hq + (int64_t)kvh * a.G + (rr - tk * a.G);
    const int kmax = a.max_blocks * KPAGE;
    const int rlo = max(a.ranges[2 * tok], 0), rhi = min(a.ranges[2 * tok + 1], kmax);
    const bool some_key = real && rlo < rhi;
    const int rsk = some_key ? min(a.sinks, rlo) : 0;
    auto least = [](int x, int y) { return min(x, y); };
    auto most = [](int x, int y) { return max(x, y); };
    const int wlo = fold32(some_key ? rlo : kmax, least), whi = fold32(some_key ? rhi : 0, most);
    const int wlo_most = __builtin_amdgcn_readfirstlane(fold32(some_key ? rlo : 0, most));
    const int whi_least = __builtin_amdgcn_readfirstlane(fold32(some_key ? rhi : kmax, least));
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

    // ---- the pool's pages (or -1) of 16 tiles at a time, one a lane, and of the 16 after them: read long before their use,
    // since a tile's page is needed to even ask for its rows
    const int32_t* bt = a.bt + (int64_t)seq * a.max_blocks;
    auto look_up = [&](int tile) {
        const int u = 4 * tile + lane, page = u < list.count ? bt[page_at(list, u)] : -1;
        return page < a.num_blocks ? page : -1;
    };
    int now = look_up(t0), then = look_up(t0 + 16);
    uint64_t gaps = __ballot(now < 0);
    int group = 0;                                 // of 16 tiles, that `now` holds
    auto page_of = [&](int tile) {                 // this wave's page of a tile of `now` or `then`
        const int x = tile - t0;
        return __builtin_amdgcn_readlane((x >> 4) == group ? now : then, (4 * x + wave) & 63);
    };
    // bit t: page t of a tile of `now` is one of the pool's
    auto held_of = [&](int tile) { return (uint32_t)~(gaps >> (4 * ((tile - t0) & 15))) & 15u; };
    struct Rows { uint4 r[VR]; uint32_t e; };
    auto load = [&](const char* pool, int page) {
        Rows y;
        const char* m = pool + ((int64_t)max(page, 0) * a.Hkv + kvh) * HEAD;
        if constexpr (FMT == FMT_FP4) {
            if constexpr (D == 128) {
                y.r[0] = ld16(m + lane * 16u);
                y.e = *reinterpret_cast<const uint8_t*>(m + (Page<FMT, D>::CODES + lane));
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(m + lane * 8u);
                y.r[0] = make_uint4(v.x, v.y, 0, 0);
                y.e = *reinterpret_cast<const uint8_t*>(m + (Page<FMT, D>::CODES + (lane >> 1)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < VR; i++) y.r[i] = ld16(m + (i * 1024 + lane * 16u));
        }
        return y;
    };
    auto sees = [&](int j) { return (j >= rlo && j < rhi) || j < rsk; };
    // a page that some row of the workgroup does not see whole
    auto partial = [&](int blk) { return blk * KPAGE < lo_most || blk * KPAGE + KPAGE > hi_least; };
    // A page's rows go to LDS in PIECES writes a lane, which the products below are mixed with.  MXFP4: a lane's block is
    // PIECES pieces of its row, which lanes take in an order (e ^ turn) by which eight of them (two rows, which a write stores
    // at once) fill the 128 bytes that LDS takes.
    constexpr int PIECES = D / 32;
    const int k_turn = D == 128 ? lane & 2 : 0, v_turn = D == 128 ? lane & 3 : (lane >> 1) & 1;
    auto piece_at = [&](int e, int turn) {         // (row of the page, piece of the row)
        if constexpr (FMT == FMT_FP4) return make_int2(lane >> 2, (lane & 3) * PIECES + (e ^ turn));
        else return make_int2((64 * e + lane) / (D / 8), lane % (D / 8));
    };
    auto piece = [&](const Rows& y, int e) {       // MXFP4: of the turned words (load)
        if constexpr (FMT == FMT_FP4) return fp4_to_16<H>(e == 0 ? y.r[0].x : e == 1 ? y.r[0].y : e == 2 ? y.r[0].z : y.r[0].w, y.e);
        else return y.r[e];
    };
    auto turn_words = [&](Rows& y, int turn) {
        if constexpr (FMT == FMT_FP4) {
            uint4 v = y.r[0];
            v = turn & 1 ? make_uint4(v.y, v.x, v.w, v.z) : v;
            if constexpr (PIECES == 4) v = turn & 2 ? make_uint4(v.z, v.w, v.x, v.y) : v;
            y.r[0] = v;
        }
    };
    auto put = [&](char* dst, int row, const Rows& y, int e, int turn) {
        const int2 at = piece_at(e, turn);
        *reinterpret_cast<uint4*>(dst + (16 * wave + at.x) * row + at.y * 16) = piece(y, e);
    };
    // A page of values that rows see in part, put once more: the values of keys that no row sees as 0, and so every value that
    // is no number (0 x NaN is NaN): the rows that do see it are given it at the end.
    auto clean = [&](int tile, const Rows& y, int page) {
        const int u = 4 * tile + wave, blk = page_at(list, u < list.count ? u : 0);
        if (page >= 0 && !partial(blk)) return;
        char* dst = vt[(tile - t0) & 1];
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            const int2 at = piece_at(e, v_turn);
            const int j = blk * KPAGE + at.x;
            const uint4 v = piece(y, e);
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            const bool none = page < 0 || !((j >= lo && j < hi) || (j < a.sinks && j < lo_most));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                constexpr uint32_t EX = H ? 0x7c00u : 0x7f80u;
                const bool low = (w[i] & EX) == EX, high = (w[i] >> 16 & EX) == EX;
                if (!none && (low || high)) odd = 1;
                w[i] = none ? 0u : (low ? 0u : w[i] & 0xffffu) | (high ? 0u : w[i] & 0xffff0000u);
            }
            *reinterpret_cast<uint4*>(dst + (16 * wave + at.x) * VROW + at.y * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };

    f32x16_t p[2];                                 // scores: keys 32 c + 8 (i / 4) + 4 h + i % 4 of the tile
    float m = -INFINITY;                           // the largest, times log2(e) / sqrt(D)
    auto largest = [&]() {
        m = p[0][0];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int i = c == 0; i < 16; i++) m = fmaxf(m, p[c][i]);
    };
    auto key_frag = [&](const char* k, int c, int s) { return *reinterpret_cast<const uint4*>(k + 32 * c * KROW + 32 * s); };
    const int k_lane = col * KROW + 16 * h;
    const int v_lane = (4 * h + ((lane & 15) >> 2)) * VROW + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    // Scores that a row does not see become -inf, in tiles that some row of the wave does not see whole; then the base.
    auto finish = [&](int tile) {
        const uint32_t held = held_of(tile);
        const int first = 4 * tile - list.sink + list.first;      // its first page, behind the sinks
        if (held != 15 || 4 * tile < list.sink || first * KPAGE < wlo_most || first * KPAGE + 64 > whi_least) {
            int b[4];
#pragma unroll
            for (int t = 0; t < 4; t++) b[t] = page_at(list, 4 * tile + t);
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = 2 * c + (i >> 3), j = b[t] * KPAGE + 8 * ((i >> 2) & 1) + 4 * h + (i & 3);
                    p[c][i] = (held >> t & 1) && sees(j) ? p[c][i] : -INFINITY;
                }
            largest();
        }
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
    };

    if (t0 < t1) {
        // A tile's life: its keys are asked for two iterations before their product and its values two before theirs; K is
        // in LDS one iteration before Q . K^T, which runs one ahead of P . V, beside the exponentials of the tile before.
        int pk = page_of(t0), p1 = page_of(t0 + 1), pn = page_of(t0 + 2);
        Rows k = load(a.kp, pk), v = load(a.vp, pk), k1 = load(a.kp, p1);
        turn_words(k, k_turn);
        turn_words(v, v_turn);
        turn_words(k1, k_turn);
#pragma unroll
        for (int e = 0; e < PIECES; e++) { put(kt[0], KROW, k, e, k_turn); put(vt[0], VROW, v, e, v_turn); put(kt[1], KROW, k1, e, k_turn); }
        clean(t0, v, pk);
        pk = p1;
        k = load(a.kp, pn);
        v = load(a.vp, pk);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
            for (int i = 0; i < 16; i++) p[c][i] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++) p[c] = mfma32<H>(key_frag(kt[0] + k_lane, c, s), qf[s], p[c]);
        }
        largest();
        finish(t0);
        __syncthreads();
        // state: kt holds tile + 1, vt tile; k is tile + 2 and v tile + 1 on their way, pn and pk their pages
        auto turn = [&](int tile, auto more) {
            constexpr bool MORE = decltype(more)::value;
            // ---- the next tile's scores, two products at a time, and between them this tile's probabilities: packed pairs,
            // eight of a lane's scores being the B operand of 16 keys.  The order is kept by the scheduling barriers.
            f32x16_t x[2] = {p[0], p[1]};
            // halves: 2^7 times the probabilities, up to 2^15, so that small ones keep their bits (the sum has it too)
            float off = (base == -INFINITY ? 0.0f : base) - (H ? 7.0f : 0.0f);
            const bool steep = fabsf(off) >= STEEP;
            if (__builtin_expect(__any(steep), 0)) {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int i = 0; i < 16; i++) x[c][i] = steep ? steep_score(x[c][i], a.scale, base) : x[c][i];
                off = steep ? (H ? -7.0f : 0.0f) : off;
            }
            uint32_t pw[16];
            const char* kb = kt[(tile + 1 - t0) & 1] + k_lane;
            const char* vb = vt[(tile - t0) & 1] + v_lane;
            uint4 kf[2][2];
            if constexpr (MORE) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    kf[0][c] = key_frag(kb, c, 0);
#pragma unroll
                    for (int i = 0; i < 16; i++) p[c][i] = 0.0f;
                }
            }
#pragma unroll
            for (int s = 0; s < KS; s++) {
                if constexpr (MORE) {
                    if (s + 1 < KS) {
#pragma unroll
                        for (int c = 0; c < 2; c++) kf[(s + 1) & 1][c] = key_frag(kb, c, s + 1);
                    }
#pragma unroll
                    for (int c = 0; c < 2; c++) p[c] = mfma32<H>(kf[s & 1][c], qf[s], p[c]);
                }
#pragma unroll
                for (int n = 0; n < 16 / KS; n++) {
                    const int w = s * (16 / KS) + n, i = 2 * (w & 7);
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[w >> 3][i], a.scale, -off));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[w >> 3][i + 1], a.scale, -off));
                    pw[w] = pack16<H>(e0, e1);
                    rsum = dot_ones<H>(pw[w], rsum);
                }
                if constexpr (MORE) {
                    pin(rsum);
                    if (KS - s == PIECES) turn_words(k, k_turn);
                    if (KS - 1 - s < PIECES) put(kt[(tile - t0) & 1], KROW, k, KS - 1 - s, k_turn);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (MORE) {
                p1 = page_of(tile + 3);
                k = load(a.kp, p1);
            }
            // ---- O^T += V^T . P^T, 16 keys at a time (16 kk + 4 h .. + 3 and 8 on), and the next tile's largest score
            auto value_frag = [&](int z) {
                const char* at = vb + 16 * (z / CT) * VROW + 64 * (z % CT);
                const uint2 y = lds_tr16(at), z8 = lds_tr16(at + 8 * VROW);
                return make_uint4(y.x, y.y, z8.x, z8.y);
            };
            constexpr int Z = 4 * CT, AHEAD = 2;
            uint4 vf[AHEAD + 1];
#pragma unroll
            for (int z = 0; z < AHEAD; z++) vf[z] = value_frag(z);
            if constexpr (MORE) {
                m = p[0][0];
                turn_words(v, v_turn);
            }
#pragma unroll
            for (int z = 0; z < Z; z++) {
                if (z + AHEAD < Z) vf[(z + AHEAD) % (AHEAD + 1)] = value_frag(z + AHEAD);
                const int kk = z / CT;
                o[z % CT] = mfma32<H>(vf[z % (AHEAD + 1)], make_uint4(pw[4 * kk], pw[4 * kk + 1], pw[4 * kk + 2], pw[4 * kk + 3]), o[z % CT]);
                if constexpr (MORE) {
#pragma unroll
                    for (int i = 0; i < 32 / Z; i++) { const int n = z * (32 / Z) + i; m = fmaxf(m, p[n >> 4][n & 15]); }
                    pin(m);
                    if (z >= 2 && z < 2 + PIECES) put(vt[(tile + 1 - t0) & 1], VROW, v, z - 2, v_turn);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (MORE) {
                clean(tile + 1, v, pk);
                v = load(a.vp, pn);
                pk = pn;
                pn = p1;
                finish(tile + 1);
                __syncthreads();
            }
        };
        for (int tile = t0; tile + 1 < t1; tile++) {
            if (((tile + 1 - t0) & 15) == 0) {     // the next tile is the first of `then`
                group++;
                now = then;
                gaps = __ballot(now < 0);
                then = look_up(t0 + 16 * (group + 1));
            }
            turn(tile, std::true_type{});
        }
        turn(t1 - 1, std::false_type{});
    }
    __syncthreads();

    const float l = some_key ? xadd32(rsum) : 0.0f;
    // Values that are no numbers, to the rows that see them: an infinity, or NaN for both signs or a NaN.  Those of pages that
    // the workgroup's rows see in part were left out of the products, and those of whole pages may have become either there
    // (0 x infinity, where a probability is 0 in 16 bits), so both are taken from the pages.  (A block of MXFP4 that is no
    // number is NaN in every product.)
    bool bad = odd;
    if constexpr (FMT != FMT_FP4) {                // (one sum: a test for each of the 64 took 0.4 us of a short prompt)
        f32x4_t t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) t[i & 3] += o[c][i];
        bad |= !__builtin_isfinite((t[0] + t[1]) + (t[2] + t[3]));
    }
    bad = bad && some_key && l == l;
    if (__builtin_expect(__any(bad), 0)) {
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float sum[4][4] = {};
            for (int u = 4 * t0; u < min(4 * t1, list.count); u++) {
                const int blk = page_at(list, u), page = bt[blk];
                if (page < 0 || page >= a.num_blocks) continue;
                bool open = false;                 // NaN is final
#pragma unroll
                for (int i = 0; i < 16; i++) open |= (odd || !__builtin_isfinite(o[c][i])) && sum[i >> 2][i & 3] == sum[i >> 2][i & 3];
                if (!__any(bad && open)) break;
                const char* v = a.vp + ((int64_t)page * a.Hkv + kvh) * HEAD;
                for (int key = 0; key < KPAGE; key++)
                    if (sees(blk * KPAGE + key)) {
#pragma unroll
                        for (int i = 0; i < 4; i++) odd_values<FMT, D>(v, key, 32 * c + 8 * i + 4 * h, sum[i]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 16; i++) o[c][i] = bad && sum[i >> 2][i & 3] != 0.0f ? sum[i >> 2][i & 3] : o[c][i];
        }
    }

    if (!real) return;
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
