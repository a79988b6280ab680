// Attention of 1 .. 8 query positions per sequence over the sinks and the sliding window of a paged cache, held in
// bf16, half or MXFP4 (include/ud_decode.h).
//
//   out[r] = sum_j softmax_j(q[r] . k[j] / sqrt(D)) v[j]   over j in [0, min(sinks, lo_r)) and [lo_r, hi_r)
//
// Bound: HBM; every visible K and V byte is read once.  One workgroup = (kv head, split of the page list, sequence);
// its rows are the M positions times the G query heads of the kv head, up to 32 (two tiles of 16), so a page is read
// once for all of them; above 32 rows a second workgroup takes the rest, on the same XCD at 8 kv heads (the rows of 64
// would not leave the registers room).  Each of the 4 or 8 waves takes chunks of its split's pages (2 pages of 16 bits, 4 of MXFP4) on its
// own, with its own running maximum and sum, so the loop has no barrier; the waves join once at the end, the splits in
// a second kernel.
//  - S^T = K . Q^T on v_mfma_f32_16x16x32: lane (c, g) loads the channels that the A operand wants of key c straight
//    into registers.  An MXFP4 lane's 16 bytes are one block of 32 channels, whose pieces serve the products over all
//    blocks in turn (the channel order within a sum is free as long as q has the same).
//  - lane (c, g) then holds row c's scores of keys 4g .. 4g + 3 of each tile, which is the B operand of
//    O^T = V^T . P^T as it stands.  V goes through the wave's own LDS tile and comes back transposed by
//    ds_read_b64_tr_b16.  MXFP4 is turned into bf16, which holds its values exactly, on the way.
//  - 16-bit operands with fp32 accuracy: a factor is split into terms (x = x0 + x1 + .., each the nearest 16-bit value
//    of what is left), one product each.  q: one term of its own type; half for bf16 products two; fp32 three of bf16 or
//    two of half (scaled by a power of two per row, so that no term leaves half's range).  Probabilities: as many terms
//    as the output's type can show.
// Measured, 32/8 heads of 128: 64 contexts of 500 .. 20,000 keys with a window of 4,096, bf16 pages (982 MB) 168 us, 5.8 TB/s;
// 64 x 4,096 keys 182 us, of which the loads alone take all but 2.  MXFP4 pages, 64 x 4,096 keys 55.5 us, the loads alone 52;
// 64 x 512 .. 8,192 keys (304 MB) 66 us, 4.6 TB/s: conversions, products and softmax in turn in each wave.  One sequence of 8,192 half
// keys is latency: 13 us in 32 splits, and 4 for the join.
#include <type_traits>

#include "paged_attention.hpp"

namespace ud {

struct WindowArgs {
    const void* q;                 // [n][M][Hq][D]
    const char* kp; const char* vp;
    const int32_t* bt;
    const int32_t* ranges;         // [n][M][2]
    void* out;                     // [n][M][Hq][D]
    float* part;                   // [n][M][Hq][splits][D], then (maximum, sum) [n][M][Hq][splits][2]
    float* stat;
    int M, G, Hq, Hkv;
    int max_blocks, num_blocks;
    int sinks, splits, pages, groups;   // pages of a split, groups of 16 RT rows
    int n, layer;                  // sequences; > 0: taken by length (rank_of_layer)
    float scale;                   // log2(e) / sqrt(D)
};

// Terms of q and of the probabilities.
template <typename E, int FMT> struct Terms {
    static constexpr bool H = FMT == FMT_F16;      // half products; else bf16
    static constexpr int Q = std::is_same<E, El32>::value ? (H ? 2 : 3) : FMT == FMT_FP4 && std::is_same<E, ElH>::value ? 2 : 1;
    static constexpr int P = std::is_same<E, El32>::value ? (H ? 2 : 3) : std::is_same<E, ElH>::value && !H ? 2 : 1;
};

// The sequence of layer z of the workgroups where a batch is taken by length (rank_of_layer, length_key).  Each wave ranks them
// by itself: a lane's sequence has as many before it as have a larger key.  Also its range, from the first lo to the last hi.
__device__ __forceinline__ int sorted_sequence(const WindowArgs& a, int z, int& lo, int& hi) {
    const int lane = threadIdx.x & 63, kmax = a.max_blocks * KPAGE;
    int key = -1, l = 0, h = 0;
    if (lane < a.n) {
        const int32_t* rg = a.ranges + (int64_t)2 * lane * a.M;
        l = max(rg[0], 0);
        h = min(max(rg[2 * a.M - 1], 0), kmax);
        key = length_key(h - l, lane);
    }
    int before = 0;
    for (int j0 = 0; j0 < a.n; j0 += 8)
#pragma unroll
        for (int j = 0; j < 8; j++) before += __builtin_amdgcn_readlane(key, j0 + j) > key;
    const int rank = rank_of_layer(z, a.layer, a.n);
    const int seq = __builtin_ctzll(__ballot(key >= 0 && before == rank));
    lo = __builtin_amdgcn_readlane(l, seq);
    hi = __builtin_amdgcn_readlane(h, seq);
    return seq;
}

template <typename E, int FMT, int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW, RT == 1 ? 2 : 1) void window_split_kernel(WindowArgs a) {
    typedef typename E::S S;
    constexpr bool H = Terms<E, FMT>::H;
    constexpr int QT = Terms<E, FMT>::Q, PT = Terms<E, FMT>::P;
    constexpr int CP = FMT == FMT_FP4 ? 4 : 2;     // pages per chunk
    constexpr int KS = D / 32;                     // products over the channels
    constexpr int DT = D / 16;                     // channel tiles
    constexpr int HEAD = Page<FMT, D>::BYTES;
    // Bytes between the rows of V in LDS: 8 rows' 32 bytes, which a product reads at once, lie on distinct banks, and every
    // product reads at a fixed distance from one address (no address arithmetic between them).  MXFP4 at D = 128: a row's
    // even pieces of 16 bytes before its odd ones (HALVES), so that the writes, four pieces a lane, are without conflicts too.
    constexpr bool HALVES = FMT == FMT_FP4 && D == 128;
    constexpr int VROW = HALVES ? 2 * D + 16 : 2 * D + 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x, split = blockIdx.y / a.groups;
    int seq_lo = 0, seq_hi = 0;
    const int seq = a.layer ? sorted_sequence(a, blockIdx.z, seq_lo, seq_hi) : (int)blockIdx.z;
    const int r0 = blockIdx.y % a.groups * (16 * RT);   // first of this workgroup's rows
    const int G = a.G, M = a.M, QR = min(M * G - r0, 16 * RT);
    __shared__ __align__(16) char tile[NW][32 * VROW];
    __shared__ float wmax[NW][16 * RT], wsum[NW][16 * RT];
    __shared__ int odd_of[NW];

    // ---- the sequence's page list, and this lane's rows (row 16 rt + col: position r / G, head r % G)
    const int32_t* rg = a.ranges + (int64_t)2 * seq * M;
    const int kmax = a.max_blocks * KPAGE;
    int lo = kmax, hi = 0, lo_most = 0, hi_least = kmax;
    const int m0 = r0 ? r0 / G : 0, m1 = a.groups == 1 ? M - 1 : (r0 + QR - 1) / G;
    for (int m = m0; m <= m1; m++) {
        const bool known = a.layer && M == 1;
        const int l = known ? seq_lo : max(rg[2 * m], 0), h = known ? seq_hi : min(rg[2 * m + 1], kmax);
        if (l < h) {
            lo = min(lo, l); hi = max(hi, h);
            lo_most = max(lo_most, l); hi_least = min(hi_least, h);
        }
    }
    // (wave-uniform values in scalar registers: addresses of pages are then a scalar base and a lane's fixed offset)
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo_most = __builtin_amdgcn_readfirstlane(lo_most);
    hi_least = __builtin_amdgcn_readfirstlane(hi_least);
    const PageList list = page_list(lo, hi, a.sinks);
    const int u0 = (int)min((int64_t)split * a.pages, (int64_t)list.count);
    const int u1 = split == a.splits - 1 ? list.count : (int)min((int64_t)u0 + a.pages, (int64_t)list.count);
    const int64_t row0 = (int64_t)seq * M * a.Hq + (int64_t)kvh * G;         // (position 0, head 0) of the group
    auto out_row = [&](int r) { return row0 + (int64_t)((r0 + r) / G) * a.Hq + (r0 + r) % G; };
    if (u0 >= u1) {                                // no key here
        if (a.splits > 1 && tid < QR)
            *reinterpret_cast<float2*>(a.stat + (out_row(tid) * a.splits + split) * 2) = make_float2(-INFINITY, 0.0f);
        if (a.splits == 1) {
            const float z[4] = {0, 0, 0, 0};
            for (int x = tid; x < QR * (D / 4); x += 64 * NW)
                store4<E>(static_cast<S*>(a.out) + out_row(x / (D / 4)) * D + x % (D / 4) * 4, z);
        }
        return;
    }
    int rlo[RT], rhi[RT], rsk[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int m = (r0 + min(16 * rt + col, QR - 1)) / G;
        rlo[rt] = max(rg[2 * m], 0);
        rhi[rt] = min(rg[2 * m + 1], kmax);
        rsk[rt] = rlo[rt] < rhi[rt] ? min(a.sinks, rlo[rt]) : 0;
    }

    // ---- q: B operand, lane (c, g): row c's channels chan(s) .. + 7 for product s
    uint4 qf[RT][KS][QT];
    float qscale[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int r = 16 * rt + col;
        const S* q = static_cast<const S*>(a.q) + out_row(min(r, QR - 1)) * D + (FMT == FMT_FP4 ? g * (D / 4) : 8 * g);
        constexpr int STEP = FMT == FMT_FP4 ? 8 : 32;
        qscale[rt] = a.scale;
        if constexpr (QT == 1) {
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const uint4 x = ld16(q + STEP * s);
                qf[rt][s][0] = r < QR ? x : make_uint4(0, 0, 0, 0);
            }
        } else {
            float x[KS][8];
            float most = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                float u[4], v[4];
                load4<E>(q + STEP * s, u);
                load4<E>(q + STEP * s + 4, v);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[s][e] = r < QR ? u[e] : 0.0f;
                    x[s][4 + e] = r < QR ? v[e] : 0.0f;
                    most = fmaxf(most, fmaxf(fabsf(x[s][e]), fabsf(x[s][4 + e])));
                }
            }
            if constexpr (H) {                     // the row's largest value to 2^10 .. 2^11
                most = xmax32(xmax16(most));
                const int ex = most > 0.0f && most < INFINITY ? 10 - max(ilogbf(most), -110) : 0;
                const float up = ldexpf(1.0f, ex);
                qscale[rt] = a.scale * ldexpf(1.0f, -ex);
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[s][e] *= up;
            }
#pragma unroll
            for (int s = 0; s < KS; s++) split8<H, QT>(x[s], qf[rt][s]);
        }
    }

    f32x4_t o[DT][RT];
    // probabilities are 2^(score - base): base follows the running maximum, but not before that is BASE_LAG ahead, so that
    // the sums are hardly ever rescaled (a probability is then at most 2^BASE_LAG)
    constexpr float BASE_LAG = 8.0f;
    float rmax[RT], rsum[RT];                      // base (all of the row), sum (this lane's keys)
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        rmax[rt] = -INFINITY;
        rsum[rt] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d][rt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // ---- the wave's chunks: pages u0 + CP wave, + NW CP, ..  Lane l holds where the l-th of the next 64 pages of the wave
    // lies in the pools (page 0 where it is none of theirs), so that the table is read once for 64 / CP chunks, not before
    // each.
    const int32_t* bt = a.bt + (int64_t)seq * a.max_blocks;
    uint32_t page_lo = 0, page_hi = 0;
    uint64_t in_pools = 0;                         // bit l: of lane l's page
    auto look_up = [&](int u) __attribute__((always_inline)) {
        const int at = u + lane / CP * (NW * CP) + lane % CP;
        const int page = at < u1 ? bt[page_at(list, at)] : -1;
        const bool ours = page >= 0 && page < a.num_blocks;
        const uint64_t base = ((uint64_t)(ours ? page : 0) * a.Hkv + kvh) * HEAD;
        page_lo = (uint32_t)base;
        page_hi = (uint32_t)(base >> 32);
        in_pools = __ballot(ours);
    };
    // 16-bit: kr[page][s], vr[page][i] rows 16 bytes a lane.  MXFP4: one piece and one exponent per page (D = 64: half).
    constexpr int KR = FMT == FMT_FP4 ? 1 : KS, VR = FMT == FMT_FP4 ? 1 : D / 32;
    uint4 kr[CP][KR], vr[CP][VR];
    uint32_t ks[CP], vs[CP];
    uint32_t held = 0;                             // bit t: the page is one of the pool's
    char* vt = tile[wave];
    // a page that every row sees whole
    auto whole = [&](int blk) { return blk * KPAGE >= lo_most && blk * KPAGE + KPAGE <= hi_least; };
    bool odd = false;                              // a value that is no number has been left out
    auto load = [&](int first) __attribute__((always_inline)) {                   // first: lane that holds the chunk's first page
        const uint32_t k_off = FMT == FMT_FP4 ? col * (D / 2) + g * (D / 8) : col * (2 * D) + 16 * g, v_off = lane * (FMT == FMT_FP4 ? D / 8 : 16);
        const uint32_t ks_off = Page<FMT, D>::CODES + col * (D / 32) + (D == 128 ? g : g >> 1);
        const uint32_t vs_off = Page<FMT, D>::CODES + (D == 128 ? lane : lane >> 1);
        held = (uint32_t)(in_pools >> first) & ((1u << CP) - 1);
#pragma unroll
        for (int t = 0; t < CP; t++) {
            const uint32_t lo32 = __builtin_amdgcn_readlane(page_lo, first + t), hi32 = __builtin_amdgcn_readlane(page_hi, first + t);
            const uint64_t base = (uint64_t)hi32 << 32 | lo32;
            const char* k = a.kp + base;
            const char* v = a.vp + base;
            if constexpr (FMT == FMT_FP4) {
                if constexpr (D == 128) {
                    kr[t][0] = ld16(k + k_off);
                    vr[t][0] = ld16(v + v_off);
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(k + k_off), y = *reinterpret_cast<const uint2*>(v + v_off);
                    kr[t][0] = make_uint4(x.x, x.y, 0, 0);
                    vr[t][0] = make_uint4(y.x, y.y, 0, 0);
                }
                ks[t] = *reinterpret_cast<const uint8_t*>(k + ks_off);
                vs[t] = *reinterpret_cast<const uint8_t*>(v + vs_off);
            } else {
#pragma unroll
                for (int s = 0; s < KS; s++) kr[t][s] = ld16(k + (k_off + 64 * s));
#pragma unroll
                for (int i = 0; i < VR; i++) vr[t][i] = ld16(v + (v_off + i * 1024));
            }
        }
    };

    int u = u0 + CP * wave, next = 0;              // next: lane of the next chunk's first page
    if (u < u1) {
        look_up(u);
        load(0);
        next = CP;
    }
    for (; u < u1; u += NW * CP) {
        // ---- scores (of q as it was scaled), row c's keys 16t + 4g + i
        // (the tiles side by side: their products do not wait for each other)
        float p[RT][CP][4];
        f32x4_t acc[RT][CP];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int t = 0; t < CP; t++) acc[rt][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int t = 0; t < CP; t++) {
                uint4 kf;
                if constexpr (FMT == FMT_FP4) {
                    const uint32_t w = s == 0 ? kr[t][0].x : s == 1 ? kr[t][0].y : s == 2 ? kr[t][0].z : kr[t][0].w;
                    kf = fp4_to_bf16(w, fp4_scale(ks[t]));
                } else {
                    kf = kr[t][s];
                }
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int x = QT - 1; x >= 0; x--) acc[rt][t] = mfma16<H>(kf, qf[rt][s][x], acc[rt][t]);
            }
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int t = 0; t < CP; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) p[rt][t][i] = acc[rt][t][i];
        const uint32_t in_pool = held;
        // a chunk that some row does not see whole (a row that sees nothing does not count: it is dropped at the end)
        const int first = u - list.sink + list.first;
        const bool some = in_pool != (1u << CP) - 1 || u < list.sink || first * KPAGE < lo_most || (first + CP) * KPAGE > hi_least;
        uint4 vb[2][VR];
        uint32_t vbs[2];
        // The V rows of 32 keys into the wave's tile (the rows of a second 32 are kept in registers until then).  MXFP4: a
        // lane's block, or (D = 64) half a block, whose two pieces are turned so that eight lanes (two rows, which a write
        // stores at once) fill the 128 bytes that LDS takes.
        const int turned = FMT == FMT_FP4 && D == 64 ? (lane >> 2) & 1 : 0;
        auto at = [&](int tt, int e) {
            const int row = FMT == FMT_FP4 ? lane >> 2 : (64 * e + lane) / (D / 8);
            const int piece = FMT == FMT_FP4 ? (lane & 3) * (D / 32) + (e ^ turned) : lane % (D / 8);
            return make_int2(row, (16 * tt + row) * VROW + (HALVES ? (piece & 1) * D + (piece >> 1) * 16 : piece * 16));
        };
        auto put_v = [&](int half) __attribute__((always_inline)) {
            __builtin_amdgcn_wave_barrier();       // the reads of the last 32 keys come first
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int e = 0; e < D / 32; e++) {
                    uint4 x;
                    if constexpr (FMT == FMT_FP4) {
                        const uint32_t w[4] = {vb[tt][0].x, vb[tt][0].y, vb[tt][0].z, vb[tt][0].w};
                        x = fp4_to_bf16(turned ? w[e ^ 1] : w[e], fp4_scale(vbs[tt]));
                    } else {
                        x = vb[tt][e];
                    }
                    *reinterpret_cast<uint4*>(vt + at(tt, e).y) = x;
                }
            if (__builtin_expect(some, 0)) {
                // In pages that rows see in part, values of keys that no row sees become 0, and so does every value that is
                // no number (0 x NaN is NaN): the rows that do see it are given it at the end.  (A loop over what this lane has
                // just written: few instructions, seldom run.)
#pragma unroll 1
                for (int i = 0; i < D / 16; i++) {
                    const int tt = i / (D / 32), t = 2 * half + tt, blk = page_at(list, u + t);
                    if ((in_pool >> t & 1) && whole(blk)) continue;
                    const int2 x = at(tt, i % (D / 32));
                    const int j = blk * KPAGE + x.x;
                    const bool none = !(in_pool >> t & 1) || !((j >= lo && j < hi) || (j < a.sinks && j < lo_most));
                    uint32_t* w = reinterpret_cast<uint32_t*>(vt + x.y);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        constexpr uint32_t EX = H ? 0x7c00u : 0x7f80u;
                        const uint32_t v = w[k];
                        const bool low = (v & EX) == EX, high = (v >> 16 & EX) == EX;
                        w[k] = none ? 0u : (low ? 0u : v & 0xffffu) | (high ? 0u : v & 0xffff0000u);
                        odd |= !none && (low || high);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        };
        auto take = [&](int half) __attribute__((always_inline)) {
#pragma unroll
            for (int tt = 0; tt < 2; tt++) {
                vbs[tt] = vs[2 * half + tt];
#pragma unroll
                for (int i = 0; i < VR; i++) vb[tt][i] = vr[2 * half + tt][i];
            }
        };
        take(0);
        put_v(0);
        if constexpr (CP > 2) take(1);
        if (u + NW * CP < u1) {
            if (next == 64) { look_up(u + NW * CP); next = 0; }
            load(next);
            next += CP;
        }
        if (__builtin_expect(some, 0)) {
#pragma unroll
            for (int t = 0; t < CP; t++) {
                const int j0 = page_at(list, u + t) * KPAGE + 4 * g;
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = j0 + i;
                        const bool in = (in_pool >> t & 1) && ((j >= rlo[rt] && j < rhi[rt]) || j < rsk[rt]);
                        p[rt][t][i] = in ? p[rt][t][i] : -INFINITY;
                    }
            }
        }
        // ---- running maximum and sum, probabilities
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float m = p[rt][0][0];
#pragma unroll
            for (int t = 0; t < CP; t++)
#pragma unroll
                for (int i = t == 0; i < 4; i++) m = fmaxf(m, p[rt][t][i]);
            m = xmax32(xmax16(m)) * qscale[rt];
            if (__any(m > rmax[rt] + BASE_LAG)) {  // the row's first key too: base is -inf
                const float to = fmaxf(rmax[rt], m), keep = to == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rmax[rt] - to);
                rsum[rt] *= keep;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[d][rt][i] *= keep;
                rmax[rt] = to;
            }
            // halves: 2^7 times the probabilities, up to 2^15, so that small ones keep their bits (the sum has it too)
            float off = (rmax[rt] == -INFINITY ? 0.0f : rmax[rt]) - (H ? 7.0f : 0.0f);
            const bool steep = fabsf(off) >= STEEP;
            if (__builtin_expect(__any(steep), 0)) {
#pragma unroll
                for (int t = 0; t < CP; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) p[rt][t][i] = steep ? steep_score(p[rt][t][i], qscale[rt], rmax[rt]) : p[rt][t][i];
                off = steep ? (H ? -7.0f : 0.0f) : off;
            }
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < CP; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[rt][t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[rt][t][i], qscale[rt], -off));
                    if constexpr (PT > 1) sum += p[rt][t][i];
                }
            rsum[rt] += sum;                       // one term: summed below, as rounded
        }
        // ---- O^T += V^T . P^T, 32 keys at a time through the wave's tile
#pragma unroll
        for (int half = 0; half < CP / 2; half++) {
            if (half) put_v(half);
            uint4 pf[RT][PT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; i++) { x[i] = p[rt][2 * half][i]; x[4 + i] = p[rt][2 * half + 1][i]; }
                split8<H, PT>(x, pf[rt]);
                if constexpr (PT == 1) {
                    const uint4 y = pf[rt][0];
                    rsum[rt] = dot_ones<H>(y.w, dot_ones<H>(y.z, dot_ones<H>(y.y, dot_ones<H>(y.x, rsum[rt]))));
                }
            }
            const char* v_lane = vt + (4 * g + (col >> 2)) * VROW + (HALVES ? 8 * (col & 1) + ((col >> 1) & 1) * D : 8 * (col & 3));
            constexpr int VD = HALVES ? 16 : 32;   // bytes between the channel tiles
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const uint2 x = lds_tr16(v_lane + VD * d), y = lds_tr16(v_lane + VD * d + 16 * VROW);
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int k = PT - 1; k >= 0; k--) o[d][rt] = mfma16<H>(make_uint4(x.x, x.y, y.x, y.y), pf[rt][k], o[d][rt]);
            }
        }
    }
    // ---- the waves joined, a row tile at a time through their LDS tiles
    if (lane == 0) odd_of[wave] = 0;
    if (odd) odd_of[wave] = 1;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const float l = xadd32(xadd16(rsum[rt]));
        const bool empty = rlo[rt] >= rhi[rt];
        if (empty) rmax[rt] = -INFINITY;
        if (g == 0) { wmax[wave][16 * rt + col] = rmax[rt]; wsum[wave][16 * rt + col] = empty ? 0.0f : l; }
    }
    __syncthreads();
    // Channels ch .. ch + 3 of row r where it sees values that are no numbers: their sum, so an infinity, or NaN for both signs or
    // a NaN.  Those of pages that rows see in part were left out of the products, and those of whole pages may have become
    // either there (a probability that is 0 in fp32, or whose second term is), so both are taken from the pages.
    auto give_odd = [&](int r, int ch, bool left_out, float (&y)[4]) {
        const int m = (r0 + r) / G, l = max(rg[2 * m], 0), e = min(rg[2 * m + 1], kmax), sk = l < e ? min(a.sinks, l) : 0;
        float sum[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (int c = u0; c < u1; c++) {
            const int blk = page_at(list, c), page = bt[blk];
            if (page < 0 || page >= a.num_blocks) continue;
            bool open = false;                     // NaN is final
            for (int i = 0; i < 4; i++) open |= (left_out || !__builtin_isfinite(y[i])) && sum[i] == sum[i];
            if (!open) break;
            const char* v = a.vp + ((int64_t)page * a.Hkv + kvh) * HEAD;
#pragma unroll 1
            for (int key = 0; key < KPAGE; key++) {
                const int j = blk * KPAGE + key;
                if (!((j >= l && j < e) || j < sk)) continue;
                odd_values<FMT, D>(v, key, ch, sum);
            }
        }
        for (int i = 0; i < 4; i++) y[i] = sum[i] != 0.0f ? sum[i] : y[i];
    };
    // a wave's share of a row with maximum m over the waves (1 where both are -inf: a sum of NaN scores stays NaN)
    auto share = [](float mine, float m) { return mine == m ? 1.0f : __builtin_amdgcn_exp2f(mine - m); };
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int rr = 16 * rt + col;
        float m = wmax[0][rr];
#pragma unroll
        for (int w = 1; w < NW; w++) m = fmaxf(m, wmax[w][rr]);
        // a wave without a key of the row adds nothing
        const bool none = rmax[rt] == -INFINITY;
        const float f = share(rmax[rt], m);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const float4 x = none ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                  : make_float4(o[d][rt][0] * f, o[d][rt][1] * f, o[d][rt][2] * f, o[d][rt][3] * f);
            *reinterpret_cast<float4*>(vt + col * (4 * D) + (((4 * d + g) ^ col) << 4)) = x;
        }
        __syncthreads();
        for (int x = tid; x < 16 * (D / 4); x += 64 * NW) {
            const int c = x / (D / 4), piece = x % (D / 4), r = 16 * rt + c;
            if (r >= QR) continue;
            float y[4] = {0, 0, 0, 0};
            float mm = wmax[0][r], l = 0.0f;
            int any_odd = 0;
#pragma unroll
            for (int w = 1; w < NW; w++) mm = fmaxf(mm, wmax[w][r]);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float4 v = *reinterpret_cast<const float4*>(tile[w] + c * (4 * D) + ((piece ^ c) << 4));
                y[0] += v.x; y[1] += v.y; y[2] += v.z; y[3] += v.w;
                l += wsum[w][r] * share(wmax[w][r], mm);
                any_odd |= odd_of[w];
            }
            // (a block of MXFP4 that is no number is NaN in every product)
            const bool odd_here = any_odd || (FMT != FMT_FP4 && !__builtin_isfinite(y[0] + y[1] + y[2] + y[3]));
            if (__builtin_expect(odd_here && l == l, 0)) give_odd(r, 4 * piece, any_odd, y);
            if (a.splits == 1) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] *= inv;
                store4<E>(static_cast<S*>(a.out) + out_row(r) * D + 4 * piece, y);
            } else {
                const int64_t at = out_row(r) * a.splits + split;
                *reinterpret_cast<float4*>(a.part + at * D + 4 * piece) = make_float4(y[0], y[1], y[2], y[3]);
                if (piece == 0) *reinterpret_cast<float2*>(a.stat + at * 2) = make_float2(mm, l);
            }
        }
        if (rt + 1 < RT) __syncthreads();
    }
}

template <typename E, int FMT, int D>
static void launch_window_d(const WindowArgs& a, const WindowPlan& plan, hipStream_t st) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(a.Hkv, a.splits * a.groups, a.n), dim3(64 * plan.waves), 0, st, a);
    };
    if constexpr (FMT != FMT_FP4)
        if (plan.waves == 8) go(window_split_kernel<E, FMT, D, 1, 8>);
    if (plan.waves == 4) {
        if (plan.tiles == 1) go(window_split_kernel<E, FMT, D, 1, 4>);
        else go(window_split_kernel<E, FMT, D, 2, 4>);
    }
    if (a.splits > 1) launch_join<E, D>(a.part, a.stat, a.out, JoinRows{(int64_t)a.n * a.M * a.Hq, 0, 0, nullptr, 1}, a.splits, st);
}
template <typename E, int FMT>
static void launch_window(const WindowArgs& a, int D, const WindowPlan& plan, hipStream_t st) {
    if (D == 128) launch_window_d<E, FMT, 128>(a, plan, st);
    else launch_window_d<E, FMT, 64>(a, plan, st);
}

}  // namespace ud

using namespace ud;

extern "C" UD_API size_t ud_gqa_window_workspace_bytes(int32_t n, int32_t n_queries, int32_t q_heads, int32_t kv_heads,
                                                       int32_t head_dim, int32_t n_sinks, int32_t max_span) {
    if (n <= 0 || n_queries <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || n_sinks < 0 || max_span < 0) return 0;
    const int s = window_most_splits(n, kv_heads, n_sinks, max_span);
    return s == 1 ? 0 : (size_t)n * n_queries * q_heads * s * (head_dim + 2) * sizeof(float);
}

extern "C" UD_API int ud_gqa_window_attention_paged(int32_t kv_format, int32_t dtype, const void* q_dev, const void* k_pages,
                                                    const void* v_pages, int32_t num_blocks, const int32_t* block_table,
                                                    int32_t max_blocks, const int32_t* ranges_dev, int32_t n_sinks, void* out_dev,
                                                    int32_t n, int32_t n_queries, int32_t q_heads, int32_t kv_heads,
                                                    int32_t head_dim, int32_t block_size, int32_t max_span, void* workspace,
                                                    size_t workspace_bytes, void* hip_stream) {
    static const char* who = "ud_gqa_window_attention_paged";
    int rc = paged_check(who, kv_format, k_pages, v_pages, num_blocks, block_table, n, max_blocks, kv_heads, head_dim, block_size);
    if (rc != UD_OK) return rc;
    if (!q_dev || !ranges_dev || !out_dev) return paged_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if (dtype != UD_F32 && dtype != UD_BF16 && dtype != UD_F16) return paged_fail(UD_ERR_INVALID, "%s: dtype %d", who, dtype);
    if (kv_format != UD_MXFP4 && dtype != UD_F32 && dtype != kv_format)
        return paged_fail(UD_ERR_INVALID, "%s: queries of dtype %d for pages of format %d (the same, or fp32, or MXFP4 pages)", who, dtype, kv_format);
    if (n_queries < 1 || n_queries > 8) return paged_fail(UD_ERR_SHAPE, "%s: %d queries per sequence (1 .. 8)", who, n_queries);
    if (q_heads < 1 || q_heads % kv_heads || (int64_t)q_heads / kv_heads * n_queries > 64)
        return paged_fail(UD_ERR_SHAPE, "%s: heads %d/%d x %d queries (at most 64 rows per kv head)", who, q_heads, kv_heads, n_queries);
    if ((int64_t)n * n_queries * q_heads > 1 << 25)
        return paged_fail(UD_ERR_SHAPE, "%s: %d sequences x %d queries x %d heads (at most 2^25 rows)", who, n, n_queries, q_heads);
    if (n_sinks < 0 || max_span < 0) return paged_fail(UD_ERR_SHAPE, "%s: %d sinks, span %d", who, n_sinks, max_span);
    if (((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) return paged_fail(UD_ERR_INVALID, "%s: buffers must be 16-byte aligned", who);
    const size_t need = ud_gqa_window_workspace_bytes(n, n_queries, q_heads, kv_heads, head_dim, n_sinks, max_span);
    if (need && !workspace) return paged_fail(UD_ERR_INVALID, "%s: null workspace", who);
    if (workspace_bytes < need) return paged_fail(UD_ERR_SHAPE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
    if ((uintptr_t)workspace & 15) return paged_fail(UD_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    const WindowPlan plan = window_plan(kv_format == UD_MXFP4, (int64_t)n_queries * (q_heads / kv_heads), n, kv_heads, n_sinks, max_span);
    WindowArgs a{};
    a.q = q_dev; a.kp = static_cast<const char*>(k_pages); a.vp = static_cast<const char*>(v_pages); a.bt = block_table;
    a.ranges = ranges_dev; a.out = out_dev;
    a.part = static_cast<float*>(workspace);
    a.stat = a.part + (size_t)n * n_queries * q_heads * plan.split.splits * head_dim;
    a.M = n_queries; a.G = q_heads / kv_heads; a.Hq = q_heads; a.Hkv = kv_heads;
    a.max_blocks = max_blocks; a.num_blocks = num_blocks; a.sinks = n_sinks; a.splits = plan.split.splits; a.pages = plan.split.pages;
    a.groups = plan.groups; a.n = n; a.layer = plan.layer;
    a.scale = (float)(1.4426950408889634 / sqrt((double)head_dim));
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (kv_format == UD_BF16) {
        if (dtype == UD_F32) launch_window<El32, FMT_BF16>(a, head_dim, plan, st);
        else launch_window<ElBf, FMT_BF16>(a, head_dim, plan, st);
    } else if (kv_format == UD_F16) {
        if (dtype == UD_F32) launch_window<El32, FMT_F16>(a, head_dim, plan, st);
        else launch_window<ElH, FMT_F16>(a, head_dim, plan, st);
    } else {
        if (dtype == UD_F32) launch_window<El32, FMT_FP4>(a, head_dim, plan, st);
        else if (dtype == UD_BF16) launch_window<ElBf, FMT_FP4>(a, head_dim, plan, st);
        else launch_window<ElH, FMT_FP4>(a, head_dim, plan, st);
    }
    return paged_launched(who);
}
