// The product of int8 rows with int8 weights, scales for each row and each channel (include/ud_layer.h):
//   out[m, n] = (sum_k codes[m, k] w[n, k]) * scales[m] * w_scales[n] + bias[n] + residual[m, n]
// The sums are exact in 32 bits, so neither the order of k nor its split over waves changes a bit.
#include "layer.hpp"
#include "linear_plan.hpp"

namespace ud {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

struct LinearArgs {
    const int8_t* a; const float* sa; const int8_t* w; const float* sw; const float* bias;
    const void* res; void* out;
    int64_t a_ld, w_ld, res_ld, out_ld;
    int M, N, K;
};

// What finishes four channels n .. n + 3 of row m, read ahead of the sums.  (The operations are those of finish8, so that a row's result does
// not follow the kernel.)
template <typename T> struct Finish4 {
    float s, sw[4], bias[4];
    T res[4];
    bool there;

    __device__ __forceinline__ void read(const LinearArgs& a, int m, int n) {
        there = m < a.M && n < a.N;
#pragma unroll
        for (int i = 0; i < 4; i++) bias[i] = 0.0f;
        if (!there) return;
        s = a.sa[m];
        const T* r = a.res ? static_cast<const T*>(a.res) + m * a.res_ld + n : nullptr;
        if (n + 4 <= a.N) {                        // as they lie: the addresses need not be those of whole pieces
            __builtin_memcpy(sw, a.sw + n, 16);
            if (a.bias) __builtin_memcpy(bias, a.bias + n, 16);
            if (r) __builtin_memcpy(res, r, sizeof res);
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++) {
                if (n + i >= a.N) continue;
                sw[i] = a.sw[n + i];
                if (a.bias) bias[i] = a.bias[n + i];
                if (r) res[i] = r[i];
            }
        }
    }
    __device__ __forceinline__ void write(const LinearArgs& a, int m, int n, const i32x4_t& acc) const {
        if (!there) return;
        T* o = static_cast<T*>(a.out) + m * a.out_ld + n;
        T y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v = fmaf((float)acc[i] * s, sw[i], bias[i]);
            if (a.res) v += to_f<T>(res[i]);
            y[i] = from_f<T>(v);
        }
        if (n + 4 <= a.N) {
            __builtin_memcpy(o, y, sizeof y);
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (n + i < a.N) o[i] = y[i];
        }
    }
};

// Eight channels n .. n + 7 of row m, `left` of them there; their scales, biases (0 for none) and residual (read already where all eight
// are there) in hand.
template <typename T>
__device__ __forceinline__ void finish8(const LinearArgs& a, int m, int n, int left, const i32x4_t& lo, const i32x4_t& hi, float s,
                                        const float (&sw)[8], const float (&bias)[8], const Raw8<T>& res) {
    T* o = static_cast<T*>(a.out) + m * a.out_ld + n;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = fmaf((float)(e < 4 ? lo[e % 4] : hi[e % 4]) * s, sw[e], bias[e]);
    if (left >= 8) {
        if (a.res) {
            float f[8];
            widen8<T>(res, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += f[e];
        }
        const Raw8<T> y = narrow8<T>(v);
        __builtin_memcpy(o, &y, sizeof y);
    } else {
        const T* r = a.res ? static_cast<const T*>(a.res) + m * a.res_ld + n : nullptr;
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) o[e] = from_f<T>(r ? v[e] + to_f<T>(r[e]) : v[e]);
    }
}

// Up to 16 rows: the time is that of the weights' way from memory.  A workgroup takes 16 channels; its WK waves take every WK-th block
// of 64 U of k, straight from memory into the matrix instruction's operands, up to 32 loads of 1 KB a wave at once, and are summed in LDS.  One row
// of 12,288 -> 4,096 takes 10.4 us, where reading the weights alone, in the same pieces, takes 9.5 - 10.2.
template <typename T, int WK, int U> __global__ __launch_bounds__(64 * WK) void i8_few_kernel(LinearArgs a) {
    __shared__ i32x4_t part[WK][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int n0 = blockIdx.x * 16;
    // rows behind the last are the last one again: read, never stored
    const int8_t* wp = a.w + min(n0 + r, a.N - 1) * a.w_ld + 16 * g;
    const int8_t* ap = a.a + min(r, a.M - 1) * a.a_ld + 16 * g;
    i32x4_t acc{0, 0, 0, 0}, wf[U], af[U];
    auto load = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = k + 64 * u;
            const bool in = at + 16 * g < a.K;     // whole pieces of 16: K is a multiple of it
            wf[u] = in ? *reinterpret_cast<const i32x4_t*>(wp + at) : i32x4_t{0, 0, 0, 0};
            af[u] = in ? *reinterpret_cast<const i32x4_t*>(ap + at) : i32x4_t{0, 0, 0, 0};
        }
    };
    int k = wave * (64 * U);
    load(k);
    // the first wave finishes; its lanes hold four channels of one row
    Finish4<T> fin;
    if (wave == 0) fin.read(a, r, n0 + 4 * g);
    for (;;) {
#pragma unroll
        for (int u = 0; u < U; u++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], af[u], acc, 0, 0, 0);
        k += WK * 64 * U;
        if (k >= a.K) break;
        load(k);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        i32x4_t s = part[0][lane];
#pragma unroll
        for (int i = 1; i < WK; i++) s += part[i][lane];
        fin.write(a, r, n0 + 4 * g, s);
    }
}

template <typename T, int WK, int U> static void launch_few(const LinearArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((i8_few_kernel<T, WK, U>), dim3((a.N + 15) / 16), dim3(64 * WK), 0, st, a);
}

// Buffer resource of `bytes` bytes at p: loads past them give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t panel_buffer(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
// 16 bytes per lane from byte voff + soff of the buffer into LDS at dst + 16 * lane.
__device__ __forceinline__ void panel_load(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, int8_t* dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, dst, 16, voff, soff, 0, 0);
}

constexpr int KB = 128;                            // bytes of k per LDS tile
constexpr uint32_t kNowhere = 1u << 31;             // an offset that is past every buffer (256 rows, 2^22 apart)

// ---------------------------------------------------------------- some rows

// Some rows: a workgroup takes S FM rows and S FN channels, each of its waves all of them for every NW-th block of 128 of k, through two LDS
// tiles of the wave's own: nothing is shared before the end, so a wave waits for its own loads alone.  A CU gets some 58 bytes a ns into LDS
// (in pieces of 128 bytes a row; straight to registers, 64 bytes a row, half of it), whichever memory they come from, so the smallest
// tiles that are one round of the chip are the fastest, though they read more: 64 rows of 14,336 -> 4,096 take 19.5 us with tiles of 32 x 32,
// 26.5 with 64 x 32, 35.2 with 64 x 64 shared by four waves; 16 rows of 4,096 -> 6,144 7.2 with 16 x 32, 10.2 from memory to registers.
// (Four LDS tiles a wave: 7.2 -> 7.5.)
template <typename T, int S, int FM, int FN, int NW>
__global__ __launch_bounds__(64 * NW) void i8_split_kernel(LinearArgs a) {
    constexpr int TM = S * FM, TN = S * FN, R = FM + FN, L = S * R / 8, TILE = S * R * KB;   // L loads per wave and tile
    constexpr int G = 64 / S, Q = KB / (16 * G), E = S * S / 64;       // pieces per row and product, products per tile, sums per lane
    __shared__ __attribute__((aligned(16))) int8_t t0[NW * TILE];
    __shared__ __attribute__((aligned(16))) int8_t t1[NW * TILE];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    // An XCD's workgroups are neighbours: the rows of a channel panel read its weights from one L2.
    const int nM = (a.M + TM - 1) / TM, nN = (a.N + TN - 1) / TN, total = nM * nN;
    const int xcd = blockIdx.x % 8, each = total / 8, more = total % 8;
    const int t = xcd * each + min(xcd, more) + blockIdx.x / 8;
    const int m0 = t % nM * TM, n0 = t / nM * TN;

    const int rows_a = min(TM, a.M - m0), rows_w = min(TN, a.N - n0);
    const __amdgpu_buffer_rsrc_t ra = panel_buffer(a.a + m0 * a.a_ld, (uint32_t)((rows_a - 1) * a.a_ld + a.K));
    const __amdgpu_buffer_rsrc_t rw = panel_buffer(a.w + n0 * a.w_ld, (uint32_t)((rows_w - 1) * a.w_ld + a.K));
    // Rows behind the last are the last one again (computed, not stored); pieces behind K are zeros.  The pieces of a row lie in the order
    // piece ^ (r / 2 % 8), against bank conflicts.
    uint32_t v[L];
    int room[L];                                   // the k before which a block holds this lane's piece
#pragma unroll
    for (int i = 0; i < L; i++) {
        const int r = i * 8 + lane / 8, piece = (lane % 8) ^ (r / 2 % 8);
        v[i] = (uint32_t)(r < TM ? min(r, rows_a - 1) * a.a_ld : min(r - TM, rows_w - 1) * a.w_ld) + 16 * piece;
        room[i] = a.K - 16 * piece;
    }
    auto load_tile = [&](int step, int8_t* at) __attribute__((always_inline)) {
        const int k = (step * NW + wave) * KB;
#pragma unroll
        for (int i = 0; i < L; i++)
            panel_load(i < TM / 8 ? ra : rw, k < room[i] ? v[i] : kNowhere, k < a.K ? k : 0, at + (wave * TILE + i * 1024));
    };
    load_tile(0, t0);
    load_tile(1, t1);
    // Four channels of a row to a thread at the end; what they need is read under the first tiles' way (before it 0.1 - 0.4 us more, behind the
    // products 0.1 - 0.3).
    constexpr int PR = TN / 4, PIECES = TM * PR, PER = (PIECES + 64 * NW - 1) / (64 * NW);
    Finish4<T> fin[PER];
#pragma unroll
    for (int f = 0; f < PER; f++) {
        const int p = tid + f * 64 * NW;
        fin[f].read(a, p < PIECES ? m0 + p / PR : a.M, n0 + p % PR * 4);
    }
    typedef int Sums __attribute__((ext_vector_type(E)));
    Sums acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int e = 0; e < E; e++) acc[i][j][e] = 0;
    const int r = lane % S, g = lane / S;
    auto tile = [&](int step, int8_t* at) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(L));  // this wave's loads of the tile have arrived (the next one's may not)
        __asm__ volatile("" ::: "memory");
        i32x4_t f[Q][R];
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int i = 0; i < R; i++)
                f[q][i] = *reinterpret_cast<const i32x4_t*>(at + wave * TILE + (S * i + r) * KB + 16 * ((G * q + g) ^ (r / 2 % 8)));
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);        // and are read (lgkmcnt 0), before the next loads overwrite them
        __asm__ volatile("" ::: "memory");
        load_tile(step + 2, at);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int i = 0; i < FN; i++)
#pragma unroll
                for (int j = 0; j < FM; j++) {
                    if constexpr (S == 32) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[q][FM + i], f[q][j], acc[i][j], 0, 0, 0);
                    else acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[q][FM + i], f[q][j], acc[i][j], 0, 0, 0);
                }
        __builtin_amdgcn_sched_barrier(0);
    };
    const int steps = ((a.K + KB - 1) / KB + NW - 1) / NW;
    int b = 0;
    for (; b + 2 <= steps; b += 2) {
        tile(b, t0);
        tile(b + 1, t1);
    }
    if (b < steps) tile(b, t0);
    __builtin_amdgcn_s_waitcnt(0);                 // the zeros behind the last tile, before LDS is used again
    __asm__ volatile("" ::: "memory");
    // A lane holds channels S / 4 i' + 4 g + (0 .. 3) of one row; a wave's sums go to its own tile, row by row (against bank conflicts four
    // channels' piece p at p ^ (row % X)).
    static_assert(TM * TN * 4 <= TILE, "a wave's sums fit its tile");
    constexpr int X = PR < 8 ? PR : 8;
    int* mine = reinterpret_cast<int*>(t0 + wave * TILE);
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int q = 0; q < E / 4; q++) {
                const int row = S * j + r, p = S / 4 * i + G * q + g;
                *reinterpret_cast<i32x4_t*>(mine + row * TN + 4 * (p ^ (row % X))) =
                    i32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < PER; f++) {
        const int p = tid + f * 64 * NW, row = p / PR;
        if (p >= PIECES) continue;
        const int8_t* at = t0 + (row * TN + 4 * (p % PR ^ (row % X))) * 4;
        i32x4_t s = *reinterpret_cast<const i32x4_t*>(at);
#pragma unroll
        for (int w = 1; w < NW; w++) s += *reinterpret_cast<const i32x4_t*>(at + w * TILE);
        fin[f].write(a, m0 + row, n0 + p % PR * 4, s);
    }
}

template <typename T, int S, int FM, int FN, int NW> static void launch_split(const LinearArgs& a, hipStream_t st) {
    const int64_t tiles = tiles_of(a.M, a.N, S * FM, S * FN);
    hipLaunchKernelGGL((i8_split_kernel<T, S, FM, FN, NW>), dim3((unsigned)tiles), dim3(64 * NW), 0, st, a);
}

// ---------------------------------------------------------------- many rows

template <int FN, int FM> __device__ __forceinline__ void pin_sums(i32x16_t (&acc)[FN][FM]) {
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++) asm volatile("" : "+a"(acc[i][j]));
}

// A workgroup of NW waves takes 64 FM rows and 16 NW FN channels, a wave 32 FM and 32 FN of them, through NS LDS tiles of 128 of k
// each.  8,192 rows of 4,096 -> 6,144 take 184 us in a loop of their own (2.2 POP/s; traced between other calls 197), 8,192^3 2.4 POP/s, where
// the library's product of the same sizes reaches 1.9 and 2.1 and the instructions alone 3.2 at the clock the card keeps under them.
//  - The tiles are loaded straight into LDS, 8 rows of 128 bytes to an instruction.  The 16-byte pieces of row r lie in the order
//    piece ^ (r / 2 % 8), so that the 16 rows that LDS serves at a time lie in different banks.  (Tiles of 64 of k, four of them: 190 -> 198.)
//  - The products are inline assembly with the sums pinned to the accumulator registers: from the builtin the compiler moved them
//    between the register files and spilled 137 registers (256 x 256).  (Finishing fp32 rows of 256 x 256 still spills 84, behind the
//    products: 209 us, of bf16 184.)  The wait states between compiled code and the products are
//    explicit at the loop's two ends; within it a sum goes from product to product in its own registers, which needs none.
//  - Reads of LDS and loads of later tiles lie between the products.  With large fragments the last quarter of a tile's products runs behind
//    the barrier: its operands are in registers by then, so the tile is free for loads, and the next tile's first operands arrive
//    under its products.  Small ones are read a whole tile ahead (1,024 rows of 4,096 -> 4,096 22.4 -> 20.4 us).
//  - Four LDS tiles where a CU holds one small workgroup: its loads are three tiles ahead (64 rows of 4,096 -> 6,144 17 -> 10 us).  Eight waves for
//    256 x 256: two per SIMD cover each other's waits (190 -> 181).
template <typename T, int FM, int FN, int NS, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 || FM * FN > 8 || (FM + FN) * NS * 8 > 80 ? 1 : 2) void i8_panel_kernel(LinearArgs a) {
    static_assert(NS == 2 || NS == 4, "the loop's body is written out for two and four LDS tiles");
    constexpr int TM = 64 * FM, TN = 16 * NW * FN;
    constexpr int LA = TM / (8 * NW), LW = TN / (8 * NW);          // loads per wave and tile
    // arrays of their own, so that the compiler can tell a tile that is read from one that is loaded
    __shared__ __attribute__((aligned(16))) int8_t a0[TM * KB];
    __shared__ __attribute__((aligned(16))) int8_t w0[TN * KB];
    __shared__ __attribute__((aligned(16))) int8_t a1[TM * KB];
    __shared__ __attribute__((aligned(16))) int8_t w1[TN * KB];
    __shared__ __attribute__((aligned(16))) int8_t a2[NS > 2 ? TM * KB : 16];
    __shared__ __attribute__((aligned(16))) int8_t w2[NS > 2 ? TN * KB : 16];
    __shared__ __attribute__((aligned(16))) int8_t a3[NS > 2 ? TM * KB : 16];
    __shared__ __attribute__((aligned(16))) int8_t w3[NS > 2 ? TN * KB : 16];
    const int tid = threadIdx.x, lane = tid % 64;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    // An XCD's workgroups are neighbours, in blocks of four row panels: what they read is shared in its L2.
    const int nM = (a.M + TM - 1) / TM, nN = (a.N + TN - 1) / TN, total = nM * nN;
    const int xcd = blockIdx.x % 8, each = total / 8, more = total % 8;
    const int t = xcd * each + min(xcd, more) + blockIdx.x / 8;
    const int grp = t / (4 * nN), rem = t - grp * 4 * nN, gm = min(4, nM - grp * 4);
    const int m0 = (grp * 4 + rem % gm) * TM, n0 = rem / gm * TN;

    const int rows_a = min(TM, a.M - m0), rows_w = min(TN, a.N - n0);
    const __amdgpu_buffer_rsrc_t ra = panel_buffer(a.a + m0 * a.a_ld, (uint32_t)((rows_a - 1) * a.a_ld + a.K));
    const __amdgpu_buffer_rsrc_t rw = panel_buffer(a.w + n0 * a.w_ld, (uint32_t)((rows_w - 1) * a.w_ld + a.K));
    uint32_t va[LA], vw[LW], last_a[LA], last_w[LW];
    const int blocks = (a.K + KB - 1) / KB, tail = a.K - (blocks - 1) * KB;
    // Rows behind the last are the last one again (computed, not stored); pieces behind K are zeros.
#pragma unroll
    for (int i = 0; i < LA; i++) {
        const int r = (wave * LA + i) * 8 + lane / 8, piece = (lane % 8) ^ (r / 2 % 8);
        va[i] = (uint32_t)(min(r, rows_a - 1) * a.a_ld) + 16 * piece;
        last_a[i] = 16 * piece < tail ? va[i] : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < LW; i++) {
        const int r = (wave * LW + i) * 8 + lane / 8, piece = (lane % 8) ^ (r / 2 % 8);
        vw[i] = (uint32_t)(min(r, rows_w - 1) * a.w_ld) + 16 * piece;
        last_w[i] = 16 * piece < tail ? vw[i] : kNowhere;
    }
    // Part i of tile b; behind the last tile zeros, which nothing reads (so that each tile counts the same loads).
    auto load_part = [&](int i, int b, int8_t* at, int8_t* wt) __attribute__((always_inline)) {
        const bool inner = b + 1 < blocks, there = b < blocks;
        const uint32_t v = i < LA ? (inner ? va[i] : last_a[i]) : inner ? vw[i - LA] : last_w[i - LA];
        if (i < LA) panel_load(ra, there ? v : kNowhere, there ? b * KB : 0, at + (wave * LA + i) * 1024);
        else panel_load(rw, there ? v : kNowhere, there ? b * KB : 0, wt + (wave * LW + i - LA) * 1024);
    };
    auto load_tile = [&](int b, int8_t* at, int8_t* wt) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LA + LW; i++) load_part(i, b, at, wt);
    };
    // Fragments of k step q (32 of k): lane l holds row l % 32, pieces 2 q + l / 32.
    const int wm = wave % 2 * (32 * FM), wn = wave / 2 * (32 * FN), r32 = lane % 32, half = lane / 32;
    // Fragments in registers: of two whole tiles with four LDS tiles, which the small ones have (a tile is read under the products of the
    // one before), else of two k steps.
    constexpr int R = FM + FN;
    constexpr bool WHOLE = NS == 4;
    static_assert(!WHOLE || (R <= 4 && NW == 4), "two whole tiles fit the registers");
    i32x4_t fa[WHOLE ? 8 : 2][FM], fw[WHOLE ? 8 : 2][FN];
    auto read_frag = [&](int i, int q, const int8_t* at, const int8_t* wt, i32x4_t (&da)[FM], i32x4_t (&dw)[FN]) __attribute__((always_inline)) {
        const int off = r32 * KB + 16 * ((2 * q + half) ^ (r32 / 2 % 8));
        if (i < FN) dw[i] = *reinterpret_cast<const i32x4_t*>(wt + (wn + 32 * i) * KB + off);
        else da[i - FN] = *reinterpret_cast<const i32x4_t*>(at + (wm + 32 * (i - FN)) * KB + off);
    };
    i32x16_t acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
    // The products of a k step, with what(0), what(1), .. between them: `work` pieces, evenly.
    constexpr int STEPS = FN * FM;
    auto products = [&](const i32x4_t (&da)[FM], const i32x4_t (&dw)[FN], int work, auto what) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int j = 0; j < FM; j++) {
                const int n = i * FM + j;
                asm volatile("v_mfma_i32_32x32x32_i8 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(dw[i]), "v"(da[j]));
#pragma unroll
                for (int k = 0; k < work; k++)
                    if (k * STEPS / work == n) what(k);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    // Tile b lies in (at, wt) with its first fragments in fa[0], fw[0] (WHOLE: with all of them, in the half `which`); the next NS - 1 tiles
    // are on their way, the first of them to (an, wnx).
    auto tile = [&](int b, int8_t* at, int8_t* wt, int8_t* an, int8_t* wnx, auto which) __attribute__((always_inline)) {
        constexpr int L = LA + LW;
        if constexpr (WHOLE) {
            constexpr int H = decltype(which)::value * 4;
            // this wave's loads of tile b + 1 have arrived, and its reads of tile b
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * L) & 0xF0FF);
            __builtin_amdgcn_s_barrier();
            __asm__ volatile("" ::: "memory");
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int first = q * L / 4;
                products(fa[H + q], fw[H + q], R + (q + 1) * L / 4 - first, [&](int k) __attribute__((always_inline)) {
                    if (k < R) read_frag(k, q, an, wnx, fa[4 - H + q], fw[4 - H + q]);
                    else load_part(first + k - R, b + 4, at, wt);
                });
            }
        } else {
            products(fa[0], fw[0], R, [&](int k) __attribute__((always_inline)) { read_frag(k, 1, at, wt, fa[1], fw[1]); });
            products(fa[1], fw[1], R, [&](int k) __attribute__((always_inline)) { read_frag(k, 2, at, wt, fa[0], fw[0]); });
            products(fa[0], fw[0], R, [&](int k) __attribute__((always_inline)) { read_frag(k, 3, at, wt, fa[1], fw[1]); });
            // this wave's loads of tile b + 1 have arrived, and its reads of tile b
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0) & 0xF0FF);
            __builtin_amdgcn_s_barrier();
            __asm__ volatile("" ::: "memory");
#pragma unroll
            for (int k = 0; k < R; k++) read_frag(k, 0, an, wnx, fa[0], fw[0]);
            __builtin_amdgcn_sched_barrier(0);
            products(fa[1], fw[1], L, [&](int k) __attribute__((always_inline)) { load_part(k, b + 2, at, wt); });
        }
    };
    const std::integral_constant<int, 0> even{};
    const std::integral_constant<int, 1> odd{};
    load_tile(0, a0, w0);
    load_tile(1, a1, w1);
    if constexpr (NS == 4) {
        load_tile(2, a2, w2);
        load_tile(3, a3, w3);
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 1) * (LA + LW)));
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
#pragma unroll
    for (int q = 0; q < (WHOLE ? 4 : 1); q++)
#pragma unroll
        for (int k = 0; k < R; k++) read_frag(k, q, a0, w0, fa[q], fw[q]);
    pin_sums<FN, FM>(acc);
    asm volatile("s_nop 7");                       // zeros -> the first product
    // (no branch in the body: where loads into LDS are on their way over one, the compiler waits for all of them before the next read of
    // LDS, which costs the last tiles little)
    int b = 0;
    for (; b + NS <= blocks; b += NS) {
        if constexpr (NS == 2) {
            tile(b, a0, w0, a1, w1, even);
            tile(b + 1, a1, w1, a0, w0, odd);
        } else {
            tile(b, a0, w0, a1, w1, even);
            tile(b + 1, a1, w1, a2, w2, odd);
            tile(b + 2, a2, w2, a3, w3, even);
            tile(b + 3, a3, w3, a0, w0, odd);
        }
    }
    if (b < blocks) tile(b, a0, w0, a1, w1, even);
    if constexpr (NS == 4) {
        if (b + 1 < blocks) tile(b + 1, a1, w1, a2, w2, odd);
        if (b + 2 < blocks) tile(b + 2, a2, w2, a3, w3, even);
    }
    __builtin_amdgcn_s_waitcnt(0);                 // the zeros behind the last tile, before LDS is used again
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7");   // the last product -> its reads below
    pin_sums<FN, FM>(acc);
    // A lane holds channels 8 q + 4 half + (0 .. 3) of one row.  32 rows of CW channels at a time go through LDS (each wave in an array of
    // its own; four channels' piece p of row r lies at p ^ r, against bank conflicts), so that a lane finishes eight channels in a row
    // and a wave writes whole lines.
    constexpr int CW = FN % 2 ? 32 : 64, CF = CW / 32, LPR = CW / 8, RPI = 64 / LPR, IT = 32 / RPI;
    static_assert(NW / 4 * 32 * CW * 4 <= TM * KB && NW / 4 * 32 * CW * 4 <= TN * KB, "a wave's rows fit each array");
    auto place = [&](int r, int p) __attribute__((always_inline)) {
        const int x = CW == 64 ? r % 16 : r / 2 % 8;
        return r * CW + 4 * (p ^ x);
    };
    __builtin_amdgcn_s_barrier();                  // every wave's reads of the last tile
    __asm__ volatile("" ::: "memory");
    const int part = wave % 4;
    int* mine = reinterpret_cast<int*>(part == 0 ? a0 : part == 1 ? w0 : part == 2 ? a1 : w1) + wave / 4 * (32 * CW);
    const int n = n0 + wn + lane % LPR * 8, mw = m0 + wm + lane / LPR;
    float sw[FN / CF][8], bias[FN / CF][8], sa[FM][IT];
#pragma unroll
    for (int c = 0; c < FN / CF; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int at = n + c * CW + e;
            sw[c][e] = at < a.N ? a.sw[at] : 0.0f;
            bias[c][e] = a.bias && at < a.N ? a.bias[at] : 0.0f;
        }
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
        for (int k = 0; k < IT; k++) sa[j][k] = a.sa[min(mw + 32 * j + k * RPI, a.M - 1)];
#pragma unroll
    for (int j = 0; j < FM; j++)
#pragma unroll
        for (int c = 0; c < FN / CF; c++) {
            const int nc = n + c * CW, left = a.N - nc, mj = mw + 32 * j;
            Raw8<T> res[IT];
            if (a.res && left >= 8) {
#pragma unroll
                for (int k = 0; k < IT; k++)
                    if (mj + k * RPI < a.M) __builtin_memcpy(&res[k], static_cast<const T*>(a.res) + (mj + k * RPI) * a.res_ld + nc, sizeof res[k]);
            }
#pragma unroll
            for (int i = 0; i < CF; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const i32x16_t& x = acc[c * CF + i][j];
                    *reinterpret_cast<i32x4_t*>(mine + place(r32, 8 * i + 2 * q + half)) =
                        i32x4_t{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
                }
            i32x4_t v[IT][2];
#pragma unroll
            for (int k = 0; k < IT; k++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    v[k][h] = *reinterpret_cast<const i32x4_t*>(mine + place(k * RPI + lane / LPR, lane % LPR * 2 + h));
#pragma unroll
            for (int k = 0; k < IT; k++)
                if (mj + k * RPI < a.M && left > 0)
                    finish8<T>(a, mj + k * RPI, nc, left, v[k][0], v[k][1], sa[j][k], sw[c], bias[c], res[k]);
        }
}

template <typename T, int FM, int FN, int NS, int NW = 4> static void launch_panel(const LinearArgs& a, hipStream_t st) {
    const int64_t tiles = tiles_of(a.M, a.N, 64 * FM, 16 * NW * FN);
    hipLaunchKernelGGL((i8_panel_kernel<T, FM, FN, NS, NW>), dim3((unsigned)tiles), dim3(64 * NW), 0, st, a);
}

template <typename T> static void launch_linear(const LinearArgs& a, hipStream_t st) {
    switch (linear_kernel(a.M, a.N, a.K)) {
        case FEW_16x16: return launch_few<T, 4, 16>(a, st);
        case FEW_16x16_DEEP: return launch_few<T, 8, 16>(a, st);
        case FEW_16x16_SHORT: return launch_few<T, 4, 8>(a, st);
        case SPLIT_16x16: return launch_split<T, 16, 1, 1, 8>(a, st);
        case SPLIT_16x32: return launch_split<T, 16, 1, 2, 4>(a, st);
        case SPLIT_32x32: return launch_split<T, 32, 1, 1, 4>(a, st);
        case SPLIT_64x32: return launch_split<T, 32, 2, 1, 4>(a, st);
        case PANEL_64x64: return launch_panel<T, 1, 1, 4>(a, st);
        case PANEL_64x128: return launch_panel<T, 1, 2, 4>(a, st);
        case PANEL_128x64: return launch_panel<T, 2, 1, 4>(a, st);
        case PANEL_128x128: return launch_panel<T, 2, 2, 4>(a, st);
        case PANEL_128x128_TWO: return launch_panel<T, 2, 2, 2>(a, st);
        case PANEL_256x192: return launch_panel<T, 4, 3, 2>(a, st);
        default: return launch_panel<T, 4, 2, 2, 8>(a, st);
    }
}

}  // namespace ud

using namespace ud;

extern "C" UD_API int ud_i8_linear(int32_t dtype, const int8_t* codes_dev, int32_t codes_ld, const float* scales_dev,
                                   const int8_t* w_dev, int32_t w_ld, const float* w_scales_dev, const float* bias_dev,
                                   const void* residual_dev, int32_t res_ld, void* out_dev, int32_t out_ld, int32_t M, int32_t N,
                                   int32_t K, void* hip_stream) {
    static const char* who = "ud_i8_linear";
    const int64_t size = type_bytes(dtype);
    if (!size) return layer_fail(UD_ERR_INVALID, "%s: dtype %d", who, dtype);
    // (a launch holds fewer than 2^32 threads, a tile's rows lie within 32-bit offsets)
    if (M < 0 || M >= (1 << 22) || N < 1 || N > (1 << 24) || (int64_t)M * N > (int64_t)1 << 38 || K < 16 || K > 131056 || K % 16)
        return layer_fail(UD_ERR_SHAPE, "%s: M %d (0 .. 2^22 - 1), N %d (1 .. 2^24, M N at most 2^38), K %d (a multiple of 16, 16 .. 131056)", who, M, N, K);
    if (codes_ld < K || w_ld < K || ((codes_ld | w_ld) & 15) || codes_ld > (1 << 22) || w_ld > (1 << 22) || out_ld < N || (residual_dev && res_ld < N))
        return layer_fail(UD_ERR_SHAPE, "%s: rows %d/%d/%d/%d elements apart for K %d (multiples of 16, at most 2^22), N %d", who, codes_ld, w_ld,
                          res_ld, out_ld, K, N);
    if (M == 0) return UD_OK;
    if (!codes_dev || !scales_dev || !w_dev || !w_scales_dev || !out_dev) return layer_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if ((((uintptr_t)codes_dev | (uintptr_t)w_dev) & 15) || (((uintptr_t)scales_dev | (uintptr_t)w_scales_dev | (uintptr_t)bias_dev) & 3) ||
        (((uintptr_t)out_dev | (uintptr_t)residual_dev) & (size - 1)))
        return layer_fail(UD_ERR_INVALID, "%s: codes and w must be 16-byte aligned, the others to their elements", who);
    const Block out{out_dev, out_ld * size, N * size, M}, res{residual_dev, res_ld * size, N * size, M};
    if ((blocks_meet(out, res) && !blocks_same(out, res)) || blocks_meet(out, Block{codes_dev, codes_ld, K, M}) ||
        blocks_meet(out, Block{w_dev, w_ld, K, N}) || blocks_meet(out, Block{scales_dev, 0, 4 * (int64_t)M, 1}) ||
        blocks_meet(out, Block{w_scales_dev, 0, 4 * (int64_t)N, 1}) || blocks_meet(out, Block{bias_dev, 0, 4 * (int64_t)N, 1}))
        return layer_fail(UD_ERR_INVALID, "%s: out overlaps an input (it may be residual, at the same ld)", who);
    LinearArgs a{};
    a.a = codes_dev; a.sa = scales_dev; a.w = w_dev; a.sw = w_scales_dev; a.bias = bias_dev; a.res = residual_dev; a.out = out_dev;
    a.a_ld = codes_ld; a.w_ld = w_ld; a.res_ld = res_ld; a.out_ld = out_ld;
    a.M = M; a.N = N; a.K = K;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == UD_F32) launch_linear<float>(a, st);
    else if (dtype == UD_BF16) launch_linear<bf16>(a, st);
    else launch_linear<f16>(a, st);
    return layer_launched(who);
}
