// The product of int8 rows with int8 weights, scales for each row and each channel (include/ud_layer.h):
//   out[m, n] = (sum_k codes[m, k] w[n, k]) * scales[m] * w_scales[n] + bias[n] + residual[m, n]
// The sums are exact in 32 bits, so neither the order of k nor its split over waves changes a bit.
#include "layer.hpp"

namespace ud {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

struct LinearArgs {
    const int8_t* a; const float* sa; const int8_t* w; const float* sw; const float* bias;
    const void* res; void* out;
    int64_t a_ld, w_ld, res_ld, out_ld;
    int M, N, K;
};

// Four channels n .. n + 3 of row m: scales, bias, residual, rounding.
template <typename T> __device__ __forceinline__ void finish4(const LinearArgs& a, int m, int n, const i32x4_t& acc) {
    if (m >= a.M || n >= a.N) return;
    const float s = a.sa[m];
    T* o = static_cast<T*>(a.out) + m * a.out_ld + n;
    const T* r = a.res ? static_cast<const T*>(a.res) + m * a.res_ld + n : nullptr;
    if (n + 4 <= a.N) {
        // as the elements lie: their addresses need not be those of whole pieces
        struct V4 { T v[4]; } x, y;
        float sw[4], b[4];
        __builtin_memcpy(sw, a.sw + n, 16);
        if (a.bias) __builtin_memcpy(b, a.bias + n, 16);
        if (r) __builtin_memcpy(&x, r, sizeof x);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v = (float)acc[i] * s * sw[i];
            if (a.bias) v += b[i];
            if (r) v += to_f<T>(x.v[i]);
            y.v[i] = from_f<T>(v);
        }
        __builtin_memcpy(o, &y, sizeof y);
    } else {
        for (int i = 0; i < a.N - n; i++) {
            float v = (float)acc[i] * s * a.sw[n + i];
            if (a.bias) v += a.bias[n + i];
            if (r) v += to_f<T>(r[i]);
            o[i] = from_f<T>(v);
        }
    }
}

// Eight channels n .. n + 7 of row m, `left` of them there, their scales and biases (0 for none) in hand.
template <typename T>
__device__ __forceinline__ void finish8(const LinearArgs& a, int m, int n, int left, const i32x4_t& lo, const i32x4_t& hi,
                                        const float (&sw)[8], const float (&bias)[8]) {
    const float s = a.sa[m];
    T* o = static_cast<T*>(a.out) + m * a.out_ld + n;
    const T* r = a.res ? static_cast<const T*>(a.res) + m * a.res_ld + n : nullptr;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)(e < 4 ? lo[e % 4] : hi[e % 4]) * s * sw[e] + bias[e];
    if (left >= 8) {
        if (r) {
            Raw8<T> x;
            float f[8];
            __builtin_memcpy(&x, r, sizeof x);
            widen8<T>(x, f);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += f[e];
        }
        const Raw8<T> y = narrow8<T>(v);
        __builtin_memcpy(o, &y, sizeof y);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) o[e] = from_f<T>(r ? v[e] + to_f<T>(r[e]) : v[e]);
    }
}

// Few rows: the time is that of the weights' way from memory.  A workgroup takes 16 NT channels and 16 MT rows; its WK waves
// take every WK-th block of 64 U of k, straight from memory into the matrix instruction's operands, and are summed in LDS.
template <typename T, int MT, int NT, int WK, int U>
__global__ __launch_bounds__(64 * WK) void i8_few_kernel(LinearArgs a) {
    __shared__ i32x4_t part[WK][MT * NT][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, r = lane % 16, g = lane / 16;
    const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * (16 * MT);
    // rows behind the last are the last one again: read, never stored
    const int8_t* wp[NT];
    const int8_t* ap[MT];
#pragma unroll
    for (int i = 0; i < NT; i++) wp[i] = a.w + min(n0 + 16 * i + r, a.N - 1) * a.w_ld + 16 * g;
#pragma unroll
    for (int i = 0; i < MT; i++) ap[i] = a.a + min(m0 + 16 * i + r, a.M - 1) * a.a_ld + 16 * g;
    i32x4_t acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = i32x4_t{0, 0, 0, 0};
    i32x4_t wf[U][NT], af[U][MT];
    for (int k = wave * (64 * U); k < a.K; k += WK * 64 * U) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = k + 64 * u;
            const bool in = at + 16 * g < a.K;     // whole pieces of 16: K is a multiple of it
#pragma unroll
            for (int i = 0; i < NT; i++) wf[u][i] = in ? *reinterpret_cast<const i32x4_t*>(wp[i] + at) : i32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < MT; j++) af[u][j] = in ? *reinterpret_cast<const i32x4_t*>(ap[j] + at) : i32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][i], af[u][j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) part[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    // a fragment's lane holds four channels of one row
    for (int e = threadIdx.x; e < MT * NT * 64; e += 64 * WK) {
        const int f = e / 64, l = e % 64;
        i32x4_t s = part[0][f][l];
#pragma unroll
        for (int i = 1; i < WK; i++) s += part[i][f][l];
        finish4<T>(a, m0 + 16 * (f % MT) + l % 16, n0 + 16 * (f / MT) + 4 * (l / 16), s);
    }
}

template <typename T, int MT, int NT, int WK, int U> static void launch_few(const LinearArgs& a, hipStream_t st) {
    const dim3 grid((a.N + 16 * NT - 1) / (16 * NT), (a.M + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((i8_few_kernel<T, MT, NT, WK, U>), grid, dim3(64 * WK), 0, st, a);
}

// ---------------------------------------------------------------- many rows

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

template <int FN, int FM> __device__ __forceinline__ void pin_sums(i32x16_t (&acc)[FN][FM]) {
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++) asm volatile("" : "+a"(acc[i][j]));
}

// A workgroup of four waves takes 64 FM rows and 64 FN channels, a wave 32 FM and 32 FN of them, through two LDS tiles of 128 of
// k each.
//  - The tiles are loaded straight into LDS, 8 rows of 128 bytes to an instruction.  The 16-byte pieces of row r lie in the order
//    piece ^ (r / 2 % 8), so that the 16 rows that LDS serves at a time lie in different banks.
//  - The products are inline assembly with the sums pinned to the accumulator registers: from the builtin the compiler moved them
//    between the register files and spilled 137 registers (256 x 256).  The wait states between compiled code and the products are
//    explicit at the loop's two ends; within it a sum is used again 4 or 16 products later.
//  - The last quarter of a tile's products runs behind the barrier: its operands are in registers by then, so the tile is free
//    for the loads after next, and the next tile's first operands arrive under its products.
template <typename T, int FM, int FN>
__global__ __launch_bounds__(256, FM * FN > 8 ? 1 : 2) void i8_panel_kernel(LinearArgs a) {
    constexpr int TM = 64 * FM, TN = 64 * FN;
    constexpr int LA = TM / 32, LW = TN / 32;      // loads per wave and tile
    __shared__ __attribute__((aligned(16))) int8_t a0[TM * KB];
    __shared__ __attribute__((aligned(16))) int8_t w0[TN * KB];
    __shared__ __attribute__((aligned(16))) int8_t a1[TM * KB];
    __shared__ __attribute__((aligned(16))) int8_t w1[TN * KB];
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
    auto load_part = [&](int i, int b, int8_t* at, int8_t* wt, bool last) __attribute__((always_inline)) {
        if (i < LA) panel_load(ra, last ? last_a[i] : va[i], b * KB, at + (wave * LA + i) * 1024);
        else panel_load(rw, last ? last_w[i - LA] : vw[i - LA], b * KB, wt + (wave * LW + i - LA) * 1024);
    };
    auto load_tile = [&](int b, int8_t* at, int8_t* wt, bool last) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LA + LW; i++) load_part(i, b, at, wt, last);
    };
    // Fragments of k step q (32 of k): lane l holds row l % 32, pieces 2 q + l / 32.
    const int wm = wave % 2 * (32 * FM), wn = wave / 2 * (32 * FN), r32 = lane % 32, half = lane / 32;
    i32x4_t fa[2][FM], fw[2][FN];
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
    // Tile b lies in (at, wt) with its first fragments in fa[0], fw[0]; tile b + 1 is on its way to (an, wnx).  INNER: tile b + 2
    // is there and not the last.
    auto tile = [&](int b, int8_t* at, int8_t* wt, int8_t* an, int8_t* wnx, auto inner) __attribute__((always_inline)) {
        constexpr bool INNER = decltype(inner)::value;
        constexpr int R = FM + FN;
        products(fa[0], fw[0], R, [&](int k) __attribute__((always_inline)) { read_frag(k, 1, at, wt, fa[1], fw[1]); });
        products(fa[1], fw[1], R, [&](int k) __attribute__((always_inline)) { read_frag(k, 2, at, wt, fa[0], fw[0]); });
        products(fa[0], fw[0], R, [&](int k) __attribute__((always_inline)) { read_frag(k, 3, at, wt, fa[1], fw[1]); });
        // this wave's loads of tile b + 1 have arrived, and its reads of tile b
        __builtin_amdgcn_s_waitcnt(0);
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
        if constexpr (INNER) {
#pragma unroll
            for (int k = 0; k < R; k++) read_frag(k, 0, an, wnx, fa[0], fw[0]);
            __builtin_amdgcn_sched_barrier(0);
            products(fa[1], fw[1], LA + LW, [&](int k) __attribute__((always_inline)) { load_part(k, b + 2, at, wt, false); });
        } else {
            if (b + 1 < blocks) {
#pragma unroll
                for (int k = 0; k < R; k++) read_frag(k, 0, an, wnx, fa[0], fw[0]);
            }
            if (b + 2 < blocks) load_tile(b + 2, at, wt, b + 2 == blocks - 1);
            __builtin_amdgcn_sched_barrier(0);
            products(fa[1], fw[1], 0, [](int) {});
        }
    };
    load_tile(0, a0, w0, blocks == 1);
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
#pragma unroll
    for (int k = 0; k < FM + FN; k++) read_frag(k, 0, a0, w0, fa[0], fw[0]);
    if (blocks > 1) load_tile(1, a1, w1, blocks == 2);
    pin_sums<FN, FM>(acc);
    asm volatile("s_nop 7");                       // zeros -> the first product
    // (without branches in the body: where loads into LDS are on their way over a branch, the compiler waits for all of them before the
    // next read of LDS)
    int b = 0;
    for (; b + 4 < blocks; b += 2) {
        tile(b, a0, w0, a1, w1, std::true_type{});
        tile(b + 1, a1, w1, a0, w0, std::true_type{});
    }
    for (; b < blocks; b += 2) {
        tile(b, a0, w0, a1, w1, std::false_type{});
        if (b + 1 < blocks) tile(b + 1, a1, w1, a0, w0, std::false_type{});
    }
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7");   // the last product -> its reads below
    pin_sums<FN, FM>(acc);
    // A lane holds channels 8 q + 4 half + (0 .. 3) of one row.  32 rows at a time go through LDS (each wave an array of its own, rows 16
    // bytes further apart than they are long, against bank conflicts), so that a lane finishes eight channels in a row and a wave writes
    // whole lines.
    constexpr int WC = 32 * FN, LPR = WC / 8, RPI = 64 / LPR, LD = WC + 4;
    static_assert(32 * LD * 4 <= TM * KB && 32 * LD * 4 <= TN * KB, "a wave's rows fit each array");
    __builtin_amdgcn_s_barrier();                  // every wave's reads of the last tile
    __asm__ volatile("" ::: "memory");
    int* mine = reinterpret_cast<int*>(wave == 0 ? a0 : wave == 1 ? w0 : wave == 2 ? a1 : w1);
    const int n = n0 + wn + lane % LPR * 8, left = a.N - n;
    float sw[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        sw[e] = e < left ? a.sw[n + e] : 0.0f;
        bias[e] = a.bias && e < left ? a.bias[n + e] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < FM; j++) {
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<i32x4_t*>(mine + r32 * LD + 32 * i + 8 * q + 4 * half) =
                    i32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int k = 0; k < 32 / RPI; k++) {
            const int r = k * RPI + lane / LPR, m = m0 + wm + 32 * j + r;
            const int* from = mine + r * LD + lane % LPR * 8;
            const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(from), hi = *reinterpret_cast<const i32x4_t*>(from + 4);
            if (m < a.M && left > 0) finish8<T>(a, m, n, left, lo, hi, sw, bias);
        }
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <typename T, int FM, int FN> static void launch_panel(const LinearArgs& a, hipStream_t st) {
    const int64_t tiles = (int64_t)((a.M + 64 * FM - 1) / (64 * FM)) * ((a.N + 64 * FN - 1) / (64 * FN));
    hipLaunchKernelGGL((i8_panel_kernel<T, FM, FN>), dim3((unsigned)tiles), dim3(256), 0, st, a);
}

template <typename T> static void launch_linear(const LinearArgs& a, hipStream_t st) {
    auto tiles = [&](int fm, int fn) { return (int64_t)((a.M + 64 * fm - 1) / (64 * fm)) * ((a.N + 64 * fn - 1) / (64 * fn)); };
    // 32-bit offsets within a tile's rows
    const bool near = a.a_ld <= (1 << 22) && a.w_ld <= (1 << 22);
    if (a.M <= 16) launch_few<T, 1, 1, 8, 4>(a, st);
    else if (a.M <= 64 || !near) launch_few<T, 4, 2, 4, 2>(a, st);
    else if (tiles(4, 4) >= 192) launch_panel<T, 4, 4>(a, st);
    else launch_panel<T, 2, 2>(a, st);
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
    if (M < 0 || M > (1 << 22) || N < 1 || N > (1 << 24) || K < 16 || K > 131056 || K % 16)
        return layer_fail(UD_ERR_SHAPE, "%s: M %d (0 .. 2^22), N %d (1 .. 2^24), K %d (a multiple of 16, 16 .. 131056)", who, M, N, K);
    if (codes_ld < K || w_ld < K || ((codes_ld | w_ld) & 15) || out_ld < N || (residual_dev && res_ld < N))
        return layer_fail(UD_ERR_SHAPE, "%s: rows %d/%d/%d/%d elements apart for K %d (multiples of 16), N %d", who, codes_ld, w_ld, res_ld,
                          out_ld, K, N);
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
