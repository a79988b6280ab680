// What the windowed attention kernels (window.hip, prefill.hip) share: products of 16-bit operands and their terms, the
// join of the splits of a query row.
#pragma once
#include <type_traits>

#include "paged.hpp"

namespace ud {

typedef short v4i16_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 lds_tr16(const char* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16_t*)p));
}

// x's two values added to acc.
template <bool H> __device__ __forceinline__ float dot_ones(uint32_t x, float acc) {
    if constexpr (H) return __builtin_amdgcn_fdot2(as_half2(x), as_half2(0x3c003c00u), acc, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc, false);
}

template <bool H> __device__ __forceinline__ f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c) {
    if constexpr (H) return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_f16x8(a), as_f16x8(b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
// Two floats as a packed pair of the products' type, and the pair's values.
template <bool H> __device__ __forceinline__ uint32_t pack16(float x, float y) {
    if constexpr (H) return __builtin_bit_cast(uint32_t, half2_t{(_Float16)x, (_Float16)y});
    else return pack_bf16x2(x, y);
}
template <bool H> __device__ __forceinline__ void unpack2(uint32_t w, float& x, float& y) {
    if constexpr (H) { x = half_lo(w); y = half_hi(w); }
    else { x = __uint_as_float(w << 16); y = __uint_as_float(w & 0xffff0000u); }
}
// Eight floats as T operands whose sum they are.
template <bool H, int T> __device__ __forceinline__ void split8(const float (&x)[8], uint4 (&t)[T]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = x[e];
#pragma unroll
    for (int k = 0; k < T; k++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w[e] = pack16<H>(r[2 * e], r[2 * e + 1]);
            if (k + 1 < T) {
                float a, b;
                unpack2<H>(w[e], a, b);
                r[2 * e] -= a;
                r[2 * e + 1] -= b;
            }
        }
        t[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A probability is 2^(x scale - off) by one fused operation, which takes the product x scale as it is, while the base in off is
// a rounded one.  From bases of STEEP on the two differ by more than 2^-4, and further up by more than a 16-bit probability has
// room for, so that the largest would become infinite or 0.  There the product is rounded as the base was: this x gives
// that by the same operation, the base left out of off.
constexpr float STEEP = 0x1p20f;
__device__ __forceinline__ float steep_score(float x, float scale, float base) {
#pragma clang fp contract(off)
    return (x * scale - base) * (1.0f / scale);
}

// Channels ch .. ch + 3 of row `key` of a head's page of values, those that are no numbers added to sum.
template <int FMT, int D> __device__ __forceinline__ void odd_values(const char* v, int key, int ch, float (&sum)[4]) {
    float x[4];
    if constexpr (FMT == FMT_FP4) {
        const uint8_t e = *reinterpret_cast<const uint8_t*>(v + Page<FMT, D>::CODES + key * (D / FP4_BLOCK) + ch / FP4_BLOCK);
        x[0] = x[1] = x[2] = x[3] = e == 255 ? NAN : 0.0f;
    } else {
        typedef typename std::conditional<FMT == FMT_BF16, ElBf, ElH>::type E;
        load4<E>(reinterpret_cast<const uint16_t*>(v) + key * D + ch, x);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) sum[i] += __builtin_isfinite(x[i]) ? 0.0f : x[i];
}

// The splits of one (query row, head) joined, 16 a wave (one round trip to memory however many there are; at most 16
// splits: four rows a workgroup): with split s's maximum m_s (of scores times log2(e)), sum l_s
// and unnormalised output x_s,  out = sum_s 2^(m_s - m) x_s / sum_s 2^(m_s - m) l_s.  A split without a key has m = -inf,
// l = 0 and its x is not looked at.  An x that is no number stays what it is, also where its weight is 0 in fp32.
// Bound: memory; of few rows the round trip.  57,600 rows of 3 splits at D = 128 (90 MB of partials) 23 us, 32 rows of 64
// splits 4 us.
// The rows: `count` of them, or (start) those of each sequence y, tokens start[y] .. start[y + 1] - 1 of `tokens`, at most
// `count` rows each.
struct JoinRows {
    int64_t count;
    int heads, tokens;
    const int32_t* start;
    int n;
};
// DEEP: splits per wave, all loads in flight at once.
template <typename E, int D, int DEEP>
__global__ __launch_bounds__(1024) void join_splits_kernel(const float* part, const float* stat, void* out, JoinRows rows, int splits) {
    typedef typename E::S S;
    constexpr int DL = D / 64, CH = MAX_SPLITS / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int each = (splits + DEEP - 1) / DEEP;                 // waves per row
    const int per = each == 1 ? 4 : 1;                           // rows per workgroup
    __shared__ float red[16][D];
    int64_t row = (int64_t)blockIdx.x * per + (each == 1 ? wave : 0);
    bool real = row < rows.count;
    if (rows.start) {
        const int s0 = min(max(rows.start[blockIdx.y], 0), rows.tokens), s1 = min(max(rows.start[blockIdx.y + 1], s0), rows.tokens);
        real = real && row < (int64_t)(s1 - s0) * rows.heads;
        row += (int64_t)s0 * rows.heads;
    }
    if (!real) return;                                           // with it the whole row's waves
    const float* st = stat + row * splits * 2;
    const int first = each == 1 ? 0 : DEEP * wave;               // this wave's splits
    const float* pr = part + (row * splits + first) * D + lane * DL;
    float x[DEEP][DL];
#pragma unroll
    for (int s = 0; s < DEEP; s++) {
        const float* p = pr + (int64_t)min(s, splits - 1 - first) * D;
        if constexpr (DL == 2) {
            const float2 v = *reinterpret_cast<const float2*>(p);
            x[s][0] = v.x; x[s][1] = v.y;
        } else {
            x[s][0] = *p;
        }
    }
    // every wave: the row's maximum and sum over all splits
    float m[CH], l[CH], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < CH; k++) {
        m[k] = -INFINITY; l[k] = 0.0f;
        if (64 * k + lane < splits) {
            const float2 v = *reinterpret_cast<const float2*>(st + 2 * (64 * k + lane));
            m[k] = v.x; l[k] = v.y;
        }
        top = fmaxf(top, m[k]);
    }
    top = wave_max(top);
    float sum = 0.0f, mine = -1.0f;                              // mine: the weights of the 64 splits that this wave's are among
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const float w = m[k] == top ? 1.0f : __builtin_amdgcn_exp2f(m[k] - top);
        sum += w * l[k];
        if (first >> 6 == k) mine = m[k] == -INFINITY ? -1.0f : w;   // -1: not looked at
    }
    sum = wave_sum(sum);
    float acc[DL];
    bool odd = false;
#pragma unroll
    for (int e = 0; e < DL; e++) acc[e] = 0.0f;
    auto weight = [&](int s) { return first + s < splits ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), (first & 63) + s)) : -1.0f; };
#pragma unroll
    for (int s = 0; s < DEEP; s++) {
        const float w = weight(s);
#pragma unroll
        for (int e = 0; e < DL; e++) acc[e] += w < 0.0f ? 0.0f : w * x[s][e];
    }
#pragma unroll
    for (int e = 0; e < DL; e++) odd |= !__builtin_isfinite(acc[e]);
    if (__builtin_expect(__any(odd), 0)) {                       // (selected in the sum above: 15.1 -> 16.0 us a call of one sequence)
#pragma unroll
        for (int e = 0; e < DL; e++) acc[e] = 0.0f;
#pragma unroll
        for (int s = 0; s < DEEP; s++) {
            const float w = weight(s);
#pragma unroll
            for (int e = 0; e < DL; e++) acc[e] += w < 0.0f ? 0.0f : __builtin_isfinite(x[s][e]) ? w * x[s][e] : x[s][e];
        }
    }
    if (each > 1) {
#pragma unroll
        for (int e = 0; e < DL; e++) red[wave][lane * DL + e] = acc[e];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int e = 0; e < DL; e++)
            for (int w = 1; w < each; w++) acc[e] += red[w][lane * DL + e];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    S* o = static_cast<S*>(out) + row * D + lane * DL;
#pragma unroll
    for (int e = 0; e < DL; e++) {
        const float y = acc[e] * inv;
        if constexpr (std::is_same<E, El32>::value) o[e] = y;
        else if constexpr (std::is_same<E, ElBf>::value) o[e] = f2bf(y);
        else o[e] = f2h(y);
    }
}
// Up to four splits (prompts) a wave asks for no more than those: 57,600 rows of 3 splits 37.2 -> 23.1 us
template <typename E, int D>
static void launch_join(const float* part, const float* stat, void* out, const JoinRows& rows, int splits, hipStream_t st) {
    const int each = splits <= 4 ? 1 : (splits + 15) / 16, per = each == 1 ? 4 : 1;
    const dim3 grid((unsigned)((rows.count + per - 1) / per), rows.start ? rows.n : 1), block(64 * (each == 1 ? 4 : each));
    if (splits <= 4) hipLaunchKernelGGL((join_splits_kernel<E, D, 4>), grid, block, 0, st, part, stat, out, rows, splits);
    else hipLaunchKernelGGL((join_splits_kernel<E, D, 16>), grid, block, 0, st, part, stat, out, rows, splits);
}

}  // namespace ud
