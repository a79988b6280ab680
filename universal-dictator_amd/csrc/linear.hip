// The product of int8 rows with int8 weights, scales for each row and each channel (include/ud_layer.h):
//   out[m, n] = (sum_k codes[m, k] w[n, k]) * scales[m] * w_scales[n] + bias[n] + residual[m, n]
// The sums are exact in 32 bits, so neither the order of k nor its split over waves changes a bit.
#include "layer.hpp"

namespace ud {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

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

template <typename T> static void launch_linear(const LinearArgs& a, hipStream_t st) {
    if (a.M <= 16) launch_few<T, 1, 1, 8, 4>(a, st);
    else launch_few<T, 4, 2, 4, 2>(a, st);
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
