// Rows between a decoder's products: the residual's addition with the root-mean-square norm, and rows to 8 bits, plain or
// gated (include/ud_layer.h).
//
// One pass: a row lies in the registers of W waves, P pieces of eight elements to a lane, between its loads and its stores; what
// depends on the whole row (the mean square, the largest magnitude) is a wave's butterfly of lane moves and, over several waves,
// one LDS exchange.
#include "layer.hpp"

namespace ud {

struct RowArgs {
    const void* x; const void* y;                  // norm: x and the residual (or null); 8 bits: x and the gate (or null)
    void* sum; const float* w;
    void* out; float* scales;
    int64_t x_ld, y_ld, out_ld;
    int rows, dim;
    float eps;
};

// The sum (or the maximum) over a row's W waves, in every lane.  `at`: an LDS array of its own for each exchange.
template <int W, typename V, typename F> __device__ __forceinline__ V row_join(V v, V* at, F join) {
    if constexpr (W > 1) {
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) at[wave] = v;
        __syncthreads();
        v = at[0];
#pragma unroll
        for (int i = 1; i < W; i++) v = join(v, at[i]);
    }
    return v;
}

// Pieces y of a row as 8-bit codes, and the row's scale.  The largest magnitude is taken as an unsigned number, so that a NaN
// is larger than all.  A code is the quotient y / scale as a division rounds it, to the nearest whole number: the product with the
// reciprocal, corrected by what it leaves of y (the product alone gives the other code to one in twelve of the values next to a border).  1.5 * 2^23 + code: the sum is
// rounded to whole numbers, and the code is its lowest byte.
template <int W, int P>
__device__ __forceinline__ void store_codes(const float (&y)[P][8], int t, int dim, uint32_t* at, int8_t* codes, float* scale_out) {
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < P; p++)
        if ((t + p * 64 * W) * 8 < dim)
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(y[p][e]) & 0x7fffffffu);
    top = row_join<W>(wave_max_u(top), at, [](uint32_t a, uint32_t b) { return max(a, b); });
    const bool bad = top >= 0x7f800000u;
    const float scale = bad ? __builtin_nanf("") : fmaxf(__uint_as_float(top) / 127.0f, 0x1p-126f);
    const float inv = bad ? 0.0f : 1.0f / scale;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (t + p * 64 * W) * 8;
        if (c >= dim) continue;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float q = y[p][e] * inv;
            const uint32_t code = __float_as_uint(fmaf(fmaf(-q, scale, y[p][e]), inv, q) + 0x1.8p23f) & 255u;
            w[e / 4] |= (bad ? 0u : code) << (8 * (e % 4));
        }
        *reinterpret_cast<uint2*>(codes + c) = make_uint2(w[0], w[1]);
    }
    if (t == 0) *scale_out = scale;
}

template <typename T, typename S, bool EIGHT, int W, int P>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void rms_norm_kernel(RowArgs a) {
    __shared__ double at_sum[W];
    __shared__ uint32_t at_top[W];
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x;
    if (row >= a.rows) return;
    const int t = W == 1 ? threadIdx.x % 64 : threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
    const S* res = a.y ? static_cast<const S*>(a.y) + row * a.y_ld : nullptr;
    Raw8<T> xr[P];
    Raw8<S> rr[P];
    float s[P][8];
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (t + p * 64 * W) * 8;
        if (c >= a.dim) continue;
        xr[p] = load8(x + c);
        if (res) rr[p] = load8(res + c);
    }
    double ss = 0.0;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (t + p * 64 * W) * 8;
        if (c >= a.dim) continue;
        widen8<T>(xr[p], s[p]);
        if (res) {
            float r[8];
            widen8<S>(rr[p], r);
#pragma unroll
            for (int e = 0; e < 8; e++) s[p][e] += r[e];
            const Raw8<S> stored = narrow8<S>(s[p]);
            store8(static_cast<S*>(a.sum) + row * a.y_ld + c, stored);
            widen8<S>(stored, s[p]);               // the norm is that of the sums as they are stored
        }
        // 64 bits: squares of rows past 2^63 or under 2^-63 stay in range
#pragma unroll
        for (int e = 0; e < 8; e++) ss = fma((double)s[p][e], (double)s[p][e], ss);
    }
    ss = row_join<W>(wave_sum_d(ss), at_sum, [](double u, double v) { return u + v; });
    const float r = (float)(1.0 / sqrt(ss / a.dim + (double)a.eps));
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (t + p * 64 * W) * 8;
        if (c >= a.dim) continue;
#pragma unroll
        for (int e = 0; e < 8; e++) s[p][e] *= r;
        if (a.w) {
            float w[8];
            widen8<float>(load8(a.w + c), w);
#pragma unroll
            for (int e = 0; e < 8; e++) s[p][e] *= w[e];
        }
        if constexpr (!EIGHT) store8(static_cast<T*>(a.out) + row * a.out_ld + c, narrow8<T>(s[p]));
    }
    if constexpr (EIGHT) store_codes<W, P>(s, t, a.dim, at_top, static_cast<int8_t*>(a.out) + row * a.out_ld, a.scales + row);
}

template <typename T, bool GATE, int W, int P>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void i8_rows_kernel(RowArgs a) {
    __shared__ uint32_t at_top[W];
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x;
    if (row >= a.rows) return;
    const int t = W == 1 ? threadIdx.x % 64 : threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
    const T* gate = GATE ? static_cast<const T*>(a.y) + row * a.x_ld : nullptr;
    Raw8<T> xr[P], gr[P];
    float y[P][8];
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int c = (t + p * 64 * W) * 8;
        if (c >= a.dim) continue;
        xr[p] = load8(x + c);
        if constexpr (GATE) gr[p] = load8(gate + c);
    }
#pragma unroll
    for (int p = 0; p < P; p++) {
        if ((t + p * 64 * W) * 8 >= a.dim) continue;
        widen8<T>(xr[p], y[p]);
        if constexpr (GATE) {
            // expf and not the short v_exp_f32 form: far gates would be off by their distance from 0 times 2^-23
            float g[8];
            widen8<T>(gr[p], g);
#pragma unroll
            for (int e = 0; e < 8; e++) y[p][e] *= g[e] * __builtin_amdgcn_rcpf(1.0f + expf(-g[e]));
        }
    }
    store_codes<W, P>(y, t, a.dim, at_top, static_cast<int8_t*>(a.out) + row * a.out_ld, a.scales + row);
}

// A row's waves and each lane's pieces, by its length: two pieces a lane where a row is long enough, so that few enough waves meet at
// the barriers and enough loads are on their way.  us, bf16 with its residual to 8 bits, W x P: 8,200 rows of 1,024 1 x 2 13.2, 4 x 1
// 16.0; of 4,096 4 x 2 39.7, 8 x 1 46.0, 16 x 1 53; of 8,192 8 x 2 85, 16 x 1 101, 4 x 4 90; 563 of 4,096 4 x 2 6.3, 16 x 1 7.7, but 256 4.8
// and 4.5, and one row (its latency, in the trace) 3.8 and 3.2.
template <template <int, int> class L> static void launch_rows(const RowArgs& a, hipStream_t st) {
    if (a.dim <= 1024) L<1, 2>::go(a, st);
    else if (a.dim <= 2048) L<4, 1>::go(a, st);
    else if (a.rows <= 256 && a.dim <= 8192) L<16, 1>::go(a, st);
    else if (a.dim <= 4096) L<4, 2>::go(a, st);
    else if (a.dim <= 8192) L<8, 2>::go(a, st);
    else if (a.dim <= 16384) L<16, 2>::go(a, st);
    else L<16, 4>::go(a, st);
}
static dim3 row_grid(int rows, int w) { return dim3((unsigned)(w == 1 ? (rows + 3) / 4 : rows)); }

template <typename T, typename S, bool EIGHT> struct Norm {
    template <int W, int P> struct L {
        static void go(const RowArgs& a, hipStream_t st) {
            hipLaunchKernelGGL((rms_norm_kernel<T, S, EIGHT, W, P>), row_grid(a.rows, W), dim3(W == 1 ? 256 : 64 * W), 0, st, a);
        }
    };
};
template <typename T, bool GATE> struct Eight {
    template <int W, int P> struct L {
        static void go(const RowArgs& a, hipStream_t st) {
            hipLaunchKernelGGL((i8_rows_kernel<T, GATE, W, P>), row_grid(a.rows, W), dim3(W == 1 ? 256 : 64 * W), 0, st, a);
        }
    };
};
template <typename T, typename S> static void launch_norm(const RowArgs& a, bool eight, hipStream_t st) {
    if (eight) launch_rows<Norm<T, S, true>::template L>(a, st);
    else launch_rows<Norm<T, S, false>::template L>(a, st);
}
template <typename T> static void launch_eight(const RowArgs& a, hipStream_t st) {
    if (a.y) launch_rows<Eight<T, true>::template L>(a, st);
    else launch_rows<Eight<T, false>::template L>(a, st);
}

// The checks that both calls make.
static int rows_check(const char* who, int32_t dtype, int32_t rows, int32_t dim) {
    if (!type_bytes(dtype)) return layer_fail(UD_ERR_INVALID, "%s: dtype %d", who, dtype);
    // (a launch holds fewer than 2^32 threads)
    if (rows < 0 || rows >= (1 << 22)) return layer_fail(UD_ERR_SHAPE, "%s: rows %d (0 .. 2^22 - 1)", who, rows);
    if (dim < 8 || dim > 32768 || dim % 8) return layer_fail(UD_ERR_SHAPE, "%s: dim %d (a multiple of 8, 8 .. 32768)", who, dim);
    return UD_OK;
}

}  // namespace ud

using namespace ud;

extern "C" UD_API int ud_rms_norm(int32_t dtype, const void* x_dev, int32_t x_ld, int32_t sum_dtype, const void* residual_dev,
                                  void* sum_out_dev, int32_t sum_ld, const float* weight_dev, float eps, int32_t out_dtype,
                                  void* out_dev, int32_t out_ld, float* scales_dev, int32_t rows, int32_t dim, void* hip_stream) {
    static const char* who = "ud_rms_norm";
    int rc = rows_check(who, dtype, rows, dim);
    if (rc != UD_OK) return rc;
    const bool eight = out_dtype == UD_I8, add = residual_dev != nullptr;
    if (!eight && out_dtype != dtype) return layer_fail(UD_ERR_INVALID, "%s: out_dtype %d (dtype %d, or UD_I8)", who, out_dtype, dtype);
    if (add && sum_dtype != dtype && sum_dtype != UD_F32)
        return layer_fail(UD_ERR_INVALID, "%s: sum_dtype %d (dtype %d, or fp32)", who, sum_dtype, dtype);
    if (!(eps >= 1e-30f) || eps > 1e30f) return layer_fail(UD_ERR_INVALID, "%s: eps %g (1e-30 .. 1e30)", who, (double)eps);
    if (add != (sum_out_dev != nullptr)) return layer_fail(UD_ERR_INVALID, "%s: residual and sum_out go together", who);
    if (eight != (scales_dev != nullptr)) return layer_fail(UD_ERR_INVALID, "%s: scales go with UD_I8", who);
    if (x_ld < dim || out_ld < dim || (add && sum_ld < dim) || ((x_ld | out_ld | (add ? sum_ld : 0)) & 7))
        return layer_fail(UD_ERR_SHAPE, "%s: rows %d/%d/%d elements apart for %d (multiples of 8)", who, x_ld, add ? sum_ld : 0, out_ld, dim);
    if (rows == 0) return UD_OK;
    if (!x_dev || !out_dev) return layer_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if ((((uintptr_t)x_dev | (uintptr_t)residual_dev | (uintptr_t)sum_out_dev | (uintptr_t)weight_dev) & 15) || ((uintptr_t)out_dev & (eight ? 7 : 15)) ||
        ((uintptr_t)scales_dev & 3))
        return layer_fail(UD_ERR_INVALID, "%s: pointers must be 16-byte aligned (codes 8, scales 4)", who);
    const int64_t size = type_bytes(dtype), ssize = add ? type_bytes(sum_dtype) : 0, osize = eight ? 1 : size;
    const Block x{x_dev, x_ld * size, dim * size, rows}, res{residual_dev, sum_ld * ssize, dim * ssize, rows},
        sum{sum_out_dev, sum_ld * ssize, dim * ssize, rows}, out{out_dev, out_ld * osize, dim * osize, rows}, w{weight_dev, 0, dim * 4, 1},
        sc{scales_dev, 4, 4, rows};
    auto clash = [](const Block& o, const Block& in, bool same_type) { return blocks_meet(o, in) && !(same_type && blocks_same(o, in)); };
    if (clash(out, x, !eight) || clash(out, res, !eight && size == ssize) || clash(sum, x, size == ssize) || clash(sum, res, true) ||
        blocks_meet(out, sum) || blocks_meet(out, w) || blocks_meet(sum, w) || blocks_meet(sc, x) || blocks_meet(sc, res) ||
        blocks_meet(sc, sum) || blocks_meet(sc, out) || blocks_meet(sc, w))
        return layer_fail(UD_ERR_INVALID, "%s: an output overlaps an input or another output (in place: the same type, place and ld)", who);
    RowArgs a{};
    a.x = x_dev; a.y = residual_dev; a.sum = sum_out_dev; a.w = weight_dev; a.out = out_dev; a.scales = scales_dev;
    a.x_ld = x_ld; a.y_ld = sum_ld; a.out_ld = out_ld; a.rows = rows; a.dim = dim; a.eps = eps;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const bool wide = add && sum_dtype == UD_F32;
    if (dtype == UD_F32) launch_norm<float, float>(a, eight, st);
    else if (dtype == UD_BF16 && wide) launch_norm<bf16, float>(a, eight, st);
    else if (dtype == UD_BF16) launch_norm<bf16, bf16>(a, eight, st);
    else if (wide) launch_norm<f16, float>(a, eight, st);
    else launch_norm<f16, f16>(a, eight, st);
    return layer_launched(who);
}

extern "C" UD_API int ud_i8_quantize(int32_t dtype, const void* x_dev, const void* gate_dev, int32_t ld, int8_t* codes_dev,
                                     int32_t codes_ld, float* scales_dev, int32_t rows, int32_t dim, void* hip_stream) {
    static const char* who = "ud_i8_quantize";
    int rc = rows_check(who, dtype, rows, dim);
    if (rc != UD_OK) return rc;
    if (ld < dim || codes_ld < dim || ((ld | codes_ld) & 7))
        return layer_fail(UD_ERR_SHAPE, "%s: rows %d/%d elements apart for %d (multiples of 8)", who, ld, codes_ld, dim);
    if (rows == 0) return UD_OK;
    if (!x_dev || !codes_dev || !scales_dev) return layer_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if ((((uintptr_t)x_dev | (uintptr_t)gate_dev) & 15) || ((uintptr_t)codes_dev & 7) || ((uintptr_t)scales_dev & 3))
        return layer_fail(UD_ERR_INVALID, "%s: x and gate must be 16-byte aligned (codes 8, scales 4)", who);
    const int64_t size = type_bytes(dtype);
    const Block x{x_dev, ld * size, dim * size, rows}, g{gate_dev, ld * size, dim * size, rows}, c{codes_dev, codes_ld, dim, rows},
        sc{scales_dev, 4, 4, rows};
    if (blocks_meet(c, x) || blocks_meet(c, g) || blocks_meet(sc, x) || blocks_meet(sc, g) || blocks_meet(sc, c))
        return layer_fail(UD_ERR_INVALID, "%s: an output overlaps an input or the other output", who);
    RowArgs a{};
    a.x = x_dev; a.y = gate_dev; a.out = codes_dev; a.scales = scales_dev;
    a.x_ld = ld; a.out_ld = codes_ld; a.rows = rows; a.dim = dim;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (dtype == UD_F32) launch_eight<float>(a, st);
    else if (dtype == UD_BF16) launch_eight<bf16>(a, st);
    else launch_eight<f16>(a, st);
    return layer_launched(who);
}
