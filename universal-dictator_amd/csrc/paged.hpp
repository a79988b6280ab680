// What the kernels over the decoder's paged cache share: page formats, their addresses, MXFP4 blocks.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/ud_decode.h"
#include "paged_plan.hpp"
#include "ud_common.hpp"

int ud_set_error(int code, const char* msg);   // encoder.hip

namespace ud {

// Page formats.  A page of one kv head: 16 rows of D 16-bit elements, or (MXFP4) 16 rows of D / 2 bytes of
// codes, the lower channel in the low nibble, and behind them 16 rows of D / 32 exponent bytes.
enum PageFormat { FMT_BF16 = 0, FMT_F16 = 1, FMT_FP4 = 2 };
constexpr int FP4_BLOCK = 32;                      // channels per shared exponent

template <int FMT, int D> struct Page {
    static constexpr int CODES = KPAGE * D / 2;                                              // FMT_FP4: bytes before the exponents
    static constexpr int BYTES = FMT == FMT_FP4 ? CODES + KPAGE * D / FP4_BLOCK : KPAGE * D * 2;   // of one kv head
};

inline int page_format(int32_t kv_format) {
    return kv_format == UD_BF16 ? FMT_BF16 : kv_format == UD_F16 ? FMT_F16 : kv_format == UD_MXFP4 ? FMT_FP4 : -1;
}

// Elements of rows outside the pages: fp32, or 16 bits wide.
struct El32 { typedef float S; };
struct ElBf { typedef uint16_t S; };
struct ElH { typedef uint16_t S; };

// Four elements as floats, and four floats stored (16-bit: rounded to nearest even; half saturates).
template <typename E> __device__ __forceinline__ void widen4(uint2 v, float (&f)[4]);
template <> __device__ __forceinline__ void widen4<ElBf>(uint2 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
}
template <> __device__ __forceinline__ void widen4<ElH>(uint2 v, float (&f)[4]) {
    f[0] = half_lo(v.x); f[1] = half_hi(v.x); f[2] = half_lo(v.y); f[3] = half_hi(v.y);
}
template <typename E> __device__ __forceinline__ void widen4(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
template <typename E> __device__ __forceinline__ void load4(const typename E::S* p, float (&f)[4]) {
    if constexpr (sizeof(typename E::S) == 4) widen4<E>(*reinterpret_cast<const uint4*>(p), f);
    else widen4<E>(*reinterpret_cast<const uint2*>(p), f);
}
template <typename E> __device__ __forceinline__ void store4(typename E::S* p, const float (&f)[4]);
template <> __device__ __forceinline__ void store4<El32>(float* p, const float (&f)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}
template <> __device__ __forceinline__ void store4<ElBf>(uint16_t* p, const float (&f)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
}
template <> __device__ __forceinline__ void store4<ElH>(uint16_t* p, const float (&f)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)f2h(f[0]) | (uint32_t)f2h(f[1]) << 16,
                                              (uint32_t)f2h(f[2]) | (uint32_t)f2h(f[3]) << 16);
}

// A block's scale as the fp32 value 2^E of its exponent byte 127 + E (bytes 1 .. 254; 255 marks a block that held
// a NaN or an infinity: the conversions below give NaN for it).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes of a block (one word, lowest nibble first) as packed bf16 pairs: exact, one conversion per pair.
__device__ __forceinline__ uint4 fp4_to_bf16(uint32_t w, float scale) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3)));
}

// A failed call's status with its message.
__attribute__((format(printf, 2, 3))) static inline int paged_fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return ud_set_error(code, buf);
}

// The checks that every call over the pages makes.
static inline int paged_check(const char* who, int32_t kv_format, const void* k_pages, const void* v_pages, int32_t num_blocks,
                              const int32_t* block_table, int32_t n, int32_t max_blocks, int32_t kv_heads, int32_t head_dim,
                              int32_t block_size) {
    if (!k_pages || !v_pages || !block_table) return paged_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if (page_format(kv_format) < 0) return paged_fail(UD_ERR_INVALID, "%s: page format %d", who, kv_format);
    if (head_dim != 64 && head_dim != 128) return paged_fail(UD_ERR_SHAPE, "%s: head_dim %d (64 or 128)", who, head_dim);
    if (block_size != KPAGE) return paged_fail(UD_ERR_SHAPE, "%s: block_size %d (16 supported)", who, block_size);
    if (n < 1 || n > 65535 || kv_heads < 1 || kv_heads > 65535)
        return paged_fail(UD_ERR_SHAPE, "%s: %d sequences, %d kv heads (1 .. 65535)", who, n, kv_heads);
    if (num_blocks < 1 || max_blocks < 1 || max_blocks > INT32_MAX / KPAGE)
        return paged_fail(UD_ERR_SHAPE, "%s: %d pages, %d table entries per sequence", who, num_blocks, max_blocks);
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15)
        return paged_fail(UD_ERR_INVALID, "%s: pages must be 16-byte aligned", who);
    return UD_OK;
}

static inline int paged_launched(const char* who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UD_OK : paged_fail(UD_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}

}  // namespace ud
