// What the calls of ud_layer.h share: element types, pieces of eight elements, wave reductions, checks of their arguments.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <type_traits>

#include "../../include/ud_layer.h"
#include "ud_common.hpp"

int ud_set_error(int code, const char* msg);   // encoder.hip

namespace ud {

// ---------------------------------------------------------------- device

// Eight elements as they lie in memory: two pieces of 16 bytes of fp32, one of 16 bits.
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); i++) r.v[i] = ld16(reinterpret_cast<const char*>(p) + 16 * i);
    return r;
}
template <typename T> __device__ __forceinline__ void widen8(const Raw8<T>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); i++) unpack16<T>(r.v[i], f + i * Vec16<T>::N);
}
// Rounded to nearest even; half saturates.
template <typename T> __device__ __forceinline__ Raw8<T> narrow8(const float (&f)[8]) {
    Raw8<T> r;
    if constexpr (sizeof(T) == 4) {
        r.v[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        r.v[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    } else if constexpr (std::is_same<T, bf16>::value) {
        r.v[0] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = (uint32_t)f2h(f[2 * i]) | (uint32_t)f2h(f[2 * i + 1]) << 16;
        r.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); i++) st16(reinterpret_cast<char*>(p) + 16 * i, r.v[i]);
}

// Sum and maximum over a wave, in every lane.
template <int CTRL> __device__ __forceinline__ double dpp_add_d(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, false);
    return v + __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_sum_d(double v) {
    v = dpp_add_d<DPP_QUAD_1032>(v);
    v = dpp_add_d<DPP_QUAD_2301>(v);
    v = dpp_add_d<DPP_ROW_HALF_MIRROR>(v);
    v = dpp_add_d<DPP_ROW_MIRROR>(v);
    auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
    auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
    v = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
    lo = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
    hi = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
    return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max_u(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    v = dpp_max_u<DPP_QUAD_1032>(v);
    v = dpp_max_u<DPP_QUAD_2301>(v);
    v = dpp_max_u<DPP_ROW_HALF_MIRROR>(v);
    v = dpp_max_u<DPP_ROW_MIRROR>(v);
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

// ---------------------------------------------------------------- host

// A failed call's status with its message.
__attribute__((format(printf, 2, 3))) static inline int layer_fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return ud_set_error(code, buf);
}
static inline int layer_launched(const char* who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UD_OK : layer_fail(UD_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
}

// Bytes of an element of a row type, 0 for none.
static inline int64_t type_bytes(int32_t dtype) { return dtype == UD_F32 ? 4 : dtype == UD_BF16 || dtype == UD_F16 ? 2 : 0; }

// `rows` rows of `width` bytes, `ld` bytes from one to the next.
struct Block {
    const void* at;
    int64_t ld, width, rows;
};
// Whether two blocks share memory.  At the same distance between rows (a single row has any) exactly; else whether the
// stretches from their first rows to their last do.
static inline bool blocks_meet(const Block& a, const Block& b) {
    if (!a.at || !b.at || a.rows < 1 || b.rows < 1) return false;
    const int64_t d = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at);
    if (!(d < (a.rows - 1) * a.ld + a.width && -d < (b.rows - 1) * b.ld + b.width)) return false;
    const int64_t ld = a.rows == 1 ? b.ld : a.ld;
    if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.ld != b.ld) || ld < 1) return true;
    // row i of a meets row i + t of b where -b.width < d + t ld < a.width, and there is one of t = 1 - a.rows .. b.rows - 1
    const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    const int64_t lo = floor_div(-b.width - d, ld) + 1, hi = -floor_div(d - a.width, ld) - 1;
    return (lo > 1 - a.rows ? lo : 1 - a.rows) <= (hi < b.rows - 1 ? hi : b.rows - 1);
}
// Whether they are the same rows in the same places, which a call that reads an element before it writes that place allows.
static inline bool blocks_same(const Block& a, const Block& b) {
    return a.at == b.at && a.width == b.width && a.rows == b.rows && (a.ld == b.ld || a.rows == 1);
}

}  // namespace ud
