// Query and key heads normalised and rotated, keys and values written into the paged cache, in one pass;
// and cache rows read back (include/ud_decode.h).
//
//   y = x / sqrt(mean_c x_c^2 + eps) * w            per head, where a weight is given
//   (y_i, y_{i+d/2}) -> (y_i cos a - y_{i+d/2} sin a, y_{i+d/2} cos a + y_i sin a),   a = position * inv_freq_i
//
// Bound: memory, with the vector units not far behind (below).  A row's heads are read once and written once (q to q_out, k
// and v to their pages).
// Layout: one workgroup per row.  A lane holds channels 4i .. 4i + 3 of a head and the four they rotate with,
// half a head on, so that the rotation stays in the lane and the norm's sum is one butterfly over the head's
// D / 8 lanes.  The D / 2 angles of a row are the same for all heads: computed once, by one lane each, into LDS.
// Angles are formed and their sine and cosine taken in 64 bits: an fp32 product of a position of 120,000 and a
// frequency near 1 is off by 0.004 rad.
// Keys for MXFP4 pages are normalised and rotated in 64 bits: a key next to a border between two codes would
// otherwise move by a whole step of its block with the order of a sum, and so would every key of a block whose
// largest value is next to a power of two's border.  That is 8 of 48 heads at 32/8.
// Measured, 32/8 heads of 128: 8,200 rows of bf16 to MXFP4 pages 45 .. 46 us (177 MB, 3.8 .. 3.9 TB/s, three quarters to four
// fifths of a large copy's 4.7 .. 5.0; vector units busy 68 % of the time), 64 rows 5.7 us, one row of fp32 to half pages 3.2 us:
// little more than an empty launch.  Read back: 17.6 (76 MB, 4.3 TB/s), 3.6 and 1.9 us.
#include <type_traits>

#include "paged.hpp"

namespace ud {

struct AppendArgs {
    const void* q; const void* k; const void* v;
    void* q_out;
    int64_t q_ld, k_ld, v_ld, qo_ld;               // elements between rows
    const float* qw; const float* kw;              // [D] norm weights, or null
    float eps;
    const float* inv_freq;                         // [D / 2], or null
    const int32_t* pos; const int32_t* seqs;
    char* kp; char* vp;
    const int32_t* bt;
    int n, max_blocks, num_blocks, Hq, Hkv;
};

// The page that holds position p of sequence s, or -1 where the row is padding or the page is none of the pool's.
__device__ __forceinline__ int row_page(int s, int p, const int32_t* bt, int n, int max_blocks, int num_blocks) {
    if (s < 0 || s >= n || p < 0 || p / KPAGE >= max_blocks) return -1;
    const int page = bt[(int64_t)s * max_blocks + p / KPAGE];
    return page >= 0 && page < num_blocks ? page : -1;
}

template <int CTRL> __device__ __forceinline__ double dpp_mov_d(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, false);
    return __hiloint2double(hi, lo);
}
// Sum over aligned groups of W lanes (8 or 16), in every lane.
template <int W> __device__ __forceinline__ double group_sum_d(double v) {
    v += dpp_mov_d<DPP_QUAD_1032>(v);
    v += dpp_mov_d<DPP_QUAD_2301>(v);
    v += dpp_mov_d<DPP_ROW_HALF_MIRROR>(v);
    if constexpr (W == 16) v += dpp_mov_d<DPP_ROW_MIRROR>(v);
    return v;
}
__device__ __forceinline__ uint32_t group_max8(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_1032, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_2301, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_HALF_MIRROR, 0xF, 0xF, false));
}

// x in fp32 by rounding to odd: not exact -> the last bit is set.  Such a value is on the same side of every
// border of fewer bits as x, so that a second rounding to nearest gives what one rounding of x would.  A finite x past
// fp32's range becomes its largest value, which is odd.
__device__ __forceinline__ float round_odd(double x) {
    const float f = (float)x;
    const double b = (double)f;
    if (b == x || x != x) return f;
    uint32_t u = __float_as_uint(f);
    if (fabs(b) > fabs(x)) u -= 1;                 // towards zero
    return __uint_as_float(u | 1);
}

// The exponent byte of a block whose largest magnitude has the bits `top`: the smallest power of two that brings
// it to 7 or less (a value in 6 .. 7 is held as 6, off by no more than a value in the next step up would be).
// Not below 2^-100, so that the values stay normal in bf16, nor above 2^125, whose 6 is the largest that fp32 holds
// (larger values saturate); 255 for a block with an infinity or a NaN.
__device__ __forceinline__ uint32_t fp4_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    const int e = (int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) > 0x600000u);
    return (uint32_t)(min(max(e, -100), 125) + 127);
}
// Four values as codes, lowest nibble first.
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[4], float scale) {
    const uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1) & 0xffffu;
}

// A lane's values (lo: channels 4i .., hi: half a head on) of row r of the kv head at `head`.
template <int FMT, int D>
__device__ __forceinline__ void store_row(char* head, int r, int i, const float (&lo)[4], const float (&hi)[4]) {
    if constexpr (FMT == FMT_FP4) {
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a = max(a, __float_as_uint(lo[e]) & 0x7fffffffu);
            b = max(b, __float_as_uint(hi[e]) & 0x7fffffffu);
        }
        const uint32_t ba = fp4_byte(group_max8(a)), bb = fp4_byte(group_max8(b));
        uint16_t* codes = reinterpret_cast<uint16_t*>(head + r * (D / 2)) + i;
        codes[0] = (uint16_t)fp4_codes(lo, fp4_scale(ba));
        codes[D / 8] = (uint16_t)fp4_codes(hi, fp4_scale(bb));
        if (i % 8 == 0) {
            char* s = head + Page<FMT, D>::CODES + r * (D / FP4_BLOCK) + i / 8;
            s[0] = (char)ba;
            s[D / 64] = (char)bb;
        }
    } else {
        typedef typename std::conditional<FMT == FMT_BF16, ElBf, ElH>::type E;
        uint16_t* row = reinterpret_cast<uint16_t*>(head) + r * D + 4 * i;
        store4<E>(row, lo);
        store4<E>(row + D / 2, hi);
    }
}

// (64 registers from 16-bit rows, eight workgroups a CU: 8,200 rows, with the read-back, 65.8 -> 64.2 us)
template <typename E, int FMT, int D>
__global__ __launch_bounds__(256, sizeof(typename E::S) == 4 ? 6 : 8) void norm_rope_append_kernel(AppendArgs a) {
    constexpr int LPH = D / 8;                     // lanes per head
    constexpr bool WIDE = FMT == FMT_FP4;          // keys in 64 bits
    typedef typename E::S S;
    __shared__ float2 turn[D / 2];
    __shared__ double2 turn_d[WIDE ? D / 2 : 1];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const int p = a.pos[row], s = a.seqs ? a.seqs[row] : (int)min(row, (int64_t)INT32_MAX);
    const int page = row_page(s, p, a.bt, a.n, a.max_blocks, a.num_blocks);
    if (page < 0) return;                          // uniform in the workgroup
    // Raw values of three passes over the heads at a time (48 heads of 128): the first are on their way while the angles are
    // made.
    constexpr int DEEP = 3, HPP = 256 / LPH;       // heads per pass
    const int i = tid % LPH, heads = a.Hq + 2 * a.Hkv;
    typedef typename std::conditional<sizeof(S) == 4, uint4, uint2>::type Raw;
    Raw raw[DEEP][2];
    auto load = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < DEEP; n++) {
            const int h = h0 + HPP * n;
            if (h >= heads) continue;
            const S* src = h < a.Hq ? static_cast<const S*>(a.q) + row * a.q_ld + (int64_t)h * D
                           : h < a.Hq + a.Hkv ? static_cast<const S*>(a.k) + row * a.k_ld + (int64_t)(h - a.Hq) * D
                                              : static_cast<const S*>(a.v) + row * a.v_ld + (int64_t)(h - a.Hq - a.Hkv) * D;
            raw[n][0] = *reinterpret_cast<const Raw*>(src + 4 * i);
            raw[n][1] = *reinterpret_cast<const Raw*>(src + 4 * i + D / 2);
        }
    };
    load(tid / LPH);
    if (a.inv_freq) {
        if (tid < D / 2) {
            double sn, cs;
            sincos((double)p * (double)a.inv_freq[tid], &sn, &cs);
            turn[tid] = make_float2((float)cs, (float)sn);
            if constexpr (WIDE) turn_d[tid] = make_double2(cs, sn);
        }
        __syncthreads();
    }
    for (int h0 = tid / LPH; h0 < heads; h0 += DEEP * HPP) {
        if (h0 >= DEEP * HPP) load(h0);
#pragma unroll
        for (int n = 0; n < DEEP; n++) {
            const int h = h0 + HPP * n;
            if (h >= heads) break;
            const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hkv;
            const int kvh = is_q ? 0 : is_k ? h - a.Hq : h - a.Hq - a.Hkv;
            float lo[4], hi[4];
            widen4<E>(raw[n][0], lo);
            widen4<E>(raw[n][1], hi);
            if (is_q || (is_k && !WIDE)) {
                const float* w = is_q ? a.qw : a.kw;
                if (w) {
                    float ss = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) ss += lo[e] * lo[e] + hi[e] * hi[e];
                    const float r = 1.0f / sqrtf(group_sum<LPH>(ss) * (1.0f / D) + a.eps);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        lo[e] *= r * w[4 * i + e];
                        hi[e] *= r * w[4 * i + e + D / 2];
                    }
                }
                if (a.inv_freq) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 t = turn[4 * i + e];
                        const float x = lo[e], y = hi[e];
                        lo[e] = x * t.x - y * t.y;
                        hi[e] = y * t.x + x * t.y;
                    }
                }
                if (is_q) {
                    S* o = static_cast<S*>(a.q_out) + row * a.qo_ld + (int64_t)h * D + 4 * i;
                    store4<E>(o, lo);
                    store4<E>(o + D / 2, hi);
                    continue;
                }
            } else if (is_k) {
                double r = 1.0;
                if (a.kw) {
                    double ss = 0.0;
#pragma unroll
                    for (int e = 0; e < 4; e++) ss += (double)lo[e] * lo[e] + (double)hi[e] * hi[e];
                    r = 1.0 / sqrt(group_sum_d<LPH>(ss) * (1.0 / D) + (double)a.eps);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    double x = lo[e], y = hi[e];
                    if (a.kw) {
                        x *= r * (double)a.kw[4 * i + e];
                        y *= r * (double)a.kw[4 * i + e + D / 2];
                    }
                    if (a.inv_freq) {
                        const double2 t = turn_d[WIDE ? 4 * i + e : 0];
                        const double z = x * t.x - y * t.y;
                        y = y * t.x + x * t.y;
                        x = z;
                    }
                    lo[e] = round_odd(x);
                    hi[e] = round_odd(y);
                }
            }
            char* pool = is_k ? a.kp : a.vp;
            store_row<FMT, D>(pool + ((int64_t)page * a.Hkv + kvh) * Page<FMT, D>::BYTES, p % KPAGE, i, lo, hi);
        }
    }
}

// Eight channels of a cache row per thread, for keys and values; a row that cannot be read is 0.
template <typename E, int FMT, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(const char* kp, const char* vp, const int32_t* bt, const int32_t* pos,
                                                      const int32_t* seqs, typename E::S* ko, typename E::S* vo, int64_t pieces,
                                                      int n, int max_blocks, int num_blocks, int Hkv) {
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= pieces) return;
    const int c = (int)(idx % (D / 8)), kvh = (int)(idx / (D / 8) % Hkv);
    const int64_t row = idx / ((D / 8) * Hkv);
    const int p = pos[row], s = seqs ? seqs[row] : (int)min(row, (int64_t)INT32_MAX);
    const int page = row_page(s, p, bt, n, max_blocks, num_blocks);
    const int64_t base = ((int64_t)max(page, 0) * Hkv + kvh) * Page<FMT, D>::BYTES;
    const int r = max(p, 0) % KPAGE;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        const char* head = (kv ? vp : kp) + base;
        uint4 v = make_uint4(0, 0, 0, 0);          // as pairs of the page's 16-bit format (MXFP4: bf16)
        if (page >= 0) {
            if constexpr (FMT == FMT_FP4) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(head + r * (D / 2) + 4 * c);
                const uint8_t e = *reinterpret_cast<const uint8_t*>(head + Page<FMT, D>::CODES + r * (D / FP4_BLOCK) + c / 4);
                v = fp4_to_bf16(w, fp4_scale(e));
            } else {
                v = ld16(head + (r * D + 8 * c) * 2);
            }
        }
        typename E::S* o = (kv ? vo : ko) + idx * 8;
        if constexpr (std::is_same<E, El32>::value) {
            float f[8];
            if constexpr (FMT == FMT_F16) unpack16<f16>(v, f);
            else unpack16<bf16>(v, f);
            *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            st16(o, v);
        }
    }
}

template <typename E, int FMT>
static void launch_append(const AppendArgs& a, int rows, int D, hipStream_t st) {
    if (D == 128) hipLaunchKernelGGL((norm_rope_append_kernel<E, FMT, 128>), dim3(rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((norm_rope_append_kernel<E, FMT, 64>), dim3(rows), dim3(256), 0, st, a);
}

struct ReadArgs {
    const char* kp; const char* vp;
    const int32_t* bt; const int32_t* pos; const int32_t* seqs;
    void* ko; void* vo;
    int n, max_blocks, num_blocks, Hkv;
};
template <typename E, int FMT, int D>
static void launch_read_d(const ReadArgs& a, int rows, hipStream_t st) {
    typedef typename E::S S;
    const int64_t pieces = (int64_t)rows * a.Hkv * (D / 8);
    hipLaunchKernelGGL((kv_read_kernel<E, FMT, D>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, a.kp, a.vp, a.bt, a.pos,
                       a.seqs, static_cast<S*>(a.ko), static_cast<S*>(a.vo), pieces, a.n, a.max_blocks, a.num_blocks, a.Hkv);
}
template <typename E, int FMT>
static void launch_read(const ReadArgs& a, int rows, int D, hipStream_t st) {
    if (D == 128) launch_read_d<E, FMT, 128>(a, rows, st);
    else launch_read_d<E, FMT, 64>(a, rows, st);
}

}  // namespace ud

using namespace ud;

extern "C" UD_API size_t ud_kv_page_bytes(int32_t kv_format, int32_t kv_heads, int32_t head_dim, int32_t block_size) {
    const int f = page_format(kv_format);
    if (f < 0 || kv_heads < 1 || (head_dim != 64 && head_dim != 128) || block_size != KPAGE) return 0;
    const size_t row = f == FMT_FP4 ? head_dim / 2 + head_dim / FP4_BLOCK : 2 * head_dim;
    return (size_t)kv_heads * KPAGE * row;
}

// Whether `rows` rows of aw elements at a, lda elements apart, share memory with rows of bw at b, ldb apart (byte
// addresses; different distances: whether the stretches from first to last row do).
static bool rows_overlap(const void* a, int64_t lda, int64_t aw, const void* b, int64_t ldb, int64_t bw, int64_t rows, int64_t size) {
    const int64_t d = (int64_t)((uintptr_t)b - (uintptr_t)a), la = aw * size, lb = bw * size;
    if (rows == 1 || lda != ldb) return d < ((rows - 1) * lda) * size + la && -d < ((rows - 1) * ldb) * size + lb;
    // row i of a meets row i + t of b where -lb < d + t lda size < la: t is one of the two around -d / (lda size)
    const int64_t step = lda * size;
    for (int64_t t = -d / step - 1; t <= -d / step + 1; t++)
        if (t > -rows && t < rows && d + t * step < la && d + t * step > -lb) return true;
    return false;
}

extern "C" UD_API int ud_qk_norm_rope_append(int32_t dtype, int32_t kv_format, const void* q_dev, int32_t q_ld, const void* k_dev,
                                             int32_t k_ld, const void* v_dev, int32_t v_ld, void* q_out_dev, int32_t q_out_ld,
                                             const float* q_weight_dev, const float* k_weight_dev, float eps,
                                             const float* inv_freq_dev, const int32_t* positions_dev, const int32_t* seqs_dev,
                                             void* k_pages, void* v_pages, int32_t num_blocks, const int32_t* block_table, int32_t n,
                                             int32_t max_blocks, int32_t rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                             int32_t block_size, void* hip_stream) {
    static const char* who = "ud_qk_norm_rope_append";
    int rc = paged_check(who, kv_format, k_pages, v_pages, num_blocks, block_table, n, max_blocks, kv_heads, head_dim, block_size);
    if (rc != UD_OK) return rc;
    // a launch holds fewer than 2^32 threads
    if (rows < 0 || rows > (1 << 23) || q_heads < 0 || q_heads > 65535)
        return paged_fail(UD_ERR_SHAPE, "%s: rows %d (at most 2^23), q_heads %d", who, rows, q_heads);
    if (rows == 0) return UD_OK;
    if (!k_dev || !v_dev || !positions_dev || (q_heads && (!q_dev || !q_out_dev))) return paged_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if (dtype != UD_F32 && dtype != UD_BF16 && dtype != UD_F16) return paged_fail(UD_ERR_INVALID, "%s: dtype %d", who, dtype);
    if (kv_format != UD_MXFP4 && dtype != UD_F32 && dtype != kv_format)
        return paged_fail(UD_ERR_INVALID, "%s: rows of dtype %d for pages of format %d (the same, or fp32 rows, or MXFP4 pages)", who, dtype, kv_format);
    if (!(eps >= 0.0f)) return paged_fail(UD_ERR_INVALID, "%s: eps %g", who, (double)eps);
    const int64_t qw = (int64_t)q_heads * head_dim, kw = (int64_t)kv_heads * head_dim;
    if (k_ld < kw || v_ld < kw || (q_heads && (q_ld < qw || q_out_ld < qw)))
        return paged_fail(UD_ERR_SHAPE, "%s: rows of %d/%d/%d/%d elements for %d/%d heads of %d", who, q_ld, k_ld, v_ld, q_out_ld, q_heads, kv_heads, head_dim);
    // a lane's four elements are one load: 16 bytes of fp32, 8 of 16 bits
    const uintptr_t piece = dtype == UD_F32 ? 15 : 7;
    uintptr_t at = (uintptr_t)k_dev | (uintptr_t)v_dev;
    int32_t lds = k_ld | v_ld;
    if (q_heads) { at |= (uintptr_t)q_dev | (uintptr_t)q_out_dev; lds |= q_ld | q_out_ld; }
    if ((at & piece) || (lds & 3)) return paged_fail(UD_ERR_INVALID, "%s: rows must be aligned to four elements", who);
    // a row's heads are read by one part of a workgroup and written by another
    const int64_t size = dtype == UD_F32 ? 4 : 2;
    if (q_heads && ((!(q_out_dev == q_dev && (q_out_ld == q_ld || rows == 1)) && rows_overlap(q_out_dev, q_out_ld, qw, q_dev, q_ld, qw, rows, size)) ||
                    rows_overlap(q_out_dev, q_out_ld, qw, k_dev, k_ld, kw, rows, size) || rows_overlap(q_out_dev, q_out_ld, qw, v_dev, v_ld, kw, rows, size)))
        return paged_fail(UD_ERR_INVALID, "%s: q_out overlaps k, v or q (it may be q, at the same distance between rows)", who);
    AppendArgs a{};
    a.q = q_dev; a.k = k_dev; a.v = v_dev; a.q_out = q_out_dev;
    a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld; a.qo_ld = q_out_ld;
    a.qw = q_weight_dev; a.kw = k_weight_dev; a.eps = eps; a.inv_freq = inv_freq_dev;
    a.pos = positions_dev; a.seqs = seqs_dev;
    a.kp = static_cast<char*>(k_pages); a.vp = static_cast<char*>(v_pages); a.bt = block_table;
    a.n = n; a.max_blocks = max_blocks; a.num_blocks = num_blocks; a.Hq = q_heads; a.Hkv = kv_heads;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (kv_format == UD_BF16) {
        if (dtype == UD_F32) launch_append<El32, FMT_BF16>(a, rows, head_dim, st);
        else launch_append<ElBf, FMT_BF16>(a, rows, head_dim, st);
    } else if (kv_format == UD_F16) {
        if (dtype == UD_F32) launch_append<El32, FMT_F16>(a, rows, head_dim, st);
        else launch_append<ElH, FMT_F16>(a, rows, head_dim, st);
    } else {
        if (dtype == UD_F32) launch_append<El32, FMT_FP4>(a, rows, head_dim, st);
        else if (dtype == UD_BF16) launch_append<ElBf, FMT_FP4>(a, rows, head_dim, st);
        else launch_append<ElH, FMT_FP4>(a, rows, head_dim, st);
    }
    return paged_launched(who);
}

extern "C" UD_API int ud_paged_kv_read(int32_t kv_format, int32_t dtype, const void* k_pages, const void* v_pages, int32_t num_blocks,
                                       const int32_t* block_table, int32_t n, int32_t max_blocks, const int32_t* positions_dev,
                                       const int32_t* seqs_dev, void* k_out, void* v_out, int32_t rows, int32_t kv_heads,
                                       int32_t head_dim, int32_t block_size, void* hip_stream) {
    static const char* who = "ud_paged_kv_read";
    int rc = paged_check(who, kv_format, k_pages, v_pages, num_blocks, block_table, n, max_blocks, kv_heads, head_dim, block_size);
    if (rc != UD_OK) return rc;
    if (rows < 0 || (int64_t)rows * kv_heads * (head_dim / 8) > (int64_t)1 << 31)
        return paged_fail(UD_ERR_SHAPE, "%s: rows %d of %d heads (2^34 elements at most)", who, rows, kv_heads);
    if (rows == 0) return UD_OK;
    if (!positions_dev || !k_out || !v_out) return paged_fail(UD_ERR_INVALID, "%s: null pointer", who);
    if (dtype != UD_F32 && dtype != (kv_format == UD_MXFP4 ? (int32_t)UD_BF16 : kv_format))
        return paged_fail(UD_ERR_INVALID, "%s: rows of dtype %d from pages of format %d (fp32, the pages' own, bf16 from MXFP4)", who, dtype, kv_format);
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return paged_fail(UD_ERR_INVALID, "%s: outputs must be 16-byte aligned", who);
    const ReadArgs a{static_cast<const char*>(k_pages), static_cast<const char*>(v_pages), block_table, positions_dev, seqs_dev,
                     k_out, v_out, n, max_blocks, num_blocks, kv_heads};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (kv_format == UD_BF16) {
        if (dtype == UD_F32) launch_read<El32, FMT_BF16>(a, rows, head_dim, st);
        else launch_read<ElBf, FMT_BF16>(a, rows, head_dim, st);
    } else if (kv_format == UD_F16) {
        if (dtype == UD_F32) launch_read<El32, FMT_F16>(a, rows, head_dim, st);
        else launch_read<ElH, FMT_F16>(a, rows, head_dim, st);
    } else {
        if (dtype == UD_F32) launch_read<El32, FMT_FP4>(a, rows, head_dim, st);
        else launch_read<ElBf, FMT_FP4>(a, rows, head_dim, st);
    }
    return paged_launched(who);
}
