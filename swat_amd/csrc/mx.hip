// swat_amd/csrc/mx.hip — packing and unpacking microscaled matrices, and the activation of an MLP with its 8-bit checkpoint.
//
//   quantize      x [rows, n] -> codes, scale bytes                  dequantize   back to values
//   act_fwd       g = act(f) and the 8-bit checkpoint of f, f read once
//   act_bwd       df = dg act'(f8) and act(f8) again (the operand of the next layer's weight gradient), f8 read once
//
// Storage: codes [rows, n rounded up to 32] (8 bits) or half of that (4 bits, the even column in the low half), scales
// [rows, blocks of 32]; the columns behind n hold zeros, so every row starts on 32 (16) bytes and products need no edge along them.
//
// All but GELU's forward (see mx_act) are bound by bytes: 8224 x 4096 QuickGELU with its checkpoint 27.5 us (6.1 TB/s), back 39 (6.0);
// 16448 x 1024 fp32 to 4 bits 13.4 us (5.7), back 14.6 (5.2; a large copy 4.95).  A thread takes 8 neighbouring columns (16 bytes of
// bfloat16, 8 or 4 of codes), four lanes make a block and agree on its scale by two lane exchanges.
#include "gemm_device.hpp"
#include "mx_device.hpp"
#include "../../include/swat_hip.h"

namespace swat {

// chunks of 8 columns, a multiple of 4 to a row; a thread takes one
struct MxMap {
    int64_t rows;
    int n, blocks;        // columns; blocks of 32 to a row
    int64_t ld;           // row stride of the values read (elements)
    unsigned mul;         // chunk / chunks per row = chunk mul >> 32 >> shift (chunk < 2^31)
    int shift;
};

// vectors at any element's address (rows of odd widths)
typedef unsigned mx_u4h __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned mx_u4f __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool mx_place(const MxMap& m, int64_t& row, int& col) {
    const unsigned cpr = 4u * (unsigned)m.blocks;
    const int64_t idx = mx_block() * 256 + threadIdx.x;
    if (idx < 0x7fffffff) {
        const unsigned i = (unsigned)idx, r = __umulhi(i, m.mul) >> m.shift;
        row = r;
        col = (int)(i - r * cpr) * 8;
    } else {
        row = idx / cpr;
        col = (int)(idx - row * cpr) * 8;
    }
    return row < m.rows;
}

// (read once by a call: non-temporal, the caches are left to what is written and to the packed form)
__device__ __forceinline__ void mx_load8(const void* p, int bf, int64_t at, int left, float (&v)[8]) {
    if (left >= 8) {
        if (bf) {
            const mx_u4h u = __builtin_nontemporal_load(reinterpret_cast<const mx_u4h*>(reinterpret_cast<const unsigned short*>(p) + at));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        } else {
            const mx_u4f a = __builtin_nontemporal_load(reinterpret_cast<const mx_u4f*>(reinterpret_cast<const float*>(p) + at));
            const mx_u4f b = __builtin_nontemporal_load(reinterpret_cast<const mx_u4f*>(reinterpret_cast<const float*>(p) + at + 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __uint_as_float(a[i]);
                v[4 + i] = __uint_as_float(b[i]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i >= left ? 0.f : bf ? bf2f(reinterpret_cast<const unsigned short*>(p)[at + i]) : reinterpret_cast<const float*>(p)[at + i];
}
__device__ __forceinline__ void mx_store8(void* p, int bf, int64_t at, int left, const float (&v)[8]) {
    if (left >= 8) {
        if (bf) {
            *reinterpret_cast<mx_u4h*>(reinterpret_cast<unsigned short*>(p) + at) =
                (mx_u4h){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
        } else {
            mx_u4f a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = __float_as_uint(v[i]);
                b[i] = __float_as_uint(v[4 + i]);
            }
            *reinterpret_cast<mx_u4f*>(reinterpret_cast<float*>(p) + at) = a;
            *reinterpret_cast<mx_u4f*>(reinterpret_cast<float*>(p) + at + 4) = b;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) {
            if (bf) reinterpret_cast<unsigned short*>(p)[at + i] = f2bf(v[i]);
            else reinterpret_cast<float*>(p)[at + i] = v[i];
        }
}

// the block's four lanes are neighbours and live or die together (chunks per row is a multiple of 4)
template <int BITS>
__device__ __forceinline__ void mx_pack8(const float (&v)[8], int64_t row, int col, const MxMap& m, unsigned char* codes, unsigned char* scales) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = mx_amax(top, v[i]);
    top = mx_amax(top, __shfl_xor(top, 1, 64));
    top = mx_amax(top, __shfl_xor(top, 2, 64));
    const int sb = mx_scale_byte<BITS>(top);
    const float inv = mx_inverse(sb);
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = v[i] * inv;
    if constexpr (BITS == 8) {
        uint2 c = make_uint2(mx_e4m3x4(t[0], t[1], t[2], t[3]), mx_e4m3x4(t[4], t[5], t[6], t[7]));
        if (sb == 255) c = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
        *reinterpret_cast<uint2*>(codes + row * (32 * (int64_t)m.blocks) + col) = c;
    } else {
        *reinterpret_cast<unsigned*>(codes + row * (16 * (int64_t)m.blocks) + col / 2) = sb == 255 ? 0u : mx_e2m1x8(t);
    }
    if (col % 32 == 0) scales[row * m.blocks + col / 32] = (unsigned char)sb;
}

template <int BITS>
__device__ __forceinline__ void mx_unpack8(const unsigned char* codes, const unsigned char* scales, int64_t row, int col, const MxMap& m, float (&v)[8]) {
    const float s = mx_scale(scales[row * m.blocks + col / 32]);
    if constexpr (BITS == 8) {
        const uint2 c = *reinterpret_cast<const uint2*>(codes + row * (32 * (int64_t)m.blocks) + col);
        mx_from_e4m3x4(c.x, s, v);
        mx_from_e4m3x4(c.y, s, v + 4);
    } else {
        mx_from_e2m1x8(*reinterpret_cast<const unsigned*>(codes + row * (16 * (int64_t)m.blocks) + col / 2), s, v);
    }
}

template <int BITS>
__global__ __launch_bounds__(256) void mx_quantize_kernel(MxMap m, const void* x, int bf, unsigned char* codes, unsigned char* scales) {
    int64_t row;
    int col;
    if (!mx_place(m, row, col)) return;
    float v[8];
    mx_load8(x, bf, row * m.ld + col, m.n - col, v);
    mx_pack8<BITS>(v, row, col, m, codes, scales);
}

template <int BITS>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxMap m, const unsigned char* codes, const unsigned char* scales, void* out, int bf) {
    int64_t row;
    int col;
    if (!mx_place(m, row, col) || col >= m.n) return;
    float v[8];
    mx_unpack8<BITS>(codes, scales, row, col, m, v);
    mx_store8(out, bf, row * m.n + col, m.n - col, v);
}

// act(x) and act'(x).  GELU: the normal distribution's tail is exp(-z^2) erfcx(z) / 2, z = |x| / sqrt 2, and erfcx(z) / 2 = t (c1 + c2 t + .. + c7 t^6),
// t = 1 / (1 + 0.512 z), with c fitted to the smallest largest RELATIVE error on 0 <= z <= 10 (a linear program): 7.7e-7, 1.1e-6 in fp32
// arithmetic, so that the tail's bfloat16 result is good to its half step down to where exp(-z^2) ends (x = -13).  Its exponential is the
// density's that the slope needs as well: one exponential and one reciprocal serve both.  8224 x 4096 there and back 73 us (105 with the
// library's erfc); the forward alone, call after call, 40 where QuickGELU takes 27.5: bound by arithmetic.
__device__ __forceinline__ void mx_act(float x, int act, float& value, float& slope) {
    if (act == 1) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-1.702f * x));
        value = x * s;
        slope = fmaf(value, 1.702f * (1.0f - s), s);   // (x s before the other factors: nothing overflows on its way to 0 or 1)
        return;
    }
    const float z = fabsf(x) * 0.70710678118654752f, e = __expf(-0.5f * x * x);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.512f, z, 1.0f));
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.0478386469f, -0.179616824f), 0.175997242f), 0.0292394273f), 0.139293984f),
                                             0.142730072f), 0.14451763f);
    const float tail = poly * e, cdf = x < 0.f ? tail : 1.0f - tail;
    value = x * cdf;
    slope = fmaf(x * 0.39894228040143268f, e, cdf);
}

__global__ __launch_bounds__(256) void mx_act_fwd_kernel(MxMap m, const unsigned short* f, int act, unsigned short* g, unsigned char* codes, unsigned char* scales) {
    int64_t row;
    int col;
    if (!mx_place(m, row, col)) return;
    float v[8], t[8];
    mx_load8(f, 1, row * m.ld + col, m.n - col, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float slope;
        mx_act(v[i], act, t[i], slope);
    }
    mx_store8(g, 1, row * m.n + col, m.n - col, t);
    mx_pack8<8>(v, row, col, m, codes, scales);
}

__global__ __launch_bounds__(256) void mx_act_bwd_kernel(MxMap m, const unsigned short* dg, const unsigned char* codes, const unsigned char* scales, int act,
                                                         unsigned short* df, unsigned short* again) {
    int64_t row;
    int col;
    if (!mx_place(m, row, col) || col >= m.n) return;
    float v[8], t[8];
    mx_load8(dg, 1, row * m.ld + col, m.n - col, t);
    mx_unpack8<8>(codes, scales, row, col, m, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float value, slope;
        // (what rounded up to 2^128 in the checkpoint was finite: taken just below, where no 0 times infinity arises)
        const float x = fabsf(v[i]) == INFINITY ? copysignf(3.4028234664e38f, v[i]) : v[i];
        mx_act(x, act, value, slope);
        t[i] *= slope;
        v[i] = value;
    }
    mx_store8(df, 1, row * m.n + col, m.n - col, t);
    if (again) mx_store8(again, 1, row * m.n + col, m.n - col, v);
}

static bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// columns of one row at most: 4 (n / 32) chunk indexes and 8 of them to a thread stay in 32 bits
static int mx_map(MxMap& m, int64_t rows, int n, int64_t ld, const char* what) {
    SWAT_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 24), "%s: %lld rows of %d columns (0 or more rows, 1 to 2^24 columns)", what, (long long)rows, n);
    SWAT_REQUIRE(ld >= n, "%s: row stride %lld under %d columns", what, (long long)ld, n);
    m.rows = rows;
    m.n = n;
    m.blocks = (n + 31) / 32;
    m.ld = ld;
    // s = ceil log2(chunks per row) and ceil(2^(31 + s) / chunks): the product is too large by under chunk 2^s, less than one step
    m.shift = 1;
    while ((2ll << m.shift) < 4ll * m.blocks) ++m.shift;
    m.mul = (unsigned)(((1ull << (32 + m.shift)) + 4ull * m.blocks - 1) / (4ull * m.blocks));
    SWAT_REQUIRE(rows * (4 * (int64_t)m.blocks) <= ((int64_t)1 << 39), "%s: %lld rows of %d columns are past one launch", what, (long long)rows, n);
    return 0;
}
static dim3 mx_grid(const MxMap& m) { return mx_grid2((m.rows * 4 * m.blocks + 255) / 256); }

}  // namespace swat

using namespace swat;

SWAT_API int swat_mx_quantize(const void* x, int64_t x_stride, int x_dtype, int bits, void* codes, void* scales, int64_t rows, int n,
                              swat_stream_t stream) {
    MxMap m;
    const int bf = x_dtype == SWAT_BF16;
    SWAT_REQUIRE(bits == 4 || bits == 8, "swat_mx_quantize: %d bits (4 or 8)", bits);
    if (const int rc = mx_map(m, rows, n, x_stride, "swat_mx_quantize")) return rc;
    if (rows == 0) return 0;
    SWAT_REQUIRE(x && codes && scales && on16(codes), "swat_mx_quantize: x, codes (on 16 bytes) and scales are needed");
    unsigned char *c = (unsigned char*)codes, *s = (unsigned char*)scales;
    if (bits == 8) mx_quantize_kernel<8><<<mx_grid(m), 256, 0, (hipStream_t)stream>>>(m, x, bf, c, s);
    else mx_quantize_kernel<4><<<mx_grid(m), 256, 0, (hipStream_t)stream>>>(m, x, bf, c, s);
    return check_launch("swat_mx_quantize");
}

SWAT_API int swat_mx_dequantize(const void* codes, const void* scales, int bits, void* out, int out_dtype, int64_t rows, int n,
                                swat_stream_t stream) {
    MxMap m;
    const int bf = out_dtype == SWAT_BF16;
    SWAT_REQUIRE(bits == 4 || bits == 8, "swat_mx_dequantize: %d bits (4 or 8)", bits);
    if (const int rc = mx_map(m, rows, n, n, "swat_mx_dequantize")) return rc;
    if (rows == 0) return 0;
    SWAT_REQUIRE(out && codes && scales && on16(codes), "swat_mx_dequantize: out, codes (on 16 bytes) and scales are needed");
    const unsigned char *c = (const unsigned char*)codes, *s = (const unsigned char*)scales;
    if (bits == 8) mx_dequantize_kernel<8><<<mx_grid(m), 256, 0, (hipStream_t)stream>>>(m, c, s, out, bf);
    else mx_dequantize_kernel<4><<<mx_grid(m), 256, 0, (hipStream_t)stream>>>(m, c, s, out, bf);
    return check_launch("swat_mx_dequantize");
}

SWAT_API int swat_mx_act_fwd(const void* f_bf16, int64_t f_stride, int act, void* g_bf16, void* codes, void* scales, int64_t rows, int n,
                             swat_stream_t stream) {
    MxMap m;
    SWAT_REQUIRE(act == 1 || act == 2, "swat_mx_act_fwd: activation %d (1 QuickGELU, 2 erf-GELU)", act);
    if (const int rc = mx_map(m, rows, n, f_stride, "swat_mx_act_fwd")) return rc;
    if (rows == 0) return 0;
    SWAT_REQUIRE(f_bf16 && g_bf16 && codes && scales && on16(codes), "swat_mx_act_fwd: f, g, codes (on 16 bytes) and scales are needed");
    mx_act_fwd_kernel<<<mx_grid(m), 256, 0, (hipStream_t)stream>>>(m, (const unsigned short*)f_bf16, act, (unsigned short*)g_bf16, (unsigned char*)codes, (unsigned char*)scales);
    return check_launch("swat_mx_act_fwd");
}

SWAT_API int swat_mx_act_bwd(const void* dg_bf16, int64_t dg_stride, const void* codes, const void* scales, int act, void* df_bf16, void* g_bf16,
                             int64_t rows, int n, swat_stream_t stream) {
    MxMap m;
    SWAT_REQUIRE(act == 1 || act == 2, "swat_mx_act_bwd: activation %d (1 QuickGELU, 2 erf-GELU)", act);
    if (const int rc = mx_map(m, rows, n, dg_stride, "swat_mx_act_bwd")) return rc;
    if (rows == 0) return 0;
    SWAT_REQUIRE(dg_bf16 && df_bf16 && codes && scales && on16(codes), "swat_mx_act_bwd: dg, df, codes (on 16 bytes) and scales are needed");
    mx_act_bwd_kernel<<<mx_grid(m), 256, 0, (hipStream_t)stream>>>(m, (const unsigned short*)dg_bf16, (const unsigned char*)codes, (const unsigned char*)scales, act,
                                                                   (unsigned short*)df_bf16, (unsigned short*)g_bf16);
    return check_launch("swat_mx_act_bwd");
}
