// swat_amd/csrc/mx_device.hpp — microscaled numbers: blocks of 32 columns of a row share a power of two, the elements are e4m3
// (8 bits, up to 448) or e2m1 (4 bits, up to 6).
//
// The scale of a block is the smallest power of two 2^E, E >= -110, with max |x| 2^-E <= the format's largest number: nothing
// saturates, and the largest element keeps the format's full precision or all but one bit of it.  E >= -110 keeps every held value
// a normal bfloat16 (the smallest e4m3 number is 2^-9), so unpacking is exact in bfloat16 and the matrix cores see what was stored.
// Byte E + 127; byte 255: the block held a NaN or an infinity and is NaN as a whole.  A matrix put together by hand may have bytes under
// 17: they mean what they say, but bfloat16 rounds such small values where they are unpacked to it.
#pragma once
#include "common.hpp"

namespace swat {

// One-dimensional work in as many workgroups as it takes: a launch holds fewer than 2^32 threads along x, the rest goes along y.  (A
// constant length along x: reading gridDim costs a kernel of one vector to a thread 6 %.)
static inline dim3 mx_grid2(int64_t blocks) {
    const int64_t x = blocks < (1 << 22) ? blocks : 1 << 22;
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ int64_t mx_block() { return ((int64_t)blockIdx.y << 22) + blockIdx.x; }

// running max |x| on raw bits: NaN and infinity win over every finite value
__device__ __forceinline__ float mx_amax(float top, float v) {
    const unsigned a = __float_as_uint(top), b = __float_as_uint(v) & 0x7fffffffu;
    return __uint_as_float(a > b ? a : b);
}
template <int BITS>
__device__ __forceinline__ int mx_scale_byte(float top) {
    const unsigned u = __float_as_uint(top);
    if (u >= 0x7f800000u) return 255;
    // 448 = 1.75 2^8, 6 = 1.5 2^2: one more where the mantissa is past the format's largest
    const int e = (int)(u >> 23) - 127 + (BITS == 8 ? -8 + ((u & 0x7fffffu) > 0x600000u) : -2 + ((u & 0x7fffffu) > 0x400000u));
    return (e < -110 ? -110 : e) + 127;
}
// (byte 0, which packing never writes: 2^-127, as the matrix instruction reads it, a subnormal float)
__device__ __forceinline__ float mx_scale(int byte) {
    const unsigned u = (unsigned)byte << 23;
    return byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(u > 0x400000u ? u : 0x400000u);
}
__device__ __forceinline__ float mx_inverse(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }  // 2^-E (byte < 255)

// four values to e4m3 / eight to e2m1, round to nearest even
__device__ __forceinline__ unsigned mx_e4m3x4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return (unsigned)r;
}
__device__ __forceinline__ unsigned mx_e2m1x8(const float (&v)[8]) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
    return r;
}
// four e4m3 / eight e2m1 codes times s
__device__ __forceinline__ void mx_from_e4m3x4(unsigned c, float s, float* v) {
    const swat_f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    v[0] = lo[0] * s; v[1] = lo[1] * s; v[2] = hi[0] * s; v[3] = hi[1] * s;
}
__device__ __forceinline__ void mx_from_e2m1x8(unsigned c, float s, float* v) {
    swat_f32x2_t t;
    t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0); v[0] = t[0] * s; v[1] = t[1] * s;
    t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1); v[2] = t[0] * s; v[3] = t[1] * s;
    t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2); v[4] = t[0] * s; v[5] = t[1] * s;
    t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3); v[6] = t[0] * s; v[7] = t[1] * s;
}

}  // namespace swat
