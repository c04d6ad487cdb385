// swat_amd/csrc/mx_wgrad.hip — the weight gradient of a linear layer whose input was kept as an 8-bit checkpoint:
//
//   dW[n, k] = sum_m dY[m, n] X8[m, k],   db[n] = sum_m dY[m, n]
//
// dY bfloat16, X8 e4m3 with a power-of-two scale to 32 columns.  An e4m3 number times such a scale is a bfloat16 number, so the
// checkpoint is unpacked on its way into LDS without a rounding and v_mfma_f32_16x16x32_bf16 sees what was stored.  The reduction
// runs over rows: both tiles lie [64 rows][columns] in LDS and are read with the transposing LDS load.
//
// 16448 rows, 4096 x 1024: 147 us call after call (940 TFLOP/s; kernel 139, join 8; the first twenty calls after a pause take 187 each, while the
// clocks rise), the same gradient from a bf16 input, without db, 153 with the GEMM kernels of gemm_*.hip, the large bf16 library product 1 425 TFLOP/s.  By
// counter a CU's matrix pipes work 43 % of the time, its LDS 37, its vector units 30: no unit is the bound, the turns they take are.  A wave's
// 64 x 64 and 8 waves to a CU leave one other wave to a SIMD to cover LDS reads, LDS writes and the unpacking; wider wave tiles spilled.
// The long side of the tile goes to X because its codes are half as many bytes: 32 KB instead of 40 from memory for the same products.
#include <math.h>
#include "gemm_device.hpp"
#include "mx_device.hpp"
#include "../../include/swat_hip.h"

namespace swat {

typedef unsigned mx_u4 __attribute__((ext_vector_type(4)));

struct MxWgradArgs {
    const unsigned short* dY;
    const unsigned char *X, *S;
    float *dW, *db;     // or the partial planes of a split reduction
    int64_t rows, ld;   // rows; row stride of dY
    int n, k, blocks;
    int tiles_n, tiles_k, splits, tiles_per_split;   // 64-row tiles to a split
};

// A workgroup computes BN x BK of dW over its share of the rows; waves of WN x WK.  64 rows at a time: both operands go through
// registers into one of two LDS buffers ([64 rows][columns], 16-byte chunks permuted so that neither the writes nor the transposing
// reads meet in a bank) while the matrix cores work on the other; the global loads run a whole tile ahead.  GROUPS of such waves share the
// rows where there are few tiles of dW (one workgroup to a CU waits for a tile's latency: 0.43 us, two 0.27 each); their sums meet in LDS,
// the first group's first.
template <int BN, int BK, int WN, int WK, int GROUPS>
__global__ __launch_bounds__((BN / WN) * (BK / WK) * 64 * GROUPS, 2) void mx_wgrad_kernel(MxWgradArgs p) {
    constexpr int NT = (BN / WN) * (BK / WK) * 64, FN = WN / 16, FK = WK / 16;
    constexpr int YB = 64 * BN * 2, XB = 64 * BK * 2;
    constexpr int YC = 64 * BN / 8 / NT, XC = 64 * BK / 16 / NT;   // chunks to a thread: 8 columns of dY, 16 of X
    static_assert(YC * NT * 8 == 64 * BN && XC * NT * 16 == 64 * BK, "whole chunks");
    __shared__ __attribute__((aligned(1024))) unsigned char shared[GROUPS * 2 * (YB + XB)];
    const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0, tid = threadIdx.x - group * NT, lane = tid & 63, wave = tid >> 6;
    unsigned char* const smem = shared + group * 2 * (YB + XB);
    const int r16 = lane & 15, g = lane >> 4, wr = wave / (BK / WK), wc = wave % (BK / WK);
    // units of one XCD (workgroups b, b + 8, ..) are neighbours: the same rows, 4 k tiles wide, so that its L2 sees few panels of dY and X
    int id;
    {
        const int total = gridDim.x, xcd = blockIdx.x & 7, q = total >> 3, r = total & 7;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (blockIdx.x >> 3);
    }
    const int tiles = p.tiles_n * p.tiles_k, split = id / tiles, in = id - split * tiles;
    const int band = in / (4 * p.tiles_n), wide = p.tiles_k - 4 * band < 4 ? p.tiles_k - 4 * band : 4;
    const int tk = 4 * band + (in - 4 * band * p.tiles_n) % wide, tn = (in - 4 * band * p.tiles_n) / wide;
    const int n0 = tn * BN, k0 = tk * BK;
    // this split's tiles, the same number to a group (those behind the last row, and behind the split's, are empty)
    const int64_t s0 = (int64_t)split * p.tiles_per_split, all = (p.rows + 63) / 64;
    const int whole = (int)(s0 + p.tiles_per_split < all ? p.tiles_per_split : all > s0 ? all - s0 : 0), nt = (whole + GROUPS - 1) / GROUPS;
    const int64_t t0 = s0 + group * nt, end_tile = t0 + nt < s0 + whole ? t0 + nt : s0 + whole, end = end_tile * 64 < p.rows ? end_tile * 64 : p.rows;

    // Global loads go through buffer descriptors that end with the matrix: rows past the last one read as zeros, columns past the edge get
    // an offset past the end.  dY may sit on any 2 bytes; the range check is by whole dwords, so with an odd n the matrix's very last
    // element reads as zero too: its products are added at the end.  A thread's offsets inside a tile are constant, the tile's base advances in scalar registers.
    struct Stage {
        mx_u4 y[YC], x[XC];
        unsigned char s[XC];
    };
    Stage st0, st1;
    float cs[8];   // this thread's 8 columns of dY, summed over its rows (at % (BN / 8) is the same for all its chunks)
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = 0.f;
    const bool sums = p.db && tk == 0;
    const int xld = 32 * p.blocks;
    constexpr unsigned OUT = 0x80000000u;
    // (a thread's chunks are YR (XR) rows apart, multiples of 16: the permutation of 16-byte chunks in LDS is the same for all of them)
    constexpr int YR = NT / (BN / 8), XR = NT / (BK / 16), YW = BN >= 128 ? 256 : 2 * BN, XW = BK >= 128 ? 256 : 2 * BK;
    static_assert(YR % 16 == 0 && XR % 16 == 0, "rows between a thread's chunks");
    const int yrow = tid / (BN / 8), ycol = n0 + 8 * (tid % (BN / 8)), xrow = tid / (BK / 16), xcol = k0 + 16 * (tid % (BK / 16));
    const unsigned oy = ycol < p.n ? 2u * (unsigned)(yrow * (int)p.ld + ycol) : OUT, ox = xcol < xld ? (unsigned)(xrow * xld + xcol) : OUT;
    const unsigned os = xcol < xld ? (unsigned)(xrow * p.blocks + (xcol >> 5)) : OUT;
    unsigned char *const wy = smem + stp_off<BN>(yrow, ycol - n0), *const wx = smem + 2 * YB + stp_off<BK>(xrow, xcol - k0);
    auto load = [&](Stage& st, int t) {
        const int64_t m0 = (t0 + t) * 64 < end ? (t0 + t) * 64 : end, left = end - m0;
        const int rows = left < 64 ? (int)left : 64;   // (a tile with rows behind it: one element more, its last dword may reach into the next)
        const bool behind = p.rows - m0 > 64;
        const __amdgpu_buffer_rsrc_t by = __builtin_amdgcn_make_buffer_rsrc((void*)(p.dY + m0 * p.ld), 0,
                                                                             !rows ? 0 : behind ? 128 * (int)p.ld + 2 : 2 * ((rows - 1) * (int)p.ld + p.n), 0x20000);
        const __amdgpu_buffer_rsrc_t bx = __builtin_amdgcn_make_buffer_rsrc((void*)(p.X + m0 * xld), 0, rows * xld, 0x20000);
        const __amdgpu_buffer_rsrc_t bs = __builtin_amdgcn_make_buffer_rsrc((void*)(p.S + m0 * p.blocks), 0, rows * p.blocks, 0x20000);
#pragma unroll
        for (int i = 0; i < YC; ++i) {
            st.y[i] = __builtin_amdgcn_raw_buffer_load_b128(by, oy + 2u * (unsigned)(i * YR * (int)p.ld), 0, 0);
        }
#pragma unroll
        for (int i = 0; i < XC; ++i) {
            st.x[i] = __builtin_amdgcn_raw_buffer_load_b128(bx, ox + (unsigned)(i * XR * xld), 0, 0);
            st.s[i] = __builtin_amdgcn_raw_buffer_load_b8(bs, os + (unsigned)(i * XR * p.blocks), 0, 0);
        }
    };
    auto put = [&](Stage& st, int buf, bool mine) {
#pragma unroll
        for (int i = 0; i < YC; ++i) *reinterpret_cast<mx_u4*>(wy + buf * YB + i * YR * YW) = st.y[i];
        if (mine) {
#pragma unroll
            for (int i = 0; i < YC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    cs[2 * e] += __uint_as_float(st.y[i][e] << 16);
                    cs[2 * e + 1] += __uint_as_float(st.y[i][e] & 0xffff0000u);
                }
        }
#pragma unroll
        for (int i = 0; i < XC; ++i) {
            const float s = mx_scale(st.s[i]);
            unsigned w[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {   // exact: an e4m3 number times a power of two of at least 2^-110
                w[2 * e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(st.x[i][e], s, false));
                w[2 * e + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(st.x[i][e], s, true));
            }
            // (a quarter wave covers 256 bytes in two writes: lanes 4 .. 7 of each eight write their second half first, so that eight
            // lanes meet all banks once)
            const bool late = tid & 4;
            *reinterpret_cast<mx_u4*>(wx + buf * XB + i * XR * XW + (late ? 16 : 0)) =
                late ? (mx_u4){w[4], w[5], w[6], w[7]} : (mx_u4){w[0], w[1], w[2], w[3]};
            *reinterpret_cast<mx_u4*>(wx + buf * XB + i * XR * XW + (late ? 0 : 16)) =
                late ? (mx_u4){w[0], w[1], w[2], w[3]} : (mx_u4){w[4], w[5], w[6], w[7]};
        }
    };
    auto bar = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // fragment of 8 rows of one column: lane (r16, g) of the 32-row half ks gets rows 32 ks + 8 g + 0 .. 7 of column base + r16
    auto frag = [&](const unsigned char* lo, int row_bytes) {
        const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(lo));
        const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(lo + 4 * row_bytes));
        const s16x8_t v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return __builtin_bit_cast(bf16x8_t, v);
    };

    f32x4_t acc[FN][FK];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FK; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

    struct Frags {
        bf16x8_t x[FK], y[FN];
    };
    Frags f0, f1;   // of the two 32-row halves of a tile
    // (the permutation depends on the low four bits of the row with bit 2 left out: rows + 4 and + 32 are at constant distances)
    const unsigned char *rx[FK], *ry[FN];
#pragma unroll
    for (int j = 0; j < FK; ++j) rx[j] = smem + 2 * YB + 8 * (r16 & 3) + stp_off<BK>(8 * g + (r16 >> 2), WK * wc + 16 * j);
#pragma unroll
    for (int i = 0; i < FN; ++i) ry[i] = smem + 8 * (r16 & 3) + stp_off<BN>(8 * g + (r16 >> 2), WN * wr + 16 * i);
    auto read = [&](Frags& f, int buf, int ks) {
#pragma unroll
        for (int j = 0; j < FK; ++j) f.x[j] = frag(rx[j] + buf * XB + ks * 32 * XW, XW);
#pragma unroll
        for (int i = 0; i < FN; ++i) f.y[i] = frag(ry[i] + buf * YB + ks * 32 * YW, YW);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](Frags& f) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FK; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.x[j], f.y[i], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // One barrier to a tile: a half's fragments are read while the matrix cores work on the half before; tile t + 1 goes into the other
    // buffer in between (whose last reads were waited for at the barrier before), t + 2 and t + 3 are on their way from memory.
    // Nothing in the loop is conditional (tiles past this split's last one are loaded, and past the matrix read as zeros, but not
    // multiplied): the waits for the loads stay exact.
    auto step = [&](Stage& st, int buf, int t) {
        read(f1, buf, 1);
        multiply(f0);
        put(st, buf ^ 1, sums && t + 1 < nt);
        load(st, t + 3);
        bar();
        read(f0, buf ^ 1, 0);
        multiply(f1);
    };
    load(st0, 0);
    load(st1, 1);
    put(st0, 0, sums && nt > 0);
    load(st0, 2);
    bar();
    read(f0, 0, 0);
    int t = 0;
    for (; t + 1 < nt; t += 2) {
        step(st1, 0, t);
        step(st0, 1, t + 1);
    }
    if (t < nt) {
        read(f1, 0, 1);
        multiply(f0);
        multiply(f1);
    }
    bar();
    const bool odd_end = (p.n & 1) && end == p.rows && t0 * 64 < end;   // (see the loads)
    if (sums) {   // the threads that share 8 columns meet in LDS (tiles are done with it), rows of threads added in order
        float* cp = reinterpret_cast<float*>(shared);
#pragma unroll
        for (int e = 0; e < 8; ++e) cp[((int)threadIdx.x / (BN / 8)) * BN + 8 * (tid % (BN / 8)) + e] = cs[e];
        bar();
        for (int c = threadIdx.x; c < BN; c += GROUPS * NT)
            if (n0 + c < p.n) {
                float t = 0.f;
#pragma unroll
                for (int r = 0; r < GROUPS * NT / (BN / 8); ++r) t += cp[r * BN + c];
                if ((p.n & 1) && whole > 0 && s0 + whole == all && n0 + c == p.n - 1) t += bf2f(p.dY[(p.rows - 1) * p.ld + n0 + c]);
                p.db[(int64_t)split * p.n + n0 + c] = t;
            }
    }
    if (odd_end) {
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            if (n0 + WN * wr + 16 * i + r16 != p.n - 1) continue;
            const float y = bf2f(p.dY[(p.rows - 1) * p.ld + p.n - 1]);
#pragma unroll
            for (int j = 0; j < FK; ++j) {
                const int k = k0 + WK * wc + 16 * j + 4 * g;
                if (k >= xld) continue;
                float x[4];
                mx_from_e4m3x4(*reinterpret_cast<const unsigned*>(p.X + (p.rows - 1) * xld + k), mx_scale(p.S[(p.rows - 1) * p.blocks + (k >> 5)]), x);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(y, x[e], acc[i][j][e]);
            }
        }
    }
    if constexpr (GROUPS > 1) {
        static_assert(GROUPS == 2 && FN * FK * NT * 16 <= 4 * (YB + XB), "one sum in LDS");
        if (sums) bar();
        f32x4_t* const other = reinterpret_cast<f32x4_t*>(shared);
        if (group)
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FK; ++j) other[(i * FK + j) * NT + tid] = acc[i][j];
        bar();
        if (group) return;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FK; ++j) acc[i][j] += other[(i * FK + j) * NT + tid];
    }
    float* dW = p.dW + (int64_t)split * p.n * p.k;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const int n = n0 + WN * wr + 16 * i + r16;
        if (n >= p.n) continue;
#pragma unroll
        for (int j = 0; j < FK; ++j) {
            const int k = k0 + WK * wc + 16 * j + 4 * g;
            float* out = dW + (int64_t)n * p.k + k;
            if (p.k % 4 == 0) {
                if (k < p.k) *reinterpret_cast<float4*>(out) = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k + e < p.k) out[e] = acc[i][j][e];
            }
        }
    }
}

// the planes of a split reduction, added in their order, eight loads under way at a time: dW's in the first w_blocks workgroups, db's (behind
// dW's in the workspace) in the others.  Four neighbours to a thread at any alignment; the last four of a count that is no multiple of 4
// are made twice, to the same values.  (Element by element with a load at a time: 6980 x 32 x 35 16.5 us in all instead of 10.)
typedef float mx_f4 __attribute__((ext_vector_type(4), aligned(4)));
__global__ __launch_bounds__(256) void mx_wgrad_join_kernel(const float* pw, const float* pb, float* dW, float* db, int64_t nk, int n, int splits, int w_blocks) {
    const bool w = (int)blockIdx.x < w_blocks;
    const float* from = w ? pw : pb;
    float* const to = w ? dW : db;
    const int64_t count = w ? nk : n;
    int64_t at = ((int64_t)(w ? (int)blockIdx.x : (int)blockIdx.x - w_blocks) * 256 + threadIdx.x) * 4;
    if (at >= count) return;
    if (count < 4) {
        for (int e = 0; e < count; ++e) {
            float s = from[e];
            for (int i = 1; i < splits; ++i) s += from[i * count + e];
            to[e] = s;
        }
        return;
    }
    if (at + 4 > count) at = count - 4;
    mx_f4 s = *reinterpret_cast<const mx_f4*>(from + at);
#pragma unroll 8
    for (int i = 1; i < splits; ++i) s += *reinterpret_cast<const mx_f4*>(from + i * count + at);
    *reinterpret_cast<mx_f4*>(to + at) = s;
}

struct MxWgradPlan {
    int form;   // 0: 64 x 64, 1: 128 x 256, 2: 64 x 64 in two groups
    int tiles_n, tiles_k, splits, per;
};
// 128 x 256 tiles (8 waves, one workgroup to a CU), 64 x 64 (4 waves, up to four) or, while those are one to a CU, 64 x 64 in two groups of
// waves, and into how many parts the rows are split, by the sum of what was measured (us): a 64-row tile takes 1.02 in the first form, 0.43
// in the second alone on its CU and 0.27 for each of several; 6.5 / 3 to start and to store; a join of up to 32 parts 3.2 and its planes' bytes at 4.5
// TB/s.  At 16448 rows, 4096 x 1024: 150 in the first form with 2 parts (259 with 1, 157 with 4), 240 in the second; at 1600 rows,
// 768 x 768: 12.5 in two groups, 15 in one (3 parts 14.5), 21.4 in the first; 6304 rows: 47.8 in one part, 26.8 in 3.
static MxWgradPlan mx_wgrad_plan(int64_t rows, int n, int k) {
    const int64_t all = (rows + 63) / 64;
    MxWgradPlan best = {};
    double cost = -1;
    for (int form = 0; form < 3; ++form) {
        const bool big = form == 1;
        const int bn = big ? 128 : 64, bk = big ? 256 : 64;
        MxWgradPlan p = {form, (n + bn - 1) / bn, (k + bk - 1) / bk, 1, 1};
        for (int s = 1; s <= 32 && (s == 1 || s <= all); ++s) {
            p.per = all > 0 ? (int)((all + s - 1) / s) : 1;
            p.splits = all > 0 ? (int)((all + p.per - 1) / p.per) : 1;
            if (p.splits != s) continue;
            const double units = (double)p.tiles_n * p.tiles_k * s, rounds = ceil(units / (big ? 256 : 1024));
            if (form == 2 && units > 256) continue;
            const double at_once = units > 1024 ? 4 : ceil(units / 256);
            const double tile = big ? 1.02 : form == 2 ? 0.27 : at_once < 2 ? 0.43 : (at_once < 3 ? 0.27 : 0.32) * at_once;
            const double c = (big ? 6.5 : form == 2 ? 4.5 : 3.0) + rounds * p.per * tile + (s > 1 ? 3.2 + (1.5 * s + 1.0) * n * k * 4 / 4.5e6 : 0.0);
            if (cost < 0 || c < cost) {
                cost = c;
                best = p;
            }
        }
    }
    return best;
}

}  // namespace swat

using namespace swat;

SWAT_API int64_t swat_mx_linear_wgrad_workspace_bytes(int64_t rows, int n_out, int n_in) {
    if (rows < 0 || rows >= (1ll << 36) || n_out < 0 || n_in < 1 || n_out > (1 << 23) || n_in > (1 << 24)) {
        set_error("swat_mx_linear_wgrad_workspace_bytes: %lld rows, %d x %d", (long long)rows, n_out, n_in);
        return -1;
    }
    const MxWgradPlan p = mx_wgrad_plan(rows, n_out, n_in);
    return p.splits > 1 ? 4 * (int64_t)p.splits * n_out * ((int64_t)n_in + 1) : 0;
}

SWAT_API int swat_mx_linear_wgrad(const void* dY_bf16, int64_t dy_stride, const void* x_codes, const void* x_scales, float* dW, float* dbias,
                                  int64_t rows, int n_out, int n_in, void* workspace, int64_t workspace_bytes, swat_stream_t stream) {
    SWAT_REQUIRE(rows >= 0 && rows < (1ll << 36) && n_out >= 0 && n_in >= 1 && n_out <= (1 << 23) && n_in <= (1 << 24), "swat_mx_linear_wgrad: %lld rows, %d x %d", (long long)rows, n_out, n_in);
    if (n_out == 0) return 0;
    SWAT_REQUIRE(dW && (rows == 0 || (dY_bf16 && x_codes && x_scales)), "swat_mx_linear_wgrad: dY, the checkpoint and dW are needed");
    SWAT_REQUIRE(rows == 0 || dy_stride >= n_out, "swat_mx_linear_wgrad: row stride %lld under %d columns", (long long)dy_stride, n_out);
    SWAT_REQUIRE(rows == 0 || dy_stride <= (1 << 23), "swat_mx_linear_wgrad: row stride %lld past 2^23", (long long)dy_stride);
    SWAT_REQUIRE(!(((uintptr_t)x_codes | (uintptr_t)dW) & 15), "swat_mx_linear_wgrad: codes and dW sit on 16 bytes");
    const MxWgradPlan pl = mx_wgrad_plan(rows, n_out, n_in);
    const int64_t grid = (int64_t)pl.tiles_n * pl.tiles_k * pl.splits, nk = (int64_t)n_out * n_in;
    SWAT_REQUIRE(grid < (1ll << 23) && nk < (1ll << 34), "swat_mx_linear_wgrad: %d x %d is past one launch", n_out, n_in);
    const int64_t want = swat_mx_linear_wgrad_workspace_bytes(rows, n_out, n_in);
    SWAT_REQUIRE(want == 0 || (workspace && workspace_bytes >= want && ((uintptr_t)workspace & 15) == 0),
                 "swat_mx_linear_wgrad: workspace of %lld bytes, %lld on 16 bytes are needed", (long long)workspace_bytes, (long long)want);
    const hipStream_t s = (hipStream_t)stream;
    float *pw = dW, *pb = dbias;
    if (pl.splits > 1) {
        pw = (float*)workspace;
        pb = dbias ? pw + pl.splits * nk : nullptr;
    }
    MxWgradArgs p = {};
    p.dY = (const unsigned short*)dY_bf16; p.X = (const unsigned char*)x_codes; p.S = (const unsigned char*)x_scales; p.dW = pw; p.db = pb;
    p.rows = rows; p.ld = dy_stride; p.n = n_out; p.k = n_in; p.blocks = (n_in + 31) / 32;
    p.tiles_n = pl.tiles_n; p.tiles_k = pl.tiles_k; p.splits = pl.splits; p.tiles_per_split = pl.per;
    if (pl.form == 1) mx_wgrad_kernel<128, 256, 64, 64, 1><<<(unsigned)grid, 512, 0, s>>>(p);
    else if (pl.form == 2) mx_wgrad_kernel<64, 64, 32, 32, 2><<<(unsigned)grid, 512, 0, s>>>(p);
    else mx_wgrad_kernel<64, 64, 32, 32, 1><<<(unsigned)grid, 256, 0, s>>>(p);
    if (pl.splits > 1) {
        const int64_t w_blocks = (nk + 1023) / 1024, b_blocks = dbias ? (n_out + 1023) / 1024 : 0;
        mx_wgrad_join_kernel<<<(unsigned)(w_blocks + b_blocks), 256, 0, s>>>(pw, pb, dW, dbias, nk, n_out, pl.splits, (int)w_blocks);
    }
    return check_launch("swat_mx_linear_wgrad");
}
