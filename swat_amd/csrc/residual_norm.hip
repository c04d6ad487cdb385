// swat_amd/csrc/residual_norm.hip — the seam between two sublayers of a transformer block as one kernel per direction:
//
//   p = Norm_post(h)  (or h);   m = gate * scale;   y = alpha x + m p;   z = Norm_pre(y)
//
// Norm: LayerNorm or root mean square, eps inside the root.  An element whose multiplier m is zero takes nothing from the branch
// (h is not looked at: a dropped row may hold anything).  z is the norm of the stream AS STORED, because the next sublayer's
// backward pass reads that y.
//
// A row lives in the registers of one team of W waves; both norms take their mean and their squared deviations from there, so
// every tensor crosses the memory bus once.  Bound by bytes in both directions.
#include <type_traits>
#include "kernels.hpp"
#include "mx_device.hpp"
#include "../../include/swat_hip.h"

namespace swat {

struct RnArgs {
    const void *x, *h, *dy, *dz, *yin;
    int64_t sx, sh, sdy, sdz, sy;           // row strides, elements
    int x_bf, h_bf, z_bf;                   // 1: bfloat16, 0: float32 (dz has z's type)
    const float *post_w, *post_b, *gate, *scale, *pre_w, *pre_b;
    int64_t rpg;                            // rows that share a gate
    int gate_mode;                          // 0 none, 1 a number per group, 2 a row of d per group
    int rms;
    float alpha, eps, inv_d;
    void *y, *z;                            // forward
    unsigned char *z8, *z8s;                // the packed z
    int z8_ld, z8s_ld;
    float* stats;                           // [4][rows]: mean, 1 / deviation of the post norm, of the pre norm
    void *dx, *dh;                          // backward
    float* part;                            // [blocks][RN_KINDS][d] column sums
    float* gate_rows;                       // [rows] (gate_mode 1) or [teams + groups][d] (gate_mode 2) partial gate gradients
    float* dgate;                           // written here when every row has its own gate
    int64_t groups;
    int rows, d, rows_per_team;
};

constexpr int RN_KINDS = 5;  // column sums of the backward pass: post_w, post_b, scale, pre_w, pre_b

template <int VEC>
__device__ __forceinline__ void rn_load(const void* p, int bf, int64_t at, float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        if (bf) {
            const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(p) + at);
            v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
            v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
        } else {
            const float4 f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        }
    } else {
        v[0] = bf ? bf2f(reinterpret_cast<const unsigned short*>(p)[at]) : reinterpret_cast<const float*>(p)[at];
    }
}

template <int VEC>
__device__ __forceinline__ void rn_store(void* p, int bf, int64_t at, const float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        if (bf) *reinterpret_cast<uint2*>(reinterpret_cast<unsigned short*>(p) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        if (bf) reinterpret_cast<unsigned short*>(p)[at] = f2bf(v[0]);
        else reinterpret_cast<float*>(p)[at] = v[0];
    }
}

// sums of N values over the team; sh: W * N floats of the team, two barriers around them (the trip count of the row loop is the
// same for every team of a workgroup when W > 1: one team is the whole workgroup)
template <int W, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* sh) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (W > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) sh[wave * N + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += sh[w * N + i];
            v[i] = s;
        }
        __syncthreads();
    }
}

// mean (layer) and 1 / deviation of a row held as v[NCH][VEC], columns c < d
template <int W, int NCH, int VEC>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][VEC], int c0, int d, const RnArgs& a, float* sh, float& mean, float& rstd) {
    mean = 0.f;
    if (!a.rms) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[0] += v[i][e];  // (columns past d hold zeros)
        team_sum<W>(s, sh);
        mean = s[0] * a.inv_d;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (c0 + i * (64 * W * VEC) < d) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = v[i][e] - mean;
                q[0] = fmaf(t, t, q[0]);
            }
        }
    team_sum<W>(q, sh);
    rstd = 1.0f / sqrtf(q[0] * a.inv_d + a.eps);
}

// W waves to a row, NCH chunks of VEC columns to a lane: rows of up to 64 W NCH VEC columns
template <int W, int NCH, int VEC>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void residual_norm_fwd_kernel(RnArgs a) {
    __shared__ float sh[W];
    const int lane = threadIdx.x & (64 * W - 1);
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= a.rows) return;
    const int d = a.d, c0 = lane * VEC;
    constexpr int STEP = 64 * W * VEC;
    float p[NCH][VEC], y[NCH][VEC];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = c0 + i * STEP;
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[i][e] = y[i][e] = 0.f;
        if (c < d) {
            rn_load<VEC>(a.h, a.h_bf, row * a.sh + c, p[i]);
            rn_load<VEC>(a.x, a.x_bf, row * a.sx + c, y[i]);
        }
    }
    float mean = 0.f, rstd = 1.f;
    if (a.post_w) {
        row_stats<W, NCH, VEC>(p, c0, d, a, sh, mean, rstd);
        if (a.stats && lane == 0) {
            a.stats[row] = mean;
            a.stats[a.rows + row] = rstd;
        }
    }
    const int64_t grp = a.gate_mode ? row / a.rpg : 0;
    const float g1 = a.gate_mode == 1 ? a.gate[grp] : 1.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = c0 + i * STEP;
        if (c >= d) continue;
        float t[VEC], m[VEC];
        if (a.post_w) {
            rn_load<VEC>(a.post_w, 0, c, t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) p[i][e] = (p[i][e] - mean) * rstd * t[e];
            if (a.post_b) {
                rn_load<VEC>(a.post_b, 0, c, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) p[i][e] += t[e];
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) m[e] = g1;
        if (a.gate_mode == 2) rn_load<VEC>(a.gate, 0, grp * d + c, m);
        if (a.scale) {
            rn_load<VEC>(a.scale, 0, c, t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) m[e] *= t[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[i][e] = m[e] == 0.f ? a.alpha * y[i][e] : fmaf(a.alpha, y[i][e], m[e] * p[i][e]);
        rn_store<VEC>(a.y, a.x_bf, row * d + c, y[i]);
        if (a.x_bf) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[i][e] = bf2f(f2bf(y[i][e]));  // the stream as stored
        }
    }
    if (!a.pre_w) return;
    row_stats<W, NCH, VEC>(y, c0, d, a, sh, mean, rstd);
    if (a.stats && lane == 0) {
        a.stats[2 * (int64_t)a.rows + row] = mean;
        a.stats[3 * (int64_t)a.rows + row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = c0 + i * STEP;
        float z[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = 0.f;
        if (c < d) {
            float t[VEC];
            rn_load<VEC>(a.pre_w, 0, c, t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) z[e] = (y[i][e] - mean) * rstd * t[e];
            if (a.pre_b) {
                rn_load<VEC>(a.pre_b, 0, c, t);
#pragma unroll
                for (int e = 0; e < VEC; ++e) z[e] += t[e];
            }
            if (a.z) rn_store<VEC>(a.z, a.z_bf, row * d + c, z);
        }
        if (a.z8) {  // blocks of 32 columns sit in 32 / VEC neighbouring lanes; the packed z is that of the z written beside it
            if (a.z_bf) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) z[e] = bf2f(f2bf(z[e]));
            }
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) top = mx_amax(top, z[e]);
#pragma unroll
            for (int o = 1; o < 32 / VEC; o <<= 1) top = mx_amax(top, __shfl_xor(top, o, 64));
            const int sb = mx_scale_byte<8>(top);
            const float inv = mx_inverse(sb);
            if (c < a.z8_ld) {
                if constexpr (VEC == 4) {
                    *reinterpret_cast<unsigned*>(a.z8 + row * a.z8_ld + c) = sb == 255 ? 0x7f7f7f7fu : mx_e4m3x4(z[0] * inv, z[1] * inv, z[2] * inv, z[3] * inv);
                } else {
                    a.z8[row * a.z8_ld + c] = sb == 255 ? 0x7f : (unsigned char)(mx_e4m3x4(z[0] * inv, 0.f, 0.f, 0.f) & 0xff);
                }
                if (c % 32 == 0) a.z8s[row * a.z8s_ld + c / 32] = (unsigned char)sb;
            }
        }
    }
}

// Backward.  With gy = dy + Norm_pre'(dz):  dx = alpha gy, and through y = alpha x + m p:
//   dp = m gy (0 where m is), dh = Norm_post'(dp), d scale = sum_rows gate p gy, d gate = sum scale p gy over what shares it,
//   Norm'(dn) = rstd (u - mean(u) - hat mean(u hat)), u = dn w  (rms: without mean(u)); d w = sum_rows dn hat, d b = sum_rows dn.
// A team walks a contiguous range of rows and keeps the column sums of its lanes' columns in registers; the workgroup's teams meet
// in LDS at the end, the workgroups in residual_norm_finish_kernel: a fixed order, no atomics.
// (TEAMS teams to a workgroup: W == 1 only)
template <int W, int NCH, int VEC, int TEAMS>
__global__ __launch_bounds__(64 * W * TEAMS) void residual_norm_bwd_kernel(RnArgs a) {
    constexpr int STEP = 64 * W * VEC, COLS = STEP * NCH;
    __shared__ float sh[TEAMS > 1 ? TEAMS * COLS : 3 * W];
    const int lane = threadIdx.x & (64 * W - 1), team_in = TEAMS > 1 ? threadIdx.x >> 6 : 0;
    const int64_t team = (int64_t)blockIdx.x * TEAMS + team_in;
    const int d = a.d, c0 = lane * VEC;
    const int64_t r0 = team * a.rows_per_team, r1 = r0 + a.rows_per_team < a.rows ? r0 + a.rows_per_team : a.rows;
    float cs[RN_KINDS][NCH][VEC], cg[NCH][VEC];
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#pragma unroll
            for (int k = 0; k < RN_KINDS; ++k) cs[k][i][e] = 0.f;
            cg[i][e] = 0.f;
        }
    int64_t grp = a.gate_mode && r0 < r1 ? r0 / a.rpg : 0, in_grp = a.gate_mode && r0 < r1 ? r0 - grp * a.rpg : 0;
    for (int64_t row = r0; row < r1; ++row) {
        float gy[NCH][VEC], hv[NCH][VEC];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * STEP;
#pragma unroll
            for (int e = 0; e < VEC; ++e) gy[i][e] = hv[i][e] = 0.f;
            if (c < d) {
                if (a.dy) rn_load<VEC>(a.dy, a.x_bf, row * a.sdy + c, gy[i]);
                rn_load<VEC>(a.h, a.h_bf, row * a.sh + c, hv[i]);
            }
        }
        if (a.pre_w) {
            float u[NCH][VEC], hat[NCH][VEC];
            const float mean = a.stats[2 * (int64_t)a.rows + row], rstd = a.stats[3 * (int64_t)a.rows + row];
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * STEP;
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[i][e] = hat[i][e] = 0.f;
                if (c < d) {
                    rn_load<VEC>(a.dz, a.z_bf, row * a.sdz + c, u[i]);
                    rn_load<VEC>(a.yin, a.x_bf, row * a.sy + c, hat[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * STEP;
                if (c >= d) continue;
                float w[VEC];
                rn_load<VEC>(a.pre_w, 0, c, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    hat[i][e] = (hat[i][e] - mean) * rstd;
                    cs[3][i][e] = fmaf(u[i][e], hat[i][e], cs[3][i][e]);
                    cs[4][i][e] += u[i][e];
                    u[i][e] *= w[e];
                    s[0] += u[i][e];
                    s[1] = fmaf(u[i][e], hat[i][e], s[1]);
                }
            }
            team_sum<W>(s, sh);
            const float m1 = a.rms ? 0.f : s[0] * a.inv_d, m2 = s[1] * a.inv_d;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) gy[i][e] = fmaf(rstd, u[i][e] - m1 - hat[i][e] * m2, gy[i][e]);
        }
        const float mean = a.post_w ? a.stats[row] : 0.f, rstd = a.post_w ? a.stats[(int64_t)a.rows + row] : 1.f;
        const float g1 = a.gate_mode == 1 ? a.gate[grp] : 1.f;
        float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * STEP;
            if (c >= d) continue;
            float t[VEC], w[VEC], b[VEC], g[VEC], sc[VEC], dp[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                t[e] = a.alpha * gy[i][e];
                w[e] = sc[e] = 1.f;
                b[e] = 0.f;
                g[e] = g1;
            }
            if (a.dx) rn_store<VEC>(a.dx, a.x_bf, row * d + c, t);
            if (a.post_w) rn_load<VEC>(a.post_w, 0, c, w);
            if (a.post_b) rn_load<VEC>(a.post_b, 0, c, b);
            if (a.gate_mode == 2) rn_load<VEC>(a.gate, 0, grp * d + c, g);
            if (a.scale) rn_load<VEC>(a.scale, 0, c, sc);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float hat = (hv[i][e] - mean) * rstd;          // post_w null: h itself
                const float p = fmaf(hat, w[e], b[e]), pg = p * gy[i][e];
                const float m = g[e] * sc[e];
                dp[e] = m == 0.f ? 0.f : m * gy[i][e];
                cs[2][i][e] = g[e] == 0.f ? cs[2][i][e] : fmaf(g[e], pg, cs[2][i][e]);
                cg[i][e] = fmaf(sc[e], pg, cg[i][e]);
                s[2] = fmaf(sc[e], pg, s[2]);
                cs[0][i][e] = dp[e] == 0.f ? cs[0][i][e] : fmaf(dp[e], hat, cs[0][i][e]);
                cs[1][i][e] += dp[e];
                const float v = dp[e] * w[e];
                s[0] += v;
                s[1] = v == 0.f ? s[1] : fmaf(v, hat, s[1]);
                gy[i][e] = v;
                hv[i][e] = hat;
            }
        }
        if (a.post_w || a.gate_mode == 1) team_sum<W>(s, sh);
        if (a.gate_mode == 1 && lane == 0) (a.groups == a.rows ? a.dgate : a.gate_rows)[row] = s[2];
        if (a.dh) {
            const float m1 = a.rms ? 0.f : s[0] * a.inv_d, m2 = s[1] * a.inv_d;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * STEP;
                if (c >= d) continue;
                if (a.post_w) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float v = gy[i][e] - m1 - (m2 == 0.f ? 0.f : hv[i][e] * m2);
                        gy[i][e] = v == 0.f ? 0.f : rstd * v;
                    }
                }
                rn_store<VEC>(a.dh, a.h_bf, row * d + c, gy[i]);
            }
        }
        if (a.gate_mode) {
            // a group's rows are neighbours: its gate's row of column sums is handed over where the group (or this team's part of
            // it) ends.  Slot team + group: both only grow along the rows, so no two (team, group) pairs share one.
            const bool last = ++in_grp == a.rpg;
            if (a.gate_mode == 2 && (last || row + 1 == r1)) {
                float* out = a.groups == a.rows ? a.dgate + grp * d : a.gate_rows + (team + grp) * d;
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int c = c0 + i * STEP;
                    if (c < d) rn_store<VEC>(out, 0, c, cg[i]);
                }
#pragma unroll
                for (int i = 0; i < NCH; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) cg[i][e] = 0.f;
            }
            if (last) {
                ++grp;
                in_grp = 0;
            }
        }
    }
    float* out = a.part + (int64_t)blockIdx.x * RN_KINDS * d;
    if constexpr (TEAMS > 1) {
#pragma unroll
        for (int k = 0; k < RN_KINDS; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sh[team_in * COLS + c0 + i * STEP + e] = cs[k][i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < d; c += 64 * TEAMS) {
                float t = 0.f;
#pragma unroll
                for (int w = 0; w < TEAMS; ++w) t += sh[w * COLS + c];
                out[k * d + c] = t;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < RN_KINDS; ++k)
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * STEP;
                if (c < d) rn_store<VEC>(out + k * d, 0, c, cs[k][i]);
            }
    }
}

struct RnFinish {
    const float* part;
    const float* gate_rows;
    float* out[RN_KINDS];
    float* dgate;
    int nblk, d, col_blocks, gate_mode, rows_per_team;
    int64_t groups, rpg, rows;
};

// workgroups 0 .. 5 col_blocks - 1: 64 columns of one column sum, four threads to a column over a quarter of the blocks each;
// behind them the gate: 4 groups to a workgroup (a number per group) or 64 columns of one group (a row per group)
__global__ __launch_bounds__(256) void residual_norm_finish_kernel(RnFinish f) {
    __shared__ float sh[4][64];
    const int col = threadIdx.x & 63, q = threadIdx.x >> 6;
    int64_t b = blockIdx.x;
    if (b < RN_KINDS * f.col_blocks) {
        const int k = (int)b / f.col_blocks, c = ((int)b % f.col_blocks) * 64 + col;
        if (!f.out[k]) return;
        float s = 0.f;
        if (c < f.d)
            for (int i = q; i < f.nblk; i += 4) s += f.part[((int64_t)i * RN_KINDS + k) * f.d + c];
        sh[q][col] = s;
        __syncthreads();
        if (q == 0 && c < f.d) f.out[k][c] = (sh[0][col] + sh[1][col]) + (sh[2][col] + sh[3][col]);
        return;
    }
    b -= RN_KINDS * f.col_blocks;
    if (f.gate_mode == 1) {
        const int64_t g = b * 4 + q;
        if (g >= f.groups) return;
        float s = 0.f;
        for (int64_t r = col; r < f.rpg; r += 64) s += f.gate_rows[g * f.rpg + r];
        s = wave_sum(s);
        if (col == 0) f.dgate[g] = s;
    } else {
        const int64_t g = b / f.col_blocks;
        const int c = (int)(b % f.col_blocks) * 64 + col;
        const int64_t t0 = g * f.rpg / f.rows_per_team, t1 = ((g + 1) * f.rpg - 1) / f.rows_per_team;
        float s = 0.f;
        if (c < f.d)
            for (int64_t t = t0 + q; t <= t1; t += 4) s += f.gate_rows[(t + g) * f.d + c];
        sh[q][col] = s;
        __syncthreads();
        if (q == 0 && c < f.d) f.dgate[g * f.d + c] = (sh[0][col] + sh[1][col]) + (sh[2][col] + sh[3][col]);
    }
}

static bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

struct RnPlan {
    int W, nch, vec, teams, rows_per_team, blocks;
};

// One wave to a row up to 1 024 columns (16 values of a tensor to a lane), whole workgroups beyond: no barrier inside a row where
// one wave holds it.  Backward: at least RN_MIN_ROWS rows to a team, so the teams' column sums stay small beside the rows, and at
// most one workgroup of eight waves to each of the 256 CUs.
constexpr int RN_MIN_ROWS = 4;
static RnPlan rn_plan(int rows, int d, bool vec4) {
    RnPlan p;
    p.vec = vec4 ? 4 : 1;
    p.W = d <= 1024 ? 1 : d <= 4096 ? 4 : 8;
    const int per = 64 * p.W * p.vec, need = (d + per - 1) / per;
    p.nch = 1;
    if (vec4 && p.W == 1) p.nch = need;
    else
        while (p.nch < need) p.nch *= 2;
    if (!vec4 && p.nch < 4) p.nch = 4;
    const int teams_blk = p.W == 1 ? 8 : 1, most = 256 * (p.W == 1 ? 8 : p.W == 4 ? 2 : 1);
    int teams = (rows + RN_MIN_ROWS - 1) / RN_MIN_ROWS;
    if (teams > most) teams = most;
    p.rows_per_team = rows ? (rows + teams - 1) / teams : 1;
    p.teams = rows ? (rows + p.rows_per_team - 1) / p.rows_per_team : 0;
    p.blocks = (p.teams + teams_blk - 1) / teams_blk;
    p.teams = p.blocks * teams_blk;
    return p;
}

#define RN_CASE(W_, N_, V_) \
    if (p.W == W_ && p.nch == N_ && p.vec == V_) return launch(std::integral_constant<int, W_>{}, std::integral_constant<int, N_>{}, std::integral_constant<int, V_>{});

template <typename F>
static bool rn_dispatch(const RnPlan& p, F&& launch) {
    RN_CASE(1, 1, 4) RN_CASE(1, 2, 4) RN_CASE(1, 3, 4) RN_CASE(1, 4, 4) RN_CASE(4, 2, 4) RN_CASE(4, 4, 4) RN_CASE(8, 4, 4)
    RN_CASE(1, 4, 1) RN_CASE(1, 8, 1) RN_CASE(1, 16, 1) RN_CASE(4, 8, 1) RN_CASE(4, 16, 1) RN_CASE(8, 16, 1)
    return false;
}
#undef RN_CASE

static int rn_common(RnArgs& a, int rows, int d, int64_t groups, int gate_channels, const char* what) {
    SWAT_REQUIRE(rows >= 0 && d >= 1 && d <= 8192, "%s: rows %d, width %d (0 rows or more, 1 to 8192 columns)", what, rows, d);
    SWAT_REQUIRE(!a.gate || (groups >= 1 && rows % groups == 0), "%s: %lld gates do not divide %d rows", what, (long long)groups, rows);
    SWAT_REQUIRE((a.post_w || !a.post_b) && (a.pre_w || !a.pre_b), "%s: a norm's bias without its weight", what);
    a.rows = rows;
    a.d = d;
    a.inv_d = 1.0f / (float)d;
    a.groups = a.gate ? groups : 1;
    a.rpg = a.gate ? rows / groups : 1;
    if (a.rpg < 1) a.rpg = 1;
    a.gate_mode = a.gate ? (gate_channels ? 2 : 1) : 0;
    return 0;
}

static bool vec_ok(const void* p, int bf, int64_t stride) { return !p || (aligned(p, bf ? 8 : 16) && stride % 4 == 0); }

}  // namespace swat

using namespace swat;

SWAT_API int swat_residual_norm_fwd(const void* x, int64_t x_stride, int x_dtype, const void* h, int64_t h_stride, int h_dtype,
                                    const float* post_w, const float* post_b, const float* gate, int64_t groups, int gate_channels,
                                    const float* scale, const float* pre_w, const float* pre_b, float alpha, int rms, float eps,
                                    void* y, void* z, int z_dtype, void* z8_codes, void* z8_scales, float* stats, int rows, int d,
                                    swat_stream_t stream) {
    RnArgs a = {};
    a.post_w = post_w; a.post_b = post_b; a.gate = gate; a.scale = scale; a.pre_w = pre_w; a.pre_b = pre_b;
    if (const int rc = rn_common(a, rows, d, groups, gate_channels, "swat_residual_norm_fwd")) return rc;
    if (rows == 0) return 0;
    SWAT_REQUIRE(x && h && y, "swat_residual_norm_fwd: x, h and y are needed");
    SWAT_REQUIRE(x_stride >= d && h_stride >= d, "swat_residual_norm_fwd: row strides %lld, %lld under %d columns", (long long)x_stride, (long long)h_stride, d);
    SWAT_REQUIRE(!pre_w == !(z || z8_codes) && !z8_codes == !z8_scales, "swat_residual_norm_fwd: z goes with the norm after the block, codes with scales");
    a.x = x; a.h = h; a.sx = x_stride; a.sh = h_stride; a.x_bf = x_dtype == SWAT_BF16; a.h_bf = h_dtype == SWAT_BF16;
    a.z_bf = z_dtype == SWAT_BF16; a.alpha = alpha; a.eps = eps; a.rms = rms != 0;
    a.y = y; a.z = z; a.z8 = (unsigned char*)z8_codes; a.z8s = (unsigned char*)z8_scales; a.stats = stats;
    a.z8s_ld = (d + 31) / 32;
    a.z8_ld = 32 * a.z8s_ld;
    const bool v = d % 4 == 0 && vec_ok(x, a.x_bf, x_stride) && vec_ok(h, a.h_bf, h_stride) && vec_ok(y, a.x_bf, d) && vec_ok(z, a.z_bf, d) &&
                   vec_ok(post_w, 0, 0) && vec_ok(post_b, 0, 0) && vec_ok(gate_channels ? gate : nullptr, 0, 0) && vec_ok(scale, 0, 0) &&
                   vec_ok(pre_w, 0, 0) && vec_ok(pre_b, 0, 0) && aligned(z8_codes, 4);
    const RnPlan p = rn_plan(rows, d, v);
    const hipStream_t s = (hipStream_t)stream;
    const bool known = rn_dispatch(p, [&](auto w, auto n, auto c) {
        constexpr int W = decltype(w)::value, N = decltype(n)::value, V = decltype(c)::value;
        const int grid = W == 1 ? (rows + 3) / 4 : rows;
        residual_norm_fwd_kernel<W, N, V><<<grid, W == 1 ? 256 : 64 * W, 0, s>>>(a);
        return true;
    });
    SWAT_REQUIRE(known, "swat_residual_norm_fwd: no kernel for %d columns", d);
    return check_launch("swat_residual_norm_fwd");
}

static int64_t rn_ws(int rows, int d, int64_t groups, int gate_mode, bool vec4, int64_t* gate_at) {
    const RnPlan p = rn_plan(rows, d, vec4);
    *gate_at = (int64_t)p.blocks * RN_KINDS * d;
    const int64_t slots = gate_mode == 1 ? rows : gate_mode == 2 ? (p.teams + groups) * (int64_t)d : 0;
    return 4 * (*gate_at + slots);
}

SWAT_API int64_t swat_residual_norm_bwd_workspace_bytes(int rows, int d, int64_t groups, int gate_channels) {
    if (rows < 0 || d < 1 || d > 8192 || groups < 0) {
        set_error("swat_residual_norm_bwd_workspace_bytes: rows %d, width %d, groups %lld", rows, d, (long long)groups);
        return -1;
    }
    int64_t at;  // (alignment decides the vector width at the call: room for either plan)
    const int mode = groups ? (gate_channels ? 2 : 1) : 0;
    const int64_t n = rn_ws(rows, d, groups, mode, true, &at), m = rn_ws(rows, d, groups, mode, false, &at);
    return n > m ? n : m;
}

SWAT_API int swat_residual_norm_bwd(const void* dy, int64_t dy_stride, const void* dz, int64_t dz_stride, int z_dtype, const void* h,
                                    int64_t h_stride, int h_dtype, const void* y, int64_t y_stride, int x_dtype, const float* stats,
                                    const float* post_w, const float* post_b, const float* gate, int64_t groups, int gate_channels,
                                    const float* scale, const float* pre_w, const float* pre_b, float alpha, int rms, void* dx, void* dh,
                                    float* dpost_w, float* dpost_b, float* dgate, float* dscale, float* dpre_w, float* dpre_b,
                                    void* workspace, int64_t workspace_bytes, int rows, int d, swat_stream_t stream) {
    RnArgs a = {};
    a.post_w = post_w; a.post_b = post_b; a.gate = gate; a.scale = scale; a.pre_w = pre_w; a.pre_b = pre_b;
    if (const int rc = rn_common(a, rows, d, groups, gate_channels, "swat_residual_norm_bwd")) return rc;
    SWAT_REQUIRE(!gate == !dgate, "swat_residual_norm_bwd: a gate goes with its gradient");
    SWAT_REQUIRE(rows == 0 || (h && dx && dh), "swat_residual_norm_bwd: h, dx and dh are needed");
    SWAT_REQUIRE(!pre_w == !dz || rows == 0, "swat_residual_norm_bwd: dz goes with the norm after the block");
    SWAT_REQUIRE(dy || pre_w || rows == 0, "swat_residual_norm_bwd: neither dy nor dz");
    SWAT_REQUIRE(rows == 0 || !pre_w || (y && y_stride >= d && dz_stride >= d), "swat_residual_norm_bwd: the norm after the block needs y and dz, strides of %d at least", d);
    SWAT_REQUIRE(rows == 0 || ((!dy || dy_stride >= d) && h_stride >= d), "swat_residual_norm_bwd: row strides under %d columns", d);
    SWAT_REQUIRE(rows == 0 || stats || !(pre_w || post_w), "swat_residual_norm_bwd: the norms need the forward's statistics");
    a.dy = dy; a.dz = dz; a.h = h; a.yin = y; a.sdy = dy_stride; a.sdz = dz_stride; a.sh = h_stride; a.sy = y_stride;
    a.x_bf = x_dtype == SWAT_BF16; a.h_bf = h_dtype == SWAT_BF16; a.z_bf = z_dtype == SWAT_BF16;
    a.alpha = alpha; a.rms = rms != 0; a.stats = const_cast<float*>(stats);
    a.dx = dx; a.dh = dh; a.dgate = dgate;
    const bool v = d % 4 == 0 && vec_ok(dy, a.x_bf, dy_stride) && vec_ok(dz, a.z_bf, dz_stride) && vec_ok(h, a.h_bf, h_stride) &&
                   vec_ok(y, a.x_bf, y_stride) && vec_ok(dx, a.x_bf, d) && vec_ok(dh, a.h_bf, d) && vec_ok(post_w, 0, 0) &&
                   vec_ok(post_b, 0, 0) && vec_ok(gate_channels ? gate : nullptr, 0, 0) && vec_ok(scale, 0, 0) && vec_ok(pre_w, 0, 0) &&
                   vec_ok(gate_channels ? dgate : nullptr, 0, 0) && aligned(workspace, 16);
    const RnPlan p = rn_plan(rows, d, v);
    int64_t gate_at;
    const int64_t want = rn_ws(rows, d, a.groups, a.gate_mode, v, &gate_at);
    SWAT_REQUIRE(rows == 0 || (workspace && workspace_bytes >= want), "swat_residual_norm_bwd: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)want);
    a.part = (float*)workspace;
    a.gate_rows = a.part + gate_at;
    a.rows_per_team = p.rows_per_team;
    const hipStream_t s = (hipStream_t)stream;
    if (rows > 0) {
        const bool known = rn_dispatch(p, [&](auto w, auto n, auto c) {
            constexpr int W = decltype(w)::value, N = decltype(n)::value, V = decltype(c)::value, T = W == 1 ? 8 : 1;
            residual_norm_bwd_kernel<W, N, V, T><<<p.blocks, 64 * W * T, 0, s>>>(a);
            return true;
        });
        SWAT_REQUIRE(known, "swat_residual_norm_bwd: no kernel for %d columns", d);
    }
    RnFinish f = {};
    f.part = a.part; f.gate_rows = a.gate_rows; f.nblk = p.blocks; f.d = d; f.col_blocks = (d + 63) / 64;
    f.out[0] = post_w ? dpost_w : nullptr; f.out[1] = post_b ? dpost_b : nullptr; f.out[2] = scale ? dscale : nullptr;
    f.out[3] = pre_w ? dpre_w : nullptr; f.out[4] = pre_b ? dpre_b : nullptr;
    f.dgate = dgate; f.groups = a.groups; f.rpg = a.rpg; f.rows = rows; f.rows_per_team = p.rows_per_team;
    f.gate_mode = a.groups != rows ? a.gate_mode : 0;
    if (rows == 0) f.rpg = 0;  // sums over nothing: zeros
    int64_t grid = RN_KINDS * f.col_blocks;
    grid += f.gate_mode == 1 ? (f.groups + 3) / 4 : f.gate_mode == 2 ? f.groups * f.col_blocks : 0;
    residual_norm_finish_kernel<<<(unsigned)grid, 256, 0, s>>>(f);
    return check_launch("swat_residual_norm_bwd");
}
