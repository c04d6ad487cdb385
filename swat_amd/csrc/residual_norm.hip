// swat_amd/csrc/residual_norm.hip — the seam between two sublayers of a transformer block as one kernel per direction:
//
//   p = Norm_post(h)  (or h);   m = gate * scale;   y = alpha x + m p;   z = Norm_pre(y)
//
// Norm: LayerNorm or root mean square, eps inside the root.  An element whose multiplier m is zero takes nothing from p: h may
// hold anything there without Norm_post, and in a row where all of m is zero (a dropped row) with it; in other rows Norm_post's mean and
// deviation are over every element, which then has its share of dh through them.  z is the norm of the stream AS STORED, because the next sublayer's
// backward pass reads that y.
//
// A row lives in the registers of one team of W waves; both norms take their mean and their squared deviations from there, so
// every tensor crosses the memory bus once.  Rows may start on any element: vector loads and stores take any address here, and the last
// columns of a width that is no multiple of 4 come as the row's last four, shifted down in registers.
//
// Bound by bytes in both directions.  fp32 stream, bf16 branch, gate, scale and both norms (us, and TB/s of what has to move; a large copy
// reaches 4.95): forward 16448 x 1024 44.5 (4.5; 49 with the packed z), 12608 x 768 28 (4.1), 4112 x 4096 45 (4.5), 2056 x 8192 50 (4.1); backward
// 74 (4.1), 47.5 (3.7), 85 (3.5) and 114 (2.7: eight waves to a row, two barriers to a sum, one workgroup to a CU), which adds the column
// sums of up to five vectors (5 of the 47.5).  All in fp32, backward: 92, 53, 108 and 165.  50 x 768 forward: 6 on the device, the latency
// of loads that wait for each other.
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

constexpr int RN_KINDS = 4;  // column sums of the backward pass: of gate gy hat, of gate gy, pre_w, pre_b

typedef unsigned rn_u4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned rn_u2 __attribute__((ext_vector_type(2), aligned(2)));

// Four neighbouring columns of a row, as they lie in memory.  T: 0 float32, 1 bfloat16, 2 by the flag.
template <int T>
struct RnRaw {
    unsigned v[T == 1 ? 2 : 4];
};
// ROW: a tensor's row, read once and never again by this call: a non-temporal load, which leaves the caches to what is written (16448 x 1024,
// tensors past the caches: forward 55.7 -> 45.6 us; with the linear layer that reads z behind it 197 -> 179.  Non-temporal stores
// gain as much alone and lose 9 us with that layer).
template <int T, bool ROW = true>
__device__ __forceinline__ void rn_raw(RnRaw<T>& r, const void* p, int bf, int64_t row, int c, int d) {
    const int cc = c + 4 <= d || d < 4 ? c : d - 4;
    const bool b = T == 1 || (T == 2 && bf);
    if (d < 4) {   // (narrower than a vector: one lane, element by element)
#pragma unroll
        for (int e = 0; e < (T == 1 ? 2 : 4); ++e) r.v[e] = 0u;
#pragma unroll
        for (int e = 0; e < 3; ++e) {
            if (e >= d) continue;
            if (b) r.v[e >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[row + e] << (16 * (e & 1));
            else if constexpr (T != 1) r.v[e] = reinterpret_cast<const unsigned*>(p)[row + e];
        }
        return;
    }
    if (b) {
        const rn_u2* q = reinterpret_cast<const rn_u2*>(reinterpret_cast<const unsigned short*>(p) + row + cc);
        const rn_u2 u = ROW ? __builtin_nontemporal_load(q) : *q;
        r.v[0] = u[0];
        r.v[1] = u[1];
    } else if constexpr (T != 1) {
        const rn_u4* q = reinterpret_cast<const rn_u4*>(reinterpret_cast<const float*>(p) + row + cc);
        const rn_u4 u = ROW ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[e] = u[e];
    }
}
// (columns past d: zeros)
template <int T>
__device__ __forceinline__ void rn_values(const RnRaw<T>& r, int bf, int c, int d, float (&v)[4]) {
    if (T == 1 || (T == 2 && bf)) {
        v[0] = __uint_as_float(r.v[0] << 16); v[1] = __uint_as_float(r.v[0] & 0xffff0000u);
        v[2] = __uint_as_float(r.v[1] << 16); v[3] = __uint_as_float(r.v[1] & 0xffff0000u);
    } else if constexpr (T != 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(r.v[e]);
    }
    const int over = d & 3;   // columns of the last vector; it was loaded 4 - over columns early
    if (over && d >= 4) {
        const bool part = c < d && c + 4 > d;
        if (over == 1) v[0] = part ? v[3] : v[0];
        else if (over == 2) {
            v[0] = part ? v[2] : v[0];
            v[1] = part ? v[3] : v[1];
        } else {
            v[0] = part ? v[1] : v[0];
            v[1] = part ? v[2] : v[1];
            v[2] = part ? v[3] : v[2];
        }
#pragma unroll
        for (int e = 1; e < 4; ++e) v[e] = part && e >= over ? 0.f : v[e];
    }
}
__device__ __forceinline__ void rn_load(const float* p, int64_t row, int c, int d, float (&v)[4]) {
    RnRaw<0> r;
    rn_raw<0, false>(r, p, 0, row, c, d);
    rn_values<0>(r, 0, c, d, v);
}
__device__ __forceinline__ void rn_store(void* p, int bf, int64_t row, int c, int d, const float (&v)[4]) {
    if (c + 4 <= d) {
        if (bf) *reinterpret_cast<rn_u2*>(reinterpret_cast<unsigned short*>(p) + row + c) = (rn_u2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else *reinterpret_cast<rn_u4*>(reinterpret_cast<float*>(p) + row + c) =
            (rn_u4){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < d) {
            if (bf) reinterpret_cast<unsigned short*>(p)[row + c + e] = f2bf(v[e]);
            else reinterpret_cast<float*>(p)[row + c + e] = v[e];
        }
}

// the wave's sum by lane shifts inside rows of 16 and two broadcasts of a row's last lane (a few cycles each; six LDS lane exchanges took
// a tenth of the backward pass)
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float row_add_sum(float v) {
    v = dpp_add<0x111, 0xf>(v);   // row_shr:1, 2, 4, 8
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);   // row_bcast:15 into rows 1 and 3
    v = dpp_add<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// sums of N values over the team; sh: W * N floats of the team, two barriers around them (the trip count of the row loop is the
// same for every team of a workgroup when W > 1: one team is the whole workgroup)
template <int W, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* sh) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = row_add_sum(v[i]);
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

// mean (layer) and 1 / deviation of a row held as v[NCH][4], columns c < d
template <int W, int NCH>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][4], int c0, int d, const RnArgs& a, float* sh, float& mean, float& rstd) {
    mean = 0.f;
    if (!a.rms) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0] += v[i][e];  // (columns past d hold zeros)
        team_sum<W>(s, sh);
        mean = s[0] * a.inv_d;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = c0 + i * (256 * W) + e < d ? v[i][e] - mean : 0.f;
            q[0] = fmaf(t, t, q[0]);
        }
    team_sum<W>(q, sh);
    rstd = 1.0f / sqrtf(q[0] * a.inv_d + a.eps);
}

// W waves to a row, NCH vectors to a lane: rows of up to 256 W NCH columns
template <int W, int NCH>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void residual_norm_fwd_kernel(RnArgs a) {
    __shared__ float sh[W];
    const int lane = threadIdx.x & (64 * W - 1);
    const int64_t row = W == 1 ? mx_block() * 4 + (threadIdx.x >> 6) : mx_block();
    if (row >= a.rows) return;
    const int d = a.d, c0 = lane * 4;
    constexpr int STEP = 256 * W;
    float p[NCH][4], y[NCH][4];
    {
        RnRaw<2> rh[NCH], rx[NCH];
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            if (c0 + i * STEP < d) rn_raw<2>(rh[i], a.h, a.h_bf, row * a.sh, c0 + i * STEP, d);
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            if (c0 + i * STEP < d) rn_raw<2>(rx[i], a.x, a.x_bf, row * a.sx, c0 + i * STEP, d);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) p[i][e] = y[i][e] = 0.f;
            if (c0 + i * STEP < d) {
                rn_values<2>(rh[i], a.h_bf, c0 + i * STEP, d, p[i]);
                rn_values<2>(rx[i], a.x_bf, c0 + i * STEP, d, y[i]);
            }
        }
    }
    float mean = 0.f, rstd = 1.f;
    if (a.post_w) {
        row_stats<W, NCH>(p, c0, d, a, sh, mean, rstd);
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
        float t[4], m[4];
        if (a.post_w) {
            rn_load(a.post_w, 0, c, d, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) p[i][e] = (p[i][e] - mean) * rstd * t[e];
            if (a.post_b) {
                rn_load(a.post_b, 0, c, d, t);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[i][e] += t[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = g1;
        if (a.gate_mode == 2) rn_load(a.gate, grp * d, c, d, m);
        if (a.scale) {
            rn_load(a.scale, 0, c, d, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] *= t[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[i][e] = c + e >= d ? 0.f : m[e] == 0.f ? a.alpha * y[i][e] : fmaf(a.alpha, y[i][e], m[e] * p[i][e]);
        rn_store(a.y, a.x_bf, row * d, c, d, y[i]);
        if (a.x_bf) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][e] = bf2f(f2bf(y[i][e]));  // the stream as stored
        }
    }
    if (!a.pre_w) return;
    row_stats<W, NCH>(y, c0, d, a, sh, mean, rstd);
    if (a.stats && lane == 0) {
        a.stats[2 * (int64_t)a.rows + row] = mean;
        a.stats[3 * (int64_t)a.rows + row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = c0 + i * STEP;
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = 0.f;
        if (c < d) {
            float t[4];
            rn_load(a.pre_w, 0, c, d, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = (y[i][e] - mean) * rstd * t[e];
            if (a.pre_b) {
                rn_load(a.pre_b, 0, c, d, t);
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] += t[e];
            }
            if (a.z) rn_store(a.z, a.z_bf, row * d, c, d, z);
        }
        if (a.z8) {  // blocks of 32 columns sit in 8 neighbouring lanes; the packed z is that of the z written beside it
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = c + e >= d ? 0.f : a.z_bf ? bf2f(f2bf(z[e])) : z[e];
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = mx_amax(top, z[e]);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = mx_amax(top, __shfl_xor(top, o, 64));
            const int sb = mx_scale_byte<8>(top);
            const float inv = mx_inverse(sb);
            if (c < a.z8_ld) {
                *reinterpret_cast<unsigned*>(a.z8 + row * a.z8_ld + c) = sb == 255 ? 0x7f7f7f7fu : mx_e4m3x4(z[0] * inv, z[1] * inv, z[2] * inv, z[3] * inv);
                if (c % 32 == 0) a.z8s[row * a.z8s_ld + c / 32] = (unsigned char)sb;
            }
        }
    }
}

// Backward.  With gy = dy + Norm_pre'(dz):  dx = alpha gy, and through y = alpha x + m p:
//   dp = m gy (0 where m is), dh = Norm_post'(dp), d scale = sum_rows gate p gy, d gate = sum scale p gy over what shares it,
//   Norm'(dn) = rstd (u - mean(u) - hat mean(u hat)), u = dn w  (rms: without mean(u)); d w = sum_rows dn hat, d b = sum_rows dn.
// With A = sum_rows gate gy hat and B = sum_rows gate gy (p = hat w + b) the weights' gradients of the first norm and of the scale are
// scale A, scale B and w A + b B: two column sums for three.
// A team walks a contiguous range of rows and keeps the column sums of its lanes' columns in registers; the workgroup's teams meet
// in LDS at the end, the workgroups in residual_norm_finish_kernel: a fixed order, no atomics.  The next row's four tensors are
// loaded before the present row is worked on; the vectors of weights wait in LDS, so that nothing but those loads is in flight.
// TEAMS teams to a workgroup (W == 1 only); TX, THZ: types of the stream and of h and dz (RnRaw; 2, 2: by the flags, no early loads);
// GC: the gate is a row per group.
template <int W, int NCH, int TEAMS, int TX, int THZ, bool GC>
__global__ __launch_bounds__(64 * W * TEAMS, 2) void residual_norm_bwd_kernel(RnArgs a) {
    constexpr int STEP = 256 * W, COLS = STEP * NCH, NT = 64 * W * TEAMS;
    constexpr bool AHEAD = TX != 2 && !(GC && NCH > 3);   // (not where the registers do not reach)
    __shared__ float red[3 * W];
    __shared__ __attribute__((aligned(16))) float sh[(TEAMS > 4 ? TEAMS : 4) * COLS];   // pre_w, post_w, post_b, scale; at the end the teams' sums
    const int lane = threadIdx.x & (64 * W - 1), team_in = TEAMS > 1 ? threadIdx.x >> 6 : 0;
    const int64_t team = (int64_t)blockIdx.x * TEAMS + team_in;
    const int d = a.d, c0 = lane * 4;
    const int64_t r0 = team * a.rows_per_team, r1 = r0 + a.rows_per_team < a.rows ? r0 + a.rows_per_team : a.rows;
    for (int c = threadIdx.x; c < COLS; c += NT) {
        sh[c] = a.pre_w && c < d ? a.pre_w[c] : 0.f;
        sh[COLS + c] = c >= d ? 0.f : a.post_w ? a.post_w[c] : 1.f;
        sh[2 * COLS + c] = a.post_b && c < d ? a.post_b[c] : 0.f;
        sh[3 * COLS + c] = c >= d ? 0.f : a.scale ? a.scale[c] : 1.f;
    }
    __syncthreads();
    auto vec = [&](int k, int i) { return *reinterpret_cast<const float4*>(sh + k * COLS + c0 + i * STEP); };
    float cs[RN_KINDS][NCH][4], cg[GC ? 2 : 1][GC ? NCH : 1][4], gate[GC ? NCH : 1][4];   // cg: A and B of a group without its gate
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int k = 0; k < RN_KINDS; ++k) cs[k][i][e] = 0.f;
            if constexpr (GC) cg[0][i][e] = cg[1][i][e] = gate[i][e] = 0.f;
        }
    struct Row {
        RnRaw<TX> dy[NCH], y[NCH];
        RnRaw<THZ> dz[NCH], h[NCH];
        float st[4], g;
    };
    auto fetch = [&](Row& r, int64_t row) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * STEP;
            if (c < d) {
                rn_raw<THZ>(r.h[i], a.h, a.h_bf, row * a.sh, c, d);
                if (a.dy) rn_raw<TX>(r.dy[i], a.dy, a.x_bf, row * a.sdy, c, d);
                if (a.pre_w) {
                    rn_raw<THZ>(r.dz[i], a.dz, a.z_bf, row * a.sdz, c, d);
                    rn_raw<TX>(r.y[i], a.yin, a.x_bf, row * a.sy, c, d);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) r.st[k] = (k < 2 ? a.post_w != nullptr : a.pre_w != nullptr) ? a.stats[k * (int64_t)a.rows + row] : 0.f;
        if constexpr (!GC) r.g = a.gate_mode == 1 ? a.gate[a.rpg == 1 ? row : row / a.rpg] : 1.f;
    };
    int64_t grp = 0, in_grp = 0;
    if (a.gate_mode && r0 < r1) {
        grp = r0 / a.rpg;
        in_grp = r0 - grp * a.rpg;
    }
    auto load_gate = [&]() {
        if constexpr (GC) {
#pragma unroll
            for (int i = 0; i < NCH; ++i)
                if (c0 + i * STEP < d) rn_load(a.gate, grp * d, c0 + i * STEP, d, gate[i]);
        }
    };
    Row next;
    if (r0 < r1) {
        if (AHEAD) fetch(next, r0);
        load_gate();
    }
    for (int64_t row = r0; row < r1; ++row) {
        Row cur;
        if constexpr (AHEAD) {
            cur = next;
            fetch(next, row + 1 < r1 ? row + 1 : row);
        } else {
            fetch(cur, row);
        }
        float gy[NCH][4], hv[NCH][4];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * STEP;
#pragma unroll
            for (int e = 0; e < 4; ++e) gy[i][e] = hv[i][e] = 0.f;
            if (c < d) {
                if (a.dy) rn_values<TX>(cur.dy[i], a.x_bf, c, d, gy[i]);
                rn_values<THZ>(cur.h[i], a.h_bf, c, d, hv[i]);
            }
        }
        if (a.pre_w) {
            float u[NCH][4], hat[NCH][4];
            const float mean = cur.st[2], rstd = cur.st[3];
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * STEP;
#pragma unroll
                for (int e = 0; e < 4; ++e) u[i][e] = hat[i][e] = 0.f;
                if (c >= d) continue;
                rn_values<THZ>(cur.dz[i], a.z_bf, c, d, u[i]);
                rn_values<TX>(cur.y[i], a.x_bf, c, d, hat[i]);
                const float4 w4 = vec(0, i);
                const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hat[i][e] = (hat[i][e] - mean) * rstd;
                    cs[2][i][e] = fmaf(u[i][e], hat[i][e], cs[2][i][e]);
                    cs[3][i][e] += u[i][e];
                    u[i][e] *= w[e];
                    s[0] += u[i][e];
                    s[1] = fmaf(u[i][e], hat[i][e], s[1]);   // (columns past d: u is zero)
                }
            }
            team_sum<W>(s, red);
            const float m1 = a.rms ? 0.f : s[0] * a.inv_d, m2 = s[1] * a.inv_d;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) gy[i][e] = fmaf(rstd, u[i][e] - m1 - hat[i][e] * m2, gy[i][e]);
        }
        const float mean = a.post_w ? cur.st[0] : 0.f, rstd = a.post_w ? cur.st[1] : 1.f;
        float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = c0 + i * STEP;
            if (c >= d) continue;
            float t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                gy[i][e] = c + e < d ? gy[i][e] : 0.f;
                t[e] = a.alpha * gy[i][e];
            }
            if (a.dx) rn_store(a.dx, TX == 2 ? a.x_bf : TX, row * d, c, d, t);
            const float4 w4 = vec(1, i), b4 = vec(2, i), s4 = vec(3, i);
            const float w[4] = {w4.x, w4.y, w4.z, w4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w}, sc[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float g = GC ? gate[GC ? i : 0][e] : cur.g;
                const float hat = (hv[i][e] - mean) * rstd;          // post_w null: h itself
                const float m = g * sc[e];
                const float dp = m == 0.f ? 0.f : m * gy[i][e];
                if constexpr (GC) {
                    cg[0][i][e] = fmaf(gy[i][e], hat, cg[0][i][e]);
                    cg[GC][i][e] += gy[i][e];
                } else {
                    const float q = g * gy[i][e];
                    cs[0][i][e] = g == 0.f ? cs[0][i][e] : fmaf(q, hat, cs[0][i][e]);
                    cs[1][i][e] += q;
                    s[2] = sc[e] != 0.f ? fmaf(sc[e] * gy[i][e], fmaf(hat, w[e], b[e]), s[2]) : s[2];   // (past d: zero)
                }
                const float v = dp * w[e];
                s[0] += v;
                s[1] = v == 0.f ? s[1] : fmaf(v, hat, s[1]);
                gy[i][e] = v;
                hv[i][e] = hat;
            }
        }
        if (a.post_w || (!GC && a.gate_mode == 1)) team_sum<W>(s, red);
        if (!GC && a.gate_mode == 1 && lane == 0) (a.groups == a.rows ? a.dgate : a.gate_rows)[row] = s[2];
        if (a.dh) {
            const float m1 = a.rms ? 0.f : s[0] * a.inv_d, m2 = s[1] * a.inv_d;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = c0 + i * STEP;
                if (c >= d) continue;
                if (a.post_w) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = gy[i][e] - m1 - (m2 == 0.f ? 0.f : hv[i][e] * m2);
                        gy[i][e] = v == 0.f ? 0.f : rstd * v;
                    }
                }
                rn_store(a.dh, THZ == 2 ? a.h_bf : THZ, row * d, c, d, gy[i]);
            }
        }
        if constexpr (GC) {
            // a group's rows are neighbours: its sums are handed over where the group (or this team's part of it) ends, its gate's row of
            // gradients into slot team + group: both only grow along the rows, so no two (team, group) pairs share one
            const bool last = ++in_grp == a.rpg;
            if (last || row + 1 == r1) {
                float* out = a.groups == a.rows ? a.dgate + grp * d : a.gate_rows + (team + grp) * d;
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    const int c = c0 + i * STEP;
                    if (c >= d) continue;
                    const float4 w4 = vec(1, i), b4 = vec(2, i), s4 = vec(3, i);
                    const float w[4] = {w4.x, w4.y, w4.z, w4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w}, sc[4] = {s4.x, s4.y, s4.z, s4.w};
                    float t[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float g = gate[i][e], A = cg[0][i][e], B = cg[GC][i][e];
                        t[e] = sc[e] == 0.f ? 0.f : sc[e] * fmaf(w[e], A, b[e] * B);
                        cs[0][i][e] = g == 0.f ? cs[0][i][e] : fmaf(g, A, cs[0][i][e]);
                        cs[1][i][e] = fmaf(g, B, cs[1][i][e]);
                        cg[0][i][e] = cg[GC][i][e] = 0.f;
                    }
                    rn_store(out, 0, 0, c, d, t);
                }
            }
            if (last) {
                ++grp;
                in_grp = 0;
                if (row + 1 < r1) load_gate();
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
                *reinterpret_cast<float4*>(sh + team_in * COLS + c0 + i * STEP) = make_float4(cs[k][i][0], cs[k][i][1], cs[k][i][2], cs[k][i][3]);
            __syncthreads();
            for (int c = threadIdx.x; c < d; c += NT) {
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
                if (c < d) rn_store(out, 0, k * (int64_t)d, c, d, cs[k][i]);
            }
    }
}

struct RnFinish {
    const float *part, *gate_rows, *post_w, *post_b, *scale;
    float *dpost_w, *dpost_b, *dscale, *dpre_w, *dpre_b, *dgate;
    int nblk, d, col_blocks, gate_mode, rows_per_team;
    int64_t groups, rpg;
};

// workgroups 0 .. 3 col_blocks - 1: 16 columns of the sums that belong together (those of the norm before, d weight and d bias of the one
// after), 16 threads to a column over a sixteenth of the blocks each, eight loads of a thread under way at a time (four threads to a
// column took 19 us, as long as a quarter of the rows' pass); behind them the gate: 4 groups to a workgroup (a number per group) or 256
// columns of one group (a row per group).  A group's rows are added by one wave, its parts of a row by one thread to a column: right for many
// groups of few rows.  A gate shared by all of 16448 x 1024 takes the whole backward from 74 us to 127 (a number) or 108 (a row).
__global__ __launch_bounds__(256) void residual_norm_finish_kernel(RnFinish f) {
    __shared__ float sh[2][16][17];
    int64_t b = blockIdx.x;
    if (b < 3 * f.col_blocks) {
        const int col = threadIdx.x & 15, q = threadIdx.x >> 4;
        const int k = (int)b / f.col_blocks, c = ((int)b % f.col_blocks) * 16 + col;
        if (k == 0 ? !(f.dpost_w || f.dpost_b || f.dscale) : k == 1 ? !f.dpre_w : !f.dpre_b) return;
        const float* p = f.part + (int64_t)(k == 0 ? 0 : k + 1) * f.d + (c < f.d ? c : 0);
        const int64_t step = (int64_t)RN_KINDS * f.d;
        float s = 0.f, t = 0.f;
        if (k == 0) {
#pragma unroll 8
            for (int i = q; i < f.nblk; i += 16) {
                s += p[i * step];
                t += p[i * step + f.d];
            }
        } else {
#pragma unroll 8
            for (int i = q; i < f.nblk; i += 16) s += p[i * step];
        }
        sh[0][q][col] = s;
        sh[1][q][col] = t;
        __syncthreads();
        if (q || c >= f.d) return;
        float A = 0.f, B = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            A += sh[0][i][col];
            B += sh[1][i][col];
        }
        if (k == 1) f.dpre_w[c] = A;
        else if (k == 2) f.dpre_b[c] = A;
        else {
            const float sc = f.scale ? f.scale[c] : 1.f;
            if (f.dpost_w) f.dpost_w[c] = sc == 0.f ? 0.f : sc * A;
            if (f.dpost_b) f.dpost_b[c] = sc == 0.f ? 0.f : sc * B;
            if (f.dscale) f.dscale[c] = fmaf(f.post_w ? f.post_w[c] : 1.f, A, f.post_b ? f.post_b[c] * B : 0.f);
        }
        return;
    }
    b -= 3 * f.col_blocks;
    const int col = threadIdx.x & 63, q = threadIdx.x >> 6;
    if (f.gate_mode == 1) {
        const int64_t g = b * 4 + q;
        if (g >= f.groups) return;
        float s = 0.f;
        for (int64_t r = col; r < f.rpg; r += 64) s += f.gate_rows[g * f.rpg + r];
        s = row_add_sum(s);
        if (col == 0) f.dgate[g] = s;
    } else {
        const int blocks = (f.d + 255) / 256;
        const int64_t g = b / blocks;
        const int c = (int)(b % blocks) * 256 + threadIdx.x;
        if (c >= f.d) return;
        const int64_t t0 = g * f.rpg / f.rows_per_team, t1 = ((g + 1) * f.rpg - 1) / f.rows_per_team;
        float s = 0.f;
#pragma unroll 8
        for (int64_t t = t0; t <= t1; ++t) s += f.gate_rows[(t + g) * f.d + c];
        f.dgate[g * f.d + c] = s;
    }
}

struct RnPlan {
    int W, nch, teams, rows_per_team, blocks;
};

// Forward: one wave to a row up to 1 024 columns (no barrier inside a row), four up to 4 096, eight beyond.  Backward: a wave to a row up to 768
// columns, four up to 2 048, eight beyond, because it keeps more of a row and the column sums in registers (16448 x 1024 with a row of
// gates: 75 us, 163 with one wave to a row and spilled registers); at most one workgroup of eight waves to each of the 256 CUs (two of
// four, four where a lane has one vector): every workgroup leaves four rows of column sums, 2 to 8 % of what the rows are.
static RnPlan rn_plan(int64_t rows, int d, bool bwd) {   // (64 bits: sums next to 2^31 rows)
    RnPlan p;
    p.W = d <= (bwd ? 768 : 1024) ? 1 : d <= (bwd ? 2048 : 4096) ? 4 : 8;
    const int need = (d + 256 * p.W - 1) / (256 * p.W);
    p.nch = need == 3 && p.W > 1 ? 4 : need;
    const int teams_blk = p.W == 1 ? 8 : 1, most = 256 * (p.W == 1 ? 8 : p.W == 4 ? (p.nch == 1 ? 4 : 2) : 1);
    const int64_t teams = rows < most ? rows : most;
    p.rows_per_team = rows ? (int)((rows + teams - 1) / teams) : 1;
    p.teams = rows ? (int)((rows + p.rows_per_team - 1) / p.rows_per_team) : 0;
    p.blocks = (p.teams + teams_blk - 1) / teams_blk;
    p.teams = p.blocks * teams_blk;
    return p;
}

template <int W, int... N, typename F>
static bool rn_try(const RnPlan& p, F&& launch) {   // W and one of N vectors to a lane
    return p.W == W && ((p.nch == N && (launch(std::integral_constant<int, W>{}, std::integral_constant<int, N>{}), true)) || ...);
}

static int rn_common(RnArgs& a, int rows, int d, int64_t groups, int gate_channels, const char* what) {
    SWAT_REQUIRE(rows >= 0 && d >= 1 && d <= 8192, "%s: rows %d, width %d (0 rows or more, 1 to 8192 columns)", what, rows, d);
    SWAT_REQUIRE(!a.gate || (groups >= 1 && rows % groups == 0), "%s: %lld gates do not divide %d rows", what, (long long)groups, rows);
    SWAT_REQUIRE(!a.gate || groups == rows || groups < (1 << 25) / (gate_channels ? 4 * ((d + 255) / 256) : 1), "%s: %lld gates are past one launch", what, (long long)groups);
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
    SWAT_REQUIRE(((uintptr_t)z8_codes & 3) == 0, "swat_residual_norm_fwd: codes sit on 4 bytes");
    const RnPlan p = rn_plan(rows, d, false);
    auto go = [&](auto w, auto n) {
        constexpr int W = decltype(w)::value, N = decltype(n)::value;
        residual_norm_fwd_kernel<W, N><<<mx_grid2(W == 1 ? ((int64_t)rows + 3) / 4 : rows), W == 1 ? 256 : 64 * W, 0, (hipStream_t)stream>>>(a);
    };
    SWAT_REQUIRE((rn_try<1, 1, 2, 3, 4>(p, go) || rn_try<4, 2, 4>(p, go) || rn_try<8, 4>(p, go)), "swat_residual_norm_fwd: no kernel for %d columns", d);
    return check_launch("swat_residual_norm_fwd");
}

static int64_t rn_ws(int rows, int d, int64_t groups, int gate_mode, int64_t* gate_at) {
    const RnPlan p = rn_plan(rows, d, true);
    *gate_at = (int64_t)p.blocks * RN_KINDS * d;
    const int64_t slots = gate_mode == 1 ? rows : gate_mode == 2 ? (p.teams + groups) * (int64_t)d : 0;
    return 4 * (*gate_at + slots);
}

SWAT_API int64_t swat_residual_norm_bwd_workspace_bytes(int rows, int d, int64_t groups, int gate_channels) {
    if (rows < 0 || d < 1 || d > 8192 || groups < 0) {
        set_error("swat_residual_norm_bwd_workspace_bytes: rows %d, width %d, groups %lld", rows, d, (long long)groups);
        return -1;
    }
    int64_t at;
    return rn_ws(rows, d, groups, groups ? (gate_channels ? 2 : 1) : 0, &at);
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
    const RnPlan p = rn_plan(rows, d, true);
    int64_t gate_at;
    const int64_t want = rn_ws(rows, d, a.groups, a.gate_mode, &gate_at);
    SWAT_REQUIRE(rows == 0 || (workspace && workspace_bytes >= want && ((uintptr_t)workspace & 15) == 0),
                 "swat_residual_norm_bwd: workspace of %lld bytes, %lld on 16 bytes are needed", (long long)workspace_bytes, (long long)want);
    a.part = (float*)workspace;
    a.gate_rows = a.part + gate_at;
    a.rows_per_team = p.rows_per_team;
    const hipStream_t s = (hipStream_t)stream;
    if (rows > 0) {
        auto run = [&](auto w, auto n) {
            constexpr int W = decltype(w)::value, N = decltype(n)::value, T = W == 1 ? 8 : 1;
            const bool hz_bf = a.h_bf && (a.z_bf || !dz), gc = a.gate_mode == 2;
            auto go = [&](auto tx, auto thz) {
                constexpr int TX = decltype(tx)::value, THZ = decltype(thz)::value;
                if (gc) residual_norm_bwd_kernel<W, N, T, TX, THZ, true><<<p.blocks, 64 * W * T, 0, s>>>(a);
                else residual_norm_bwd_kernel<W, N, T, TX, THZ, false><<<p.blocks, 64 * W * T, 0, s>>>(a);
            };
            using I0 = std::integral_constant<int, 0>;
            using I1 = std::integral_constant<int, 1>;
            using I2 = std::integral_constant<int, 2>;
            if (hz_bf && !a.x_bf) go(I0{}, I1{});
            else if (hz_bf) go(I1{}, I1{});
            else go(I2{}, I2{});
        };
        SWAT_REQUIRE((rn_try<1, 1, 2, 3>(p, run) || rn_try<4, 1, 2>(p, run) || rn_try<8, 2, 4>(p, run)), "swat_residual_norm_bwd: no kernel for %d columns", d);
    }
    RnFinish f = {};
    f.part = a.part; f.gate_rows = a.gate_rows; f.nblk = p.blocks; f.d = d; f.col_blocks = (d + 15) / 16;
    f.post_w = post_w; f.post_b = post_b; f.scale = scale;
    f.dpost_w = post_w ? dpost_w : nullptr; f.dpost_b = post_b ? dpost_b : nullptr; f.dscale = scale ? dscale : nullptr;
    f.dpre_w = pre_w ? dpre_w : nullptr; f.dpre_b = pre_b ? dpre_b : nullptr;
    f.dgate = dgate; f.groups = a.groups; f.rpg = a.rpg; f.rows_per_team = p.rows_per_team;
    f.gate_mode = a.groups != rows ? a.gate_mode : 0;
    if (rows == 0) f.rpg = 0;  // sums over nothing: zeros
    int64_t grid = 3 * f.col_blocks;
    grid += f.gate_mode == 1 ? (f.groups + 3) / 4 : f.gate_mode == 2 ? f.groups * ((d + 255) / 256) : 0;
    residual_norm_finish_kernel<<<(unsigned)grid, 256, 0, s>>>(f);
    return check_launch("swat_residual_norm_bwd");
}
