// swat_amd/csrc/mx_wgrad.hip — the weight gradient of a linear layer whose input was kept as an 8-bit checkpoint:
//
//   dW[n, k] = sum_m dY[m, n] X8[m, k],   db[n] = sum_m dY[m, n]
//
// dY bfloat16, X8 e4m3 with a power-of-two scale to 32 columns.  An e4m3 number times such a scale is a bfloat16 number, so the
// checkpoint is unpacked on its way into LDS without a rounding and v_mfma_f32_16x16x32_bf16 sees what was stored.  The reduction
// runs over rows: both tiles lie [64 rows][128 columns] in LDS and are read with the transposing LDS load.
#include "gemm_device.hpp"
#include "mx_device.hpp"
#include "../../include/swat_hip.h"

namespace swat {

struct MxWgradArgs {
    const unsigned short* dY;
    const unsigned char *X, *S;
    float *dW, *db;
    int64_t rows, ld;   // rows; row stride of dY
    int n, k, blocks;
    int tiles_n, tiles_k;
    int vec;            // dY rows on 16 bytes, n % 8 == 0
};

__global__ __launch_bounds__(256) void mx_wgrad_kernel(MxWgradArgs p) {
    __shared__ __attribute__((aligned(1024))) unsigned char ty[64 * 256], tx[64 * 256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r16 = lane & 15, g = lane >> 4, wr = wave >> 1, wc = wave & 1;
    const int n0 = (blockIdx.x % p.tiles_n) * 128, k0 = (blockIdx.x / p.tiles_n) * 128;
    f32x4_t acc[4][4], accs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        accs[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    const bool sums = p.db && k0 == 0 && wc == 0;
    bf16x8_t ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (__bf16)1.0f;
    for (int64_t m0 = 0; m0 < p.rows; m0 += 64) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = i * 256 + tid, row = at >> 4, c = at & 15;   // 16 chunks of 8 columns to a row
            const int64_t m = m0 + row;
            {
                const int col = n0 + 8 * c;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (m < p.rows && col < p.n) {
                    const unsigned short* src = p.dY + m * p.ld + col;
                    if (p.vec) v = *reinterpret_cast<const uint4*>(src);
                    else {
                        unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + e < p.n) w[e >> 1] |= (unsigned)src[e] << (16 * (e & 1));
                        v = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                *reinterpret_cast<uint4*>(ty + st_off<128>(row, c)) = v;
            }
            {
                const int col = k0 + 8 * c;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (m < p.rows && col < 32 * p.blocks) {
                    const uint2 q = *reinterpret_cast<const uint2*>(p.X + m * (32 * (int64_t)p.blocks) + col);
                    const float s = mx_scale(p.S[m * p.blocks + (col >> 5)]);
                    float f[8];
                    mx_from_e4m3x4(q.x, s, f);
                    mx_from_e4m3x4(q.y, s, f + 4);
                    v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
                }
                *reinterpret_cast<uint4*>(tx + st_off<128>(row, c)) = v;
            }
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8_t fx[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) fx[j] = read_frag<false, 128>(tx, 64 * wc + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8_t fy = read_frag<false, 128>(ty, 64 * wr + 16 * i, ks, lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[j], fy, acc[i][j], 0, 0, 0);
                if (sums) accs[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, fy, accs[i], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + 64 * wr + 16 * i + r16;
        if (n >= p.n) continue;
        if (sums && g == 0) p.db[n] = accs[i][0];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + 64 * wc + 16 * j + 4 * g;
            float* out = p.dW + (int64_t)n * p.k + k;
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

}  // namespace swat

using namespace swat;

SWAT_API int64_t swat_mx_linear_wgrad_workspace_bytes(int64_t rows, int n_out, int n_in) { return 0; }

SWAT_API int swat_mx_linear_wgrad(const void* dY_bf16, int64_t dy_stride, const void* x_codes, const void* x_scales, float* dW, float* dbias,
                                  int64_t rows, int n_out, int n_in, void* workspace, int64_t workspace_bytes, swat_stream_t stream) {
    SWAT_REQUIRE(rows >= 0 && n_out >= 0 && n_in >= 0 && n_out <= (1 << 24) && n_in <= (1 << 24), "swat_mx_linear_wgrad: %lld rows, %d x %d", (long long)rows, n_out, n_in);
    if (n_out == 0 || n_in == 0) return 0;
    SWAT_REQUIRE(dW && (rows == 0 || (dY_bf16 && x_codes && x_scales)), "swat_mx_linear_wgrad: dY, the checkpoint and dW are needed");
    SWAT_REQUIRE(rows == 0 || dy_stride >= n_out, "swat_mx_linear_wgrad: row stride %lld under %d columns", (long long)dy_stride, n_out);
    SWAT_REQUIRE(!(((uintptr_t)x_codes | (uintptr_t)dW) & 15), "swat_mx_linear_wgrad: codes and dW sit on 16 bytes");
    MxWgradArgs p = {};
    p.dY = (const unsigned short*)dY_bf16; p.X = (const unsigned char*)x_codes; p.S = (const unsigned char*)x_scales; p.dW = dW; p.db = dbias;
    p.rows = rows; p.ld = dy_stride; p.n = n_out; p.k = n_in; p.blocks = (n_in + 31) / 32;
    p.vec = n_out % 8 == 0 && dy_stride % 8 == 0 && ((uintptr_t)dY_bf16 & 15) == 0;
    p.tiles_n = (n_out + 127) / 128; p.tiles_k = (n_in + 127) / 128;
    const int64_t grid = (int64_t)p.tiles_n * p.tiles_k;
    SWAT_REQUIRE(grid < (1ll << 31), "swat_mx_linear_wgrad: %d x %d is past one launch", n_out, n_in);
    mx_wgrad_kernel<<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(p);
    return check_launch("swat_mx_linear_wgrad");
}
