// swat_amd/csrc/mx_gemm.hip — C[m, n] = sum_k A[m, k] B[n, k] (+ bias[n]) of two packed matrices (4 or 8 bits each).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 columns of packed elements and applies both operands' block scales inside, with
// fp32 accumulation: nothing is unpacked.  Inside, it adds the products of eight neighbouring columns after aligning them to the largest
// (13 binary places below it are kept, the rest is cut off; measured with cancelling pairs), and those sums, 64 columns at a time, to
// the fp32 accumulator.  e2m1 by e2m1 loses nothing by it (multiples of 1/4 up to 36); with an e4m3 operand up to 2^-13 of the largest
// product can go, which a bfloat16 result does not show and a float32 one would: those products come out in bfloat16 only.
// Lane (r = lane & 15, g = lane >> 4) feeds row r; e2m1: columns 32 g .. + 31 (16 bytes); e4m3: columns 16 g .. + 15 and 64 + 16 g .. + 15; its
// scale operand is the byte of block g of the 128 columns in both.
#include <math.h>
#include <type_traits>
#include "gemm_device.hpp"
#include "mx_device.hpp"
#include "../../include/swat_hip.h"

namespace swat {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef unsigned mx_u4 __attribute__((ext_vector_type(4)));

struct MxGemmArgs {
    const unsigned char *A, *B, *sA, *sB;
    const float* bias;
    void* C;
    int64_t M, N;
    int blocks, out_bf;   // blocks of 32 along k
    int tiles_m, tiles_n;
    int m_begin;          // first row of this launch
};

template <int BITS>
__device__ __forceinline__ constexpr int mx_lds_off(int row, int c) {  // 16-byte chunk c of a row of 128 packed columns
    if constexpr (BITS == 4) return row * 64 + ((c ^ ((row >> 2) & 3)) << 4);
    else return row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
}
// D[n][m] += B[n] . A[m]; the scales are byte S of sb, sa
template <int AB, int BB, int S>
__device__ __forceinline__ f32x4_t mx_mfma(mx_v8i b, mx_v8i a, f32x4_t c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, BB == 4 ? 4 : 0, AB == 4 ? 4 : 0, S, sb, S, sa);
}

// bias[n .. n + 3], n a multiple of 4 (columns past the last: zeros)
__device__ __forceinline__ f32x4_t mx_bias4(const MxGemmArgs& p, int64_t n) {
    f32x4_t b = {0.f, 0.f, 0.f, 0.f};
    if (p.bias) {
        if (n + 4 <= p.N) b = *reinterpret_cast<const f32x4_t*>(p.bias + n);
        else
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (n + e < p.N) b[e] = p.bias[n + e];
    }
    return b;
}
typedef unsigned mx_u2h __attribute__((ext_vector_type(2), aligned(2)));
typedef float mx_f4f __attribute__((ext_vector_type(4), aligned(4)));
// A wave's tile: the lane holds C[m + 16 i][n + 16 j .. + 3].  What the whole launch shares is decided outside the loops and the bias is
// loaded before the first store (which no load would be moved across).
template <int FM, int FN>
__device__ __forceinline__ void mx_store_tile(const MxGemmArgs& p, int64_t m, int64_t n, f32x4_t (&acc)[FM][FN]) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const f32x4_t b = mx_bias4(p, n + 16 * j);
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][j] += b;
    }
    auto rows = [&](auto four, auto one) {   // (rows start on any element where N is no multiple of 4)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            if (m + 16 * i >= p.M) return;
            const int64_t at = (m + 16 * i) * p.N + n;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if (n + 16 * j + 4 <= p.N) four(at + 16 * j, acc[i][j]);
                else
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (n + 16 * j + e < p.N) one(at + 16 * j + e, acc[i][j][e]);
            }
        }
    };
    unsigned short* const cb = (unsigned short*)p.C;
    float* const cf = (float*)p.C;
    if (p.out_bf)
        rows([&](int64_t at, f32x4_t v) { *reinterpret_cast<mx_u2h*>(cb + at) = (mx_u2h){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}; },
             [&](int64_t at, float v) { cb[at] = f2bf(v); });
    else rows([&](int64_t at, f32x4_t v) { *reinterpret_cast<mx_f4f*>(cf + at) = v; }, [&](int64_t at, float v) { cf[at] = v; });
}

// 16 scale bytes of a row from block `first` on.  Rows sit on any byte: where 16 bytes would reach past the matrix's end (last: the row's last
// block with 15 behind it in the matrix, may be negative) the load is moved back and its bytes shifted down (the matrix has 16 bytes at least).
__device__ __forceinline__ mx_u4 mx_scales16(const unsigned char* row, int first, int last) {
    const int to = first <= last ? first : last, sh = first - to;
    uint64_t v[2];
    __builtin_memcpy(v, row + to, 16);
    if (__builtin_amdgcn_ballot_w64(sh != 0)) {   // (a branch of the whole wave: a divergent one in the loop over k would restructure the loop)
        const int by = 8 * (sh & 7);
        const uint64_t lo = sh & 8 ? v[1] : v[0], hi = sh & 8 ? 0 : v[1];
        v[0] = lo >> by | (hi << 1) << (63 - by);
        v[1] = hi >> by;
    }
    return (mx_u4){(unsigned)v[0], (unsigned)(v[0] >> 32), (unsigned)v[1], (unsigned)(v[1] >> 32)};
}

// The tile of this workgroup.  Units of one XCD (workgroups b, b + 8, ..) are neighbours, 4 column tiles wide: its L2 sees few panels of
// either operand.
template <int BM, int BN>
__device__ __forceinline__ void mx_tile(const MxGemmArgs& p, int64_t& m0, int64_t& n0) {
    const int total = gridDim.x, xcd = blockIdx.x & 7, q = total >> 3, r = total & 7;
    const int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (blockIdx.x >> 3);
    const int band = id / (4 * p.tiles_m), wide = p.tiles_n - 4 * band < 4 ? p.tiles_n - 4 * band : 4;
    const int tn = 4 * band + (id - 4 * band * p.tiles_m) % wide, tm = (id - 4 * band * p.tiles_m) / wide;
    m0 = p.m_begin + (int64_t)tm * BM;
    n0 = (int64_t)tn * BN;
}

// The scales of a tile's rows: 16 bytes (four tiles of k) of each at a time, on their way from memory to LDS; a thread takes one or two rows.
// LDS: [A rows | B rows][block of the tile][tile of four].
template <int BM, int BN, int NT>
struct MxScales {
    static constexpr int ROWS = BM + BN, SR = (ROWS + NT - 1) / NT;
    mx_u4 sc[SR];
    const unsigned char* row[SR];
    int last[SR];
    int next;   // group of four tiles to load next
    int blocks;
    __device__ __forceinline__ MxScales(const MxGemmArgs& p, int64_t m0, int64_t n0) : next(0), blocks(p.blocks) {
#pragma unroll
        for (int i = 0; i < SR; ++i) {
            const int r = threadIdx.x + i * NT;
            const bool isa = r < BM;
            const int64_t most = isa ? p.M : p.N, at = isa ? m0 + r : n0 + (r - BM), to = at < most ? at : most - 1;   // (rows past the matrix: any scale)
            row[i] = (isa ? p.sA : p.sB) + to * blocks;
            const int64_t left = (most - to) * blocks - 16;
            last[i] = left < (1 << 30) ? (int)left : 1 << 30;
        }
    }
    __device__ __forceinline__ void load() {
        const int first = 16 * next < blocks ? 16 * next : 0;
#pragma unroll
        for (int i = 0; i < SR; ++i) sc[i] = mx_scales16(row[i], first, last[i]);
    }
    __device__ __forceinline__ void put(unsigned char* to) {
        const int have = blocks - 16 * next;   // blocks of this group inside the row; the rest gets scale byte 0 (zeros times 2^-127)
#pragma unroll
        for (int i = 0; i < SR; ++i) {
            const int r = threadIdx.x + i * NT;
            if (ROWS % NT && r >= ROWS) break;
            unsigned w[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int n = have - 4 * d;
                w[d] = sc[i][d] & (n >= 4 ? ~0u : (1u << 8 * (n > 0 ? n : 0)) - 1u);
            }
            // bytes [tile][block] -> [block][tile]
            const unsigned p0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), p1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
            const unsigned q0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), q1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
            const mx_u4 t = {__builtin_amdgcn_perm(q0, p0, 0x05040100), __builtin_amdgcn_perm(q0, p0, 0x07060302),
                             __builtin_amdgcn_perm(q1, p1, 0x05040100), __builtin_amdgcn_perm(q1, p1, 0x07060302)};
            *reinterpret_cast<mx_u4*>(to + r * 16) = t;
        }
        ++next;
    }
};

// A workgroup computes BM x BN of C in waves of WM x WN, 128 columns at a time: codes go through registers into one of two LDS buffers while
// the matrix cores work on the other, loads two tiles ahead.  A row's scales come 16 bytes (four tiles) at a time, are transposed to
// [block of the tile][tile] and kept in LDS, so that one 4-byte read gives a lane the scales of its row and block for four tiles, which
// the instruction picks by byte.  16384 x 1024 x 4096 in 256 x 256 (8 waves of 128 x 64): 8 by 8 bits 67 us (2.1
// PFLOP/s; matrix pipes busy 45 % of the time by counter, LDS 31), 8 by 4 59.
template <int AB, int BB, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, 2) void mx_gemm_kernel(MxGemmArgs p) {
    constexpr int NT = (BM / WM) * (BN / WN) * 64, FM = WM / 16, FN = WN / 16;
    constexpr int RA = 16 * AB, RB = 16 * BB, CRA = RA / 16, CRB = RB / 16;          // bytes, chunks of a tile's row
    constexpr int CA = BM * CRA / NT, CB = BN * CRB / NT, RSA = NT / CRA, RSB = NT / CRB;   // chunks to a thread and the rows between them
    constexpr int BUF = BM * RA + BN * RB, ROWS = BM + BN;
    static_assert(CA * NT == BM * CRA && CB * NT == BN * CRB && RSA % 16 == 0 && RSB % 16 == 0 && ROWS <= 2 * NT, "whole chunks");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * BUF + 2 * ROWS * 16];
    unsigned char* const ssc = smem + 2 * BUF;   // two groups of scales
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r16 = lane & 15, g = lane >> 4, wr = wave / (BN / WN), wc = wave % (BN / WN);
    int64_t m0, n0;
    mx_tile<BM, BN>(p, m0, n0);
    const int rowA = p.blocks * 4 * AB, rowB = p.blocks * 4 * BB;   // bytes of a packed row
    const int nk = (p.blocks + 3) / 4;

    // codes: buffer descriptors that start at the tile's rows and end with the matrix (rows past it read as zeros), advanced along k;
    // chunks past a row's end get an offset past the end
    constexpr unsigned OUT = 0x80000000u;
    const int rowsA = p.M - m0 < BM ? (int)(p.M - m0) : BM, rowsB = p.N - n0 < BN ? (int)(p.N - n0) : BN;
    const unsigned char *ga = p.A + m0 * rowA, *gb = p.B + n0 * rowB;
    int left = 4 * p.blocks * 4;   // 4-bit bytes of a row still to load: AB / 4 times that of A
    const int ra = tid / CRA, ca = tid % CRA, rb = tid / CRB, cb = tid % CRB;
    const unsigned oa = (unsigned)(ra * rowA + ca * 16), ob = (unsigned)(rb * rowB + cb * 16);
    unsigned char *const wa = smem + mx_lds_off<AB>(ra, ca), *const wb = smem + BM * RA + mx_lds_off<BB>(rb, cb);
    struct Stage {
        mx_u4 a[CA], b[CB];
    };
    constexpr bool DEEP = WM * WN <= 4096 && AB + BB < 16;   // two tiles of loads in flight; one where the registers do not reach
    Stage st0, st1_;
    Stage& st1 = DEEP ? st1_ : st0;
    auto load = [&](Stage& st) {
        const int la = left * (AB / 4), lb = left * (BB / 4);   // (<= 0: past the last tile)
        const __amdgpu_buffer_rsrc_t da = __builtin_amdgcn_make_buffer_rsrc((void*)ga, 0, la > 0 ? (rowsA - 1) * rowA + la : 0, 0x20000);
        const __amdgpu_buffer_rsrc_t db = __builtin_amdgcn_make_buffer_rsrc((void*)gb, 0, lb > 0 ? (rowsB - 1) * rowB + lb : 0, 0x20000);
        const unsigned pa = ca * 16 < la ? oa : OUT, pb = cb * 16 < lb ? ob : OUT;
#pragma unroll
        for (int i = 0; i < CA; ++i) st.a[i] = __builtin_amdgcn_raw_buffer_load_b128(da, pa + (unsigned)(i * RSA * rowA), 0, 0);
#pragma unroll
        for (int i = 0; i < CB; ++i) st.b[i] = __builtin_amdgcn_raw_buffer_load_b128(db, pb + (unsigned)(i * RSB * rowB), 0, 0);
        ga += RA;
        gb += RB;
        left -= 64;
    };
    auto put = [&](const Stage& st, int buf) {
#pragma unroll
        for (int i = 0; i < CA; ++i) *reinterpret_cast<mx_u4*>(wa + buf * BUF + i * RSA * RA) = st.a[i];
#pragma unroll
        for (int i = 0; i < CB; ++i) *reinterpret_cast<mx_u4*>(wb + buf * BUF + i * RSB * RB) = st.b[i];
    };
    MxScales<BM, BN, NT> sc(p, m0, n0);
    auto bar = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    int sa[FM], sb[FN];
    auto read_scales = [&](int buf) {
        const unsigned char* q = ssc + buf * ROWS * 16 + 4 * g;
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = *reinterpret_cast<const int*>(q + (WM * wr + 16 * i + r16) * 16);
#pragma unroll
        for (int j = 0; j < FN; ++j) sb[j] = *reinterpret_cast<const int*>(q + (BM + WN * wc + 16 * j + r16) * 16);
    };
    // (fragment rows are 16 apart: the chunk permutation depends on r16 alone)
    const unsigned char* const pa0 = smem + WM * wr * RA + mx_lds_off<AB>(r16, g);
    const unsigned char* const pa1 = smem + WM * wr * RA + mx_lds_off<AB>(r16, AB == 8 ? 4 + g : g);
    const unsigned char* const pb0 = smem + BM * RA + WN * wc * RB + mx_lds_off<BB>(r16, g);
    const unsigned char* const pb1 = smem + BM * RA + WN * wc * RB + mx_lds_off<BB>(r16, BB == 8 ? 4 + g : g);
    auto frag = [&](const unsigned char* lo, const unsigned char* hi, auto bits) {
        const mx_u4 l = *reinterpret_cast<const mx_u4*>(lo);
        mx_v8i v = {(int)l[0], (int)l[1], (int)l[2], (int)l[3], 0, 0, 0, 0};
        if constexpr (decltype(bits)::value == 8) {
            const mx_u4 h = *reinterpret_cast<const mx_u4*>(hi);
            v[4] = (int)h[0]; v[5] = (int)h[1]; v[6] = (int)h[2]; v[7] = (int)h[3];
        }
        return v;
    };
    auto multiply = [&](int buf, auto tile) {
        constexpr int S = decltype(tile)::value;
        mx_v8i fb[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = frag(pb0 + buf * BUF + 16 * j * RB, pb1 + buf * BUF + 16 * j * RB, std::integral_constant<int, BB>{});
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const mx_v8i fa = frag(pa0 + buf * BUF + 16 * i * RA, pa1 + buf * BUF + 16 * i * RA, std::integral_constant<int, AB>{});
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mx_mfma<AB, BB, S>(fb[j], fa, acc[i][j], sb[j], sa[i]);
        }
    };

    sc.load();
    load(st0);
    if constexpr (DEEP) load(st1);
    sc.put(ssc);
    sc.load();
    put(st0, 0);
    load(st0);
    bar();
    int t = 0;
    for (int sbuf = 0;; sbuf ^= 1) {
        read_scales(sbuf);
        put(st1, 1);
        load(st1);
        multiply(0, std::integral_constant<int, 0>{});
        bar();
        if (++t >= nk) break;
        put(st0, 0);
        load(st0);
        multiply(1, std::integral_constant<int, 1>{});
        bar();
        if (++t >= nk) break;
        put(st1, 1);
        load(st1);
        sc.put(ssc + (sbuf ^ 1) * ROWS * 16);   // (read last two tiles ago)
        sc.load();
        multiply(0, std::integral_constant<int, 2>{});
        bar();
        if (++t >= nk) break;
        put(st0, 0);
        load(st0);
        multiply(1, std::integral_constant<int, 3>{});
        bar();
        if (++t >= nk) break;
    }
    mx_store_tile(p, m0 + WM * wr + r16, n0 + WN * wc + 4 * g, acc);
}

// The same for 4 by 4 bits in tiles of 128 and more, whose codes come straight into LDS, three tiles ahead, in a ring of four buffers: the loads
// cost no registers, so that there is room to read the next tile's B and half of its A while this tile's second half multiplies, and they
// may take the time of two tiles.  16448 x 1024 x 4096: 54.5 -> 47.7 us, 8192^3 323 -> 273 (4.0 PFLOP/s; in 128 x 128 405 -> 386).  Bound by
// the matrix cores and LDS in turn (busy 42 and 37 % of the time by counter): 16384 x 1024 x 4096 takes 42 us, 72 % of its time without loads and
// LDS reads, and 16 is what the matrix instructions take from registers with every CU on them (8.7 PFLOP/s).
// What a load past an edge leaves in LDS (the next row's codes, zeros or older codes) is multiplied by block scales of zero bytes, 2^-127 on
// both sides, or belongs to rows that are not stored: an e2m1 code is always finite.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, 2) void mx_ring_kernel(MxGemmArgs p) {
    constexpr int NW = (BM / WM) * (BN / WN), NT = 64 * NW, FM = WM / 16, FN = WN / 16;
    constexpr int ROWS = BM + BN, BUF = 64 * ROWS, LOADS = ROWS / NW / 16;   // a tile: 64 bytes of each row; loads to a wave
    static_assert(BM % (16 * NW) == 0 && BN % (16 * NW) == 0 && 2 * LOADS < 16, "whole loads; their count fits the wait");
    __shared__ __attribute__((aligned(1024))) unsigned char ring0[BUF], ring1[BUF], ring2[BUF], ring3[BUF];
    __shared__ __attribute__((aligned(1024))) unsigned char ssc[2 * ROWS * 16];   // two groups of scales
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4, wr = wave / (BN / WN), wc = wave % (BN / WN);
    int64_t m0, n0;
    mx_tile<BM, BN>(p, m0, n0);
    const int row = p.blocks * 16;   // bytes of a packed row
    const int nk = (p.blocks + 3) / 4;

    // codes: buffer descriptors that start at the tile's rows and end with the matrix, advanced along k
    const int rowsA = p.M - m0 < BM ? (int)(p.M - m0) : BM, rowsB = p.N - n0 < BN ? (int)(p.N - n0) : BN;
    const unsigned char *ga = p.A + m0 * row, *gb = p.B + n0 * row;
    int left = row;   // bytes of a row still to load (<= 0: past the last tile)
    // a load fills 16 rows in LDS, lane l bytes 16 l .. of them: the permutation is on what a lane loads
    const int lr = lane >> 2, lc = (lane & 3) ^ ((lane >> 4) & 3);
    const unsigned oa = (unsigned)((wave * (BM / NW) + lr) * row + lc * 16), ob = (unsigned)((wave * (BN / NW) + lr) * row + lc * 16);
    auto ring = [&](auto n) -> unsigned char* {
        constexpr int R = decltype(n)::value & 3;
        if constexpr (R == 0) return ring0;
        else if constexpr (R == 1) return ring1;
        else if constexpr (R == 2) return ring2;
        else return ring3;
    };
    auto load = [&](auto n) {
        unsigned char* to = ring(n);
        const __amdgpu_buffer_rsrc_t da = __builtin_amdgcn_make_buffer_rsrc((void*)ga, 0, left > 0 ? (rowsA - 1) * row + left : 0, 0x20000);
        const __amdgpu_buffer_rsrc_t db = __builtin_amdgcn_make_buffer_rsrc((void*)gb, 0, left > 0 ? (rowsB - 1) * row + left : 0, 0x20000);
#pragma unroll
        for (int i = 0; i < BM / NW / 16; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(da, (__attribute__((address_space(3))) void*)(to + (wave * (BM / NW) + 16 * i) * 64), 16, oa + (unsigned)(16 * i * row), 0, 0, 0);
#pragma unroll
        for (int i = 0; i < BN / NW / 16; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(db, (__attribute__((address_space(3))) void*)(to + BM * 64 + (wave * (BN / NW) + 16 * i) * 64), 16, ob + (unsigned)(16 * i * row), 0, 0, 0);
        ga += 64;
        gb += 64;
        left -= 64;
    };
    MxScales<BM, BN, NT> sc(p, m0, n0);
    auto bar = [&]() {   // (all but the newest two tiles' loads)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x70 | (2 * LOADS));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    int sa[FM], sb[FN];
    auto read_scales = [&](int buf) {
        const unsigned char* q = ssc + buf * ROWS * 16 + 4 * g;
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = *reinterpret_cast<const int*>(q + (WM * wr + 16 * i + r16) * 16);
#pragma unroll
        for (int j = 0; j < FN; ++j) sb[j] = *reinterpret_cast<const int*>(q + (BM + WN * wc + 16 * j + r16) * 16);
    };
    int fa0 = WM * wr * 64 + mx_lds_off<4>(r16, g), fb0 = (BM + WN * wc) * 64 + mx_lds_off<4>(r16, g);
    mx_u4 qa[FM], qb[2][FN];
    auto read_a = [&](auto n, auto half) {
        constexpr int I0 = decltype(half)::value * (FM / 2);
        const unsigned char* q = ring(n) + fa0;
#pragma unroll
        for (int i = I0; i < I0 + FM / 2; ++i) qa[i] = *reinterpret_cast<const mx_u4*>(q + 16 * i * 64);
    };
    auto read_b = [&](auto n) {
        const unsigned char* q = ring(n) + fb0;
#pragma unroll
        for (int j = 0; j < FN; ++j) qb[decltype(n)::value & 1][j] = *reinterpret_cast<const mx_u4*>(q + 16 * j * 64);
    };
    auto four = [](mx_u4 v) { return (mx_v8i){(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };
    auto half_tile = [&](auto n, auto half) {
        constexpr int I0 = decltype(half)::value * (FM / 2), S = decltype(n)::value;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = I0; i < I0 + FM / 2; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mx_mfma<4, 4, S>(four(qb[S & 1][j]), four(qa[i]), acc[i][j], sb[j], sa[i]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, 0> H0{};
    constexpr std::integral_constant<int, 1> H1{};
    auto step = [&](auto n, int sbuf) {
        constexpr int S = decltype(n)::value;
        constexpr std::integral_constant<int, (S + 1) & 3> N1{};
        constexpr std::integral_constant<int, (S + 3) & 3> N3{};
        asm volatile("" : "+v"(fa0), "+v"(fb0));   // (sums of these and a buffer's address are made anew, not kept in registers)
        if constexpr (S == 0) read_scales(sbuf);
        read_a(n, H1);
        __builtin_amdgcn_sched_barrier(0);
        load(N3);
        if constexpr (S == 2) {
            sc.put(ssc + (sbuf ^ 1) * ROWS * 16);   // (read last two tiles ago)
            sc.load();
        }
        __builtin_amdgcn_sched_barrier(0);
        half_tile(n, H0);
        bar();
        read_b(N1);
        read_a(N1, H0);
        __builtin_amdgcn_sched_barrier(0);
        half_tile(n, H1);
    };
    constexpr std::integral_constant<int, 0> T0{};
    constexpr std::integral_constant<int, 1> T1{};
    constexpr std::integral_constant<int, 2> T2{};
    constexpr std::integral_constant<int, 3> T3{};
    sc.load();
    load(T0);
    load(T1);
    load(T2);
    sc.put(ssc);
    sc.load();
    bar();
    read_b(T0);
    read_a(T0, H0);
    int t = 0;
    for (int sbuf = 0;; sbuf ^= 1) {   // (a tile past the last one multiplies by scales of zero)
        step(T0, sbuf);
        step(T1, sbuf);
        if ((t += 2) >= nk) break;
        step(T2, sbuf);
        step(T3, sbuf);
        if ((t += 2) >= nk) break;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load may reach LDS after the workgroup has left it)
    mx_store_tile(p, m0 + WM * wr + r16, n0 + WN * wc + 4 * g, acc);
}

// Few rows: a workgroup computes 16 columns of 16 FM rows, its 8 waves take the 128-column tiles of k in turn, straight from memory into
// registers (nothing is used twice), and their sums meet in LDS in the order of the waves.  Bound by latency and B's bytes.  Addresses past
// an edge are moved to readable ones and what they load is replaced by zeros, so that all loads of several tiles go out together.
template <int AB, int BB, int FM>
__global__ __launch_bounds__(512, 2) void mx_rows_kernel(MxGemmArgs p) {
    __shared__ f32x4_t part[8][FM][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    p.m_begin += (int)blockIdx.x / p.tiles_n * (16 * FM);
    const int64_t n0 = (int64_t)((int)blockIdx.x % p.tiles_n) * 16, n = n0 + r16;
    const int64_t rowA = (int64_t)p.blocks * 4 * AB, rowB = (int64_t)p.blocks * 4 * BB;
    f32x4_t acc[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    auto piece = [&](const unsigned char* row, int at, bool live) {
        mx_u4 v = *reinterpret_cast<const mx_u4*>(row + (live ? at : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = live ? v[e] : 0u;
        return v;
    };
    auto frag = [&](const unsigned char* row, int kt, bool live, auto bits) {
        constexpr int BITS = decltype(bits)::value;
        mx_v8i v = {0, 0, 0, 0, 0, 0, 0, 0};
        if constexpr (BITS == 4) {
            const mx_u4 l = piece(row, 64 * kt + 16 * g, live && 4 * kt + g < p.blocks);
            v[0] = (int)l[0]; v[1] = (int)l[1]; v[2] = (int)l[2]; v[3] = (int)l[3];
        } else {   // columns 16 g .. and 64 + 16 g ..: half a block each
            const mx_u4 l = piece(row, 128 * kt + 16 * g, live && 4 * kt + g / 2 < p.blocks);
            const mx_u4 h = piece(row, 128 * kt + 64 + 16 * g, live && 4 * kt + 2 + g / 2 < p.blocks);
            v[0] = (int)l[0]; v[1] = (int)l[1]; v[2] = (int)l[2]; v[3] = (int)l[3];
            v[4] = (int)h[0]; v[5] = (int)h[1]; v[6] = (int)h[2]; v[7] = (int)h[3];
        }
        return v;
    };
    const int nk = (p.blocks + 3) / 4;
    const bool live_n = n < p.N;
    const int64_t nn = live_n ? n : n0;
    const unsigned char *bp = p.B + nn * rowB, *bs = p.sB + nn * p.blocks;
    const unsigned char *ap[FM], *as[FM];
    bool live_m[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t m = p.m_begin + 16 * i + r16;
        live_m[i] = m < p.M;
        const int64_t mm = live_m[i] ? m : p.m_begin;
        ap[i] = p.A + mm * rowA;
        as[i] = p.sA + mm * p.blocks;
    }
    auto tiles = [&](int kt0, auto count) {   // `count` tiles of k, 8 apart: loads first, then the products in order
        constexpr int C = decltype(count)::value;
        mx_v8i fb[C], fa[C][FM];
        int sb[C], sa[C][FM];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int kt = kt0 + 8 * c;
            const bool inside = 4 * kt + g < p.blocks;
            const int ks = inside ? 4 * kt + g : 0;
            fb[c] = frag(bp, kt, live_n, std::integral_constant<int, BB>{});
            sb[c] = bs[ks];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                fa[c][i] = frag(ap[i], kt, live_m[i], std::integral_constant<int, AB>{});
                sa[c][i] = as[i][ks];
            }
            sb[c] = inside ? sb[c] : 0;
#pragma unroll
            for (int i = 0; i < FM; ++i) sa[c][i] = inside ? sa[c][i] : 0;
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[i] = mx_mfma<AB, BB, 0>(fb[c], fa[c][i], acc[i], sb[c], sa[c][i]);
    };
    int kt = wave;
    constexpr int AHEAD = FM == 4 && AB + BB > 8 ? 2 : 4;
    for (; kt + 8 * (AHEAD - 1) < nk; kt += 8 * AHEAD) tiles(kt, std::integral_constant<int, AHEAD>{});
    for (; kt < nk; kt += 8) tiles(kt, std::integral_constant<int, 1>{});
#pragma unroll
    for (int i = 0; i < FM; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave < FM) {
        f32x4_t s = part[0][wave][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) s += part[w][wave][lane];
        f32x4_t one[1][1] = {{s}};
        mx_store_tile(p, p.m_begin + 16 * wave + r16, n0 + 4 * g, one);
    }
}

template <int AB, int BB>
static bool mx_rows(MxGemmArgs p, int64_t m_begin, int rows, hipStream_t s) {
    // a workgroup to each 16-row part while they stay within 2 to a CU (64 rows, 4 bits, k 4096: 1024 columns 5.7 us with 256 workgroups,
    // 10.9 with 64; k 1024: 4096 columns 5.8 with 1024, 4.8 with 256)
    p.m_begin = (int)m_begin;
    p.tiles_n = (int)((p.N + 15) / 16);
    const int64_t parts = (rows + 15) / 16, few = p.tiles_n * parts, many = p.tiles_n * ((parts + 3) / 4);
    if (many >= 1 << 23) return false;   // (2^32 threads)
    if (few <= 512) mx_rows_kernel<AB, BB, 1><<<(unsigned)few, 512, 0, s>>>(p);
    else mx_rows_kernel<AB, BB, 4><<<(unsigned)many, 512, 0, s>>>(p);
    return true;
}
template <int AB, int BB, int BM, int BN, int WM, int WN>
static bool mx_tiles(MxGemmArgs p, int64_t rows, hipStream_t s) {
    p.M = rows;   // (rows behind them, if any, go to mx_rows)
    p.tiles_m = (int)((rows + BM - 1) / BM);
    p.tiles_n = (int)((p.N + BN - 1) / BN);
    const int64_t grid = (int64_t)p.tiles_m * p.tiles_n;
    if (grid >= 1 << 23) return false;
    if constexpr (AB + BB == 8 && BM >= 128) mx_ring_kernel<BM, BN, WM, WN><<<(unsigned)grid, (BM / WM) * (BN / WN) * 64, 0, s>>>(p);
    else mx_gemm_kernel<AB, BB, BM, BN, WM, WN><<<(unsigned)grid, (BM / WM) * (BN / WN) * 64, 0, s>>>(p);
    return true;
}

// Which tile, by the sum of what was measured (us): a 128-column step takes a CU, 4 by 4 bits, 0.8 with five 64 x 64 workgroups on it (0.25
// with one), 0.73 with two of 128 x 128 (0.4 with one), 0.97 with one of 256 x 256; with 8-bit operands 0.8, 0.78 (0.45), 1.2 and 28 % more
// for each of them; a round of workgroups 2.5, 3.5, 7 more (the last is alone on its CU while it stores).  Up to 64 rows past whole tiles
// may go to mx_rows (5) instead of a round of their own.  Few rows and columns: mx_rows.
//   4 x 4 bits, 64 x 64 / 128 x 128 / 256 x 256: 1600 x 768 x 768 10.4 / 10.1 / 17.1; 4096 x 1024 x 1024 11.6 / 10.1 / 16.9; 2048 x 4096 x 4096 62 /
//   31.9 / 36.2; 8239 x 2048 x 1000 36 / 27.9 / 25.6; 16448 x 1024 x 4096 108 / 66 / 47.7; 8192^3 797 / 386 / 273.   64 rows, 1024 x 4096 5.7 in
//   mx_rows, 11.1 in 64 x 64; 64 rows, 65536 x 512 20 and 8.2
struct MxGemmPlan {
    int size;        // 0: mx_rows, 1: 64 x 64, 2: 128 x 128, 3: 256 x 256
    int64_t rows;    // those of the tile kernel; what is behind goes to mx_rows
};
static MxGemmPlan mx_plan(int64_t M, int64_t N, int blocks, int ab, int bb) {
    const int64_t cols16 = (N + 15) / 16;
    // (fewer than 16 scale bytes in an operand: the tile kernels load them by 16)
    if ((M <= 64 && cols16 <= 512) || M * blocks < 16 || N * blocks < 16) return {0, 0};
    static const double full4[4] = {0, 0.8, 0.73, 0.97}, alone4[4] = {0, 0.25, 0.4, 0.97}, full8[4] = {0, 0.8, 0.78, 1.2}, alone8[4] = {0, 0.25, 0.45, 1.2};
    static const double round[4] = {0, 2.5, 3.5, 7.0};
    const double *full = ab + bb == 8 ? full4 : full8, *alone = ab + bb == 8 ? alone4 : alone8;
    static const int slots[4] = {0, 5, 2, 1};
    const double f = 1.0 + 0.07 * (ab + bb - 8), steps = (blocks + 3) / 4;
    MxGemmPlan best = {};
    double cost = -1;
    for (int size = 1; size <= 3; ++size) {
        const int b = 32 << size;
        const int64_t tn = (N + b - 1) / b, rem = M % b;
        for (int tail = 0; tail < 2; ++tail) {
            if (tail && !(rem > 0 && rem <= 64 && M > b && size > 1)) continue;
            const double tiles = (double)tn * (tail ? M / b : (M + b - 1) / b), per = 256.0 * slots[size];
            const double whole = floor(tiles / per), rest = ceil((tiles - whole * per) / 256.0);   // workgroups to a CU in the last round
            const double one = slots[size] > 1 ? (full[size] - alone[size]) / (slots[size] - 1) : 0.0;
            double c = 4.0 + whole * (steps * full[size] * f + round[size]);
            if (rest > 0) c += steps * (slots[size] > 1 ? alone[size] + (rest - 1) * one : full[size]) * f + round[size];
            if (tail) c += 5.0;
            if (cost < 0 || c < cost) {
                cost = c;
                best = {size, tail ? M - rem : M};
            }
        }
    }
    return best;
}
template <int AB, int BB>
static bool mx_product(const MxGemmArgs& p, hipStream_t s) {
    const MxGemmPlan pl = mx_plan(p.M, p.N, p.blocks, AB, BB);
    const bool ok = pl.size == 1   ? mx_tiles<AB, BB, 64, 64, 32, 32>(p, pl.rows, s)
                    : pl.size == 2 ? mx_tiles<AB, BB, 128, 128, 64, 64>(p, pl.rows, s)
                    : pl.size == 3 ? mx_tiles<AB, BB, 256, 256, 128, 64>(p, pl.rows, s)
                                   : true;
    return ok && (pl.rows == p.M || mx_rows<AB, BB>(p, pl.rows, (int)(p.M - pl.rows), s));
}

}  // namespace swat

using namespace swat;

SWAT_API int swat_mx_matmul(const void* a_codes, const void* a_scales, int a_bits, const void* b_codes, const void* b_scales, int b_bits,
                            const float* bias, void* c, int c_dtype, int64_t M, int64_t N, int K, swat_stream_t stream) {
    SWAT_REQUIRE((a_bits == 4 || a_bits == 8) && (b_bits == 4 || b_bits == 8), "swat_mx_matmul: %d and %d bits (4 or 8 each)", a_bits, b_bits);
    SWAT_REQUIRE(M >= 0 && N >= 0 && K >= 1 && K <= (1 << 22) && M <= (1 << 30) && N <= (1 << 30), "swat_mx_matmul: %lld x %lld x %d", (long long)M, (long long)N, K);
    SWAT_REQUIRE(c_dtype == SWAT_BF16 || (c_dtype == SWAT_F32 && a_bits == 4 && b_bits == 4), "swat_mx_matmul: output type %d of %d by %d bits (bf16; fp32 where both have 4 bits)", c_dtype, a_bits, b_bits);
    if (M == 0 || N == 0) return 0;
    SWAT_REQUIRE(a_codes && a_scales && b_codes && b_scales && c, "swat_mx_matmul: both operands and the output are needed");
    SWAT_REQUIRE(!(((uintptr_t)a_codes | (uintptr_t)b_codes | (uintptr_t)c | (uintptr_t)bias) & 15), "swat_mx_matmul: codes, bias and output sit on 16 bytes");
    MxGemmArgs p = {};
    p.A = (const unsigned char*)a_codes; p.sA = (const unsigned char*)a_scales; p.B = (const unsigned char*)b_codes; p.sB = (const unsigned char*)b_scales;
    p.bias = bias; p.C = c; p.M = M; p.N = N; p.blocks = (K + 31) / 32; p.out_bf = c_dtype == SWAT_BF16;
    const hipStream_t s = (hipStream_t)stream;
    const bool ok = a_bits == 4 ? (b_bits == 4 ? mx_product<4, 4>(p, s) : mx_product<4, 8>(p, s))
                                : (b_bits == 4 ? mx_product<8, 4>(p, s) : mx_product<8, 8>(p, s));
    SWAT_REQUIRE(ok, "swat_mx_matmul: %lld x %lld is past one launch", (long long)M, (long long)N);
    return check_launch("swat_mx_matmul");
}
