// sdh_dense.hip — dense Q8_0 weight x 8-bit activations: y[t][o] = sum_b dw[o][b] dx[t][b] sum_{k in b} qw[o][k] qx[t][k].
//
// The integer sum of a block of 32 is exact (at most 32 * 127 * 128 < 2^20); the two scales multiply it once in F32 and the
// blocks are summed in F32.
//
//   dense_few_kernel   one token: bound by the stream of the weight; v_dot4_i32_i8.
//   dense_thin_kernel, dense_mid_kernel
//                      a batch: 16 to 64 rows of v_mfma_i32_16x16x32_i8 or 32 x 32 tiles of v_mfma_i32_32x32x32_i8, whose K is exactly
//                      one block, straight from memory.
//   dense_mfma_kernel  a prompt: tiles of 64 x 64 to 128 x 128 through LDS; most of its time is the vector pipe's (integers to F32).
#include "sdh_internal.h"

#include <algorithm>
#include <hip/hip_fp16.h>

namespace sdh {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v32f __attribute__((ext_vector_type(32)));

struct DenseArgs {
    const int8_t * wq; const __half * wd;      // [n_out][n_in], [n_out][nblk]
    const int8_t * xq; int64_t ldq;
    const float * xd; int64_t ldd;
    int n_out, nblk;                           // n_in = 32 * nblk
    int64_t T;
    float * y; int64_t ldy;
};

// A wave owns R rows; chunk c of 16 bytes (half a block) of a row belongs to lane c & 63, so a load instruction takes 1 KB of
// consecutive bytes, U of them per row in flight; neighbouring lanes join their halves of a block as integers. The tokens' chunks
// come from the cache; no LDS, no barrier. One token x 4096 -> 14336: 11.6 us, 5.4 TB/s (62.4 MB; torch's copy of a large tensor 4.95);
// a block per lane, two loads 32 bytes apart, took 22.8 us, four rows per wave 13.3 to 13.9 us, one row 10.5 us without the
// exchange of halves against 10.6 for two.
template <int TT, int R, int U>
__global__ __launch_bounds__(256) void dense_few_kernel(const DenseArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o0 = ((int) blockIdx.x * 4 + wave) * R;
    const int64_t t0 = (int64_t) blockIdx.y * TT;
    if (o0 >= a.n_out) return;
    const int64_t n_in = (int64_t) a.nblk * 32;
    const int n_ch = 2 * a.nblk;
    float acc[TT][R];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[t][r] = 0.0f;
    const int8_t * wp[R];
    const __half * dp[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {                             // rows past the end: the last one, not stored
        const int64_t row = min(o0 + r, a.n_out - 1);
        wp[r] = a.wq + row * n_in;
        dp[r] = a.wd + row * a.nblk;
    }
    for (int c0 = lane; c0 < n_ch; c0 += 64 * U) {
        v4i w[U][R];
        float dw[U][R];
        int c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {                         // even lanes count; chunks past the end: the last one, both scales zero (one may be infinite)
            c[u] = min(c0 + 64 * u, n_ch - 1);
            const int counts = c0 + 64 * u < n_ch && !(lane & 1) ? -1 : 0;      // as a mask: a choice would make the load conditional (16.4 us for one token)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                w[u][r] = __builtin_nontemporal_load(reinterpret_cast<const v4i *>(wp[r] + (int64_t) c[u] * 16));
                dw[u][r] = __int_as_float(__float_as_int(__half2float(dp[r][c[u] >> 1])) & counts);
            }
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int64_t tt = min(t0 + t, a.T - 1);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const v4i x = *reinterpret_cast<const v4i *>(a.xq + tt * a.ldq + (int64_t) c[u] * 16);
                const float dx = c0 + 64 * u < n_ch && !(lane & 1) ? a.xd[tt * a.ldd + (c[u] >> 1)] : 0.0f;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    int s = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) s = __builtin_amdgcn_sdot4(w[u][r][k], x[k], s, false);
                    s += __builtin_amdgcn_update_dpp(0, s, 0xB1, 0xF, 0xF, true);      // the neighbour's half of the block
                    acc[t][r] = fmaf((float) s, dw[u][r] * dx, acc[t][r]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v = acc[t][r];
            for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
            if (lane == 0 && t0 + t < a.T && o0 + r < a.n_out) a.y[(t0 + t) * a.ldy + o0 + r] = v;
        }
}

// 32 tokens x 32 rows per workgroup: still the stream of the weight. The waves split K in groups of four blocks (128 bytes, a whole
// line of a row) and are joined in LDS at the end; the next group is asked for before the present one is multiplied, without a
// barrier anywhere in the loop.
//   loads      128 consecutive bytes of 8 rows per instruction, turned into fragments in a corner of LDS of the wave's own (16-byte
//              chunks at chunk ^ ((row >> 1) & 7): no bank twice; LDS works in order within a wave). Fragments straight from memory put
//              neighbouring lanes into different rows, a cache access per lane: 27.4 us against 22.1 for 11 tokens x 14336 -> 4096,
//              39 against 23 for 32 tokens.
//   fragments  v_mfma_i32_32x32x32_i8: lane = row (or token) lane & 31, the 16 bytes of half lane >> 5 of the block; the result has
//              token 8 (i / 4) + 4 (lane >> 5) + i % 4 in register i and row lane & 31.
//   scales     four of a row as one 8-byte load (whatever its alignment; one by one they took as long as the weight); the tokens' are
//              transposed through LDS.
//   tail       the last group of a row is its last four blocks, with both scales zero (one may be infinite) for those that an earlier
//              group has taken.
__global__ __launch_bounds__(512, 4) void dense_mid_kernel(const DenseArgs a) {
    constexpr int NW = 8;
    __shared__ v4i turn[NW][2][256];                             // per wave: 32 rows of the weight, 32 of x
    __shared__ __align__(16) float dxs[NW][4][32];
    static_assert(sizeof(turn) >= NW * 32 * 33 * 4, "room for the join");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 31, h = lane >> 5, lr = lane >> 3, lc = lane & 7;
    const int o0 = (int) blockIdx.x * 32;
    const int64_t t0 = (int64_t) blockIdx.y * 32;
    const int8_t * wp[4], * xp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        wp[i] = a.wq + (int64_t) min(o0 + 8 * i + lr, a.n_out - 1) * a.nblk * 32 + 16 * lc;
        xp[i] = a.xq + min(t0 + 8 * i + lr, a.T - 1) * a.ldq + 16 * lc;
    }
    const __half * dwp = a.wd + (int64_t) min(o0 + m, a.n_out - 1) * a.nblk;
    const float * dxp = a.xd + min(t0 + m, a.T - 1) * a.ldd + 2 * h;
    const int st = lr * 8 + (lc ^ (lr >> 1)), key = (m >> 1) & 7;       // rows 8 i + lr: 8 more rows flip bit 2 of the key
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    v4i wn[4], xn[4];
    __half dw[4];
    float dx[2];
    auto load = [&](int b0) {
        const int bs = min(b0, a.nblk - 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) wn[i] = *reinterpret_cast<const v4i *>(wp[i] + (int64_t) bs * 32);
        __builtin_memcpy(dw, dwp + bs, 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) xn[i] = *reinterpret_cast<const v4i *>(xp[i] + (int64_t) bs * 32);
        __builtin_memcpy(dx, dxp + bs, 8);
    };
    load(4 * wave);
    for (int b0 = 4 * wave; b0 < a.nblk; b0 += 4 * NW) {
        const int bs = min(b0, a.nblk - 4);
        float dc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            turn[wave][0][64 * i + (i & 1 ? st ^ 4 : st)] = wn[i];
            turn[wave][1][64 * i + (i & 1 ? st ^ 4 : st)] = xn[i];
            dc[i] = bs + i >= b0 ? __half2float(dw[i]) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) dxs[wave][2 * h + i][m] = bs + 2 * h + i >= b0 ? dx[i] : 0.0f;
        load(b0 + 4 * NW);                                       // past the end: in bounds and not used
        wave_lds_order();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = m * 8 + ((2 * k + h) ^ key);
            v16i z = {};
            z = __builtin_amdgcn_mfma_i32_32x32x32_i8(turn[wave][1][at], turn[wave][0][at], z, 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 d = *reinterpret_cast<const float4 *>(&dxs[wave][k][8 * q + 4 * h]);
                acc[4 * q + 0] = fmaf((float) z[4 * q + 0], d.x * dc[k], acc[4 * q + 0]);
                acc[4 * q + 1] = fmaf((float) z[4 * q + 1], d.y * dc[k], acc[4 * q + 1]);
                acc[4 * q + 2] = fmaf((float) z[4 * q + 2], d.z * dc[k], acc[4 * q + 2]);
                acc[4 * q + 3] = fmaf((float) z[4 * q + 3], d.w * dc[k], acc[4 * q + 3]);
            }
        }
        wave_lds_order();
    }
    __syncthreads();
    float * part = reinterpret_cast<float *>(turn);              // [NW][32][33]
#pragma unroll
    for (int i = 0; i < 16; ++i) part[(wave * 32 + 8 * (i / 4) + 4 * h + (i & 3)) * 33 + m] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += 64 * NW) {
        const int t = e >> 5, c = e & 31;
        if (t0 + t < a.T && o0 + c < a.n_out) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += part[(w * 32 + t) * 33 + c];
            a.y[(t0 + t) * a.ldy + o0 + c] = v;
        }
    }
}

// The same with 16 RR rows and 16 TT tokens per workgroup, for two things that 32 x 32 tiles do badly: a weight of some thousand rows
// leaves CUs without work (RR = 1: 11 tokens x 14336 -> 4096 11.7 us, 5.4 TB/s, against 22.5), and one of very many rows reads x so often
// that its way from the L2 counts as much as the weight (RR = 4, one workgroup per CU: 11 tokens x 4096 -> 14336 13.2 us against 16.8, 18.7
// with RR = 1). RR = 3 where that fills the CUs better. 16 waves instead of 8 gain nothing (13.5 us for the former), nor does starting
// each workgroup at another column (20.5 us for the latter: x is then no longer shared in the cache).
//   fragments  v_mfma_i32_16x16x32_i8: lane = row (or token) lane & 15, the 8 bytes lane >> 4 of the block; the result has token
//              4 (lane >> 4) + i in register i and row lane & 15.
template <int TT, int RR>
__global__ __launch_bounds__(512, TT * RR == 1 ? 8 : TT + RR <= 4 ? 4 : 2) void dense_thin_kernel(const DenseArgs a) {
    constexpr int NW = 8;
    __shared__ v4i turn[NW][RR + TT][128];                       // per wave: 16 RR rows of the weight, 16 TT of x
    __shared__ __align__(16) float dxs[NW][4][16 * TT];
    static_assert(sizeof(turn) >= NW * 16 * TT * (16 * RR + 1) * 4, "room for the join");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4, lr = lane >> 3, lc = lane & 7;
    const int o0 = (int) blockIdx.x * (16 * RR);
    const int64_t t0 = (int64_t) blockIdx.y * (16 * TT);
    const int8_t * wp[2 * RR], * xp[2 * TT];
    const __half * dwp[RR];
#pragma unroll
    for (int i = 0; i < 2 * RR; ++i) wp[i] = a.wq + (int64_t) min(o0 + 8 * i + lr, a.n_out - 1) * a.nblk * 32 + 16 * lc;
#pragma unroll
    for (int i = 0; i < 2 * TT; ++i) xp[i] = a.xq + min(t0 + 8 * i + lr, a.T - 1) * a.ldq + 16 * lc;
#pragma unroll
    for (int r = 0; r < RR; ++r) dwp[r] = a.wd + (int64_t) min(o0 + 16 * r + m, a.n_out - 1) * a.nblk;
    const int dxt = TT == 2 ? lane & 31 : m, dxb = TT == 2 ? 2 * (lane >> 5) : g;         // this lane's token and first block (TT: as many)
    const float * dxp = a.xd + min(t0 + dxt, a.T - 1) * a.ldd + dxb;
    const int st = lr * 8 + (lc ^ (lr >> 1)), key = (m >> 1) & 7;       // rows 8 i + lr: 8 more rows flip bit 2 of the key
    float acc[RR][TT][4];
#pragma unroll
    for (int r = 0; r < RR; ++r)
#pragma unroll
        for (int j = 0; j < TT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][j][i] = 0.0f;
    v4i wn[2 * RR], xn[2 * TT];
    __half dw[RR][4];
    float dx[TT];
    auto load = [&](int b0) {
        const int bs = min(b0, a.nblk - 4);
#pragma unroll
        for (int i = 0; i < 2 * RR; ++i) wn[i] = *reinterpret_cast<const v4i *>(wp[i] + (int64_t) bs * 32);
#pragma unroll
        for (int r = 0; r < RR; ++r) __builtin_memcpy(dw[r], dwp[r] + bs, 8);
#pragma unroll
        for (int i = 0; i < 2 * TT; ++i) xn[i] = *reinterpret_cast<const v4i *>(xp[i] + (int64_t) bs * 32);
        __builtin_memcpy(dx, dxp + bs, 4 * TT);
    };
    load(4 * wave);
    for (int b0 = 4 * wave; b0 < a.nblk; b0 += 4 * NW) {
        const int bs = min(b0, a.nblk - 4);
        float dc[RR][4];
#pragma unroll
        for (int i = 0; i < 2 * RR; ++i) turn[wave][i / 2][64 * (i & 1) + (i & 1 ? st ^ 4 : st)] = wn[i];
#pragma unroll
        for (int i = 0; i < 2 * TT; ++i) turn[wave][RR + i / 2][64 * (i & 1) + (i & 1 ? st ^ 4 : st)] = xn[i];
#pragma unroll
        for (int r = 0; r < RR; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) dc[r][i] = bs + i >= b0 ? __half2float(dw[r][i]) : 0.0f;
#pragma unroll
        for (int i = 0; i < TT; ++i) dxs[wave][dxb + i][dxt] = bs + dxb + i >= b0 ? dx[i] : 0.0f;
        load(b0 + 4 * NW);                                       // past the end: in bounds and not used
        wave_lds_order();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = 2 * (m * 8 + ((2 * k + (g >> 1)) ^ key)) + (g & 1);         // 8 bytes
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                const long xf = reinterpret_cast<const long *>(turn[wave][RR + j])[at];
                const float4 d = *reinterpret_cast<const float4 *>(&dxs[wave][k][16 * j + 4 * g]);
#pragma unroll
                for (int r = 0; r < RR; ++r) {
                    v4i z = {};
                    z = __builtin_amdgcn_mfma_i32_16x16x32_i8(xf, reinterpret_cast<const long *>(turn[wave][r])[at], z, 0, 0, 0);
                    acc[r][j][0] = fmaf((float) z[0], d.x * dc[r][k], acc[r][j][0]);
                    acc[r][j][1] = fmaf((float) z[1], d.y * dc[r][k], acc[r][j][1]);
                    acc[r][j][2] = fmaf((float) z[2], d.z * dc[r][k], acc[r][j][2]);
                    acc[r][j][3] = fmaf((float) z[3], d.w * dc[r][k], acc[r][j][3]);
                }
            }
        }
        wave_lds_order();
    }
    __syncthreads();
    float * part = reinterpret_cast<float *>(turn);              // [NW][16 TT][16 RR + 1]
#pragma unroll
    for (int r = 0; r < RR; ++r)
#pragma unroll
        for (int j = 0; j < TT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[(wave * 16 * TT + 16 * j + 4 * g + i) * (16 * RR + 1) + 16 * r + m] = acc[r][j][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * TT * RR; e += 64 * NW) {
        const int t = e / (16 * RR), c = e % (16 * RR);
        if (t0 + t < a.T && o0 + c < a.n_out) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += part[(w * 16 * TT + t) * (16 * RR + 1) + c];
            a.y[(t0 + t) * a.ldy + o0 + c] = v;
        }
    }
}

template <int TT, int RR>
static void launch_thin(const DenseArgs & a, hipStream_t s) {
    hipLaunchKernelGGL((dense_thin_kernel<TT, RR>), dim3((unsigned) ((a.n_out + 16 * RR - 1) / (16 * RR)), (unsigned) ((a.T + 16 * TT - 1) / (16 * TT))), dim3(512), 0, s, a);
}

// Many tokens: BM tokens x BN rows per workgroup, both operands through LDS in steps of SB blocks, two stages. A wave owns 32 tokens x
// 32 NN rows; with KS = 2 two waves share them, each with every other block, joined at the end.
//
// 2048 tokens x 4096 -> 14336 take 357 us, 674 TOP/s. Of 741,000 busy cycles per SIMD the vector pipe works 562,000 (76 %) and the matrix pipe
// 229,000 (31 %): two pipes that can run at once, so neither alone is the bound yet. A wave waits for its MFMAs and converts then, and a
// barrier per step keeps its neighbours in phase. The vector pipe alone would be about 270 us: a 32x32x32 MFMA takes 32 cycles and leaves
// 16 integers per lane, each of which costs a conversion and a fused multiply-add (packed F32 being off). The products of the scales come from v_mfma_f32_32x32x1_2b_f32, two
// tiles in 64 cycles (32 vector instructions of 4 cycles otherwise); a step's addresses are one operation each, and the operands' way
// through registers is left out (loads to LDS), so two tiles take 128 cycles of the matrix pipe and 72 vector instructions, 288 cycles
// (products by vector instructions and operands through registers: 424 us).
//   waves      four per SIMD: a wave waits for LDS, MFMA and conversions in turn (four waves of 64 x 64 in the place of eight of 32 x 64:
//              559 us against 463).
//   steps      four blocks (128 bytes a row); eight for 64 x 64, which has half the work between two barriers (512 tokens x 2560 ->
//              10240: 50 us against 78, with four and two stages ahead 62).
//   LDS        16-byte chunks of a row at chunk ^ ((row >> 1) & 7), or ^ (row & 15) for 256 bytes a row: the 16 rows of a fragment read
//              hit all 64 banks once.
//   scales     [block][row], a lane's row of the product's operand.
//   workgroups XCD k (round-robin dispatch) takes the row panels k, k + 8, ... with all their token tiles: a panel of the weight
//              comes from memory once and stays in that XCD's L2.

// 16 bytes per lane from memory straight to LDS: the wave's 1 KB from `to` (the same in all lanes) on, in the order of its lanes
__device__ __forceinline__ void to_lds(const int8_t * from, int8_t * to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned *) from, (__attribute__((address_space(3))) unsigned *) to, 16, 0, 0);
}

template <int BM, int BN, int NN, int KS, int SB>
__global__ __launch_bounds__(BM * BN / 16 / NN * KS, 4) void dense_mfma_kernel(const DenseArgs a, int n_tt) {
    constexpr int NT = BM * BN / 16 / NN * KS;                      // threads
    constexpr int CH = 2 * SB, RB = 16 * CH;                        // chunks and bytes of a row in a stage
    constexpr int XL = BM * CH / NT, WL = BN * CH / NT;             // 16-byte loads per thread and stage
    constexpr int XS = (SB * BM + NT - 1) / NT, WS = (SB * BN + NT - 1) / NT;    // scales per thread and stage
    constexpr int KP = 2 / NN;                                      // blocks per pair of products
    static_assert(NT * XL == BM * CH && NT * WL == BN * CH && NT / CH % 16 == 0 && KP * NN == 2 && SB % (KP * KS) == 0, "whole loads, whole pairs");
    // one array: with several the compiler waits for loads on their way to the next stage before it reads the present one
    __shared__ __align__(16) int8_t lds[2 * (BM + BN) * (RB + 4 * SB)];
    int8_t (* const xs)[BM * RB] = reinterpret_cast<int8_t (*)[BM * RB]>(lds);
    int8_t (* const ws)[BN * RB] = reinterpret_cast<int8_t (*)[BN * RB]>(lds + 2 * BM * RB);
    float (* const dxs)[SB * BM] = reinterpret_cast<float (*)[SB * BM]>(lds + 2 * (BM + BN) * RB);
    float (* const dws)[SB * BN] = reinterpret_cast<float (*)[SB * BN]>(lds + 2 * (BM + BN) * RB + 2 * SB * BM * 4);
    const int id = (int) blockIdx.x, seq = id >> 3;
    const int o_tile = ((seq / n_tt) * 8 + (id & 7)) * BN;
    const int64_t t_tile = (int64_t) (seq % n_tt) * BM;
    if (o_tile >= a.n_out) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 31, h = lane >> 5;
    const int wt = (wave % (BM / 32)) * 32, wo = (wave / (BM / 32)) % (BN / 32 / NN) * 32 * NN, ks = KS == 1 ? 0 : wave / (BM * BN / 1024 / NN);
    const int64_t n_in = (int64_t) a.nblk * 32;
    const auto key = [](int row) { return SB == 4 ? (row >> 1) & 7 : row & 15; };
    const int lr = tid / CH, lc = tid % CH ^ key(lr);               // staging: rows lr + NT / CH i (the same key), chunk lc into slot tid % CH
    const int dst = __builtin_amdgcn_readfirstlane(wave) * 1024;
    const int8_t * xp[XL], * wp[WL];
#pragma unroll
    for (int i = 0; i < XL; ++i) xp[i] = a.xq + min(t_tile + lr + NT / CH * i, a.T - 1) * a.ldq;
#pragma unroll
    for (int i = 0; i < WL; ++i) wp[i] = a.wq + (int64_t) min(o_tile + lr + NT / CH * i, a.n_out - 1) * n_in;
    const float * dxp = a.xd + min(t_tile + tid % BM, a.T - 1) * a.ldd;               // scale e of a stage: row e % BM (BN), block e / BM (BN)
    const __half * dwp = a.wd + (int64_t) min(o_tile + tid % BN, a.n_out - 1) * a.nblk;
    float dx[XS];
    __half dw[WS];
    auto load = [&](int b0, int st) {
#pragma unroll
        for (int k = 0; k < XS; ++k) dx[k] = dxp[min(b0 + (tid + NT * k) / BM % SB, a.nblk - 1)];
#pragma unroll
        for (int k = 0; k < WS; ++k) dw[k] = dwp[min(b0 + (tid + NT * k) / BN % SB, a.nblk - 1)];
        const int64_t off = (int64_t) min(b0 + (lc >> 1), a.nblk - 1) * 32 + (lc & 1) * 16;       // blocks past the end: the last one, with scales of zero
#pragma unroll
        for (int i = 0; i < XL; ++i) to_lds(xp[i] + off, &xs[st][dst + i * 16 * NT]);
#pragma unroll
        for (int i = 0; i < WL; ++i) to_lds(wp[i] + off, &ws[st][dst + i * 16 * NT]);
    };
    auto store = [&](int b0, int st) {                              // the choices stand here: at the load they would wait for it
#pragma unroll
        for (int k = 0; k < XS; ++k) if (tid + NT * k < SB * BM) dxs[st][tid + NT * k] = b0 + (tid + NT * k) / BM < a.nblk ? dx[k] : 0.0f;
#pragma unroll
        for (int k = 0; k < WS; ++k) if (tid + NT * k < SB * BN) dws[st][tid + NT * k] = b0 + (tid + NT * k) / BN < a.nblk ? __half2float(dw[k]) : 0.0f;
    };
    float acc[NN][16];
#pragma unroll
    for (int j = 0; j < NN; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[j][q] = 0.0f;
    const int c0 = ((2 * ks + h) ^ key(m)) << 4;                    // tiles start at multiples of 32 rows: the key is the lane's
    load(0, 0);
    store(0, 0);
    for (int b0 = 0, st = 0; b0 < a.nblk; b0 += SB, st ^= 1) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); // the stage has arrived, this wave's part; after the barrier all of it
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load(b0 + SB, st ^ 1);                                      // past the end: in bounds and not used
        // chunk 2 k + h of row m is at (h ^ key) * 16 with its bits from 5 on flipped by k
        const int8_t * const xa = &xs[st][(wt + m) * RB], * const wa = &ws[st][(wo + m) * RB];
        const float * const dxa = &dxs[st][ks * BM + wt + m + (NN == 2 ? 0 : h * KS * BM)], * const dwa = &dws[st][ks * BN + wo + (NN == 2 ? lane : m + h * KS * BN)];
#pragma unroll
        for (int k = 0; k < SB; k += KP * KS) {
            // products of the scales, two 32 x 32 outer products an instruction: NN == 2 the wave's two tiles, else two of its blocks
            v32f dd = {};
            dd = __builtin_amdgcn_mfma_f32_32x32x1f32(dxa[k * BM], dwa[k * BN], dd, 0, 0, 0);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int at = c0 ^ ((NN == 2 ? k : k + KS * p) << 5), j = NN == 2 ? p : 0;
                const v4i xf = *reinterpret_cast<const v4i *>(xa + at);
                const v4i wf = *reinterpret_cast<const v4i *>(wa + 32 * j * RB + at);
                v16i z = {};
                z = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf, wf, z, 0, 0, 0);
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[j][q] = fmaf((float) z[q], dd[16 * p + q], acc[j][q]);
            }
#pragma unroll
            for (int j = 0; j < NN; ++j)                            // one pair after the other, or every MFMA of the step is started first and registers spill
#pragma unroll
                for (int q = 0; q < 16; ++q) asm volatile("" : "+v"(acc[j][q]) :: "memory");
        }
        if (b0 + SB < a.nblk) store(b0 + SB, st ^ 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                // nothing is still on its way to LDS when it changes its use, or its owner
    if constexpr (KS > 1) {                                         // the waves that share a tile: 4 KB of each tile and wave but the first
        constexpr int TW = NT / 64 / KS;                            // waves per part
        static_assert((KS - 1) * TW * NN * 4096 <= 2 * (BM + BN) * RB, "room for the parts");
        float * red = reinterpret_cast<float *>(lds) + wave % TW * NN * 1024 + lane;
        __syncthreads();
        if (ks) {
#pragma unroll
            for (int j = 0; j < NN; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) red[((ks - 1) * TW * NN + j) * 1024 + 64 * q] = acc[j][q];
        }
        __syncthreads();
        if (ks) return;
#pragma unroll
        for (int i = 0; i < KS - 1; ++i)
#pragma unroll
            for (int j = 0; j < NN; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[j][q] += red[(i * TW * NN + j) * 1024 + 64 * q];
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int64_t t = t_tile + wt + 8 * (q / 4) + 4 * h + (q & 3);
        if (t < a.T) {
#pragma unroll
            for (int j = 0; j < NN; ++j) {
                const int o = o_tile + wo + 32 * j + m;
                if (o < a.n_out) a.y[t * a.ldy + o] = acc[j][q];
            }
        }
    }
}

template <int TT, int R, int U>
static void launch_few(const DenseArgs & a, hipStream_t s) {
    hipLaunchKernelGGL((dense_few_kernel<TT, R, U>), dim3((unsigned) ((a.n_out + 4 * R - 1) / (4 * R)), (unsigned) ((a.T + TT - 1) / TT)), dim3(256), 0, s, a);
}

template <int BM, int BN, int NN, int KS, int SB>
static void launch_mfma(const DenseArgs & a, hipStream_t s) {
    const int n_tt = (int) ((a.T + BM - 1) / BM), n_pan = (a.n_out + BN - 1) / BN;
    hipLaunchKernelGGL((dense_mfma_kernel<BM, BN, NN, KS, SB>), dim3((unsigned) ((n_pan + 7) / 8 * 8 * n_tt)), dim3(BM * BN / 16 / NN * KS), 0, s, a, n_tt);
}

static void launch_mid(const DenseArgs & a, hipStream_t s) {
    hipLaunchKernelGGL(dense_mid_kernel, dim3((unsigned) ((a.n_out + 31) / 32), (unsigned) ((a.T + 31) / 32)), dim3(512), 0, s, a);
}

// The forms from 2 tokens on: tile of tokens x rows, and its time in us per 128 bytes of K: per round in which the workgroups fill the CUs
// (workgroups per CU, rounded up), plus `add`, `least` at least. `blocks`: the fewest blocks of a row; before that the start and the end
// of a large tile count for more than its rounds (48 tokens x 1152 -> 6912: 32 x 64 8.9 us, 32 x 32 6.6). Fitted to nine shapes between 1152 and 28672 at 2 to 2048 tokens (a
// call's time less 2 us); between these shapes nothing says how far the choice is from the best form. What the choice is worth, us:
//   14336 -> 4096    11 tokens  16 x 16 11.7, 16 x 48 23, 16 x 64 29, 32 x 32 22.5;    32 tokens  32 x 16 17, 32 x 32 23, 32 x 64 39;
//                    64 / 256 / 512 / 2048 tokens  32 x 32 23 / 79 / 156 / 642, 64 x 64 65 / 66 / 103 / 447, 64 x 128 120 / 114 / 116 / 425,
//                    128 x 128 189 / 205 / 205 / 340
//   4096 -> 14336    11 tokens  16 x 16 18.7, 16 x 48 18.3, 16 x 64 13.2, 32 x 32 16.8;  32 tokens  32 x 16 21, 32 x 32 18.3, 32 x 48 24, 32 x 64 17.1;
//                    64 / 256 / 512 / 2048 tokens  32 x 32 30 / 96 / 183 / 723, 64 x 64 23 / 57 / 103 / 465, 64 x 128 38 / 55 / 104 / 426,
//                    128 x 128 55 / 61 / 94 / 348
//   2560 -> 10240    16 tokens  16 x 16 8.3, 16 x 48 7.8, 16 x 64 9.0, 32 x 32 10.5;    32 tokens  32 x 16 11.0, 32 x 32 11.7, 32 x 48 10.0, 32 x 64 11.5
struct DenseForm {
    int tokens, rows, blocks;
    double per, add, least;
    void (*launch)(const DenseArgs &, hipStream_t);
};
static const DenseForm dense_forms[] = {
    {16, 16, 4, 0.115, 0, 0, launch_thin<1, 1>},
    {16, 48, 64, 0.29, 0, 0, launch_thin<1, 3>},
    {16, 64, 64, 0.37, 0, 0, launch_thin<1, 4>},
    {32, 16, 4, 0.145, 0, 0, launch_thin<2, 1>},
    {32, 32, 4, 0.24, 0, 0, launch_mid},
    {32, 48, 64, 0.42, 0, 0, launch_thin<2, 3>},
    {32, 64, 64, 0.47, 0, 0, launch_thin<2, 4>},
    {64, 64, 4, 0.46, 0.1, 0, launch_mfma<64, 64, 1, 2, 8>},
    {64, 128, 4, 0.92, 0, 1.05, launch_mfma<64, 128, 1, 1, 4>},
    {128, 128, 4, 1.54, 0, 1.85, launch_mfma<128, 128, 2, 1, 4>},
};

static int launch_dense(const DenseArgs & all, hipStream_t s) {
    const DenseForm * form = nullptr;                       // none with fewer than four blocks
    double best = 0.0;
    for (const DenseForm & f : dense_forms) {
        if (all.nblk < f.blocks) continue;
        const int64_t wg = ((all.T + f.tokens - 1) / f.tokens) * ((all.n_out + f.rows - 1) / f.rows), cu = lib().num_cu;
        const double cost = std::max(f.least, f.per * (double) ((wg + cu - 1) / cu) + f.add);
        if (!form || cost < best) { form = &f; best = cost; }
    }
    // a launch has fewer than 2^32 threads, 65535 workgroups in its second dimension: tokens in chunks for very many of them
    const int64_t n_pan = (all.n_out + 63) / 64, chunk = std::max<int64_t>(1, std::min<int64_t>(1000, (1 << 21) / n_pan)) * 128;
    for (int64_t t0 = 0; t0 < all.T; t0 += chunk) {
        DenseArgs a = all;
        a.T = std::min(chunk, all.T - t0);
        a.xq += t0 * a.ldq; a.xd += t0 * a.ldd; a.y += t0 * a.ldy;
        // one token takes the stream of rows whatever the shape: 4096 -> 14336 11.6 us (16 x 64 tiles 12.7), 6912 -> 1152 5.1 (6.3). Of the
        // shapes measured 14336 -> 4096 loses by it: 13.3 us, 11.5 with 16 x 16 tiles; the costs above do not have this form yet
        if (all.T == 1)       { if (a.nblk >= 96) launch_few<1, 2, 4>(a, s); else launch_few<1, 2, 2>(a, s); }
        else if (form)        form->launch(a, s);
        else                  launch_few<2, 2, 4>(a, s);
    }
    SDH_HIP_CHECK(hipGetLastError());
    return SDH_OK;
}

} // namespace sdh

using namespace sdh;

static int sdh_dense_forward_q8_impl(const sdh_dense * W, const sdh_q8 * x, int64_t T, float * y, int64_t ldy, void * stream) {
    static const char * who = "sdh_dense_forward_q8";
    if (T == 0) return ready_on_device(who);
    if (!W || !x || !x->q || !x->d || !y) { set_error("%s: null argument", who); return SDH_ERR_INVALID; }
    const DenseQ8 w = dense_q8(W);
    if (w.type != SDH_TYPE_Q8_0) { set_error("%s: the weight is not Q8_0 (type %d)", who, w.type); return SDH_ERR_UNSUPPORTED; }
    if (w.n_out > (1 << 26)) { set_error("%s: %lld rows, more than a launch has threads for", who, (long long) w.n_out); return SDH_ERR_UNSUPPORTED; }
    if (T < 0 || ldy < w.n_out || x->ldq < w.n_in || x->ldd < w.n_in / 32) {
        set_error("%s: bad shape: T=%lld ldq=%lld ldd=%lld (n_in=%lld) ldy=%lld (n_out=%lld)", who, (long long) T, (long long) x->ldq, (long long) x->ldd, (long long) w.n_in, (long long) ldy, (long long) w.n_out);
        return SDH_ERR_INVALID;
    }
    if (!aligned(x->q, 16) || x->ldq % 16 || !aligned(x->d, 4) || !aligned(y, 4)) { set_error("%s: x->q needs 16-byte aligned rows, x->d and y 4-byte ones", who); return SDH_ERR_INVALID; }
    const int rc = ready_on_device(who);
    if (rc != SDH_OK) return rc;
    if (w.device != lib().device) { set_error("%s: the weight was made on device %d, the library is bound to %d", who, w.device, lib().device); return SDH_ERR_INVALID; }
    const DenseArgs a{w.q, (const __half *) w.d, x->q, x->ldq, x->d, x->ldd, (int) w.n_out, (int) (w.n_in / 32), T, y, ldy};
    return launch_dense(a, (hipStream_t) stream);
}

extern "C" int sdh_dense_forward_q8(const sdh_dense * W, const sdh_q8 * x, int64_t n_tokens, float * y, int64_t ldy, void * stream) {
    SDH_NO_THROW(sdh_dense_forward_q8_impl(W, x, n_tokens, y, ldy, stream));
}
