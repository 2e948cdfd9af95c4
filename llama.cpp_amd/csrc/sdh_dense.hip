// sdh_dense.hip — dense Q8_0 weight x 8-bit activations: y[t][o] = sum_b dw[o][b] dx[t][b] sum_{k in b} qw[o][k] qx[t][k].
//
// The integer sum of a block of 32 is exact (at most 32 * 127 * 128 < 2^20); the two scales multiply it once in F32 and the
// blocks are summed in F32.
//
//   dense_few_kernel   few tokens: bound by the stream of the weight. A wave owns R rows, a lane a block of 32 per step (two
//                      16-byte loads per row), v_dot4_i32_i8, the tokens' blocks from the cache; no LDS, no barrier.
//   dense_tile_kernel  many tokens: v_mfma_i32_32x32x32_i8, whose K is exactly one block.
#include "sdh_internal.h"

#include <algorithm>
#include <hip/hip_fp16.h>

namespace sdh {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

struct DenseArgs {
    const int8_t * wq; const __half * wd;      // [n_out][n_in], [n_out][nblk]
    const int8_t * xq; int64_t ldq;
    const float * xd; int64_t ldd;
    int n_out, nblk;                           // n_in = 32 * nblk
    int64_t T;
    float * y; int64_t ldy;
};

// U chunks of 16 bytes (half a block) per lane and row in flight; chunk c of a row belongs to lane c & 63.
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
        for (int u = 0; u < U; ++u) {                         // chunks past the end: the last one, with a scale of zero
            c[u] = min(c0 + 64 * u, n_ch - 1);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                w[u][r] = __builtin_nontemporal_load(reinterpret_cast<const v4i *>(wp[r] + (int64_t) c[u] * 16));
                dw[u][r] = __half2float(dp[r][c[u] >> 1]);
            }
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int64_t tt = min(t0 + t, a.T - 1);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const v4i x = *reinterpret_cast<const v4i *>(a.xq + tt * a.ldq + (int64_t) c[u] * 16);
                const float dx = c0 + 64 * u < n_ch && !(lane & 1) ? a.xd[tt * a.ldd + (c[u] >> 1)] : 0.0f;     // even lanes count
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

// 32 NT tokens x 32 rows per workgroup: the stream of the weight again. The waves split K in groups of four blocks (128 bytes, a
// whole line of a row) and are joined in LDS at the end; every fragment goes from memory to registers, the next group's before the
// present one is multiplied, so that a CU has 64 KB in flight without a barrier anywhere in the loop.
//   fragments  v_mfma_i32_32x32x32_i8: lane = row (or token) lane & 31, the 16 bytes of half lane >> 5 of the block; the result has
//              token 8 (i / 4) + 4 (lane >> 5) + i % 4 in register i and row lane & 31.
//   scales     four of a row as one 8-byte load (whatever its alignment); the tokens' are transposed through LDS (each wave its own
//              corner; LDS works in order within a wave).
//   tail       the last group of a row is its last four blocks, with scales of zero for those that an earlier group has taken.
template <int NT, int NW>
__global__ __launch_bounds__(64 * NW, NT == 1 ? 4 : 2) void dense_mid_kernel(const DenseArgs a) {
    __shared__ __align__(16) float dxs[NW][NT][4][32];
    __shared__ float part[NW][32][33];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 31, h = lane >> 5;
    const int o = (int) blockIdx.x * 32 + m;
    const int64_t t0 = (int64_t) blockIdx.y * (32 * NT), orow = min(o, a.n_out - 1);
    const int8_t * wp = a.wq + orow * a.nblk * 32 + 16 * h;
    const __half * dwp = a.wd + orow * a.nblk;
    const int8_t * xp[NT];
    const float * dxp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int64_t t = min(t0 + 32 * n + m, a.T - 1);
        xp[n] = a.xq + t * a.ldq + 16 * h;
        dxp[n] = a.xd + t * a.ldd + 2 * h;
    }
    float acc[NT][16];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = 0.0f;
    v4i wf[4], xf[NT][4];
    __half dw[4];
    float dx[NT][2];
    auto load = [&](int b0) {
        const int bs = min(b0, a.nblk - 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) wf[k] = *reinterpret_cast<const v4i *>(wp + (int64_t) (bs + k) * 32);
        __builtin_memcpy(dw, dwp + bs, 8);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < 4; ++k) xf[n][k] = *reinterpret_cast<const v4i *>(xp[n] + (int64_t) (bs + k) * 32);
            __builtin_memcpy(dx[n], dxp[n] + bs, 8);
        }
    };
    load(4 * wave);
    for (int b0 = 4 * wave; b0 < a.nblk; b0 += 4 * NW) {
        const int bs = min(b0, a.nblk - 4);
        v4i wc[4], xc[NT][4];
        float dc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) { wc[k] = wf[k]; dc[k] = bs + k >= b0 ? __half2float(dw[k]) : 0.0f; }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < 4; ++k) xc[n][k] = xf[n][k];
            dxs[wave][n][2 * h][m] = dx[n][0];
            dxs[wave][n][2 * h + 1][m] = dx[n][1];
        }
        load(b0 + 4 * NW);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                v16i z = {};
                z = __builtin_amdgcn_mfma_i32_32x32x32_i8(xc[n][k], wc[k], z, 0, 0, 0);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 d = *reinterpret_cast<const float4 *>(&dxs[wave][n][k][8 * q + 4 * h]);
                    acc[n][4 * q + 0] = fmaf((float) z[4 * q + 0], d.x * dc[k], acc[n][4 * q + 0]);
                    acc[n][4 * q + 1] = fmaf((float) z[4 * q + 1], d.y * dc[k], acc[n][4 * q + 1]);
                    acc[n][4 * q + 2] = fmaf((float) z[4 * q + 2], d.z * dc[k], acc[n][4 * q + 2]);
                    acc[n][4 * q + 3] = fmaf((float) z[4 * q + 3], d.w * dc[k], acc[n][4 * q + 3]);
                }
            }
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (n) __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[wave][8 * (i / 4) + 4 * h + (i & 3)][m] = acc[n][i];
        __syncthreads();
        for (int e = threadIdx.x; e < 1024; e += 64 * NW) {
            const int t = e >> 5, c = e & 31;
            const int64_t tt = t0 + 32 * n + t;
            if (tt < a.T && (int) blockIdx.x * 32 + c < a.n_out) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) v += part[w][t][c];
                a.y[tt * a.ldy + (int) blockIdx.x * 32 + c] = v;
            }
        }
    }
}

// Many tokens: BM tokens x 128 rows per workgroup of four waves, both operands through LDS in steps of four blocks (128 bytes a
// row), two stages. A wave owns 64 tokens x 16 BM / 32 rows as 32x32 tiles.
//
// What bounds it is the vector pipe: a 32x32x32 MFMA takes 32 cycles and leaves 16 integers per lane, each of which costs a
// conversion, the product of its two scales and a fused multiply-add (48 instructions of 4 cycles, packed F32 being off).
//   LDS        16-byte chunks of a row at chunk ^ ((row >> 1) & 7): the 16 rows of a fragment read hit all 64 banks once.
//   scales     [block][row] as F32: a lane reads the four tokens of a register group as one broadcast.
//   workgroups XCD k (round-robin dispatch) takes the row panels k, k + 8, ... with all their token tiles: a panel of the weight
//              comes from memory once and stays in that XCD's L2.
template <int BM, int NN /* 32x32 tiles per wave, along the rows */>
__global__ __launch_bounds__(8 * BM / NN, NN == 1 ? 4 : BM == 128 ? 4 : 3) void dense_mfma_kernel(const DenseArgs a, int n_tt) {
    constexpr int BN = 128, NM = 1;
    constexpr int NT = 8 * BM / NN, XL = NN, WL = 128 * NN / BM, SL = 512 / NT;                      // 16-byte loads per thread and stage
    __shared__ __align__(16) int8_t xs[2][BM * 128];
    __shared__ __align__(16) int8_t ws[2][BN * 128];
    __shared__ __align__(16) float dxs[2][4][BM];
    __shared__ __half dws[2][4][BN];
    const int id = (int) blockIdx.x, seq = id >> 3;
    const int o_tile = ((seq / n_tt) * 8 + (id & 7)) * BN;
    const int64_t t_tile = (int64_t) (seq % n_tt) * BM;
    if (o_tile >= a.n_out) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 31, h = lane >> 5;
    const int wt = (wave % (BM / 32)) * 32, wo = (wave / (BM / 32)) * 32 * NN;
    const int64_t n_in = (int64_t) a.nblk * 32;
    const int lr = tid >> 3, lc = tid & 7;                          // staging: rows lr + NT / 8 i, chunk lc
    const int8_t * xp[XL], * wp[WL];
#pragma unroll
    for (int i = 0; i < XL; ++i) xp[i] = a.xq + min(t_tile + lr + NT / 8 * i, a.T - 1) * a.ldq;
#pragma unroll
    for (int i = 0; i < WL; ++i) wp[i] = a.wq + (int64_t) min(o_tile + lr + NT / 8 * i, a.n_out - 1) * n_in;
    const int sr = tid & 127, sb = (tid >> 7) * SL;                 // scales: row sr, blocks sb .. sb + SL - 1
    const float * dxp = a.xd + min(t_tile + (sr < BM ? sr : 0), a.T - 1) * a.ldd;
    const __half * dwp = a.wd + (int64_t) min(o_tile + sr, a.n_out - 1) * a.nblk;
    const int st_off = lr * 128 + ((lc ^ ((lr >> 1) & 7)) << 4);    // rows 16 apart have the same key

    // stages asked for ahead of the one in use: with one workgroup per CU a step's arithmetic (0.8 us) does not cover a load
    constexpr int D = BM == 128 ? 1 : 2;
    struct Stage { v4i x[XL], w[WL]; float dx[SL]; __half dw[SL]; } pre[D];
    auto load = [&](int b0, Stage & r) {
        const int cb = min(b0 + (lc >> 1), a.nblk - 1);             // blocks past the end: the last one, with scales of zero
        const int64_t off = (int64_t) cb * 32 + (lc & 1) * 16;
#pragma unroll
        for (int i = 0; i < XL; ++i) r.x[i] = *reinterpret_cast<const v4i *>(xp[i] + off);
#pragma unroll
        for (int i = 0; i < WL; ++i) r.w[i] = *reinterpret_cast<const v4i *>(wp[i] + off);
#pragma unroll
        for (int k = 0; k < SL; ++k) {
            const int b = min(b0 + sb + k, a.nblk - 1);
            r.dx[k] = dxp[b]; r.dw[k] = dwp[b];
            if (b0 + sb + k >= a.nblk) { r.dx[k] = 0.0f; r.dw[k] = __half(0.0f); }
        }
    };
    auto store = [&](int st, const Stage & r) {
#pragma unroll
        for (int i = 0; i < XL; ++i) *reinterpret_cast<v4i *>(&xs[st][st_off + i * 16 * NT]) = r.x[i];
#pragma unroll
        for (int i = 0; i < WL; ++i) *reinterpret_cast<v4i *>(&ws[st][st_off + i * 16 * NT]) = r.w[i];
#pragma unroll
        for (int k = 0; k < SL; ++k) {
            if (sr < BM) dxs[st][sb + k][sr] = r.dx[k];
            dws[st][sb + k][sr] = r.dw[k];
        }
    };
    float acc[NM][NN][16];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int j = 0; j < NN; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
    const int n_step = (a.nblk + 3) / 4, key = (m >> 1) & 7;        // tiles start at multiples of 32 rows: the key is the lane's
    load(0, pre[0]);
    store(0, pre[0]);
#pragma unroll
    for (int d = 1; d < D; ++d) load(4 * d, pre[d - 1]);
    for (int s0 = 0; s0 < n_step; s0 += D)
#pragma unroll
    for (int d = 0; d < D; ++d) {                                   // stage s + 1 is in pre[d], stage s + D goes to pre[(d + D - 1) % D]
        const int s = s0 + d;
        if (s >= n_step) break;
        __syncthreads();
        const int st = s & 1;
        load(4 * (s + D), pre[(d + D - 1) % D]);                    // past the end: in bounds, with scales of zero, and not stored
#pragma unroll 1                                                    // or every MFMA of the step is started first, and registers spill
        for (int k = 0; k < 4; ++k) {
            const int ch = ((2 * k + h) ^ key) << 4;
            v4i xf[NM], wf[NN];
            float dw[NN];
#pragma unroll
            for (int i = 0; i < NM; ++i) xf[i] = *reinterpret_cast<const v4i *>(&xs[st][(wt + 32 * i + m) * 128 + ch]);
#pragma unroll
            for (int j = 0; j < NN; ++j) { wf[j] = *reinterpret_cast<const v4i *>(&ws[st][(wo + 32 * j + m) * 128 + ch]); dw[j] = __half2float(dws[st][k][wo + 32 * j + m]); }
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                v16i z[NN];
#pragma unroll
                for (int j = 0; j < NN; ++j) {
                    v16i zero = {};
                    z[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[i], wf[j], zero, 0, 0, 0);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 d4 = *reinterpret_cast<const float4 *>(&dxs[st][k][wt + 32 * i + 8 * g + 4 * h]);
                    const float d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                    for (int j = 0; j < NN; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[i][j][4 * g + q] = fmaf((float) z[j][4 * g + q], d[q] * dw[j], acc[i][j][4 * g + q]);
                }
            }
        }
        if (s + 1 < n_step) store(st ^ 1, pre[d]);
    }
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int64_t t = t_tile + wt + 32 * i + 8 * (q / 4) + 4 * h + (q & 3);
            if (t < a.T) {
#pragma unroll
                for (int j = 0; j < NN; ++j) {
                    const int o = o_tile + wo + 32 * j + m;
                    if (o < a.n_out) a.y[t * a.ldy + o] = acc[i][j][q];
                }
            }
        }
}

template <int TT, int R, int U>
static void launch_few(const DenseArgs & a, hipStream_t s) {
    hipLaunchKernelGGL((dense_few_kernel<TT, R, U>), dim3((unsigned) ((a.n_out + 4 * R - 1) / (4 * R)), (unsigned) ((a.T + TT - 1) / TT)), dim3(256), 0, s, a);
}

template <int NT, int NW>
static void launch_mid(const DenseArgs & a, hipStream_t s) {
    hipLaunchKernelGGL((dense_mid_kernel<NT, NW>), dim3((unsigned) ((a.n_out + 31) / 32), (unsigned) ((a.T + 32 * NT - 1) / (32 * NT))), dim3(64 * NW), 0, s, a);
}

static int launch_dense(const DenseArgs & all, hipStream_t s) {
    // a launch has fewer than 2^32 threads: tokens in chunks for very many of them
    const int64_t n_pan = (all.n_out + 127) / 128, chunk = std::max<int64_t>(1, std::min<int64_t>(8192, (1 << 22) / n_pan)) * 128;
    for (int64_t t0 = 0; t0 < all.T; t0 += chunk) {
        DenseArgs a = all;
        a.T = std::min(chunk, all.T - t0);
        a.xq += t0 * a.ldq; a.xd += t0 * a.ldd; a.y += t0 * a.ldy;
        if (all.T == 1)       { if (a.nblk >= 96) launch_few<1, 2, 4>(a, s); else launch_few<1, 2, 2>(a, s); }
        else if (all.T == 2 || a.nblk < 4) launch_few<2, 2, 4>(a, s);
        else if (all.T <= 32) launch_mid<1, 8>(a, s);
        else if (all.T <= 64) launch_mid<2, 8>(a, s);
        else {
            const bool half = n_pan * ((all.T + 127) / 128) < 4 * lib().num_cu;
            const int n_tt = (int) (half ? (a.T + 63) / 64 : (a.T + 127) / 128);
            const dim3 grid((unsigned) ((n_pan + 7) / 8 * 8 * n_tt));
            if (half) hipLaunchKernelGGL((dense_mfma_kernel<64, 1>), grid, dim3(512), 0, s, a, n_tt);
            else      hipLaunchKernelGGL((dense_mfma_kernel<128, 2>), grid, dim3(512), 0, s, a, n_tt);
        }
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
    const DenseArgs a{w.q, (const __half *) w.d, x->q, x->ldq, x->d, x->ldd, (int) w.n_out, (int) (w.n_in / 32), T, y, ldy};
    return launch_dense(a, (hipStream_t) stream);
}

extern "C" int sdh_dense_forward_q8(const sdh_dense * W, const sdh_q8 * x, int64_t n_tokens, float * y, int64_t ldy, void * stream) {
    SDH_NO_THROW(sdh_dense_forward_q8_impl(W, x, n_tokens, y, ldy, stream));
}
