// sdh_lora.hip — low-rank adapters of many requests beside one projection: y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t].
//
// Two steps: u = A x for the tokens of an adapter (lora_shrink_kernel, K = n_in, split over workgroups), y = base + B (scale u)
// (lora_expand_kernel, K = rank). Tokens are taken by adapter, 32 at a time, so an adapter is read once per 32 of its tokens in
// whatever order they stand. ids live on the device (a captured graph sees the ids of the replay), so the sorting does too:
//   up to 64 tokens   a wave sees all ids at once: the first token of an adapter does the work of all of them (no launch for it);
//   more              of few adapters the same up to 256 tokens; else lora_plan_kernel sorts the tokens by adapter and cuts them into
//                     tiles (no ids, one adapter: nothing to sort).
// One to four tokens of small adapters take one launch (lora_fused_kernel) in which every workgroup forms u for itself.
//
// Kernel times (plan + shrink + expand), and what bounds them: 1 token, rank 16, 4096 -> 14336: 6.3 us (one launch and its chain of
// loads: id, record, A, B). 48 tokens, 32 adapters of rank 32 and less: 5.8 + 11.1 us (the same chains, made again by each of 33 x 56
// workgroups; 22 MB). 512 tokens, rank 64 in F32, 14336 -> 4096: 4.7 + 19.4 + 13 us (the products alone are 6.1 and 1.8 us at the rate of a
// large F32 product; one step of loads in flight per wave; x comes from the caches twice, once per 32 ranks). 4096 tokens, rank 16,
// 4096 -> 14336: 7.4 + 22.7 + 93.6 us; the last one is 470 MB of base and y, 5.0 TB/s.
//
// Everything is F32: v_mfma_f32_16x16x4_f32 does 2048 operations in 32 cycles, and both steps move far more bytes than that costs
// (8 bytes of y per 2 * rank operations, 4 of x per 2 * rank). Which k an MFMA takes is free as long as both operands agree: lane
// group g = lane >> 4 holds consecutive columns and MFMA j multiplies its j-th, so every operand load is a vector.
#include "sdh_internal.h"

#include <algorithm>
#include <cstring>
#include <hip/hip_fp16.h>

namespace sdh {

typedef float v4f __attribute__((ext_vector_type(4)));

// A in the order of the shrink kernel's fragments: per 16 ranks (8 up to rank 8), per 32 columns, lane' = 16 (or 8) * group + rank with
// columns 4 group .. and 16 + 4 group ..: eight consecutive halves, or four floats in each of two halves of the block. B in the order of
// the expand kernel's fragments: per 16 output rows, per 16 ranks, [lane][4] with row lane & 15 and ranks 4 (lane >> 4) ..; up to
// rank 8 one [lane][2] with ranks 2 (lane >> 4) ... Whatever lies past n_in, n_out or `rank` is zero.
struct LoraAdapter {
    const void * a;
    const void * b;
    float scale;
    int rank, r_ld, f32;   // r_ld: 8, or rank rounded up to 16
};

struct LoraSet {
    int64_t n_in = 0, n_out = 0, a_ld = 0;
    int n = 0, u_ld = 0;                   // adapters; row pitch of u: the largest r_ld
    bool any_f32 = false;
    int device = -1;
    uint8_t * dev = nullptr;               // the LoraAdapter table, then the matrices
    int64_t stored_bytes = 0;
};

constexpr int LT = 32;                     // tokens per tile of the shrink kernel
constexpr int ET = 16;                     // ... of the expand kernel
constexpr int LORA_RC = 32;                // ranks per workgroup of the shrink kernel
constexpr int LORA_SPLITS = 16;            // its most splits of the columns
constexpr int LORA_SCAN_T = 256;           // most tokens that a wave deals from the ids alone
constexpr int64_t LORA_WGS = 384;          // no more splits where tiles times splits would pass this

struct LoraTile { int adapter, start, count, pad; };       // adapter -1: none

// the caller's workspace
struct LoraWs {
    int * perm; LoraTile * tiles; LoraTile * etiles; int * n_tiles; float * u;
    int64_t max_tiles, max_etiles; int splits; int64_t bytes;
};

static LoraWs lora_ws(const LoraSet & l, int64_t T, uint8_t * base) {
    LoraWs w{};
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    w.max_tiles = (T + LT - 1) / LT + std::min<int64_t>(T, l.n + 1);
    w.max_etiles = (T + ET - 1) / ET + std::min<int64_t>(T, l.n + 1);
    // K splits of the shrink step: a workgroup per CU and more, at least 256 columns each; a power of two, so that from 8 on a split
    // stays on one XCD (round-robin dispatch) with its slice of A for all tiles. Not more than that needs, as the expand step adds them
    // up: 4096 tokens at rank 16, 2 splits 123 us, 8 (1056 workgroups) 129; 512 tokens at rank 64, 8 instead of 16 makes the expand step
    // 1.2 us faster and this one 5 slower
    const int64_t tiles = (T + LT - 1) / LT;
    for (w.splits = 1; w.splits < LORA_SPLITS && 2 * w.splits * tiles <= LORA_WGS && l.a_ld / (2 * w.splits) >= 256;) w.splits *= 2;
    int64_t at = 0;
    w.perm = (int *) (base + at);         at += up(T * 4);
    w.tiles = (LoraTile *) (base + at);   at += up(w.max_tiles * (int64_t) sizeof(LoraTile));
    w.etiles = (LoraTile *) (base + at);  at += up(w.max_etiles * (int64_t) sizeof(LoraTile));
    w.n_tiles = (int *) (base + at);      at += 256;
    w.u = (float *) (base + at);          at += up((int64_t) w.splits * T * l.u_ld * 4);
    w.bytes = at;
    return w;
}

// ---- tokens sorted by adapter, cut into tiles -----------------------------------------------------------------------
// One workgroup: count, scan, tiles, scatter. The place of a token inside its adapter's run depends on the order of the atomics; no
// result depends on the place.
__global__ __launch_bounds__(1024)
void lora_plan_kernel(const int * __restrict__ ids, int64_t T, int n, int * __restrict__ perm, LoraTile * __restrict__ tiles, LoraTile * __restrict__ etiles, int * __restrict__ n_tiles) {
    extern __shared__ int lds[];
    int * run = lds, * toff = lds + (n + 2), * eoff = lds + 2 * (n + 2);     // per adapter (bin n: none): tokens, then first place; first tiles
    __shared__ int wsum[3][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int b = tid; b <= n + 1; b += 1024) run[b] = 0;
    __syncthreads();
    auto bin = [&](int64_t t) { const int a = t < T && ids ? ids[t] : 0; return t >= T ? -1 : (unsigned) a < (unsigned) n ? a : n; };
    // adds the wave's tokens to the counters of their adapters, one LDS atomic per adapter -> this lane's place
    auto count_in = [&](int b) {
        int place = 0;
        for (unsigned long long left = __ballot(b >= 0); left;) {
            const int first = __ffsll(left) - 1, one = __shfl(b, first, 64);
            const unsigned long long m = __ballot(b == one);
            int at = 0;
            if (lane == first) at = atomicAdd(&run[one], __popcll(m));
            at = __shfl(at, first, 64);
            if (b == one) place = at + __popcll(m & ((1ull << lane) - 1));
            left &= ~m;
        }
        return place;
    };
    // four ids in flight per thread; all lanes take part
    const int64_t t_end = (T + 4095) / 4096 * 4096;
    int bk[4], at[4];
    for (int64_t t = tid; t < t_end; t += 4096) {
#pragma unroll
        for (int i = 0; i < 4; ++i) bk[i] = bin(t + 1024 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = count_in(bk[i]);
    }
    __syncthreads();
    // exclusive sums of the counts and of both tile counts, a contiguous share of the bins per thread
    const int per = (n + 1 + 1023) / 1024, b0 = min(n + 1, tid * per), b1 = min(n + 1, b0 + per);
    int v[3] = {0, 0, 0}, in[3];
    for (int b = b0; b < b1; ++b) { v[0] += run[b]; v[1] += (run[b] + LT - 1) / LT; v[2] += (run[b] + ET - 1) / ET; }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        in[i] = v[i];
        for (int m = 1; m < 64; m <<= 1) { const int up = __shfl_up(in[i], m, 64); if (lane >= m) in[i] += up; }
        if (lane == 63) wsum[i][wave] = in[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        v[i] = in[i] - v[i];
        for (int w = 0; w < wave; ++w) v[i] += wsum[i][w];
    }
    for (int b = b0; b < b1; ++b) {
        const int c = run[b];
        run[b] = v[0]; toff[b] = v[1]; eoff[b] = v[2];
        v[0] += c; v[1] += (c + LT - 1) / LT; v[2] += (c + ET - 1) / ET;
    }
    if (tid == 1023) { run[n + 1] = v[0]; toff[n + 1] = n_tiles[0] = v[1]; eoff[n + 1] = n_tiles[1] = v[2]; }
    __syncthreads();
    // every tile finds its adapter in the sums
    const auto fill = [&](const int * first, LoraTile * out, int size) {
        for (int i = tid; i < first[n + 1]; i += 1024) {
            int lo = 0, hi = n;                             // the last adapter whose first tile is not past i
            while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (first[mid] <= i) lo = mid; else hi = mid - 1; }
            const int at = run[lo] + (i - first[lo]) * size;
            out[i] = LoraTile{lo < n ? lo : -1, at, min(size, run[lo + 1] - at), 0};
        }
    };
    fill(toff, tiles, LT);
    fill(eoff, etiles, ET);
    __syncthreads();
    if (t_end <= 4096) {                                    // every thread still has its tokens and their places in the runs
#pragma unroll
        for (int i = 0; i < 4; ++i) if (bk[i] >= 0) perm[run[bk[i]] + at[i]] = tid + 1024 * i;
        return;
    }
    for (int64_t t = tid; t < t_end; t += 4096) {
        const int b[4] = {bin(t), bin(t + 1024), bin(t + 2 * 1024), bin(t + 3 * 1024)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int place = count_in(b[i]);
            if (b[i] >= 0) perm[place] = (int) (t + 1024 * i);
        }
    }
}

template <int N> __device__ __forceinline__ void load_n(const __half * p, float (&v)[N]) {
    __half h[N];
    __builtin_memcpy(h, __builtin_assume_aligned(p, 2 * N), 2 * N);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __half2float(h[i]);
}
template <int N> __device__ __forceinline__ void load_n(const float * p, float (&v)[N]) { __builtin_memcpy(v, __builtin_assume_aligned(p, 4 * N), 4 * N); }

// a lane's eight values of a fragment of A, as stored; `at`: the block, `lane`: lane'
template <typename W> struct AFrag;
template <> struct AFrag<__half> {
    __half v[8];
    __device__ __forceinline__ void load(const __half * at, int, int lane) { __builtin_memcpy(v, __builtin_assume_aligned(at + lane * 8, 16), 16); }
    __device__ __forceinline__ float get(int h, int q) const { return __half2float(v[4 * h + q]); }
};
template <> struct AFrag<float> {
    float v[8];
    __device__ __forceinline__ void load(const float * at, int rw, int lane) {
        __builtin_memcpy(v, __builtin_assume_aligned(at + lane * 4, 16), 16);
        __builtin_memcpy(v + 4, __builtin_assume_aligned(at + rw * 16 + lane * 4, 16), 16);
    }
    __device__ __forceinline__ float get(int h, int q) const { return v[4 * h + q]; }
};

// four consecutive activations (4-byte aligned; a 16-byte load takes that); CHECK: past n zero
template <bool CHECK>
__device__ __forceinline__ v4f load4x(const float * p, int64_t k, int64_t n) {
    v4f v;
    if (!CHECK || k + 4 <= n) { __builtin_memcpy(&v, p + k, 16); return v; }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < n ? p[k + i] : 0.0f;
    return v;
}

// ---- the tokens of a workgroup --------------------------------------------------------------------------------------
// How the tokens are dealt to workgroups:
//   LORA_FEW   up to 64 tokens: all tokens of one adapter; with fewer adapters than tokens of adapter `at` (n: none), else of the adapter
//              of token `at`, if that is the first of them;
//   LORA_SCAN  up to LORA_SCAN_T tokens of few adapters (n < 64): tile `at` of `size` tokens, found by every wave from the ids. Lane b
//              counts adapter b (n: none);
//   LORA_PLAN  tile `at` of the plan, or without ids of `size` tokens of adapter 0.
// -> the tokens in `list` (a row of LDS of each wave's own: LDS works in order within a wave, no barrier), their number (0: nothing to do
// here) and the adapter (-1: none)
enum LoraDeal { LORA_FEW, LORA_SCAN, LORA_PLAN };
template <LoraDeal DEAL>
__device__ __forceinline__ int lora_tokens(const LoraTile * tiles, const int * n_tiles, const int * perm, const int * ids, int T, int n, int at, int size, int * list, int * adapter) {
    const int lane = threadIdx.x & 63;
    if constexpr (DEAL == LORA_PLAN) {
        if (!ids) {                                         // all tokens in their order
            const int start = at * size, count = max(0, min(size, T - start));
            for (int i = lane; i < count; i += 64) list[i] = start + i;
            *adapter = 0;
            return count;
        }
        const LoraTile tile = tiles[at];
        if (at >= *n_tiles) return 0;
        for (int i = lane; i < tile.count; i += 64) list[i] = perm[tile.start + i];
        *adapter = tile.adapter;
        return tile.count;
    }
    if constexpr (DEAL == LORA_SCAN) {
        constexpr int C = LORA_SCAN_T / 64;
        int a[C], count = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            a[c] = -1;                                      // no token
            if (64 * c + lane < T) { a[c] = ids[64 * c + lane]; if ((unsigned) a[c] >= (unsigned) n) a[c] = n; }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
            for (unsigned long long left = __ballot(a[c] >= 0); left;) {
                const int one = __builtin_amdgcn_readlane(a[c], __ffsll(left) - 1);
                const unsigned long long m = __ballot(a[c] == one);
                if (lane == one) count += __popcll(m);
                left &= ~m;
            }
        const int n_t = (count + size - 1) / size;
        int first = n_t;
        for (int m = 1; m < 64; m <<= 1) { const int up = __shfl_up(first, m, 64); if (lane >= m) first += up; }
        first -= n_t;
        const unsigned long long own = __ballot(at >= first && at < first + n_t);
        if (!own) return 0;
        const int mine = __ffsll(own) - 1, from = (at - __builtin_amdgcn_readlane(first, mine)) * size;
        int seen = -from;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const unsigned long long m = __ballot(a[c] == mine);
            const int i = seen + __popcll(m & ((1ull << lane) - 1));
            if (a[c] == mine && i >= 0 && i < size) list[i] = 64 * c + lane;
            seen += __popcll(m);
        }
        *adapter = mine < n ? mine : -1;
        return min(seen, size);
    }
    int a = lane < T ? (ids ? ids[lane] : 0) : -2;          // -2: no token
    if (lane < T && (unsigned) a >= (unsigned) n) a = -1;
    const bool by_adapter = n + 1 < T;
    const int mine = by_adapter ? (at < n ? at : -1) : __builtin_amdgcn_readfirstlane(__shfl(a, at, 64));
    const unsigned long long m = __ballot(a == mine);
    *adapter = mine;
    if (!by_adapter && (m & ((1ull << at) - 1))) return 0;
    if (a == mine) list[__popcll(m & ((1ull << lane) - 1))] = lane;
    return __popcll(m);
}

// ---- u[split][token][r] = sum over the split's columns of A[r][k] x[token][k] -------------------------------------------
// A workgroup: one tile, LORA_RC ranks, one split of the columns; its four waves take steps of 32 columns in turn and are joined in
// LDS. 16x16x4 operands: row / column lane & 15, k = lane >> 4; in a step lane group g holds columns 4 g .. 4 g + 3 and 16 + 4 g ...
// Fragments of x read from memory would put neighbouring lanes into different rows, a cache access per lane (28 us against 20 for 512
// tokens of rank 64): a wave loads 128 consecutive bytes of 8 rows per instruction and turns them in a corner of LDS of
// its own (16-byte chunks of a row at chunk ^ ((row >> 1) & 7): no bank twice; LDS works in order within a wave, so no barrier).
// A is stored as its fragments are.
constexpr int SU = 1;                                       // steps in flight per wave; two: 24.2 us against 20.4 for 512 tokens at rank 64

// NS: groups of 16 tokens, NJ: fragments of A. Steps k, k + 128, ... below k_end; CHECK: some columns of a step may lie past n_in.
template <typename W, int NS, int NJ, bool CHECK>
__device__ __forceinline__ void shrink_steps(const float * const (&xr)[4], const W * A, int rw, int64_t tile_ld, int64_t n_in, int64_t k, int64_t k_end, v4f * turn, v4f (&acc)[2][LORA_RC / 16]) {
    constexpr int U = CHECK ? 1 : SU;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, lr = lane >> 3, lc = lane & 7;
    const int al = g * rw + (m & (rw - 1)), st = lr * 8 + (lc ^ ((lr >> 1) & 7)), key = (m >> 1) & 7;
    v4f xn[U][2 * NS];
    AFrag<W> an[U][NJ];
    const auto load = [&](int64_t k0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = CHECK ? k0 : min(k0 + 128 * u, k_end - 32);       // past the end: in bounds and not used
#pragma unroll
            for (int i = 0; i < 2 * NS; ++i) xn[u][i] = load4x<CHECK>(xr[i], at + 4 * lc, n_in);
#pragma unroll
            for (int j = 0; j < NJ; ++j) an[u][j].load(A + j * tile_ld + at * rw, rw, al);
        }
    };
    load(k);
    for (; k < k_end; k += 128 * U) {
        AFrag<W> ac[U][NJ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < 2 * NS; ++i) turn[u * 256 + i * 64 + (i & 1 ? st ^ 4 : st)] = xn[u][i];     // rows 8 i + lr: 8 more rows flip bit 2 of the key
#pragma unroll
            for (int j = 0; j < NJ; ++j) ac[u][j] = an[u][j];
        }
        if (k + 128 * U < k_end) load(k + 128 * U);
        wave_lds_order();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u && k + 128 * u >= k_end) break;
            v4f xv[NS][2];
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) xv[i][h] = turn[u * 256 + (16 * i + m) * 8 + ((4 * h + g) ^ key)];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int i = 0; i < NS; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[i][h][q], ac[u][j].get(h, q), acc[i][j], 0, 0, 0);
        }
        wave_lds_order();
    }
}

template <typename W>
__device__ void shrink_tile(const LoraAdapter & ad, const int * list, int count, int rc, const float * x, int64_t ldx, int64_t n_in, int64_t a_ld,
                            int64_t k_begin, int64_t k_end, float * u, int u_ld, v4f * lds) {
    constexpr int NJ = LORA_RC / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
    const int rw = ad.r_ld == 8 ? 8 : 16;
    const int64_t tile_ld = a_ld * rw;
    const W * A = (const W *) ad.a + (rc / 16) * tile_ld;
    v4f * turn = lds + wave * SU * 256;
    const float * xr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xr[i] = x + (int64_t) list[min(8 * i + (lane >> 3), count - 1)] * ldx;
    v4f acc[2][NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const bool two = count > 16, more = ad.rank - rc > 16;
    const int64_t k = k_begin + 32 * wave, whole = min(k_end, n_in / 32 * 32);                 // from `whole` on with checks
    if (k < whole) {
        if (two && more) shrink_steps<W, 2, 2, false>(xr, A, rw, tile_ld, n_in, k, whole, turn, acc);
        else if (two)    shrink_steps<W, 2, 1, false>(xr, A, rw, tile_ld, n_in, k, whole, turn, acc);
        else if (more)   shrink_steps<W, 1, 2, false>(xr, A, rw, tile_ld, n_in, k, whole, turn, acc);
        else             shrink_steps<W, 1, 1, false>(xr, A, rw, tile_ld, n_in, k, whole, turn, acc);
    }
    const int64_t rest = k < whole ? k + (whole - k + 127) / 128 * 128 : k;                    // this wave's first step at or past it
    if (rest < k_end) {
        if (more) shrink_steps<W, 2, 2, true>(xr, A, rw, tile_ld, n_in, rest, k_end, turn, acc);
        else      shrink_steps<W, 2, 1, true>(xr, A, rw, tile_ld, n_in, rest, k_end, turn, acc);
    }
    __syncthreads();
    float * red = reinterpret_cast<float *>(lds);           // [4][LT][LORA_RC + 1]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) red[(wave * LT + 16 * i + 4 * g + q) * (LORA_RC + 1) + 16 * j + m] = acc[i][j][q];
    __syncthreads();
    const int nr = min(LORA_RC, ad.r_ld - rc);
    for (int e = threadIdx.x; e < count * LORA_RC; e += 256) {
        const int t = e / LORA_RC, r = e % LORA_RC;
        const auto part = [&](int w) { return red[(w * LT + t) * (LORA_RC + 1) + r]; };
        if (r < nr)                                         // columns between rank and r_ld are zero, whatever x holds
            u[(int64_t) list[t] * u_ld + rc + r] = rc + r < ad.rank ? (part(0) + part(1)) + (part(2) + part(3)) : 0.0f;
    }
    __syncthreads();
}

template <LoraDeal DEAL>
__global__ __launch_bounds__(256, 3)
void lora_shrink_kernel(const LoraAdapter * __restrict__ ads, int n, const int * __restrict__ ids, const LoraTile * __restrict__ tiles, const int * __restrict__ n_tiles,
                        const int * __restrict__ perm, const float * __restrict__ x, int64_t ldx, int64_t n_in, int64_t a_ld, int64_t T, int splits, int64_t k_split, int n_z,
                        float * __restrict__ u, int u_ld) {
    __shared__ v4f lds[std::max(4 * SU * 256, LT * (LORA_RC + 1))];          // the waves' corners, then the join
    __shared__ int lists[4][64];
    int * list = lists[threadIdx.x >> 6];
    // the split is the fastest index, then the ranks: all workgroups of a split on one XCD (8 splits and more), those that read the
    // same columns of x one after the other
    const int split = (int) (blockIdx.x % (unsigned) splits), rest = (int) (blockIdx.x / (unsigned) splits), rc = rest % n_z * LORA_RC;
    int a = -1;
    const int count = lora_tokens<DEAL>(tiles, n_tiles, perm, ids, (int) T, n, rest / n_z, LT, list, &a);
    wave_lds_order();                                       // the list
    const LoraAdapter ad = ads[max(a, 0)];                  // on its way beside the ids where `a` does not come from them
    if (!count || a < 0 || rc >= ad.rank) return;
    const int64_t k0 = split * k_split, k1 = min(a_ld, k0 + k_split);
    float * us = u + split * T * u_ld;
    for (int t0 = 0; t0 < count; t0 += LT) {
        if (ad.f32) shrink_tile<float>(ad, list + t0, min(LT, count - t0), rc, x, ldx, n_in, a_ld, k0, k1, us, u_ld, lds);
        else        shrink_tile<__half>(ad, list + t0, min(LT, count - t0), rc, x, ldx, n_in, a_ld, k0, k1, us, u_ld, lds);
    }
}

// ---- y[token][o] = base[token][o] + sum_r (scale sum_split u[split][token][r]) B[o][r] ----------------------------------
// A wave owns 64 columns (four fragments of 16) and takes its tokens 16 at a time. u is the A operand, so the result has token
// 4 (lane >> 4) + i in register i and column lane & 15: a load or store of base and y takes 64 consecutive bytes of 4 tokens, four
// cache accesses. (The other way round a lane has four columns and an instruction moves 16 bytes per lane, but neighbouring lanes
// are in different rows, which costs an access per lane: 106 us against 100 for 4096 tokens x 4096 -> 14336. Asking for B before u and the
// base gains nothing: 13.0 us against 12.5 for 48 tokens.)
struct ExpandWave {
    const int * list; int count;           // tokens
    const float * us; int us_ld;           // scale * u of them, in LDS
    int64_t o0, n_out;                     // columns, o0 the same in all lanes
    const float * base; int64_t ldb; float * y; int64_t ldy;
};
__device__ __forceinline__ void expand_base(const ExpandWave & e, v4f (&acc)[4]) {
    const int m = (int) threadIdx.x & 15, t = ((int) threadIdx.x & 63) >> 4 << 2;
    const int left = (int) min(e.n_out - e.o0, (int64_t) 64) - m;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (!e.base) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float * p = e.base + e.list[min(t + i, e.count - 1)] * e.ldb + e.o0 + m;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (16 * j < left && t + i < e.count) acc[j][i] = p[16 * j];
    }
}
__device__ __forceinline__ void expand_store(const ExpandWave & e, const v4f (&acc)[4]) {
    const int m = (int) threadIdx.x & 15, t = ((int) threadIdx.x & 63) >> 4 << 2;
    const int left = (int) min(e.n_out - e.o0, (int64_t) 64) - m;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (t + i < e.count) {
            float * p = e.y + e.list[t + i] * e.ldy + e.o0 + m;
#pragma unroll
            for (int j = 0; j < 4; ++j) if (16 * j < left) p[16 * j] = acc[j][i];
        }
}
// KQ: ranks per lane of a fragment: 4, or 2 for the one of 8 ranks
template <typename W, int KQ>
__device__ __forceinline__ void expand_mult(const ExpandWave & e, const W * b_all, int r_ld, v4f (&acc)[4]) {
    const int lane = threadIdx.x & 63;
    const int last = (int) ((e.n_out - 1) >> 4), tile = (int) (e.o0 >> 4);
    const float * ur = e.us + (lane & 15) * e.us_ld + KQ * (lane >> 4);
#pragma unroll 1
    for (int r = 0; r < r_ld; r += 4 * KQ) {
        float b[4][KQ], uv[KQ];
#pragma unroll
        for (int j = 0; j < 4; ++j) load_n<KQ>(b_all + ((int64_t) min(tile + j, last) * r_ld + r) * 16 + KQ * lane, b[j]);
        load_n<KQ>(ur + r, uv);
#pragma unroll
        for (int q = 0; q < KQ; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(uv[q], b[j][q], acc[j], 0, 0, 0);
    }
}

template <LoraDeal DEAL>
__global__ __launch_bounds__(256, 5)
void lora_expand_kernel(const LoraAdapter * __restrict__ ads, int n, const int * __restrict__ ids, const LoraTile * __restrict__ tiles, const int * __restrict__ n_tiles,
                        const int * __restrict__ perm, const float * __restrict__ u, int u_ld, int splits, int64_t T, int64_t n_out,
                        const float * base, int64_t ldb, float * y, int64_t ldy) {
    extern __shared__ __align__(16) float us[];             // [16][r_ld + 4]
    __shared__ int lists[4][DEAL == LORA_FEW ? 64 : ET];
    // neighbouring workgroups take neighbouring columns of the same tokens
    const int n_col = (int) ((n_out + 255) >> 8), at = (int) (blockIdx.x / (unsigned) n_col), col = (int) (blockIdx.x % (unsigned) n_col);
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    int * list = lists[wave];
    int a = -1;
    const int all = lora_tokens<DEAL>(tiles, n_tiles, perm, ids, (int) T, n, at, ET, list, &a);
    wave_lds_order();                                       // the list
    const LoraAdapter ad = ads[max(a, 0)];
    if (!all || (a < 0 && base == y)) return;
    ExpandWave e{list, all, us, 0, 0, n_out, base, ldb, y, ldy};
    e.us_ld = ad.r_ld + 4;                                  // 16-byte rows that start on different banks
    const int n4 = ad.r_ld >> 2;
#pragma unroll 1
    for (int t0 = 0; t0 < all; t0 += 16) {
        e.list = list + t0;
        e.count = min(16, all - t0);
        int64_t o0 = (int64_t) col * 256 + 64 * wave;
        asm volatile("" : "+s"(o0));                        // addresses are formed here, not kept across (and spilled) by the loop
        e.o0 = o0;
        v4f acc[4];
        expand_base(e, acc);                        // asked for first: it takes the longest way
        if (a >= 0) {                                       // no adapter: y is the base
            if (t0) __syncthreads();
#pragma unroll 1
            for (int i = threadIdx.x; i < 16 * n4; i += 256) {
                const int t = i / n4, r = 4 * (i - t * n4);
                v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
                if (t < e.count) {
                    const float * up = u + (int64_t) e.list[t] * u_ld + r;
#pragma unroll 1
                    for (int s0 = 0; s0 < splits; s0 += 4) {            // four at a time in flight; past the last split: the last one, not added
                        v4f p[4];
#pragma unroll
                        for (int s = 0; s < 4; ++s) p[s] = *reinterpret_cast<const v4f *>(up + min(s0 + s, splits - 1) * T * u_ld);
#pragma unroll
                        for (int s = 0; s < 4; ++s) if (s0 + s < splits) v += p[s];
                    }
                }
                *reinterpret_cast<v4f *>(us + t * e.us_ld + r) = ad.scale * v;
            }
            __syncthreads();
            if (ad.f32) {
                if (ad.r_ld == 8) expand_mult<float, 2>(e, (const float *) ad.b, ad.r_ld, acc);
                else              expand_mult<float, 4>(e, (const float *) ad.b, ad.r_ld, acc);
            } else {
                if (ad.r_ld == 8) expand_mult<__half, 2>(e, (const __half *) ad.b, ad.r_ld, acc);
                else              expand_mult<__half, 4>(e, (const __half *) ad.b, ad.r_ld, acc);
            }
        }
        expand_store(e, acc);
    }
}

// ---- one launch for one to four tokens ----------------------------------------------------------------------------------
// us[r] = scale * sum_k A[r][k] x[k], 16 (or 8) ranks at a time: a wave takes every eighth block of 32 columns, a lane its rank and
// eight of them; joined over the lane groups by exchanges and over the waves in LDS.
template <typename W>
__device__ void fused_u(const LoraAdapter & ad, const float * x, int64_t n_in, int64_t a_ld, float * us, float (*red)[16]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const int rw = ad.r_ld == 8 ? 8 : 16, al = g * rw + (m & (rw - 1));
    for (int rc = 0; rc < ad.r_ld; rc += rw) {
        const W * A = (const W *) ad.a + (int64_t) (rc / rw) * rw * a_ld;
        float acc = 0.0f;
#pragma unroll 4
        for (int64_t k = 32 * wave; k < a_ld; k += 256) {
            AFrag<W> av;
            av.load(A + k * rw, rw, al);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4f xv = load4x<true>(x, k + 16 * h + 4 * g, n_in);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc = fmaf(av.get(h, q), xv[q], acc);
            }
        }
        acc += __shfl_xor(acc, 16, 64);
        acc += __shfl_xor(acc, 32, 64);
        if (lane < rw) red[wave][lane] = acc;
        __syncthreads();
        if ((int) threadIdx.x < rw) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) v += red[w][threadIdx.x];
            us[rc + threadIdx.x] = rc + (int) threadIdx.x < ad.rank ? ad.scale * v : 0.0f;     // between rank and r_ld zero, whatever x holds
        }
        __syncthreads();
    }
}

// one column: v + sum_r us[r] B[o][r]
template <typename W>
__device__ __forceinline__ float fused_column(const LoraAdapter & ad, int64_t o, const float * us, float v) {
    const W * B = (const W *) ad.b + (o >> 4) * 16 * ad.r_ld;
    if (ad.r_ld == 8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float b[2];
            load_n<2>(B + g * 32 + 2 * (o & 15), b);
            v = fmaf(us[2 * g], b[0], v);
            v = fmaf(us[2 * g + 1], b[1], v);
        }
        return v;
    }
    for (int r = 0; r < ad.r_ld; r += 16)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float b[4];
            load_n<4>(B + r * 16 + g * 64 + 4 * (o & 15), b);
#pragma unroll
            for (int q = 0; q < 4; ++q) v = fmaf(us[r + 4 * g + q], b[q], v);
        }
    return v;
}

__global__ __launch_bounds__(512)
void lora_fused_kernel(const LoraAdapter * __restrict__ ads, int n, const int * __restrict__ ids, const float * __restrict__ x, int64_t ldx, int64_t n_in, int64_t a_ld,
                       int64_t n_out, const float * base, int64_t ldb, float * y, int64_t ldy) {
    __shared__ __align__(16) float us[SDH_LORA_MAX_RANK];
    __shared__ float red[8][16];
    const int64_t t = blockIdx.x, o = (int64_t) blockIdx.y * 512 + threadIdx.x;
    const int a = ids ? ids[t] : 0;
    const float v = base && o < n_out ? base[t * ldb + o] : 0.0f;
    if ((unsigned) a >= (unsigned) n) {
        if (o < n_out && base != y) y[t * ldy + o] = v;
        return;
    }
    const LoraAdapter ad = ads[a];
    if (ad.f32) fused_u<float>(ad, x + t * ldx, n_in, a_ld, us, red);
    else        fused_u<__half>(ad, x + t * ldx, n_in, a_ld, us, red);
    if (o >= n_out) return;
    y[t * ldy + o] = ad.f32 ? fused_column<float>(ad, o, us, v) : fused_column<__half>(ad, o, us, v);
}

// ---- host -----------------------------------------------------------------------------------------------------------
static int lora_check(const char * what, int i, const sdh_tensor & t, int64_t ne0, int64_t ne1) {
    if (!t.data || (t.type != SDH_TYPE_F16 && t.type != SDH_TYPE_F32)) { set_error("sdh_lora_create: adapter %d: %s is missing or not F16 / F32", i, what); return SDH_ERR_INVALID; }
    if (t.ne[0] != ne0 || t.ne[1] != ne1 || t.ne[2] > 1 || t.ne[3] > 1) {
        set_error("sdh_lora_create: adapter %d: %s is [%lld, %lld], expected [%lld, %lld]", i, what, (long long) t.ne[0], (long long) t.ne[1], (long long) ne0, (long long) ne1);
        return SDH_ERR_INVALID;
    }
    return SDH_OK;
}

// t (F16 / F32, any strides) as contiguous rows, as it is (in place, or copied to `keep`) or widened
static const void * lora_rows(const sdh_tensor & t, bool f32, std::vector<uint8_t> & keep) {
    const size_t n0 = (size_t) t.ne[0], n1 = (size_t) t.ne[1], es = f32 ? 4 : 2;
    if ((t.type == SDH_TYPE_F32) == f32 && t.nb[0] == (int64_t) es && t.nb[1] == (int64_t) (n0 * es)) return t.data;
    keep.resize(n0 * n1 * es);
    if (f32) {
        const std::vector<float> v = tensor_f32(t);
        memcpy(keep.data(), v.data(), keep.size());
        return keep.data();
    }
    for (size_t i1 = 0; i1 < n1; ++i1) {
        const uint8_t * row = (const uint8_t *) t.data + (int64_t) i1 * t.nb[1];
        if (t.nb[0] == 2) memcpy(keep.data() + i1 * n0 * 2, row, n0 * 2);
        else for (size_t i0 = 0; i0 < n0; ++i0) memcpy(keep.data() + (i1 * n0 + i0) * 2, row + (int64_t) i0 * t.nb[0], 2);
    }
    return keep.data();
}

// rows of A [rank][n_in] into fragment order (LoraAdapter), E: the element
template <typename E>
static void lora_pack_a(const E * rows, int rank, int r_ld, int64_t n_in, int64_t a_ld, E * out) {
    const int rw = r_ld == 8 ? 8 : 16;
    const bool f32 = sizeof(E) == 4;
    for (int r = 0; r < rank; ++r)
        for (int64_t k0 = 0; k0 < n_in; k0 += 32) {
            E * block = out + (r / rw) * a_ld * rw + k0 * rw;
            for (int i = 0; i < 8; ++i) {                   // four columns stay neighbours: half h = i >> 2 of the block, lane group g = i & 3
                const int64_t k = k0 + 4 * i, n = std::min<int64_t>(4, n_in - k);
                const int lane = (i & 3) * rw + r % rw, h = i >> 2;
                if (n > 0) memcpy(block + (f32 ? h * rw * 16 + lane * 4 : lane * 8 + h * 4), rows + r * n_in + k, n == 4 ? 4 * sizeof(E) : (size_t) n * sizeof(E));
            }
        }
}
// rows of B [n_out][rank]
template <typename E>
static void lora_pack_b(const E * rows, int rank, int r_ld, int64_t n_out, E * out) {
    const int kq = r_ld == 8 ? 2 : 4;                       // ranks of a lane
    for (int64_t o = 0; o < n_out; ++o) {
        E * tile = out + (o >> 4) * 16 * r_ld + (o & 15) * kq;
        for (int r = 0; r < rank; r += kq)
            memcpy(tile + (r / (4 * kq)) * 256 + (r / kq & 3) * 16 * kq, rows + o * rank + r, r + kq <= rank ? (size_t) kq * sizeof(E) : (size_t) (rank - r) * sizeof(E));
    }
}

static int lora_create(int64_t n_in, int64_t n_out, const sdh_lora_desc * d, int n, LoraSet ** out) {
    if (n_in < 1 || n_out < 1 || n_in > (1 << 24) || n_out > (1 << 24)) { set_error("sdh_lora_create: bad dims n_in=%lld n_out=%lld", (long long) n_in, (long long) n_out); return SDH_ERR_INVALID; }
    if (n < 1 || n > SDH_LORA_MAX_ADAPTERS) { set_error("sdh_lora_create: %d adapters (1 .. %d)", n, SDH_LORA_MAX_ADAPTERS); return SDH_ERR_INVALID; }
    LoraSet l;
    l.n_in = n_in; l.n_out = n_out; l.n = n;
    l.a_ld = (n_in + 31) / 32 * 32;
    const int64_t b_rows = (n_out + 15) / 16 * 16;
    std::vector<LoraAdapter> tab((size_t) n);
    std::vector<size_t> at_a((size_t) n), at_b((size_t) n);
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    size_t total = up(tab.size() * sizeof(LoraAdapter));
    for (int i = 0; i < n; ++i) {
        const int64_t r = d[i].a.ne[1];
        if (r < 1 || r > SDH_LORA_MAX_RANK) { set_error("sdh_lora_create: adapter %d: rank %lld (1 .. %d)", i, (long long) r, SDH_LORA_MAX_RANK); return SDH_ERR_INVALID; }
        int rc = lora_check("lora_a", i, d[i].a, n_in, r);
        if (rc == SDH_OK) rc = lora_check("lora_b", i, d[i].b, r, n_out);
        if (rc != SDH_OK) return rc;
        LoraAdapter & a = tab[(size_t) i];
        a.rank = (int) r; a.r_ld = r <= 8 ? 8 : (int) (r + 15) / 16 * 16; a.scale = d[i].scale;
        a.f32 = d[i].a.type == SDH_TYPE_F32 || d[i].b.type == SDH_TYPE_F32;
        l.u_ld = std::max(l.u_ld, a.r_ld);
        l.stored_bytes += r * n_in * (d[i].a.type == SDH_TYPE_F32 ? 4 : 2) + r * n_out * (d[i].b.type == SDH_TYPE_F32 ? 4 : 2);
        const size_t es = a.f32 ? 4 : 2;
        at_a[(size_t) i] = total; total += up((size_t) (a.r_ld * l.a_ld) * es);
        at_b[(size_t) i] = total; total += up((size_t) b_rows * (size_t) a.r_ld * es);
        l.any_f32 |= a.f32 != 0;
    }
    if (const int rc = ready_on_device("sdh_lora_create")) return rc;
    l.device = lib().device;
    SDH_HIP_CHECK(hipMalloc((void **) &l.dev, total));
    struct Guard { uint8_t * p; ~Guard() { if (p) (void) hipFree(p); } } guard{l.dev};
    std::vector<uint8_t> buf, keep;
    auto upload = [&](size_t at, size_t bytes) { return hipMemcpy(l.dev + at, buf.data(), bytes, hipMemcpyHostToDevice); };
    for (int i = 0; i < n; ++i) {
        LoraAdapter & a = tab[(size_t) i];
        const size_t es = a.f32 ? 4 : 2;
        a.a = l.dev + at_a[(size_t) i]; a.b = l.dev + at_b[(size_t) i];
        const void * rows = lora_rows(d[i].a, a.f32 != 0, keep);
        buf.assign((size_t) (a.r_ld * l.a_ld) * es, 0);
        if (a.f32) lora_pack_a((const float *) rows, a.rank, a.r_ld, n_in, l.a_ld, (float *) buf.data());
        else       lora_pack_a((const uint16_t *) rows, a.rank, a.r_ld, n_in, l.a_ld, (uint16_t *) buf.data());
        SDH_HIP_CHECK(upload(at_a[(size_t) i], buf.size()));
        rows = lora_rows(d[i].b, a.f32 != 0, keep);
        buf.assign((size_t) b_rows * (size_t) a.r_ld * es, 0);
        if (a.f32) lora_pack_b((const float *) rows, a.rank, a.r_ld, n_out, (float *) buf.data());
        else       lora_pack_b((const uint16_t *) rows, a.rank, a.r_ld, n_out, (uint16_t *) buf.data());
        SDH_HIP_CHECK(upload(at_b[(size_t) i], buf.size()));
    }
    buf.resize(tab.size() * sizeof(LoraAdapter));
    memcpy(buf.data(), tab.data(), buf.size());
    SDH_HIP_CHECK(upload(0, buf.size()));
    *out = new LoraSet(l);
    guard.p = nullptr;
    return SDH_OK;
}

static int sdh_lora_create_impl(int64_t n_in, int64_t n_out, const sdh_lora_desc * d, int n, sdh_lora ** out) {
    if (!d || !out) { set_error("sdh_lora_create: null argument"); return SDH_ERR_INVALID; }
    *out = nullptr;
    LoraSet * l = nullptr;
    const int rc = lora_create(n_in, n_out, d, n, &l);
    if (rc == SDH_OK) *out = reinterpret_cast<sdh_lora *>(l);
    return rc;
}

struct LoraCall { const int * ids; const float * x; int64_t ldx, T; const float * base; int64_t ldb; float * y; int64_t ldy; };

template <LoraDeal DEAL>
static void lora_two_steps(const LoraSet & l, const LoraWs & w, const LoraCall & c, hipStream_t s) {
    const LoraAdapter * ads = (const LoraAdapter *) l.dev;
    const int64_t k_split = ((l.a_ld + w.splits - 1) / w.splits + 31) / 32 * 32;      // the last ones may be empty
    const int n_z = (l.u_ld + LORA_RC - 1) / LORA_RC;
    const auto along = [&](int size, int64_t planned) {                               // workgroups along the tokens, as lora_tokens deals them
        return DEAL == LORA_FEW ? std::min<int64_t>(c.T, l.n + 1) : c.ids ? planned : (c.T + size - 1) / size;
    };
    const auto shrink = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned) (along(LT, w.max_tiles) * n_z * w.splits)), dim3(256), 0, s, ads, l.n, c.ids, w.tiles, w.n_tiles, w.perm, c.x, c.ldx, l.n_in, l.a_ld, c.T, w.splits, k_split, n_z, w.u, l.u_ld);
    };
    shrink(lora_shrink_kernel<DEAL>);
    const unsigned n_col = (unsigned) ((l.n_out + 255) / 256);
    const auto expand = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned) along(ET, w.max_etiles) * n_col), dim3(256), (size_t) (16 * (l.u_ld + 4)) * 4, s,
                           ads, l.n, c.ids, w.etiles, w.n_tiles + 1, w.perm, w.u, l.u_ld, w.splits, c.T, l.n_out, c.base, c.ldb, c.y, c.ldy);
    };
    expand(lora_expand_kernel<DEAL>);
}

static void lora_launch(const LoraSet & l, const LoraWs & w, const LoraCall & c, hipStream_t s) {
    // one launch while every workgroup can read all of A in about the time of a launch: 1 and 4 tokens in a replayed graph, A of 128 KB
    // 5.5 and 5.7 us (two launches 8.9 and 9.0), 256 KB 9.1 and 11.4 (9.8), 512 KB 20.2 (10.7 and 11.0)
    if (c.T <= 4 && (int64_t) l.u_ld * l.a_ld * (l.any_f32 ? 4 : 2) <= (192 << 10)) {
        hipLaunchKernelGGL(lora_fused_kernel, dim3((unsigned) c.T, (unsigned) ((l.n_out + 511) / 512)), dim3(512), 0, s, (const LoraAdapter *) l.dev, l.n, c.ids, c.x, c.ldx, l.n_in, l.a_ld, l.n_out, c.base, c.ldb, c.y, c.ldy);
    } else if (c.T <= 64) lora_two_steps<LORA_FEW>(l, w, c, s);
    // a wave finds its tokens in a step per adapter and 64 tokens, while these steps take less than the plan's launch: 128 / 256 tokens of 3
    // adapters in any order 20.5 / 26.6 us against 24.3 / 29.7 (rank 64, 14336 -> 4096), 128 of 15 16.5 against 20.0 (rank 16, 4096 -> 14336),
    // but 256 of 15 27.0 against 23.7 and 512 of 3 30.4 against 29.3
    else if (c.ids && c.T <= LORA_SCAN_T && (c.T + 63) / 64 * (l.n + 1) <= 32) lora_two_steps<LORA_SCAN>(l, w, c, s);
    else {
        if (c.ids) hipLaunchKernelGGL(lora_plan_kernel, dim3(1), dim3(1024), (size_t) (l.n + 2) * 12, s, c.ids, c.T, l.n, w.perm, w.tiles, w.etiles, w.n_tiles);
        lora_two_steps<LORA_PLAN>(l, w, c, s);
    }
}

// The most tokens of a pass: a launch has fewer than 2^32 threads, 256 for every tile and 256 columns of y
static int64_t lora_chunk(const LoraSet & l) {
    const int64_t most = (1 << 24) / ((l.n_out + 255) / 256 + 1) - 1;            // tiles, at least 250
    int64_t c = 1 << 20;
    while (c > 64 && (c + ET - 1) / ET + std::min<int64_t>(c, l.n + 1) > most) c = c / 2;
    return c;
}

static int sdh_lora_apply_impl(const sdh_lora * h, const int32_t * ids, const float * x, int64_t ldx, int64_t T,
                               const float * base, int64_t ldb, float * y, int64_t ldy, void * ws, int64_t ws_bytes, void * stream) {
    static const char * who = "sdh_lora_apply";
    if (T == 0) return ready_on_device(who);
    if (!h || !x || !y || !ws) { set_error("%s: null argument", who); return SDH_ERR_INVALID; }
    const LoraSet & l = *reinterpret_cast<const LoraSet *>(h);
    if (T < 0 || T > INT32_MAX / 2 || ldx < l.n_in || ldy < l.n_out || (base && ldb < l.n_out) || (base == y && ldb != ldy) || y == x) {
        set_error("%s: bad shape: T=%lld ldx=%lld (n_in=%lld) ldb=%lld ldy=%lld (n_out=%lld)", who, (long long) T, (long long) ldx, (long long) l.n_in, (long long) ldb, (long long) ldy, (long long) l.n_out);
        return SDH_ERR_INVALID;
    }
    if (!aligned(ids, 4) || !aligned(x, 4) || !aligned(base, 4) || !aligned(y, 4) || !aligned(ws, 16)) { set_error("%s: pointers need 4-byte alignment, the workspace 16", who); return SDH_ERR_INVALID; }
    const int rc = ready_on_device(who);
    if (rc != SDH_OK) return rc;
    if (l.device != lib().device) { set_error("%s: the set was made on device %d, the library is bound to %d", who, l.device, lib().device); return SDH_ERR_INVALID; }
    const int64_t need = sdh_lora_workspace_bytes(h, T);
    if (ws_bytes < need) { set_error("%s: the workspace holds %lld bytes, %lld are needed", who, (long long) ws_bytes, (long long) need); return SDH_ERR_INVALID; }
    const int64_t chunk = lora_chunk(l);
    for (int64_t t0 = 0; t0 < T; t0 += chunk) {
        const int64_t n = std::min(chunk, T - t0);
        lora_launch(l, lora_ws(l, n, (uint8_t *) ws), LoraCall{ids ? ids + t0 : nullptr, x + t0 * ldx, ldx, n, base ? base + t0 * ldb : nullptr, ldb, y + t0 * ldy, ldy}, (hipStream_t) stream);
    }
    SDH_HIP_CHECK(hipGetLastError());
    return SDH_OK;
}

} // namespace sdh

using namespace sdh;

extern "C" int sdh_lora_create(int64_t n_in, int64_t n_out, const sdh_lora_desc * adapters, int n_adapters, sdh_lora ** out) {
    SDH_NO_THROW(sdh_lora_create_impl(n_in, n_out, adapters, n_adapters, out));
}

extern "C" void sdh_lora_destroy(sdh_lora * h) {
    if (!h) return;
    LoraSet * l = reinterpret_cast<LoraSet *>(h);
    (void) hipDeviceSynchronize();
    (void) hipFree(l->dev);
    delete l;
}

extern "C" int64_t sdh_lora_bytes(const sdh_lora * h) { return h ? reinterpret_cast<const LoraSet *>(h)->stored_bytes : (int64_t) SDH_ERR_INVALID; }

extern "C" int64_t sdh_lora_workspace_bytes(const sdh_lora * h, int64_t T) {
    if (!h || T < 0 || T > INT32_MAX / 2) { set_error("sdh_lora_workspace_bytes: bad argument"); return SDH_ERR_INVALID; }
    if (T == 0) return 0;
    const LoraSet & l = *reinterpret_cast<const LoraSet *>(h);
    // what any number of tokens up to T needs: fewer tokens can have more splits, so the most tokens of each number of splits count
    const int64_t most = std::min(T, lora_chunk(l));
    int64_t bytes = lora_ws(l, most, nullptr).bytes;
    for (int64_t splits = 2; splits <= LORA_SPLITS; splits *= 2) bytes = std::max(bytes, lora_ws(l, std::min(most, LORA_WGS / splits * LT), nullptr).bytes);
    return bytes;
}

extern "C" int sdh_lora_apply(const sdh_lora * l, const int32_t * ids, const float * x, int64_t ldx, int64_t n_tokens,
                              const float * base, int64_t ldb, float * y, int64_t ldy, void * ws, int64_t ws_bytes, void * stream) {
    SDH_NO_THROW(sdh_lora_apply_impl(l, ids, x, ldx, n_tokens, base, ldb, y, ldy, ws, ws_bytes, stream));
}
