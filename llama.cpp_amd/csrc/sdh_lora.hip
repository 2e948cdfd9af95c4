// sdh_lora.hip — low-rank adapters of many requests beside one projection: y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t].
//
// Three steps: the tokens are sorted by adapter and cut into tiles of 32 of one adapter each (lora_plan_kernel; ids live on the
// device, so a captured graph sees the ids of the replay), u = A x for every tile (lora_shrink_kernel), y = base + scale B u
// (lora_expand_kernel). An adapter is then read once per tile of its tokens, whatever the order of the tokens.
//
// Everything is F32: v_mfma_f32_16x16x4_f32 for u, whose K is long (n_in), fused multiply-adds for y, whose K is the rank: that
// step moves 8 bytes per output for 2 * rank operations.
#include "sdh_internal.h"

#include <algorithm>
#include <cstring>
#include <hip/hip_fp16.h>

namespace sdh {

typedef float v4f __attribute__((ext_vector_type(4)));

struct LoraAdapter {
    const void * a;        // [rank][a_ld]   f16 / f32, columns past n_in zero
    const void * b;        // [n_out][r_ld]  f16 / f32, columns past rank zero
    float scale;
    int rank, r_ld, f32;
};

struct LoraSet {
    int64_t n_in = 0, n_out = 0, a_ld = 0;
    int n = 0, u_ld = 0;                   // adapters; row pitch of u: the largest r_ld
    uint8_t * dev = nullptr;               // the LoraAdapter table, then the matrices
    int64_t stored_bytes = 0;
};

constexpr int LT = 32;                     // tokens per tile
constexpr int LORA_RC = 64;                // ranks per pass of the shrink kernel

struct LoraTile { int adapter, start, count, pad; };       // adapter -1: none

// the caller's workspace
struct LoraWs {
    int * perm; LoraTile * tiles; int * n_tiles; float * u;
    int64_t max_tiles; int splits; int64_t bytes;
};

static LoraWs lora_ws(const LoraSet & l, int64_t T, uint8_t * base) {
    LoraWs w{};
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    w.max_tiles = (T + LT - 1) / LT + std::min<int64_t>(T, l.n + 1);
    // K splits of the shrink step: about two workgroups per CU, at least 128 columns each
    const int64_t tiles = (T + LT - 1) / LT, most = std::max<int64_t>(1, l.n_in / 128);
    w.splits = (int) std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(16, most), 512 / tiles));
    int64_t at = 0;
    w.perm = (int *) (base + at);         at += up(T * 4);
    w.tiles = (LoraTile *) (base + at);   at += up(w.max_tiles * (int64_t) sizeof(LoraTile));
    w.n_tiles = (int *) (base + at);      at += 256;
    w.u = (float *) (base + at);          at += up((int64_t) w.splits * T * l.u_ld * 4);
    w.bytes = at;
    return w;
}

// ---- tokens sorted by adapter, cut into tiles -----------------------------------------------------------------------
// One workgroup: count, scan, scatter. The place of a token inside its adapter's run depends on the order of the atomics; no
// result depends on the place.
__global__ __launch_bounds__(1024)
void lora_plan_kernel(const int * __restrict__ ids, int64_t T, int n, int * __restrict__ perm, LoraTile * __restrict__ tiles, int * __restrict__ n_tiles) {
    extern __shared__ int lds[];
    int * cnt = lds, * off = lds + (n + 1), * toff = lds + 2 * (n + 1);      // bin n: no adapter
    __shared__ int wsum[2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int b = tid; b <= n; b += 1024) cnt[b] = 0;
    __syncthreads();
    auto bin = [&](int64_t t) { const int a = ids ? ids[t] : 0; return (unsigned) a < (unsigned) n ? a : n; };
    for (int64_t t = tid; t < T; t += 1024) atomicAdd(&cnt[bin(t)], 1);
    __syncthreads();
    // exclusive sums of the counts and of the tile counts, a contiguous share of the bins per thread
    const int per = (n + 1 + 1023) / 1024, b0 = tid * per, b1 = min(n + 1, b0 + per);
    int c = 0, k = 0;
    for (int b = b0; b < b1; ++b) { c += cnt[b]; k += (cnt[b] + LT - 1) / LT; }
    int ci = c, ki = k;
    for (int m = 1; m < 64; m <<= 1) {
        const int cu = __shfl_up(ci, m, 64), ku = __shfl_up(ki, m, 64);
        if (lane >= m) { ci += cu; ki += ku; }
    }
    if (lane == 63) { wsum[0][wave] = ci; wsum[1][wave] = ki; }
    __syncthreads();
    int cb = ci - c, kb = ki - k;
    for (int w = 0; w < wave; ++w) { cb += wsum[0][w]; kb += wsum[1][w]; }
    for (int b = b0; b < b1; ++b) {
        off[b] = cb; toff[b] = kb;
        for (int j = 0; j * LT < cnt[b]; ++j) tiles[kb + j] = LoraTile{b < n ? b : -1, cb + j * LT, min(LT, cnt[b] - j * LT), 0};
        cb += cnt[b]; kb += (cnt[b] + LT - 1) / LT;
    }
    if (tid == 1023) *n_tiles = kb;
    __syncthreads();
    for (int64_t t = tid; t < T; t += 1024) perm[atomicAdd(&off[bin(t)], 1)] = (int) t;
}

// eight consecutive weights as F32
__device__ __forceinline__ void load8(const __half * p, float (&v)[8]) {
    const uint4 q = *reinterpret_cast<const uint4 *>(p);
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 h; __builtin_memcpy(&h, &w[i], 4);
        v[2 * i] = __low2float(h); v[2 * i + 1] = __high2float(h);
    }
}
__device__ __forceinline__ void load8(const float * p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// eight consecutive activations; past n: zero
template <bool VEC>
__device__ __forceinline__ void load8x(const float * p, int64_t k, int64_t n, float (&v)[8]) {
    if (VEC && k + 8 <= n) { load8(p + k, v); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < n ? p[k + i] : 0.0f;
}

// ---- u[split][place][r] = sum over the split's columns of A[r][k] x[token][k] -----------------------------------------
// 16x16x4 operands: row / column lane & 15, k = lane >> 4. Which k an MFMA takes is free as long as both operands agree: lane
// group g holds columns 8 g .. 8 g + 7 of a 32-column step and MFMA j multiplies column 8 g + j, so every load is 16 bytes.
template <typename W, bool VEC>
__device__ void shrink_body(const LoraAdapter & ad, const LoraTile & tile, const int * perm, const float * x, int64_t ldx, int64_t n_in, int64_t a_ld,
                            int64_t k_begin, int64_t k_end, float * u, int u_ld, float (*red)[LT][LORA_RC + 1]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const W * A = (const W *) ad.a;
    const float * xr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) xr[i] = x + (int64_t) perm[tile.start + min(16 * i + m, tile.count - 1)] * ldx;
    for (int rc = 0; rc < ad.rank; rc += LORA_RC) {
        const int nj = min(4, (ad.rank - rc + 15) / 16);
        const W * ar[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ar[j] = A + (int64_t) min(rc + 16 * j + m, ad.rank - 1) * a_ld;
        v4f acc[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t k = k_begin + 32 * wave; k < k_end; k += 128) {
            float xv[2][8];
#pragma unroll
            for (int i = 0; i < 2; ++i) load8x<VEC>(xr[i], k + 8 * g, n_in, xv[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j < nj) {
                    float av[8];
                    load8(ar[j] + k + 8 * g, av);
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        acc[0][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[0][q], av[q], acc[0][j], 0, 0, 0);
                        acc[1][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[1][q], av[q], acc[1][j], 0, 0, 0);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) red[wave][16 * i + 4 * g + q][16 * j + m] = acc[i][j][q];
        __syncthreads();
        const int nr = min(LORA_RC, ad.r_ld - rc);
        for (int e = threadIdx.x; e < tile.count * LORA_RC; e += 256) {
            const int t = e / LORA_RC, r = e % LORA_RC;
            if (r < nr)                                     // columns between rank and r_ld are zero, whatever x holds
                u[(int64_t) (tile.start + t) * u_ld + rc + r] = rc + r < ad.rank ? (red[0][t][r] + red[1][t][r]) + (red[2][t][r] + red[3][t][r]) : 0.0f;
        }
        __syncthreads();
    }
}

template <bool VEC>
__global__ __launch_bounds__(256)
void lora_shrink_kernel(const LoraAdapter * __restrict__ ads, const LoraTile * __restrict__ tiles, const int * __restrict__ n_tiles, const int * __restrict__ perm,
                        const float * __restrict__ x, int64_t ldx, int64_t n_in, int64_t a_ld, int64_t T, int64_t k_split, float * __restrict__ u, int u_ld) {
    __shared__ float red[4][LT][LORA_RC + 1];
    if ((int) blockIdx.x >= *n_tiles) return;
    const LoraTile tile = tiles[blockIdx.x];
    if (tile.adapter < 0) return;
    const LoraAdapter ad = ads[tile.adapter];
    const int64_t k0 = (int64_t) blockIdx.y * k_split, k1 = min(a_ld, k0 + k_split);
    float * us = u + (int64_t) blockIdx.y * T * u_ld;
    if (ad.f32) shrink_body<float, VEC>(ad, tile, perm, x, ldx, n_in, a_ld, k0, k1, us, u_ld, red);
    else        shrink_body<__half, VEC>(ad, tile, perm, x, ldx, n_in, a_ld, k0, k1, us, u_ld, red);
}

// ---- y[token][o] = base[token][o] + sum_r (scale sum_split u[split][place][r]) B[o][r] --------------------------------
template <bool VEC>
__device__ __forceinline__ float4 row_load4(const float * p, int64_t o, int64_t n) {
    if constexpr (VEC) return *reinterpret_cast<const float4 *>(p + o);
    float4 v = make_float4(p[o], 0.0f, 0.0f, 0.0f);
    if (o + 1 < n) v.y = p[o + 1];
    if (o + 2 < n) v.z = p[o + 2];
    if (o + 3 < n) v.w = p[o + 3];
    return v;
}
template <bool VEC>
__device__ __forceinline__ void row_store4(float * p, int64_t o, int64_t n, float4 v) {
    if constexpr (VEC) { *reinterpret_cast<float4 *>(p + o) = v; return; }
    p[o] = v.x;
    if (o + 1 < n) p[o + 1] = v.y;
    if (o + 2 < n) p[o + 2] = v.z;
    if (o + 3 < n) p[o + 3] = v.w;
}

template <typename W, bool VEC>
__device__ void expand_body(const LoraAdapter & ad, const LoraTile & tile, const int * perm, const float * us, int64_t o, int64_t n_out,
                            const float * base, int64_t ldb, float * y, int64_t ldy) {
    constexpr int TC = 8;                                   // tokens per pass over the rank
    const W * B = (const W *) ad.b;
    const W * br[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) br[c] = B + min(o + c, n_out - 1) * ad.r_ld;
    for (int t0 = 0; t0 < tile.count; t0 += TC) {
        int64_t tok[TC];
        float4 acc[TC];
#pragma unroll
        for (int t = 0; t < TC; ++t) {
            tok[t] = perm[tile.start + min(t0 + t, tile.count - 1)];
            acc[t] = base ? row_load4<VEC>(base + tok[t] * ldb, o, n_out) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (int r = 0; r < ad.r_ld; r += 8) {
            float b[4][8];
#pragma unroll
            for (int c = 0; c < 4; ++c) load8(br[c] + r, b[c]);
#pragma unroll
            for (int t = 0; t < TC; ++t) {
                float uv[8];
                load8(us + (t0 + t) * ad.r_ld + r, uv);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    acc[t].x = fmaf(uv[q], b[0][q], acc[t].x); acc[t].y = fmaf(uv[q], b[1][q], acc[t].y);
                    acc[t].z = fmaf(uv[q], b[2][q], acc[t].z); acc[t].w = fmaf(uv[q], b[3][q], acc[t].w);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < TC; ++t)
            if (t0 + t < tile.count) row_store4<VEC>(y + tok[t] * ldy, o, n_out, acc[t]);
    }
}

template <bool VEC>
__global__ __launch_bounds__(256)
void lora_expand_kernel(const LoraAdapter * __restrict__ ads, const LoraTile * __restrict__ tiles, const int * __restrict__ n_tiles, const int * __restrict__ perm,
                        const float * __restrict__ u, int u_ld, int splits, int64_t T, int64_t n_out, const float * base, int64_t ldb, float * y, int64_t ldy) {
    extern __shared__ __align__(16) float us[];             // [LT][r_ld]
    if ((int) blockIdx.x >= *n_tiles) return;
    const LoraTile tile = tiles[blockIdx.x];
    const int64_t o = 4 * ((int64_t) blockIdx.y * 256 + threadIdx.x);
    if (tile.adapter < 0) {                                 // no adapter: y is the base
        if (base == y || o >= n_out) return;
        for (int t = 0; t < tile.count; ++t) {
            const int64_t tok = perm[tile.start + t];
            row_store4<VEC>(y + tok * ldy, o, n_out, base ? row_load4<VEC>(base + tok * ldb, o, n_out) : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        }
        return;
    }
    const LoraAdapter ad = ads[tile.adapter];
    for (int e = threadIdx.x; e < LT * ad.r_ld; e += 256) {
        const int t = e / ad.r_ld, r = e - t * ad.r_ld;
        float v = 0.0f;
        if (t < tile.count)
            for (int s = 0; s < splits; ++s) v += u[((int64_t) s * T + tile.start + t) * u_ld + r];
        us[e] = ad.scale * v;
    }
    __syncthreads();
    if (o >= n_out) return;
    if (ad.f32) expand_body<float, VEC>(ad, tile, perm, us, o, n_out, base, ldb, y, ldy);
    else        expand_body<__half, VEC>(ad, tile, perm, us, o, n_out, base, ldb, y, ldy);
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

// rows of t (F16 / F32, any strides) to dst with `ld` elements a row, as they are or widened
static void lora_pack(const sdh_tensor & t, bool f32, uint8_t * dst, int64_t ld) {
    if (f32) {
        const std::vector<float> v = tensor_f32(t);
        for (int64_t i1 = 0; i1 < t.ne[1]; ++i1) memcpy(dst + i1 * ld * 4, v.data() + i1 * t.ne[0], (size_t) t.ne[0] * 4);
        return;
    }
    for (int64_t i1 = 0; i1 < t.ne[1]; ++i1) {
        const uint8_t * row = (const uint8_t *) t.data + i1 * t.nb[1];
        if (t.nb[0] == 2) memcpy(dst + i1 * ld * 2, row, (size_t) t.ne[0] * 2);
        else for (int64_t i0 = 0; i0 < t.ne[0]; ++i0) memcpy(dst + (i1 * ld + i0) * 2, row + i0 * t.nb[0], 2);
    }
}

static int lora_create(int64_t n_in, int64_t n_out, const sdh_lora_desc * d, int n, LoraSet ** out) {
    if (n_in < 1 || n_out < 1 || n_in > INT32_MAX / 2 || n_out > INT32_MAX / 2) { set_error("sdh_lora_create: bad dims n_in=%lld n_out=%lld", (long long) n_in, (long long) n_out); return SDH_ERR_INVALID; }
    if (n < 1 || n > SDH_LORA_MAX_ADAPTERS) { set_error("sdh_lora_create: %d adapters (1 .. %d)", n, SDH_LORA_MAX_ADAPTERS); return SDH_ERR_INVALID; }
    LoraSet l;
    l.n_in = n_in; l.n_out = n_out; l.n = n;
    l.a_ld = (n_in + 31) / 32 * 32;
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
        a.rank = (int) r; a.r_ld = (int) (r + 7) / 8 * 8; a.scale = d[i].scale;
        a.f32 = d[i].a.type == SDH_TYPE_F32 || d[i].b.type == SDH_TYPE_F32;
        l.u_ld = std::max(l.u_ld, a.r_ld);
        l.stored_bytes += r * n_in * (d[i].a.type == SDH_TYPE_F32 ? 4 : 2) + r * n_out * (d[i].b.type == SDH_TYPE_F32 ? 4 : 2);
        const size_t es = a.f32 ? 4 : 2;
        at_a[(size_t) i] = total; total += up((size_t) (r * l.a_ld) * es);
        at_b[(size_t) i] = total; total += up((size_t) n_out * (size_t) a.r_ld * es);
    }
    if (const int rc = ready_on_device("sdh_lora_create")) return rc;
    SDH_HIP_CHECK(hipMalloc((void **) &l.dev, total));
    struct Guard { uint8_t * p; ~Guard() { if (p) (void) hipFree(p); } } guard{l.dev};
    std::vector<uint8_t> buf;
    auto upload = [&](size_t at, size_t bytes) { return hipMemcpy(l.dev + at, buf.data(), bytes, hipMemcpyHostToDevice); };
    for (int i = 0; i < n; ++i) {
        LoraAdapter & a = tab[(size_t) i];
        const size_t es = a.f32 ? 4 : 2;
        a.a = l.dev + at_a[(size_t) i]; a.b = l.dev + at_b[(size_t) i];
        buf.assign((size_t) (a.rank * l.a_ld) * es, 0);
        lora_pack(d[i].a, a.f32 != 0, buf.data(), l.a_ld);
        SDH_HIP_CHECK(upload(at_a[(size_t) i], buf.size()));
        buf.assign((size_t) n_out * (size_t) a.r_ld * es, 0);
        lora_pack(d[i].b, a.f32 != 0, buf.data(), a.r_ld);
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

template <bool VX, bool VY>
static void lora_launch(const LoraSet & l, const LoraWs & w, const int * ids, const float * x, int64_t ldx, int64_t T,
                        const float * base, int64_t ldb, float * y, int64_t ldy, hipStream_t s) {
    const LoraAdapter * ads = (const LoraAdapter *) l.dev;
    const int64_t k_split = ((l.a_ld + w.splits - 1) / w.splits + 127) / 128 * 128;
    const unsigned splits = (unsigned) ((l.a_ld + k_split - 1) / k_split);
    hipLaunchKernelGGL(lora_plan_kernel, dim3(1), dim3(1024), (size_t) (l.n + 1) * 12, s, ids, T, l.n, w.perm, w.tiles, w.n_tiles);
    hipLaunchKernelGGL((lora_shrink_kernel<VX>), dim3((unsigned) w.max_tiles, splits), dim3(256), 0, s, ads, w.tiles, w.n_tiles, w.perm, x, ldx, l.n_in, l.a_ld, T, k_split, w.u, l.u_ld);
    hipLaunchKernelGGL((lora_expand_kernel<VY>), dim3((unsigned) w.max_tiles, (unsigned) ((l.n_out + 1023) / 1024)), dim3(256), (size_t) (LT * l.u_ld) * 4, s,
                       ads, w.tiles, w.n_tiles, w.perm, w.u, l.u_ld, (int) splits, T, l.n_out, base, ldb, y, ldy);
}

static int sdh_lora_apply_impl(const sdh_lora * h, const int32_t * ids, const float * x, int64_t ldx, int64_t T,
                               const float * base, int64_t ldb, float * y, int64_t ldy, void * ws, int64_t ws_bytes, void * stream) {
    static const char * who = "sdh_lora_apply";
    if (T == 0) return ready_on_device(who);
    if (!h || !x || !y || !ws) { set_error("%s: null argument", who); return SDH_ERR_INVALID; }
    const LoraSet & l = *reinterpret_cast<const LoraSet *>(h);
    if (T < 0 || T > INT32_MAX / 2 || ldx < l.n_in || ldy < l.n_out || (base && ldb < l.n_out) || (base == y && ldb != ldy)) {
        set_error("%s: bad shape: T=%lld ldx=%lld (n_in=%lld) ldb=%lld ldy=%lld (n_out=%lld)", who, (long long) T, (long long) ldx, (long long) l.n_in, (long long) ldb, (long long) ldy, (long long) l.n_out);
        return SDH_ERR_INVALID;
    }
    if (!aligned(ids, 4) || !aligned(x, 4) || !aligned(base, 4) || !aligned(y, 4) || !aligned(ws, 16)) { set_error("%s: pointers need 4-byte alignment, the workspace 16", who); return SDH_ERR_INVALID; }
    const int rc = ready_on_device(who);
    if (rc != SDH_OK) return rc;
    const LoraWs w = lora_ws(l, T, (uint8_t *) ws);
    if (ws_bytes < w.bytes) { set_error("%s: the workspace holds %lld bytes, %lld are needed", who, (long long) ws_bytes, (long long) w.bytes); return SDH_ERR_INVALID; }
    const bool vx = aligned(x, 16) && ldx % 4 == 0;
    const bool vy = aligned(y, 16) && ldy % 4 == 0 && l.n_out % 4 == 0 && (!base || (aligned(base, 16) && ldb % 4 == 0));
    hipStream_t s = (hipStream_t) stream;
    if (vx && vy)      lora_launch<true, true>(l, w, ids, x, ldx, T, base, ldb, y, ldy, s);
    else if (vx)       lora_launch<true, false>(l, w, ids, x, ldx, T, base, ldb, y, ldy, s);
    else if (vy)       lora_launch<false, true>(l, w, ids, x, ldx, T, base, ldb, y, ldy, s);
    else               lora_launch<false, false>(l, w, ids, x, ldx, T, base, ldb, y, ldy, s);
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
    return T == 0 ? 0 : lora_ws(*reinterpret_cast<const LoraSet *>(h), T, nullptr).bytes;
}

extern "C" int sdh_lora_apply(const sdh_lora * l, const int32_t * ids, const float * x, int64_t ldx, int64_t n_tokens,
                              const float * base, int64_t ldb, float * y, int64_t ldy, void * ws, int64_t ws_bytes, void * stream) {
    SDH_NO_THROW(sdh_lora_apply_impl(l, ids, x, ldx, n_tokens, base, ldb, y, ldy, ws, ws_bytes, stream));
}
