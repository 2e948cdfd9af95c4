// sdh_norm.hip — residual addition + root-mean-square norm + weight, outputs in F32 and / or 8 bits with scales, and the
// 8-bit conversion alone. Per token
//   s = x + res,  z = s * w / sqrt(mean(s^2) + eps),  per 32 values d = max|z| / 127, q = rint(z / d).
//
// One workgroup per token, the row in registers between the sum of squares and the outputs: every input is read once and the memory
// bounds it. 8192 rows of 4096 with residual and 8-bit output: 76.7 us, 5.7 TB/s (torch's copy of a large tensor: 4.95); the conversion
// alone of 2048 rows of 14336: 33.8 us, 4.5 TB/s, of one row 4.4 us. A lane holds 4 consecutive
// values per step, so eight neighbouring lanes hold a block of 32 and its maximum is three lane exchanges.
//
// Arithmetic: s is rounded to F32 (the next layer reads it); from there on everything is in double and rounded once per output.
// gfx950 issues double multiplies and adds at the F32 rate, the kernel waits for memory, and q then does not depend on how the
// sum of squares was split (in F32 about one value in 40,000 lands on the other side of a rounding border).
#include "sdh_internal.h"

#include <type_traits>

namespace sdh {

struct NormArgs {
    const float * x; int64_t ldx;
    const float * res; int64_t ldr;      // or null
    const float * w;                     // or null
    double eps;
    int n;
    float * sum; int64_t lds;            // or null
    float * y; int64_t ldy;              // or null
    int8_t * q; int64_t ldq;             // or null
    float * d; int64_t ldd;
};

typedef float v4f __attribute__((ext_vector_type(4)));

// NT: past the caches (rows that are more than the L2 holds together): 76.7 us against 87.5 for the prompt above
template <bool VEC, bool NT = false>
__device__ __forceinline__ float4 load4(const float * p, int i, int n) {
    if constexpr (VEC && NT) { const v4f v = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(p + i)); return make_float4(v.x, v.y, v.z, v.w); }
    if constexpr (VEC) return *reinterpret_cast<const float4 *>(p + i);
    float4 v;
    if (i + 4 <= n) { __builtin_memcpy(&v, p + i, 16); return v; }          // 4-byte aligned: still one load
    v.x = p[i];
    v.y = i + 1 < n ? p[i + 1] : 0.0f; v.z = i + 2 < n ? p[i + 2] : 0.0f; v.w = i + 3 < n ? p[i + 3] : 0.0f;
    return v;
}
template <bool VEC, bool NT = false>
__device__ __forceinline__ void store4(float * p, int i, int n, float4 v) {
    if constexpr (VEC && NT) { __builtin_nontemporal_store(v4f{v.x, v.y, v.z, v.w}, reinterpret_cast<v4f *>(p + i)); return; }
    if constexpr (VEC) { *reinterpret_cast<float4 *>(p + i) = v; return; }
    if (i + 4 <= n) { __builtin_memcpy(p + i, &v, 16); return; }
    p[i] = v.x;
    if (i + 1 < n) p[i + 1] = v.y;
    if (i + 2 < n) p[i + 2] = v.z;
}

// magnitude bits of a double: ordered as unsigned integers, every NaN above infinity, so a maximum keeps a NaN
__device__ __forceinline__ unsigned long long mag(double z) { return (unsigned long long) __double_as_longlong(z) & 0x7fffffffffffffffull; }
__device__ __forceinline__ unsigned long long umax64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

__device__ __forceinline__ double block_sum(double v, double * red) {
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
    const int nw = (int) blockDim.x >> 6;
    if (nw == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}

// n / d, given 1 / d within 2^-40: one Newton step on the quotient. The remainder of the first one is exact (or rounds past its 50th bit), so
// what is left is rounded once, to n / d itself where that is a double. 2048 x 14336 in 8 bits 33.7 us; with the compiler's divisions for the scale
// and the reciprocal 36.9.
__device__ __forceinline__ double quotient(double n, double d, double inv) {
    const double p = n * inv;
    return fma(fma(-p, d, n), inv, p);
}

// outputs of four consecutive values i .. i + 3 of one row; live: i < n. All lanes of the wave come here (lane exchanges).
template <bool VEC, bool NORM, bool NT>
__device__ __forceinline__ void emit4(const NormArgs & a, int64_t t, int i, bool live, float4 s, double r) {
    double z[4] = {(double) s.x, (double) s.y, (double) s.z, (double) s.w};
    if constexpr (NORM) {
        float4 w = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (a.w && live) w = load4<VEC>(a.w, i, a.n);
        z[0] = z[0] * r * (double) w.x; z[1] = z[1] * r * (double) w.y; z[2] = z[2] * r * (double) w.z; z[3] = z[3] * r * (double) w.w;
        if (a.y && live) store4<VEC, NT>(a.y + t * a.ldy, i, a.n, make_float4((float) z[0], (float) z[1], (float) z[2], (float) z[3]));
    }
    if (a.q) {                                              // n % 32 == 0: the eight lanes of a block are live together
        unsigned long long m = live ? umax64(umax64(mag(z[0]), mag(z[1])), umax64(mag(z[2]), mag(z[3]))) : 0;
        m = umax64(m, __shfl_xor(m, 1, 64)); m = umax64(m, __shfl_xor(m, 2, 64)); m = umax64(m, __shfl_xor(m, 4, 64));
        const double amax = __longlong_as_double((long long) m);
        const float d = (float) (m < 0x7ff0000000000000ull ? quotient(amax, 127.0, 1.0 / 127.0) : amax);
        const bool fine = d > 0.0f && d < INFINITY;          // zeros, and blocks that are not finite (the scale of F32 decides): quants of 0
        unsigned b = 0;
        if (fine) {
            // z / d = 127 z / amax. z times a rounded 127 / amax would not do: a tie (z F32: 127 z is exact) has to come out as itself,
            // and 73.5 / 49 falls below 1.5 that way.
            double inv = __builtin_amdgcn_rcp(amax);         // 2^-22 and better, after a Newton step 2^-44
            inv = fma(fma(-amax, inv, 1.0), inv, inv);
            for (int k = 0; k < 4; ++k) {
                const double v = quotient(z[k] * 127.0, amax, inv) + 0x1.8p52;       // rounds to an integer, ties to even; it is in the low word
                b |= ((unsigned) __double_as_longlong(v) & 0xffu) << (8 * k);
            }
        }
        if (live) {
            *reinterpret_cast<unsigned *>(a.q + t * a.ldq + i) = b;
            if ((i & 31) == 0) a.d[t * a.ldd + (i >> 5)] = d;
        }
    }
}

// NV: steps of 4 values per thread, n <= 4 * NV * blockDim.x
template <int NV, bool VEC, bool NORM, bool NT>
__global__ __launch_bounds__(1024) void norm_rows_kernel(const NormArgs a) {
    __shared__ double red[16];
    const int64_t t = blockIdx.x;
    const float * x = a.x + t * a.ldx;
    float4 s[NV];
    double ss = 0.0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = 4 * ((int) threadIdx.x + v * (int) blockDim.x);
        s[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < a.n) {
            s[v] = load4<VEC, NT>(x, i, a.n);
            if (NORM && a.res) { const float4 r = load4<VEC, NT>(a.res + t * a.ldr, i, a.n); s[v].x += r.x; s[v].y += r.y; s[v].z += r.z; s[v].w += r.w; }
        }
    }
    double r = 1.0;
    if constexpr (NORM) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = 4 * ((int) threadIdx.x + v * (int) blockDim.x);
            ss += (double) s[v].x * s[v].x + (double) s[v].y * s[v].y + ((double) s[v].z * s[v].z + (double) s[v].w * s[v].w);
            if (a.sum && i < a.n) store4<VEC, NT>(a.sum + t * a.lds, i, a.n, s[v]);
        }
        r = 1.0 / sqrt(block_sum(ss, red) / a.n + a.eps);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = 4 * ((int) threadIdx.x + v * (int) blockDim.x);
        emit4<VEC, NORM, NT>(a, t, i, i < a.n, s[v], r);
    }
}

// rows that do not fit the registers of a workgroup: two passes; the second reads s where the first one stored it
template <bool VEC, bool NORM>
__global__ __launch_bounds__(1024) void norm_long_kernel(const NormArgs a) {
    __shared__ double red[16];
    const int64_t t = blockIdx.x;
    const float * x = a.x + t * a.ldx;
    double ss = 0.0, r = 1.0;
    const int end = (a.n + 4095) / 4096 * 4096;             // every lane takes part in the exchanges of the last step
    if constexpr (NORM) {
        for (int i = 4 * (int) threadIdx.x; i < a.n; i += 4096) {
            float4 s = load4<VEC>(x, i, a.n);
            if (a.res) { const float4 q = load4<VEC>(a.res + t * a.ldr, i, a.n); s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w; }
            ss += (double) s.x * s.x + (double) s.y * s.y + ((double) s.z * s.z + (double) s.w * s.w);
            if (a.sum) store4<VEC>(a.sum + t * a.lds, i, a.n, s);
        }
        r = 1.0 / sqrt(block_sum(ss, red) / a.n + a.eps);
    }
    for (int i = 4 * (int) threadIdx.x; i < end; i += 4096) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < a.n) {
            if (NORM && a.sum) s = load4<VEC>(a.sum + t * a.lds, i, a.n);      // this thread's own stores
            else {
                s = load4<VEC>(x, i, a.n);
                if (NORM && a.res) { const float4 q = load4<VEC>(a.res + t * a.ldr, i, a.n); s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w; }
            }
        }
        emit4<VEC, NORM, false>(a, t, i, i < a.n, s, r);
    }
}

template <int NV, bool VEC, bool NORM>
static void launch_rows(const NormArgs & a, int64_t T, bool nt, hipStream_t s) {
    const dim3 grid((unsigned) T), block((unsigned) (((a.n + 4 * NV - 1) / (4 * NV) + 63) / 64 * 64));
    if (VEC && nt) hipLaunchKernelGGL((norm_rows_kernel<NV, VEC, NORM, VEC>), grid, block, 0, s, a);
    else           hipLaunchKernelGGL((norm_rows_kernel<NV, VEC, NORM, false>), grid, block, 0, s, a);
}

template <bool NORM>
static int launch_norm(const NormArgs & all, int64_t T, hipStream_t s) {
    // 16-byte accesses where every row of every tensor starts on 16 bytes and the row length is a multiple of 4
    auto ok = [](const float * p, int64_t ld) { return !p || (aligned(p, 16) && ld % 4 == 0); };
    const bool vec = all.n % 4 == 0 && ok(all.x, all.ldx) && ok(all.res, all.ldr) && ok(all.sum, all.lds) && ok(all.y, all.ldy) && ok(all.w, 0);
    const int q4 = (all.n + 3) / 4;
    // few rows: as many threads as there are groups of four values (one row of 4096: 4.8 us); many: four groups a thread, four
    // workgroups of 256 for one of 1024 (8192 rows of 4096: 76.7 us against 88.6)
    const int nv = q4 > 4096 ? 0 : q4 > 2048 || (T > 2 * lib().num_cu && q4 >= 1024) ? 4 : q4 > 1024 ? 2 : 1;
    const bool nt = (int64_t) 4 * all.n * T > (32 << 20);
    constexpr int64_t CHUNK = 1 << 21;                      // a launch has fewer than 2^32 threads
    for (int64_t t0 = 0; t0 < T; t0 += CHUNK) {
        NormArgs a = all;
        const int64_t rows = T - t0 < CHUNK ? T - t0 : CHUNK;
        a.x += t0 * a.ldx;
        if (a.res) a.res += t0 * a.ldr;
        if (a.sum) a.sum += t0 * a.lds;
        if (a.y) a.y += t0 * a.ldy;
        if (a.q) { a.q += t0 * a.ldq; a.d += t0 * a.ldd; }
        const auto go = [&](auto v) {
            constexpr bool V = decltype(v)::value;
            if (nv == 1)      launch_rows<1, V, NORM>(a, rows, nt, s);
            else if (nv == 2) launch_rows<2, V, NORM>(a, rows, nt, s);
            else if (nv == 4) launch_rows<4, V, NORM>(a, rows, nt, s);
            else hipLaunchKernelGGL((norm_long_kernel<V, NORM>), dim3((unsigned) rows), dim3(1024), 0, s, a);
        };
        if (vec) go(std::true_type{}); else go(std::false_type{});
    }
    SDH_HIP_CHECK(hipGetLastError());
    return SDH_OK;
}

static int check_q8(const char * who, const sdh_q8 * o, int64_t n) {
    if (!o->q || !o->d) { set_error("%s: null plane of the 8-bit output", who); return SDH_ERR_INVALID; }
    if (n % 32) { set_error("%s: 8-bit outputs need n %% 32 == 0 (n=%lld)", who, (long long) n); return SDH_ERR_INVALID; }
    if (o->ldq < n || o->ldd < n / 32) { set_error("%s: ldq=%lld ldd=%lld are too short for n=%lld", who, (long long) o->ldq, (long long) o->ldd, (long long) n); return SDH_ERR_INVALID; }
    if (!aligned(o->q, 4) || o->ldq % 4 || !aligned(o->d, 4)) { set_error("%s: the 8-bit plane needs 4-byte aligned rows", who); return SDH_ERR_INVALID; }
    return SDH_OK;
}

} // namespace sdh

using namespace sdh;

static int sdh_rms_norm_impl(const float * x, int64_t ldx, const float * res, int64_t ldr, const float * weight, float eps,
                             int64_t n, int64_t T, float * sum, int64_t lds, float * y, int64_t ldy, const sdh_q8 * o8, void * stream) {
    static const char * who = "sdh_rms_norm";
    if (T == 0) return ready_on_device(who);
    int rc;
    if (!x || (!sum && !y && !o8)) { set_error("%s: null argument (x, or every output)", who); return SDH_ERR_INVALID; }
    if (n < 1 || n > INT32_MAX / 2 || T < 0 || T > INT32_MAX || !(eps >= 0.0f)) { set_error("%s: bad shape or eps: n=%lld T=%lld eps=%g", who, (long long) n, (long long) T, (double) eps); return SDH_ERR_INVALID; }
    if (ldx < n || (res && ldr < n) || (sum && lds < n) || (y && ldy < n)) { set_error("%s: a row stride is shorter than n=%lld", who, (long long) n); return SDH_ERR_INVALID; }
    if (!aligned(x, 4) || !aligned(res, 4) || !aligned(weight, 4) || !aligned(sum, 4) || !aligned(y, 4)) { set_error("%s: a pointer is not 4-byte aligned", who); return SDH_ERR_INVALID; }
    if (o8 && (rc = check_q8(who, o8, n)) != SDH_OK) return rc;
    auto in_place = [&](const float * o, int64_t ldo) { return !o || ((o != x || ldo == ldx) && (o != res || ldo == ldr)); };
    if (!in_place(sum, lds) || !in_place(y, ldy) || (y && y == sum)) { set_error("%s: outputs overlap (sum or y may be x or res with the same stride, and not each other)", who); return SDH_ERR_INVALID; }
    if ((rc = ready_on_device(who)) != SDH_OK) return rc;
    NormArgs a{x, ldx, res, ldr, weight, (double) eps, (int) n, sum, lds, y, ldy, nullptr, 0, nullptr, 0};
    if (o8) { a.q = o8->q; a.ldq = o8->ldq; a.d = o8->d; a.ldd = o8->ldd; }
    return launch_norm<true>(a, T, (hipStream_t) stream);
}

static int sdh_q8_quantize_impl(const float * x, int64_t ldx, int64_t n, int64_t T, const sdh_q8 * o8, void * stream) {
    static const char * who = "sdh_q8_quantize";
    if (T == 0) return ready_on_device(who);
    int rc;
    if (!x || !o8) { set_error("%s: null argument", who); return SDH_ERR_INVALID; }
    if (n < 1 || n > INT32_MAX / 2 || T < 0 || T > INT32_MAX || ldx < n || !aligned(x, 4)) { set_error("%s: bad shape: n=%lld T=%lld ldx=%lld", who, (long long) n, (long long) T, (long long) ldx); return SDH_ERR_INVALID; }
    if ((rc = check_q8(who, o8, n)) != SDH_OK) return rc;
    if ((rc = ready_on_device(who)) != SDH_OK) return rc;
    NormArgs a{x, ldx, nullptr, 0, nullptr, 0.0, (int) n, nullptr, 0, nullptr, 0, o8->q, o8->ldq, o8->d, o8->ldd};
    return launch_norm<false>(a, T, (hipStream_t) stream);
}

extern "C" int sdh_rms_norm(const float * x, int64_t ldx, const float * res, int64_t ldr, const float * weight, float eps,
                            int64_t n, int64_t n_tokens, float * sum, int64_t lds, float * y, int64_t ldy, const sdh_q8 * out8, void * stream) {
    SDH_NO_THROW(sdh_rms_norm_impl(x, ldx, res, ldr, weight, eps, n, n_tokens, sum, lds, y, ldy, out8, stream));
}

extern "C" int sdh_q8_quantize(const float * x, int64_t ldx, int64_t n, int64_t n_tokens, const sdh_q8 * out8, void * stream) {
    SDH_NO_THROW(sdh_q8_quantize_impl(x, ldx, n, n_tokens, out8, stream));
}
