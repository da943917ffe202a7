// The output head in front of the losses: layer norm, counter-based dropout, and the projection x W^T + b ended either in
// log-probabilities (what DenseFsaVec takes) or in a softmax cross entropy that never keeps the logits.
//
// N = rows (frames or tokens), D = features, V = outputs.  All sums, softmax statistics and norms are fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/wf_dwfst.h"

int wf_fail(int code, const char* fmt, ...);   // wf_graph.cpp

#define HIP_TRY(expr)                                                                         \
    do {                                                                                      \
        hipError_t e_ = (expr);                                                               \
        if (e_ != hipSuccess) return wf_fail(WF_EHIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glb_void;

constexpr int kBK = 64;       // K extent of a staged tile
constexpr int kRowPad = 256;  // rows of padded operands: a multiple of every tile

__device__ inline float to_f(float v) { return v; }
__device__ inline float to_f(bf16 v) { return (float)v; }
__device__ inline float to_f(f16 v) { return (float)v; }

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ inline float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// W elements that may sit at any address a T may sit at (rows of odd length): global memory takes wide accesses at the
// element's own alignment.
template <class T, int W> struct Pack { T v[W]; };
template <class T, int W> __device__ inline Pack<T, W> load_n(const T* p, int n) {   // n valid elements, zeros behind them
    Pack<T, W> r;
    if (n >= W) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
    }
    return r;
}
template <class T, int W> __device__ inline void store_n(T* p, const Pack<T, W>& r, int n) {
    if (n >= W) {
        __builtin_memcpy(p, &r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < n) p[i] = r.v[i];
    }
}

__device__ inline float load_any(const void* p, int type, int64_t i) {
    return type == WF_F32 ? ((const float*)p)[i] : type == WF_BF16 ? (float)((const bf16*)p)[i] : (float)((const f16*)p)[i];
}
template <int W> __device__ inline void load_params(const void* p, int type, int64_t i, int n, float none, float (&out)[W]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < W; ++j) out[j] = none;
    } else if (type == WF_F32) {
        const auto q = load_n<float, W>((const float*)p + i, n);
#pragma unroll
        for (int j = 0; j < W; ++j) out[j] = q.v[j];
    } else if (type == WF_BF16) {
        const auto q = load_n<bf16, W>((const bf16*)p + i, n);
#pragma unroll
        for (int j = 0; j < W; ++j) out[j] = (float)q.v[j];
    } else {
        const auto q = load_n<f16, W>((const f16*)p + i, n);
#pragma unroll
        for (int j = 0; j < W; ++j) out[j] = (float)q.v[j];
    }
}
__device__ inline void store_any(void* p, int type, int64_t i, float v) {
    if (type == WF_F32) ((float*)p)[i] = v;
    else if (type == WF_BF16) ((bf16*)p)[i] = (bf16)v;
    else ((f16*)p)[i] = (f16)v;
}

// =====================================================================================================================
// layer norm
//
// y = (x - mean) rstd w + b over a row of D.  One pass over HBM: the row stays in registers between the mean, the variance
// about that mean (two sums, no E[x^2] - mean^2 cancellation) and the result.  WAVES waves share a row (1, 4 or 16 by D);
// a workgroup of max(4, WAVES) waves.  Backward in one pass as well: with xh = (x - mean) rstd and g = dy w,
//   dx = rstd (g - mean(g) - xh mean(g xh)),   dw = sum_n dy xh,   db = sum_n dy;
// every thread keeps the dw / db sums of its own columns in registers over the rows its workgroup walks, one partial row
// per workgroup goes to the workspace and a second kernel adds the partial rows in a fixed order (no atomics).

constexpr int kLnVecs = 4;                 // 16-byte pieces of a row that a lane holds at most
template <class T> constexpr int vec_of() { return 16 / (int)sizeof(T); }

template <int WAVES> __device__ inline float row_sum(float v, float* red, int slot) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
        const int w = threadIdx.x >> 6;
        __syncthreads();                   // the slots' last readers are done
        if ((threadIdx.x & 63) == 0) red[slot * WAVES + w] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) v += red[slot * WAVES + i];
    }
    return v;
}

struct LnArgs {
    const void *x, *dy, *w, *b;
    int64_t ldx, lddy;
    void* y;                 // y or dx, rows of D
    float* stats;            // [N][2] mean, rstd
    float* part;             // [gridDim][2][D] (backward)
    int64_t N;
    int D, ptype;
    float eps;
};

template <class T, int WAVES, int C> __global__ void __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64)
layer_norm_kernel(LnArgs a) {
    constexpr int VEC = vec_of<T>(), TPR = WAVES * 64, RPB = WAVES == 1 ? 4 : 1;
    __shared__ float red[WAVES > 1 ? 2 * WAVES : 1];
    const int tr = WAVES == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    float w[C][VEC], b[C][VEC];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = (c * TPR + tr) * VEC;
        load_params<VEC>(a.w, a.ptype, d, a.D - d, 1.f, w[c]);
        load_params<VEC>(a.b, a.ptype, d, a.D - d, 0.f, b[c]);
    }
    const float count = (float)a.D;      // divided by, not multiplied with its inverse: a row of equal values whose sum is exact gives y = b
    // (with WAVES > 1 the trip count is the same for the whole workgroup: barriers inside)
    for (int64_t r = (int64_t)blockIdx.x * RPB + (WAVES == 1 ? (threadIdx.x >> 6) : 0); r < a.N; r += (int64_t)gridDim.x * RPB) {
        const T* x = (const T*)a.x + r * a.ldx;
        float v[C][VEC];
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = (c * TPR + tr) * VEC;
            const auto p = load_n<T, VEC>(x + d, a.D - d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) { v[c][i] = to_f(p.v[i]); s += v[c][i]; }
        }
        const float mean = row_sum<WAVES>(s, red, 0) / count;
        s = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = (c * TPR + tr) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) { v[c][i] -= mean; s += d + i < a.D ? v[c][i] * v[c][i] : 0.f; }
        }
        const float rstd = 1.f / sqrtf(row_sum<WAVES>(s, red, 1) / count + a.eps);
        T* y = (T*)a.y + r * (int64_t)a.D;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = (c * TPR + tr) * VEC;
            if (d >= a.D) break;
            Pack<T, VEC> p;
#pragma unroll
            for (int i = 0; i < VEC; ++i) p.v[i] = (T)(v[c][i] * rstd * w[c][i] + b[c][i]);
            store_n<T, VEC>(y + d, p, a.D - d);
        }
        if (a.stats && tr == 0) { a.stats[2 * r] = mean; a.stats[2 * r + 1] = rstd; }
    }
}

template <class T, int WAVES, int C> __global__ void __launch_bounds__(1024)
layer_norm_backward_kernel(LnArgs a) {
    constexpr int VEC = vec_of<T>(), TPR = WAVES * 64, RPB = 16 / WAVES;   // rows a workgroup of 16 waves has in hand
    __shared__ float red[WAVES > 1 ? 2 * 16 : 1];
    __shared__ float fold[WAVES == 16 ? 1 : 16 * 64 * VEC];
    const int tr = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    float dw[C][VEC] = {}, db[C][VEC] = {}, w[C][VEC];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int d = (c * TPR + tr) * VEC;
        load_params<VEC>(a.w, a.ptype, d, a.D - d, 1.f, w[c]);
    }
    const float inv = 1.f / (float)a.D;
    // rounds of gridDim * RPB rows; the trip count is the same for all waves of a workgroup (barriers inside)
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.N; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + slot;
        const bool live = r < a.N;
        const T* x = (const T*)a.x + (live ? r : 0) * a.ldx;
        const T* dy = (const T*)a.dy + (live ? r : 0) * a.lddy;
        const float mean = live ? a.stats[2 * r] : 0.f, rstd = live ? a.stats[2 * r + 1] : 0.f;
        float xh[C][VEC], g[C][VEC];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int d = (c * TPR + tr) * VEC;
            const int n = live ? a.D - d : 0;
            const auto p = load_n<T, VEC>(x + d, n);
            const auto q = load_n<T, VEC>(dy + d, n);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xi = i < n ? (to_f(p.v[i]) - mean) * rstd : 0.f, gi = to_f(q.v[i]);
                dw[c][i] += gi * xi;
                db[c][i] += gi;
                xh[c][i] = xi;
                g[c][i] = gi * w[c][i];
                s1 += g[c][i];
                s2 += g[c][i] * xi;
            }
        }
        if constexpr (WAVES == 1) {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
        } else {                           // the waves of one row meet in LDS
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            const int wv = threadIdx.x >> 6;
            __syncthreads();
            if ((threadIdx.x & 63) == 0) { red[wv] = s1; red[16 + wv] = s2; }
            __syncthreads();
            s1 = s2 = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) { s1 += red[slot * WAVES + i]; s2 += red[16 + slot * WAVES + i]; }
        }
        s1 *= inv;
        s2 *= inv;
        if (live) {
            T* dx = (T*)a.y + r * (int64_t)a.D;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int d = (c * TPR + tr) * VEC;
                if (d >= a.D) break;
                Pack<T, VEC> p;
#pragma unroll
                for (int i = 0; i < VEC; ++i) p.v[i] = (T)(rstd * (g[c][i] - s1 - xh[c][i] * s2));
                store_n<T, VEC>(dx + d, p, a.D - d);
            }
        }
    }
    if (!a.part) return;
    // the workgroup's partial rows: [2][D]
    float* part = a.part + (size_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float(&v)[C][VEC] = k ? db : dw;
            if constexpr (WAVES == 16) {
                const int d = (c * TPR + tr) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (d + i < a.D) part[(size_t)k * a.D + d + i] = v[c][i];
            } else {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < VEC; ++i) fold[(slot * TPR + tr) * VEC + i] = v[c][i];
                __syncthreads();
                for (int j = threadIdx.x; j < TPR * VEC; j += 1024) {
                    float s = 0.f;
#pragma unroll
                    for (int q = 0; q < RPB; ++q) s += fold[q * TPR * VEC + j];
                    const int d = c * TPR * VEC + j;
                    if (d < a.D) part[(size_t)k * a.D + d] = s;
                }
            }
        }
}

// dw / db = the sum of G partial rows [G][2][D], column by column in a fixed order: a workgroup owns 16 columns, 64 threads
// walk the partial rows of each.
__global__ void __launch_bounds__(1024) layer_norm_fold_kernel(const float* part, int G, int D, void* dw, void* db, int ptype) {
    __shared__ float s[64][17];
    const int c = threadIdx.x & 15, q = threadIdx.x >> 4, d = blockIdx.x * 16 + c, k = blockIdx.y;
    float v = 0.f;
    if (d < D)
        for (int g = q; g < G; g += 64) v += part[((size_t)g * 2 + k) * D + d];
    s[q][c] = v;
    __syncthreads();
    for (int o = 32; o; o >>= 1) {
        if (q < o) s[q][c] += s[q + o][c];
        __syncthreads();
    }
    if (q == 0 && d < D) {
        void* out = k ? db : dw;
        if (out) store_any(out, ptype, d, s[0][c]);
    }
}

// =====================================================================================================================
// dropout
//
// Element i (row-major) is kept iff word i % 4 of Philox4x32-7 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy
// as 1, 2, 3; 2011 -- seven rounds are the fewest the authors found to pass every test of BigCrush) under the key `seed` and
// the counter i / 4 is at least p 2^32; kept elements are multiplied by 1 / (1 - p), the others are exactly 0 whatever they
// hold.  The mask is a function of (seed, i): backward computes it again, nothing is stored.
struct Philox { uint32_t w[4]; };
__device__ inline Philox philox7(uint64_t counter, uint64_t key) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

template <class T> __global__ void __launch_bounds__(256)
dropout_kernel(const T* x, T* y, int64_t n, uint32_t below, float scale, uint64_t seed, const uint64_t* seed_dev) {
    constexpr int VEC = vec_of<T>();
    if (seed_dev) seed = *seed_dev;
    const int64_t step = (int64_t)gridDim.x * 256 * VEC;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC; i < n; i += step) {
        const int m = (int)min((int64_t)VEC, n - i);
        auto p = load_n<T, VEC>(x + i, m);
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const Philox u = philox7((uint64_t)(i + j) >> 2, seed);
#pragma unroll
            for (int q = 0; q < 4; ++q) p.v[j + q] = u.w[q] >= below ? (T)(to_f(p.v[j + q]) * scale) : (T)0.f;
        }
        store_n<T, VEC>(y + i, p, m);
    }
}

__global__ void __launch_bounds__(256) zero_kernel(uint16_t* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

// ---- host side --------------------------------------------------------------------------------------------------------
constexpr int kCUs = 256;
constexpr int kLnMaxD = 32768;      // 16 waves x 64 lanes x 32 elements of a lane
constexpr int kLnParts = kCUs;      // workgroups (= partial rows) of the backward pass: one per CU

bool known_type(int t) { return t == WF_F32 || t == WF_BF16 || t == WF_F16; }

// waves of a row and 16-byte pieces of a lane: the fewest waves that hold the row in kLnVecs pieces each
template <class T, class F> void with_ln_shape(int D, F&& f) {
    constexpr int VEC = vec_of<T>();
    auto in = [&](int waves, int c) { return D <= waves * 64 * VEC * c; };
    using std::integral_constant;
    if (in(1, 1)) f(integral_constant<int, 1>(), integral_constant<int, 1>());
    else if (in(1, 2)) f(integral_constant<int, 1>(), integral_constant<int, 2>());
    else if (in(1, 4)) f(integral_constant<int, 1>(), integral_constant<int, 4>());
    else if (in(4, 2)) f(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if (in(4, 4)) f(integral_constant<int, 4>(), integral_constant<int, 4>());
    else if (in(16, 4)) f(integral_constant<int, 16>(), integral_constant<int, 4>());
    else f(integral_constant<int, 16>(), integral_constant<int, 8>());      // fp32 rows above 16384
}
template <class F> void with_type(int type, F&& f) {
    if (type == WF_F32) f(float());
    else if (type == WF_BF16) f(bf16());
    else f(f16());
}

int ln_check(const char* who, const void* x, int64_t ldx, int64_t N, int32_t D, int32_t type, int32_t ptype) {
    if (!known_type(type) || !known_type(ptype)) return wf_fail(WF_EINVAL, "%s: unknown element type", who);
    if (N < 0 || D < 1 || ldx < 0) return wf_fail(WF_EINVAL, "%s: bad size (N %lld, D %d)", who, (long long)N, D);
    if (D > kLnMaxD) return wf_fail(WF_EUNSUPPORTED, "%s: rows of %d elements (at most %d)", who, D, kLnMaxD);
    if (N > 0 && !x) return wf_fail(WF_EINVAL, "%s: null pointer", who);
    return WF_OK;
}
}  // namespace

extern "C" int wf_layer_norm(const void* x, int64_t ldx, int64_t N, int32_t D, int32_t type, const void* weight, const void* bias,
                             int32_t param_type, float eps, void* y, float* stats, void* stream) {
    int rc = ln_check("wf_layer_norm", x, ldx, N, D, type, param_type);
    if (rc) return rc;
    if (N == 0) return WF_OK;
    if (!y) return wf_fail(WF_EINVAL, "wf_layer_norm: null pointer");
    LnArgs a = {x, nullptr, weight, bias, ldx, 0, y, stats, nullptr, N, D, param_type, eps};
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_ln_shape<T>(D, [&](auto waves, auto c) {
            constexpr int W = decltype(waves)::value, C = decltype(c)::value, RPB = W == 1 ? 4 : 1;
            const int64_t blocks = std::min<int64_t>((N + RPB - 1) / RPB, (int64_t)kCUs * (W == 1 ? 8 : W == 4 ? 8 : 2));
            layer_norm_kernel<T, W, C><<<(unsigned)blocks, W == 1 ? 256 : W * 64, 0, (hipStream_t)stream>>>(a);
        });
    });
    HIP_TRY(hipGetLastError());
    return WF_OK;
}

extern "C" int wf_layer_norm_backward_workspace_bytes(int64_t N, int32_t D, int32_t type, size_t* bytes) {
    if (!bytes) return wf_fail(WF_EINVAL, "null bytes");
    int rc = ln_check("wf_layer_norm_backward_workspace_bytes", bytes, 0, N, D, type, type);
    if (rc) return rc;
    *bytes = sizeof(float) * 2 * (size_t)D * kLnParts;
    return WF_OK;
}

extern "C" int wf_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t N, int32_t D, int32_t type,
                                      const void* weight, int32_t param_type, const float* stats, void* dx, void* dweight,
                                      void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = ln_check("wf_layer_norm_backward", x, ldx, N, D, type, param_type);
    if (rc) return rc;
    if (N > 0 && (!dy || !stats || !dx || lddy < 0)) return wf_fail(WF_EINVAL, "wf_layer_norm_backward: null pointer");
    const bool sums = dweight || dbias;
    if (sums && (!workspace || workspace_bytes < sizeof(float) * 2 * (size_t)D * kLnParts))
        return wf_fail(WF_ENOSPC, "wf_layer_norm_backward: workspace too small");
    LnArgs a = {x, dy, weight, nullptr, ldx, lddy, dx, (float*)stats, sums ? (float*)workspace : nullptr, N, D, param_type, 0.f};
    hipStream_t st = (hipStream_t)stream;
    unsigned blocks = 0;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_ln_shape<T>(D, [&](auto waves, auto c) {
            constexpr int W = decltype(waves)::value, C = decltype(c)::value, RPB = 16 / W;
            blocks = (unsigned)std::min<int64_t>((N + RPB - 1) / RPB, kLnParts);
            if (blocks) layer_norm_backward_kernel<T, W, C><<<blocks, 1024, 0, st>>>(a);
        });
    });
    if (sums)   // (no rows: the sums of nothing are zeros)
        layer_norm_fold_kernel<<<dim3((unsigned)(D + 15) / 16, 2), 1024, 0, st>>>((const float*)workspace, (int)blocks, D, dweight, dbias, param_type);
    HIP_TRY(hipGetLastError());
    return WF_OK;
}

extern "C" int wf_dropout(const void* x, int64_t n, int32_t type, double p, uint64_t seed, const uint64_t* seed_dev, void* y,
                          void* stream) {
    if (!known_type(type)) return wf_fail(WF_EINVAL, "wf_dropout: unknown element type");
    if (n < 0 || !(p >= 0.0 && p <= 1.0)) return wf_fail(WF_EINVAL, "wf_dropout: bad size or probability %g", p);
    if (n == 0) return WF_OK;
    if (!x || !y) return wf_fail(WF_EINVAL, "wf_dropout: null pointer");
    hipStream_t st = (hipStream_t)stream;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const int64_t per = 256 * (int64_t)vec_of<T>();
        const unsigned blocks = (unsigned)std::min<int64_t>((n + per - 1) / per, kCUs * 16);
        if (p == 1.0)      // nothing is kept, whatever the words say
            zero_kernel<<<blocks, 256, 0, st>>>((uint16_t*)y, n * (int64_t)(sizeof(T) / 2));
        else
            dropout_kernel<T><<<blocks, 256, 0, st>>>((const T*)x, (T*)y, n, (uint32_t)(p * 4294967296.0), (float)(1.0 / (1.0 - p)), seed, seed_dev);
    });
    HIP_TRY(hipGetLastError());
    return WF_OK;
}
