// Group normalisation with an activation over channels-last images, forward
// and backward (an extension: the reference has no normalisation layer).
//
//   x [n][rows][C], G groups of cpg = C / G channels, M = rows * cpg
//   mean, var over (rows, cpg);  rstd = 1 / sqrt(var + eps)
//   h = (x - mean) rstd;  z = h weight_c + bias_c;  y = act(z)
//   dz = dy act'(z);  A_c = sum_rows dz,  B_c = sum_rows dz h
//   dbias_c = sum_n A_c,  dweight_c = sum_n B_c
//   dx = rstd (weight_c dz - mean_g(weight A) - h mean_g(weight B))
//
// All of it is bound by memory: 2 values moved per value forward, 3 backward,
// if what the statistics pass reads is still on chip when the second pass
// wants it. Statistics are 32-bit per thread about the thread's own first
// value (no cancellation where |mean| >> deviation) and merged in 64 bits by
// the pairwise update of Chan, Golub and LeVeque; sums are taken in a fixed
// order, so reruns give the same bits.
//
// Mapping. A thread owns VEC consecutive values and steps by a multiple of a
// whole row, so it meets the same channels in every step and keeps its sums
// and its scales in registers. "Flat": the threads of a block cover whole
// rows back to back, vectors may straddle rows (needs C / gcd(C, VEC) <=
// threads). "Slab": wider rows are cut into slabs of whole groups, or of
// pieces of one group.
#include <algorithm>
#include <cstdint>
#include <numeric>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"

namespace dressi {

namespace {

constexpr int kGnThreads = 512;

struct GnDims {
    uint64_t n, rows;
    int C, G, cpg;
    float eps;
    // mapping
    int slabs;         // column slabs of a row (1: flat)
    int slab_cols;     // columns of a full slab
    int pieces;        // slabs per group (1 unless a group exceeds a slab)
    uint32_t chunks;   // row chunks of a sample
    uint64_t chunk_rows;
    int threads;       // threads that work (flat: a multiple of a row cover)
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) {
    return __float2bfloat16_rn(v);
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

// Columns [col0, col0 + cols) of slab s.
__device__ __forceinline__ void slab_of(const GnDims& d, int s, int* col0,
                                        int* cols) {
    if (d.pieces > 1) {
        const int g = s / d.pieces, k = s % d.pieces;
        *col0 = g * d.cpg + k * d.slab_cols;
        *cols = min(d.slab_cols, d.cpg - k * d.slab_cols);
    } else {
        *col0 = s * d.slab_cols;
        *cols = min(d.slab_cols, d.C - *col0);
    }
}

// What a thread walks over: values base, base + step, ... below end of a
// sample, each VEC wide; its first value is column `col` of the slab.
struct Walk {
    uint64_t base, step, end;
    int col0, cols, lanes, col;
    bool works;
};

template <int VEC>
__device__ __forceinline__ Walk walk_of(const GnDims& d, int slab,
                                        uint32_t chunk) {
    Walk w;
    const uint64_t r0 = uint64_t(chunk) * d.chunk_rows;
    const uint64_t r1 = min(r0 + d.chunk_rows, d.rows);
    w.end = r1 * d.C;
    if (d.slabs == 1) {
        w.col0 = 0;
        w.cols = d.C;
        w.lanes = int(int64_t(d.threads) * VEC / d.C);
        w.works = int(threadIdx.x) < d.threads;
        w.base = r0 * d.C + uint64_t(threadIdx.x) * VEC;
        w.step = uint64_t(d.threads) * VEC;
        w.col = int(uint32_t(threadIdx.x) * VEC % uint32_t(d.C));
    } else {
        slab_of(d, slab, &w.col0, &w.cols);
        const int per_row = w.cols / VEC;
        w.lanes = max(1, kGnThreads / per_row);
        const int lane = threadIdx.x / per_row;
        w.works = lane < w.lanes;
        w.col = (threadIdx.x % per_row) * VEC;
        w.base = (r0 + lane) * d.C + w.col0 + w.col;
        w.step = uint64_t(w.lanes) * d.C;
    }
    return w;
}

// Number of steps of the walk that starts at base.
__device__ __forceinline__ uint32_t steps_of(const Walk& w, uint64_t base) {
    return base < w.end ? uint32_t((w.end - base + w.step - 1) / w.step) : 0u;
}

// Rounding below 0 is 0; NaN stays.
__device__ __forceinline__ float nonneg(float v) { return v < 0.f ? 0.f : v; }

struct Moments {
    double n, mean, m2;
};
__device__ __forceinline__ void merge(Moments* a, double n, double mean,
                                      double m2) {
    if (n == 0.0) return;
    const double t = a->n + n, d = mean - a->mean;
    a->mean += d * (n / t);
    a->m2 += m2 + d * d * (a->n * (n / t));
    a->n = t;
}
__device__ __forceinline__ void merge_warp(Moments* a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double n = __shfl_xor_sync(0xffffffffu, a->n, o);
        const double mean = __shfl_xor_sync(0xffffffffu, a->mean, o);
        const double m2 = __shfl_xor_sync(0xffffffffu, a->m2, o);
        // both sides in one order: the same bits in every lane
        const bool up = threadIdx.x & o;
        Moments lo = up ? Moments{n, mean, m2} : *a;
        const Moments hi = up ? *a : Moments{n, mean, m2};
        merge(&lo, hi.n, hi.mean, hi.m2);
        *a = lo;
    }
}

// act 0: none, 1: relu, 2: silu. NaN stays NaN.
__device__ __forceinline__ float sigmoid_(float z) {
    return __fdividef(1.f, 1.f + __expf(-z));
}
template <int ACT>
__device__ __forceinline__ float act_(float z) {
    if (ACT == 1) return z < 0.f ? 0.f : z;
    if (ACT == 2) return z * sigmoid_(z);
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float dy, float z) {
    if (ACT == 1) return z <= 0.f ? 0.f : dy;
    if (ACT == 2) {
        const float s = sigmoid_(z);
        return dy * (s * (1.f + z * (1.f - s)));
    }
    return dy;
}

// ------------------------------------------------------------------ forward

// Statistics of one (sample, chunk, slab): part[n][g][chunk * pieces + piece]
// = (mean less the group's first value in the sample, sum of squares about
// the mean). Means of 1e4 deviations would lose digits of the variance in 32
// bits; their distances from a common value do not.
template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_stats(GnDims d, const T* x, float2* part) {
    __shared__ float2 sm[kGnThreads * VEC];
    __shared__ uint32_t cnt[kGnThreads];
    uint64_t i = blockIdx.x;
    const int slab = int(i % d.slabs);
    i /= d.slabs;
    const uint32_t chunk = uint32_t(i % d.chunks);
    const uint64_t n = i / d.chunks;
    const Walk w = walk_of<VEC>(d, slab, chunk);
    const T* xs = x + n * d.rows * d.C;
    float k[VEC], s1[VEC], s2[VEC], k0[VEC];
    const uint32_t steps = w.works ? steps_of(w, w.base) : 0u;
    if (steps > 0) {
        const Pack<T, VEC> f = load_pack<T, VEC>(xs + w.base);
        int c = w.col;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            k[j] = to_f<T>(f.v[j]);
            s1[j] = s2[j] = 0.f;
            k0[j] = to_f<T>(xs[(w.col0 + c) / d.cpg * d.cpg]);
            if (++c == w.cols) c = 0;
        }
        const T* p = xs + w.base;
#pragma unroll 4
        for (uint32_t t = 1; t < steps; t++) {
            p += w.step;
            const Pack<T, VEC> v = load_pack<T, VEC>(p);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float e = to_f<T>(v.v[j]) - k[j];
                s1[j] += e;
                s2[j] += e * e;
            }
        }
        const float inv = 1.f / float(steps);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float m = s1[j] * inv;
            sm[threadIdx.x * VEC + j] =
                    make_float2(k[j] - k0[j] + m, nonneg(s2[j] - s1[j] * m));
        }
    }
    cnt[threadIdx.x] = steps;
    __syncthreads();
    // sm[lane * cols + c]: one warp per group merges its lanes x channels
    const int per = d.pieces > 1 ? w.cols : d.cpg;
    const int groups = w.cols / per, g0 = w.col0 / d.cpg;
    for (int g = threadIdx.x / 32; g < groups; g += kGnThreads / 32) {
        Moments a{0.0, 0.0, 0.0};
        for (int e = threadIdx.x & 31; e < w.lanes * per; e += 32) {
            const int at = e / per * w.cols + g * per + e % per;
            const float2 v = sm[at];
            merge(&a, double(cnt[at / VEC]), v.x, v.y);
        }
        merge_warp(&a);
        if ((threadIdx.x & 31) == 0)
            part[(n * d.G + g0 + g) * d.chunks * d.pieces +
                 size_t(chunk) * d.pieces + slab % d.pieces] =
                    make_float2(float(a.mean), float(a.m2));
    }
}

// mean[n][g], rstd[n][g] from the parts; one warp each.
template <typename T>
__global__ void k_gn_finish(GnDims d, uint64_t n, const T* x,
                            const float2* part, float* mean, float* rstd) {
    const uint64_t i = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
    if (i >= n * d.G) return;
    Moments a{0.0, 0.0, 0.0};
    const uint32_t np = d.chunks * d.pieces;
    for (uint32_t e = threadIdx.x & 31; e < np; e += 32) {
        const uint32_t chunk = e / d.pieces, piece = e % d.pieces;
        const uint64_t r0 = chunk * d.chunk_rows;
        const uint64_t rows = min(d.chunk_rows, d.rows - r0);
        const int cols = d.pieces > 1
                                 ? min(d.slab_cols,
                                       d.cpg - int(piece) * d.slab_cols)
                                 : d.cpg;
        const float2 v = part[i * np + e];
        merge(&a, double(rows) * cols, v.x, v.y);
    }
    merge_warp(&a);
    if ((threadIdx.x & 31) == 0) {
        const T first = x[i / d.G * d.rows * d.C + i % d.G * d.cpg];
        mean[i] = float(a.mean + to_f<T>(first));
        rstd[i] = float(1.0 / sqrt(a.m2 / a.n + double(d.eps)));
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_apply(GnDims d, const T* x, const float* weight,
                   const float* bias, const float* mean, const float* rstd,
                   T* y) {
    // the last chunks first: they are what the statistics pass left on chip
    uint64_t i = gridDim.x - 1 - blockIdx.x;
    const int slab = int(i % d.slabs);
    i /= d.slabs;
    const uint32_t chunk = uint32_t(i % d.chunks);
    const uint64_t n = i / d.chunks;
    const Walk w = walk_of<VEC>(d, slab, chunk);
    if (!w.works) return;
    const T* xs = x + n * d.rows * d.C;
    T* ys = y + n * d.rows * d.C;
    float mu[VEC], a[VEC], b[VEC];
    int c = w.col;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int ch = w.col0 + c, g = ch / d.cpg;
        mu[j] = mean[n * d.G + g];
        a[j] = rstd[n * d.G + g] * (weight ? weight[ch] : 1.f);
        b[j] = bias ? bias[ch] : 0.f;
        if (++c == w.cols) c = 0;
    }
    const uint32_t steps = steps_of(w, w.base);
    uint64_t at = w.base;
#pragma unroll 4
    for (uint32_t t = 0; t < steps; t++, at += w.step) {
        const Pack<T, VEC> v = load_pack<T, VEC>(xs + at);
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; j++)
            o.v[j] = from_f<T>(
                    act_<ACT>((to_f<T>(v.v[j]) - mu[j]) * a[j] + b[j]));
        *reinterpret_cast<Pack<T, VEC>*>(ys + at) = o;
    }
}

// ----------------------------------------------------------------- backward

// part[n][chunk][c] = (sum dz, sum dz h) over the chunk's rows.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_grad_sums(GnDims d, const T* dy, const T* x, const float* weight,
                       const float* bias, const float* mean,
                       const float* rstd, float2* part) {
    __shared__ float2 sm[kGnThreads * VEC];
    uint64_t i = blockIdx.x;
    const int slab = int(i % d.slabs);
    i /= d.slabs;
    const uint32_t chunk = uint32_t(i % d.chunks);
    const uint64_t n = i / d.chunks;
    const Walk w = walk_of<VEC>(d, slab, chunk);
    const T* xs = x + n * d.rows * d.C;
    const T* gs = dy + n * d.rows * d.C;
    if (w.works) {
        float mu[VEC], r[VEC], wt[VEC], b[VEC], A[VEC], B[VEC];
        int c = w.col;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int ch = w.col0 + c, g = ch / d.cpg;
            mu[j] = mean[n * d.G + g];
            r[j] = rstd[n * d.G + g];
            wt[j] = weight ? weight[ch] : 1.f;
            b[j] = bias ? bias[ch] : 0.f;
            A[j] = B[j] = 0.f;
            if (++c == w.cols) c = 0;
        }
        const uint32_t steps = steps_of(w, w.base);
        uint64_t at = w.base;
#pragma unroll 2
        for (uint32_t t = 0; t < steps; t++, at += w.step) {
            const Pack<T, VEC> v = load_pack<T, VEC>(xs + at);
            const Pack<T, VEC> e = load_pack<T, VEC>(gs + at);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float h = (to_f<T>(v.v[j]) - mu[j]) * r[j];
                const float dz =
                        act_grad<ACT>(to_f<T>(e.v[j]), h * wt[j] + b[j]);
                A[j] += dz;
                B[j] += dz * h;
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; j++)
            sm[threadIdx.x * VEC + j] = make_float2(A[j], B[j]);
    }
    __syncthreads();
    float2* out = part + (n * d.chunks + chunk) * d.C + w.col0;
    for (int c = threadIdx.x; c < w.cols; c += kGnThreads) {
        double a = 0.0, b = 0.0;
        for (int l = 0; l < w.lanes; l++) {
            a += sm[l * w.cols + c].x;
            b += sm[l * w.cols + c].y;
        }
        out[c] = make_float2(float(a), float(b));
    }
}

// sums[n][c] = sum of the parts over chunks; means[n][g] = the group's means
// of weight * sums. One block per (sample, bundle of whole groups); 32
// columns x 16 chunk lanes at a time.
__global__ void __launch_bounds__(512)
        k_gn_grad_finish(GnDims d, int bundle, const float2* part,
                         const float* weight, float2* sums, float2* means) {
    __shared__ double sa[16][33], sb[16][33];
    const int bundles = (d.G + bundle - 1) / bundle;
    const uint64_t n = blockIdx.x / bundles;
    const int g0 = int(blockIdx.x % bundles) * bundle;
    const int groups = min(bundle, d.G - g0);
    const int lane = threadIdx.x & 31, row = threadIdx.x / 32;
    const int c0 = g0 * d.cpg, c1 = c0 + groups * d.cpg;
    double ga = 0.0, gb = 0.0;  // of the group that this thread closes
    for (int c = c0; c < c1; c += 32) {
        double a = 0.0, b = 0.0;
        if (c + lane < c1)
            for (uint32_t k = row; k < d.chunks; k += 16) {
                const float2 v = part[(n * d.chunks + k) * d.C + c + lane];
                a += v.x;
                b += v.y;
            }
        sa[row][lane] = a;
        sb[row][lane] = b;
        __syncthreads();
        if (row == 0) {
            for (int k = 1; k < 16; k++) {
                a += sa[k][lane];
                b += sb[k][lane];
            }
            if (c + lane < c1) {
                sums[n * d.C + c + lane] = make_float2(float(a), float(b));
                const double wt = weight ? weight[c + lane] : 1.f;
                sa[0][lane] = a * wt;
                sb[0][lane] = b * wt;
            }
            __syncwarp();
            if (lane < groups) {  // this tile's columns of group lane
                const int lo = max(c, (g0 + lane) * d.cpg);
                const int hi = min(min(c + 32, c1), (g0 + lane + 1) * d.cpg);
                for (int q = lo; q < hi; q++) {
                    ga += sa[0][q - c];
                    gb += sb[0][q - c];
                }
            }
        }
        __syncthreads();
    }
    if (row == 0 && lane < groups) {
        const double m = double(d.rows) * d.cpg;
        means[n * d.G + g0 + lane] =
                make_float2(float(ga / m), float(gb / m));
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_grad_apply(GnDims d, const T* dy, const T* x,
                        const float* weight, const float* bias,
                        const float* mean, const float* rstd,
                        const float2* means, T* dx) {
    uint64_t i = gridDim.x - 1 - blockIdx.x;
    const int slab = int(i % d.slabs);
    i /= d.slabs;
    const uint32_t chunk = uint32_t(i % d.chunks);
    const uint64_t n = i / d.chunks;
    const Walk w = walk_of<VEC>(d, slab, chunk);
    if (!w.works) return;
    const T* xs = x + n * d.rows * d.C;
    const T* gs = dy + n * d.rows * d.C;
    T* os = dx + n * d.rows * d.C;
    float mu[VEC], r[VEC], wt[VEC], b[VEC], ma[VEC], mb[VEC];
    int c = w.col;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int ch = w.col0 + c, g = ch / d.cpg;
        mu[j] = mean[n * d.G + g];
        r[j] = rstd[n * d.G + g];
        wt[j] = weight ? weight[ch] : 1.f;
        b[j] = bias ? bias[ch] : 0.f;
        const float2 m = means[n * d.G + g];
        ma[j] = m.x;
        mb[j] = m.y;
        if (++c == w.cols) c = 0;
    }
    const uint32_t steps = steps_of(w, w.base);
    uint64_t at = w.base;
#pragma unroll 2
    for (uint32_t t = 0; t < steps; t++, at += w.step) {
        const Pack<T, VEC> v = load_pack<T, VEC>(xs + at);
        const Pack<T, VEC> e = load_pack<T, VEC>(gs + at);
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float h = (to_f<T>(v.v[j]) - mu[j]) * r[j];
            const float dz = act_grad<ACT>(to_f<T>(e.v[j]), h * wt[j] + b[j]);
            o.v[j] = from_f<T>(r[j] * (wt[j] * dz - ma[j] - h * mb[j]));
        }
        *reinterpret_cast<Pack<T, VEC>*>(os + at) = o;
    }
}

// dweight[c], dbias[c] = the sums over samples (in order).
__global__ void k_gn_grad_affine(GnDims d, const float2* sums, float* dweight,
                                 float* dbias) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= d.C) return;
    double a = 0.0, b = 0.0;
#pragma unroll 8
    for (uint64_t n = 0; n < d.n; n++) {
        const float2 v = sums[n * d.C + c];
        a += v.x;
        b += v.y;
    }
    if (dbias) dbias[c] = float(a);
    if (dweight) dweight[c] = float(b);
}

// --------------------------------------------------------------------- host

struct GnPlan {
    GnDims d;
    int vec;
    uint64_t batch;  // samples per round of launches
};

// A round of launches covers as many samples as stay in L2 between its two
// passes.
constexpr uint64_t kGnRoundBytes = 64ull << 20;

bool aligned(const void* p, size_t a) {
    return p == nullptr || reinterpret_cast<uintptr_t>(p) % a == 0;
}

GnPlan make_plan(const GroupNormArgs& a, std::initializer_list<const void*> ps,
                 bool grad) {
    const int es = a.dtype == 0 ? 4 : 2;
    GnPlan p{};
    GnDims& d = p.d;
    d.n = a.n;
    d.rows = a.rows;
    d.C = a.C;
    d.G = a.G;
    d.cpg = a.C / a.G;
    d.eps = a.eps;
    d.pieces = 1;
    int vec = 16 / es;
    const uint64_t sample = a.rows * uint64_t(a.C);
    auto fits = [&](int v) {
        for (const void* q : ps)
            if (!aligned(q, size_t(v) * es)) return false;
        return true;
    };
    // flat: vectors need only the sample's size to be a multiple of them
    while (vec > 1 && (sample % vec != 0 || !fits(vec))) vec /= 2;
    int cover = a.C / std::gcd(a.C, vec);  // threads that cover whole rows
    uint64_t row_unit = 1;                 // rows a chunk is a multiple of
    if (cover <= kGnThreads) {
        d.slabs = 1;
        d.slab_cols = a.C;
        const uint64_t want = (sample / vec + cover - 1) / cover;
        d.threads = cover * int(std::min<uint64_t>(kGnThreads / cover,
                                                   std::max<uint64_t>(want, 1)));
        row_unit = vec / std::gcd(a.C, vec);
    } else {
        // slabs start at multiples of the vector in a row of such
        for (;; vec /= 2) {
            if (vec > 1 && a.C % vec != 0) continue;
            const int most = kGnThreads * vec;
            if (d.cpg <= most) {
                const int unit = vec / std::gcd(d.cpg, vec);  // groups
                const int k = most / d.cpg / unit * unit;
                if (k > 0) {
                    d.slab_cols = k * d.cpg;
                    d.slabs = (a.C + d.slab_cols - 1) / d.slab_cols;
                    break;
                }
            } else if (d.cpg % vec == 0) {
                d.slab_cols = most;
                d.pieces = (d.cpg + most - 1) / most;
                d.slabs = d.G * d.pieces;
                break;
            }
            // vec = 1 always ends in one of the two
        }
        d.threads = kGnThreads;
    }
    p.vec = vec;
    const uint64_t bytes = std::max<uint64_t>(1, sample * es * (grad ? 2 : 1));
    p.batch = std::min<uint64_t>(std::max<uint64_t>(1, kGnRoundBytes / bytes),
                                 a.n);
    // two resident blocks an SM, one wave; a thread takes 4 steps or more
    const uint64_t wave = 148 * 2;
    uint64_t chunks = std::max<uint64_t>(
            1, wave / std::max<uint64_t>(1, p.batch * d.slabs));
    const uint64_t lanes = std::max<uint64_t>(
            1, uint64_t(d.threads) * vec /
                       std::max(1, std::min(d.slab_cols, a.C)));
    const uint64_t least = lanes * 4;  // rows
    chunks = std::min(chunks, std::max<uint64_t>(1, a.rows / least));
    d.chunk_rows = (a.rows + chunks - 1) / chunks;
    d.chunk_rows = (d.chunk_rows + row_unit - 1) / row_unit * row_unit;
    d.chunks = uint32_t((a.rows + d.chunk_rows - 1) / d.chunk_rows);
    // a launch's blocks fit the grid
    const uint64_t per = uint64_t(d.chunks) * d.slabs;
    p.batch = std::max<uint64_t>(
            1, std::min<uint64_t>(p.batch, ((1ull << 31) - 1) / per));
    return p;
}

struct GnWorkspace {
    float2* part;
    float* mean;
    float* rstd;
    float2* sums;
    float2* means;
    size_t bytes;
};

// The most that any alignment of the pointers needs.
GnWorkspace carve(const GroupNormArgs& a, const GnPlan& p, bool grad,
                  char* base) {
    Arena ar;
    ar.base = base;
    ar.size = ~size_t(0);
    GnWorkspace w{};
    const size_t nb = size_t(p.batch), parts = size_t(p.d.chunks);
    if (grad) {
        w.part = ar.take<float2>(nb * parts * a.C);
        w.sums = ar.take<float2>(size_t(a.n) * a.C);
        w.means = ar.take<float2>(size_t(a.n) * a.G);
    } else {
        w.part = ar.take<float2>(nb * a.G * parts * p.d.pieces);
        w.mean = ar.take<float>(size_t(a.n) * a.G);
        w.rstd = ar.take<float>(size_t(a.n) * a.G);
    }
    w.bytes = ar.used;
    return w;
}

template <typename T, int VEC>
void forward_t(const GnPlan& p, const GroupNormArgs& a, const void* x,
               const float* weight, const float* bias, void* y, float* mean,
               float* rstd, const GnWorkspace& w, cudaStream_t s) {
    const size_t sample = size_t(a.rows) * a.C;
    for (uint64_t n0 = 0; n0 < a.n; n0 += p.batch) {
        const uint64_t nb = std::min<uint64_t>(p.batch, a.n - n0);
        const unsigned grid = unsigned(nb * p.d.chunks * p.d.slabs);
        const T* xb = static_cast<const T*>(x) + n0 * sample;
        T* yb = static_cast<T*>(y) + n0 * sample;
        float* mb = mean + n0 * a.G;
        float* rb = rstd + n0 * a.G;
        k_gn_stats<T, VEC><<<grid, kGnThreads, 0, s>>>(p.d, xb, w.part);
        k_gn_finish<T><<<unsigned((nb * a.G + 7) / 8), 256, 0, s>>>(
                p.d, nb, xb, w.part, mb, rb);
        switch (a.act) {
            case 1:
                k_gn_apply<T, VEC, 1><<<grid, kGnThreads, 0, s>>>(
                        p.d, xb, weight, bias, mb, rb, yb);
                break;
            case 2:
                k_gn_apply<T, VEC, 2><<<grid, kGnThreads, 0, s>>>(
                        p.d, xb, weight, bias, mb, rb, yb);
                break;
            default:
                k_gn_apply<T, VEC, 0><<<grid, kGnThreads, 0, s>>>(
                        p.d, xb, weight, bias, mb, rb, yb);
        }
        DRESSI_CUDA(cudaGetLastError());
    }
}

template <typename T, int VEC, int ACT>
void backward_a(const GnPlan& p, const GroupNormArgs& a, const void* dy,
                const void* x, const float* weight, const float* bias,
                const float* mean, const float* rstd, void* dx,
                float* dweight, float* dbias, const GnWorkspace& w,
                cudaStream_t s) {
    const size_t sample = size_t(a.rows) * a.C;
    const int bundle = std::min(32, std::max(1, 32 / p.d.cpg));
    const int bundles = (a.G + bundle - 1) / bundle;
    for (uint64_t n0 = 0; n0 < a.n; n0 += p.batch) {
        const uint64_t nb = std::min<uint64_t>(p.batch, a.n - n0);
        const unsigned grid = unsigned(nb * p.d.chunks * p.d.slabs);
        const T* xb = static_cast<const T*>(x) + n0 * sample;
        const T* gb = static_cast<const T*>(dy) + n0 * sample;
        const float* mb = mean + n0 * a.G;
        const float* rb = rstd + n0 * a.G;
        float2* means = w.means + n0 * a.G;
        k_gn_grad_sums<T, VEC, ACT><<<grid, kGnThreads, 0, s>>>(
                p.d, gb, xb, weight, bias, mb, rb, w.part);
        k_gn_grad_finish<<<unsigned(nb * bundles), 512, 0, s>>>(
                p.d, bundle, w.part, weight, w.sums + n0 * a.C, means);
        if (dx)
            k_gn_grad_apply<T, VEC, ACT><<<grid, kGnThreads, 0, s>>>(
                    p.d, gb, xb, weight, bias, mb, rb, means,
                    static_cast<T*>(dx) + n0 * sample);
        DRESSI_CUDA(cudaGetLastError());
    }
    if (dweight || dbias) {
        k_gn_grad_affine<<<unsigned((a.C + 127) / 128), 128, 0, s>>>(
                p.d, w.sums, dweight, dbias);
        DRESSI_CUDA(cudaGetLastError());
    }
}

template <typename T, int VEC>
void backward_t(const GnPlan& p, const GroupNormArgs& a, const void* dy,
                const void* x, const float* weight, const float* bias,
                const float* mean, const float* rstd, void* dx,
                float* dweight, float* dbias, const GnWorkspace& w,
                cudaStream_t s) {
    auto* f = a.act == 1   ? backward_a<T, VEC, 1>
              : a.act == 2 ? backward_a<T, VEC, 2>
                           : backward_a<T, VEC, 0>;
    f(p, a, dy, x, weight, bias, mean, rstd, dx, dweight, dbias, w, s);
}

// Calls fn.template operator()<T, VEC>() for the plan's type and width.
template <typename F>
void by_type(int dtype, int vec, F&& fn) {
    if (dtype == 0) {
        if (vec == 4) fn(float(), std::integral_constant<int, 4>());
        else if (vec == 2) fn(float(), std::integral_constant<int, 2>());
        else fn(float(), std::integral_constant<int, 1>());
        return;
    }
    auto half = [&](auto t) {
        if (vec == 8) fn(t, std::integral_constant<int, 8>());
        else if (vec == 4) fn(t, std::integral_constant<int, 4>());
        else if (vec == 2) fn(t, std::integral_constant<int, 2>());
        else fn(t, std::integral_constant<int, 1>());
    };
    if (dtype == 1) half(__half());
    else half(__nv_bfloat16());
}

}  // namespace

size_t group_norm_workspace(const GroupNormArgs& a, bool grad) {
    if (a.n == 0 || a.rows == 0) return 256;
    // vectors get narrower with a pointer's alignment; the parts are most
    // with the narrowest
    size_t most = 256;
    for (int align = 16; align >= 1; align /= 2) {
        const GnPlan p = make_plan(
                a, {reinterpret_cast<const void*>(uintptr_t(align))}, grad);
        most = std::max(most, carve(a, p, grad, nullptr).bytes);
    }
    return most;
}

void group_norm_op(const GroupNormArgs& a, const void* x, const float* weight,
                   const float* bias, void* y, float* mean, float* rstd,
                   void* workspace, cudaStream_t s) {
    if (a.n == 0 || a.rows == 0) return;
    const GnPlan p = make_plan(a, {x, y}, false);
    const GnWorkspace w = carve(a, p, false, static_cast<char*>(workspace));
    ProfScope ps("group_norm", s);
    by_type(a.dtype, p.vec, [&](auto t, auto v) {
        forward_t<decltype(t), decltype(v)::value>(
                p, a, x, weight, bias, y, mean ? mean : w.mean,
                rstd ? rstd : w.rstd, w, s);
    });
}

void group_norm_grad_op(const GroupNormArgs& a, const void* dy, const void* x,
                        const float* weight, const float* bias,
                        const float* mean, const float* rstd, void* dx,
                        float* dweight, float* dbias, void* workspace,
                        cudaStream_t s) {
    if (a.n == 0 || a.rows == 0) {
        if (dweight) DRESSI_CUDA(cudaMemsetAsync(dweight, 0, 4ull * a.C, s));
        if (dbias) DRESSI_CUDA(cudaMemsetAsync(dbias, 0, 4ull * a.C, s));
        return;
    }
    const GnPlan p = make_plan(a, {dy, x, dx}, true);
    const GnWorkspace w = carve(a, p, true, static_cast<char*>(workspace));
    ProfScope ps("group_norm_grad", s);
    by_type(a.dtype, p.vec, [&](auto t, auto v) {
        backward_t<decltype(t), decltype(v)::value>(
                p, a, dy, x, weight, bias, mean, rstd, dx, dweight, dbias, w,
                s);
    });
}

}  // namespace dressi
