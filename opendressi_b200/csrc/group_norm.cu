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
// wants it (8x256x256x64 bf16 forward: 45 us, against 20.5 for its bytes at the
// copy rate; 2x1024x1024x64 bf16 with its gradient: 414 us, a sample being
// larger than L2). Samples of a few values are not what it is made for: a block
// takes them one by one (10^6 x 32 f32: 6.6 ms, 21 ms backward). Statistics are
// 32-bit per thread about the mean of the thread's values so far (no
// cancellation where |mean| >> deviation), merged in 32 bits
// within a block as distances from a common value and in 64 bits between
// blocks; sums are taken in a fixed order, so reruns give the same bits.
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
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"

namespace dressi {

namespace {

constexpr int kGnThreads = 256;
constexpr int kGnSms = 148;  // of a B200; another number would cost time alone
constexpr int kGnResident = 4;      // resident blocks an SM, forward
constexpr int kGnResidentGrad = 2;  // backward

struct GnDims {
    uint64_t rows;
    int C, G, cpg;
    float eps;
    // mapping
    int slabs;         // column slabs of a row (1: flat)
    int slab_cols;     // columns of a full slab
    int pieces;        // slabs per group (1 unless a group exceeds a slab)
    uint32_t chunks;   // row chunks of a sample
    uint64_t chunk_rows;
    int threads;       // flat: threads that work (they cover whole rows)
    int lanes;         // flat: rows they cover
    int run;           // channels of a group that a vector holds side by side
    int slots;         // resident: steps that a block keeps
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

// Two 32-bit values in one register pair and one instruction.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
    Two d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ float2 of_two(Two d) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(d));
    return f;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// A vector as pairs of 32-bit values (one and a zero where VEC is 1).
template <int VEC>
constexpr int kPairs = (VEC + 1) / 2;

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& v, Two* o) {
    if constexpr (VEC == 1) {
        o[0] = two(to_f<T>(v.v[0]), 0.f);
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 2; k++) {
            if constexpr (sizeof(T) == 4) {
                o[k] = two(v.v[2 * k], v.v[2 * k + 1]);
            } else {
                const uint32_t w = reinterpret_cast<const uint32_t*>(&v)[k];
                if constexpr (std::is_same<T, __half>::value) {
                    const float2 f = __half22float2(
                            *reinterpret_cast<const __half2*>(&w));
                    o[k] = two(f.x, f.y);
                } else {
                    o[k] = two(__uint_as_float(w << 16),
                               __uint_as_float(w & 0xffff0000u));
                }
            }
        }
    }
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const Two* o) {
    Pack<T, VEC> v;
    if constexpr (VEC == 1) {
        v.v[0] = from_f<T>(of_two(o[0]).x);
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 2; k++) {
            const float2 f = of_two(o[k]);
            if constexpr (sizeof(T) == 4) {
                v.v[2 * k] = f.x;
                v.v[2 * k + 1] = f.y;
            } else if constexpr (std::is_same<T, __half>::value) {
                reinterpret_cast<__half2*>(&v)[k] =
                        __floats2half2_rn(f.x, f.y);
            } else {
                reinterpret_cast<__nv_bfloat162*>(&v)[k] =
                        __floats2bfloat162_rn(f.x, f.y);
            }
        }
    }
    return v;
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
    uint64_t base, step;
    int col0, cols, lanes, col;
    uint32_t steps;
    bool works;
};

// Blocks are (slab, chunk) along x and samples along y.
template <int VEC>
__device__ __forceinline__ Walk walk_of(const GnDims& d, uint32_t chunk,
                                        int slab) {
    Walk w;
    const uint64_t r0 = uint64_t(chunk) * d.chunk_rows;
    const uint64_t end = min(r0 + d.chunk_rows, d.rows) * d.C;
    if (d.slabs == 1) {
        w.col0 = 0;
        w.cols = d.C;
        w.lanes = d.lanes;
        w.works = int(threadIdx.x) < d.threads;
        w.base = r0 * d.C + threadIdx.x * VEC;
        w.step = uint64_t(d.threads) * VEC;
        w.col = int(threadIdx.x * VEC % uint32_t(d.C));
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
    w.steps = 0;
    if (w.works && w.base < end) {
        const uint64_t left = end - w.base + w.step - 1;
        w.steps = left >> 32 ? uint32_t(left / w.step)
                             : uint32_t(left) / uint32_t(w.step);
    }
    return w;
}

// Calls fn(j, channel, group) for the values of a thread's vector.
template <int VEC, typename F>
__device__ __forceinline__ void each_channel(const GnDims& d, const Walk& w,
                                             F&& fn) {
    int c = w.col0 + w.col, g = c / d.cpg, k = c - g * d.cpg;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        fn(j, c, g);
        if (++c == w.col0 + w.cols) {  // rows of a flat walk follow each other
            c = w.col0;
            g = c / d.cpg;
            k = c - g * d.cpg;
        } else if (++k == d.cpg) {
            k = 0;
            g++;
        }
    }
}

// Rounding below 0 is 0; NaN stays.
__device__ __forceinline__ float nonneg(float v) { return v < 0.f ? 0.f : v; }

template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Stages on their way to a thread at a time, of two vectors of each image.
constexpr int kGnStages = 4;

template <typename T, int VEC>
constexpr bool whole_vectors() {
    return VEC * sizeof(T) == 16;
}
// Bytes of shared memory of a block that walks over `images`.
// (and then writes VEC pairs of sums there).
template <typename T, int VEC>
constexpr int ring_bytes(int images) {
    return whole_vectors<T, VEC>()
                   ? images * kGnStages * 2 * kGnThreads * 16
                   : VEC * kGnThreads * int(sizeof(float2));
}

__device__ __forceinline__ void copy_16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         uint32_t(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
}

// Calls ready() once the first loads are under way, then fn(a, b) for `steps`
// vectors of one image (q null) or two. Whole vectors come through a ring in
// shared memory, each thread's its own: loads into registers would be a quarter
// as many.
template <typename T, int VEC, int IMAGES, typename R, typename F>
__device__ __forceinline__ void walk_over(const T* p, const T* q,
                                          uint64_t step, uint32_t steps,
                                          char* ring, R&& ready, F&& fn) {
    using V = Pack<T, VEC>;
    if constexpr (whole_vectors<T, VEC>()) {
        constexpr int stage = 2 * IMAGES * kGnThreads;
        V* own = reinterpret_cast<V*>(ring) + threadIdx.x;
        uint32_t sent = 0;
        auto send = [&](V* to) {
            if (sent + 1 < steps) {
                copy_16(to, p);
                copy_16(to + kGnThreads, p + step);
                p += 2 * step;
                if (IMAGES == 2) {
                    copy_16(to + 2 * kGnThreads, q);
                    copy_16(to + 3 * kGnThreads, q + step);
                    q += 2 * step;
                }
            } else if (sent < steps) {
                copy_16(to, p);
                if (IMAGES == 2) copy_16(to + 2 * kGnThreads, q);
            }
            sent += 2;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < kGnStages; k++) send(own + k * stage);
        ready();
        V* slot = own;
        for (uint32_t t = 0; t < steps; t += 2) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kGnStages - 1)
                         : "memory");
            const V a = *slot, b = IMAGES == 2 ? slot[2 * kGnThreads] : V{};
            if (t + 1 < steps) {
                const V a1 = slot[kGnThreads];
                const V b1 = IMAGES == 2 ? slot[3 * kGnThreads] : V{};
                send(slot);
                fn(a, b);
                fn(a1, b1);
            } else {
                fn(a, b);
            }
            slot += stage;
            if (slot == own + kGnStages * stage) slot = own;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        constexpr int kBatch = 4 / IMAGES;  // loads under way together
        ready();
        uint32_t t = 0;
        for (; t + kBatch <= steps; t += kBatch) {
            V a[kBatch], b[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                a[k] = load_pack<T, VEC>(p + k * step);
                if (IMAGES == 2) b[k] = load_pack<T, VEC>(q + k * step);
            }
            p += kBatch * step;
            if (IMAGES == 2) q += kBatch * step;
#pragma unroll
            for (int k = 0; k < kBatch; k++) fn(a[k], b[k]);
        }
        for (; t < steps; t++, p += step) {
            const V a = load_pack<T, VEC>(p);
            V b{};
            if (IMAGES == 2) {
                b = load_pack<T, VEC>(q);
                q += step;
            }
            fn(a, b);
        }
    }
}

// act 0: none, 1: relu, 2: silu. NaN stays NaN.
__device__ __forceinline__ Two sigmoid2(Two z) {
    const float2 t = of_two(mul2(z, two(-1.4426950408889634f)));
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = of_two(add2(two(e.x, e.y), two(1.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
    return two(e.x, e.y);
}
template <int ACT>
__device__ __forceinline__ Two act2(Two z) {
    if (ACT == 1) {
        const float2 f = of_two(z);
        return two(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);
    }
    if (ACT == 2) return mul2(z, sigmoid2(z));
    return z;
}
template <int ACT>
__device__ __forceinline__ Two act_grad2(Two dy, Two z) {
    if (ACT == 1) {
        const float2 f = of_two(z), g = of_two(dy);
        return two(f.x <= 0.f ? 0.f : g.x, f.y <= 0.f ? 0.f : g.y);
    }
    if (ACT == 2) {  // s (1 + z (1 - s))
        const Two s = sigmoid2(z);
        const Two t = fma2(s, two(-1.f), two(1.f));
        return mul2(dy, mul2(s, fma2(z, t, two(1.f))));
    }
    return dy;
}

// ------------------------------------------------------------------ forward

// Statistics of one (sample, chunk, slab): part[n][g][chunk * pieces + piece]
// = (mean, sum of squares about it). A thread sums distances from its own
// first value; runs of `run` channels of a group are merged in the thread, the
// threads' results by some lanes a group: the group's mean is an average of
// theirs, its sum of squares theirs plus count times (their mean - the mean)^2
// (the pairwise update of Chan, Golub and LeVeque, all at once). Means enter
// as distances from one of them: the square of a mean of many deviations would
// leave no digits of the variance in 32 bits.
//
// Where the first value is far from the others (a bright corner), a sum of
// squares about it is N times the variance's: so the sums are moved to the mean
// so far after 4, 16, 64, ... values. Squares are then at most 4 times what they
// are about the mean of all: of 4 n values, with d from the first n's mean to
// the others', they sum up to m about their own mean, 3/4 n d^2 or more, and to
// m + 9/4 n d^2 about the first n's.
template <int VEC>
struct ThreadMoments {
    static constexpr int P = kPairs<VEC>;
    Two k[P], s1[P], s2[P];  // -centre, sums of distances from it and squares
    uint32_t left;           // values until the next move
    float count;             // values that there are then

    // At the first value, which counts as met or comes again.
    template <typename T>
    __device__ __forceinline__ void begin(const Pack<T, VEC>& first,
                                          bool met) {
        unpack<T, VEC>(first, k);
#pragma unroll
        for (int j = 0; j < P; j++) {
            k[j] = mul2(k[j], two(-1.f));
            s1[j] = s2[j] = two(0.f);
        }
        left = met ? 3 : 4;
        count = 4.f;
    }
    // The sums about c + d from those about c, d the values' mean distance.
    __device__ __forceinline__ void move() {
        const float inv = -1.f / count;
#pragma unroll
        for (int j = 0; j < P; j++) {
            const Two old = k[j];
            k[j] = fma2(s1[j], two(inv), old);
            const Two d = fma2(k[j], two(-1.f), old);  // as it was rounded
            const Two nd = mul2(d, two(-count));
            s2[j] = fma2(mul2(d, two(-1.f)),
                         add2(s1[j], add2(s1[j], nd)), s2[j]);
            s1[j] = add2(s1[j], nd);
        }
        left = 3 * uint32_t(count);
        count *= 4.f;
    }
    template <typename T>
    __device__ __forceinline__ void add(const Pack<T, VEC>& v) {
        Two e[P];
        unpack<T, VEC>(v, e);
#pragma unroll
        for (int j = 0; j < P; j++) {
            e[j] = add2(e[j], k[j]);
            s1[j] = add2(s1[j], e[j]);
            s2[j] = fma2(e[j], e[j], s2[j]);
        }
        if (--left == 0) move();
    }
    // (mean, sum of squares) of each run of channels to sm.
    __device__ __forceinline__ void put(uint32_t steps, int run, float2* sm) {
        float mean[2 * P], m2[2 * P];
        const float inv = 1.f / float(steps);
#pragma unroll
        for (int j = 0; j < P; j++) {
            const Two m = mul2(s1[j], two(inv));
            const float2 q = of_two(fma2(mul2(s1[j], two(-1.f)), m, s2[j]));
            const float2 c = of_two(add2(m, mul2(k[j], two(-1.f))));
            mean[2 * j] = c.x;
            mean[2 * j + 1] = c.y;
            m2[2 * j] = nonneg(q.x);
            m2[2 * j + 1] = nonneg(q.y);
        }
        // neighbours of a group: equal counts
        float half = 0.5f * float(steps);
#pragma unroll
        for (int h = 1; h < VEC; h *= 2) {
            if (h < run) {
#pragma unroll
                for (int j = 0; j < VEC; j += 2 * h) {
                    const float e = mean[j + h] - mean[j];
                    m2[j] += m2[j + h] + e * e * half;
                    mean[j] += 0.5f * e;
                }
                half *= 2.f;
            }
        }
        sm += int(threadIdx.x) * (VEC / run);
#pragma unroll
        for (int j = 0; j < VEC; j++)
            if ((j & (run - 1)) == 0) sm[j / run] = make_float2(mean[j], m2[j]);
    }
};

// How many lanes add up a group where all `groups` are added up at once.
__device__ __forceinline__ int lanes_for(int groups) {
    int lanes = 32;
    while (lanes > 1 && kGnThreads / lanes < groups) lanes /= 2;
    return lanes;
}
template <typename F>
__device__ __forceinline__ F lane_sum(F v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Calls fn(g, mean, sum of squares) in one lane for each group g of the slab,
// from what the threads have put into sm and their counts of steps.
template <int VEC, typename F>
__device__ __forceinline__ void merge_block(const GnDims& d, const Walk& w,
                                            const float2* sm,
                                            const uint32_t* cnt, F&& fn) {
    // sm[lane * cols + c] with runs of 2^shift channels for columns
    const int shift = __ffs(d.run) - 1, runs_shift = __ffs(VEC) - 1 - shift;
    const int cols = w.cols >> shift;
    const int per = d.pieces > 1 ? cols : d.cpg >> shift;
    const int groups = d.pieces > 1 ? 1 : w.cols / d.cpg;
    const int lanes = lanes_for(groups), lane = threadIdx.x & (lanes - 1);
    // entry e = row * per + column: where a lane starts and how far it steps
    const int l0 = lane / per, c0 = lane - l0 * per;
    const int dl = lanes / per, dc = lanes - dl * per;
    for (int b = 0; b < groups; b += kGnThreads / lanes) {
        const int g = b + threadIdx.x / lanes;
        auto each = [&](auto&& add) {
            int l = g < groups ? l0 : w.lanes, c = c0;
            while (l < w.lanes) {
                const int at = l * cols + g * per + c;
                const uint32_t n = cnt[at >> runs_shift];
                if (n > 0) add(float(n << shift), sm[at]);
                l += dl;
                c += dc;
                if (c >= per) {
                    c -= per;
                    l++;
                }
            }
        };
        const float ref = g < groups ? sm[g * per].x : 0.f;
        float count = 0.f, sum = 0.f, all = 0.f;
        each([&](float n, float2 v) {
            count += n;
            sum += n * (v.x - ref);
        });
        const float off = lane_sum(sum, lanes) / lane_sum(count, lanes);
        each([&](float n, float2 v) {
            const float e = v.x - ref - off;
            all += v.y + n * e * e;
        });
        all = lane_sum(all, lanes);
        if (g < groups && lane == 0)
            fn(g, double(ref) + double(off), double(all));
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_stats(GnDims d, const T* __restrict__ x,
                   double2* __restrict__ part) {
    extern __shared__ __align__(16) char ring[];
    __shared__ uint32_t cnt[kGnThreads];
    const int slab = d.slabs == 1 ? 0 : int(blockIdx.x % uint32_t(d.slabs));
    const uint32_t chunk =
            d.slabs == 1 ? blockIdx.x : blockIdx.x / uint32_t(d.slabs);
    const uint64_t n = blockIdx.y;
    start_next();
    const Walk w = walk_of<VEC>(d, chunk, slab);
    ThreadMoments<VEC> m;
    if (w.steps > 0) {
        const T* own = x + n * d.rows * d.C + w.base;
        walk_over<T, VEC, 1>(
                own, static_cast<const T*>(nullptr), w.step, w.steps, ring,
                [&] { m.begin(load_pack<T, VEC>(own), false); },
                [&](const Pack<T, VEC>& v, const Pack<T, VEC>&) { m.add(v); });
    }
    // the ring is free once every thread has left it
    __syncthreads();
    float2* const sm = reinterpret_cast<float2*>(ring);
    if (w.steps > 0) m.put(w.steps, d.run, sm);
    cnt[threadIdx.x] = w.steps;
    __syncthreads();
    merge_block<VEC>(d, w, sm, cnt, [&](int g, double mean, double m2) {
        part[(n * d.G + w.col0 / d.cpg + g) * d.chunks * d.pieces +
             size_t(chunk) * d.pieces + slab % d.pieces] =
                make_double2(mean, m2);
    });
}

// Values of a group in part e of its d.chunks * d.pieces.
__device__ __forceinline__ double part_count(const GnDims& d, uint32_t e) {
    uint32_t chunk = e, piece = 0;
    if (d.pieces > 1) {
        chunk = e / d.pieces;
        piece = e - chunk * d.pieces;
    }
    const uint64_t rows = min(d.chunk_rows, d.rows - chunk * d.chunk_rows);
    return double(rows) *
           (d.pieces > 1 ? min(d.slab_cols, d.cpg - int(piece) * d.slab_cols)
                         : d.cpg);
}

// mean[n][g], rstd[n][g] from the parts; one warp each.
__global__ void k_gn_finish(GnDims d, uint32_t n,
                            const double2* part,
                            float* __restrict__ mean,
                            float* __restrict__ rstd) {
    const uint64_t i = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
    start_next();
    await_previous();
    if (i >= uint64_t(n) * d.G) return;
    const uint32_t np = d.chunks * d.pieces;
    const double2* own = part + i * np;
    const double all = double(d.rows) * d.cpg;
    double sum = 0.0, m2 = 0.0;
    for (uint32_t e = threadIdx.x & 31; e < np; e += 32)
        sum += part_count(d, e) * own[e].x;
    const double mu = warp_sum(sum) / all;
    for (uint32_t e = threadIdx.x & 31; e < np; e += 32) {
        const double off = own[e].x - mu;
        m2 += own[e].y + part_count(d, e) * off * off;
    }
    m2 = warp_sum(m2);
    if ((threadIdx.x & 31) == 0) {
        mean[i] = float(mu);
        rstd[i] = float(1.0 / sqrt(m2 / all + double(d.eps)));
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_apply(GnDims d, const T* __restrict__ x,
                   const float* __restrict__ weight,
                   const float* __restrict__ bias,
                   const float* mean,
                   const float* rstd, T* __restrict__ y) {
    extern __shared__ __align__(16) char ring[];
    // the last chunks first: they are what the statistics pass left on chip
    const uint32_t i = gridDim.x - 1 - blockIdx.x;
    const uint64_t n = gridDim.y - 1 - blockIdx.y;
    const int slab = d.slabs == 1 ? 0 : int(i % uint32_t(d.slabs));
    const uint32_t chunk = d.slabs == 1 ? i : i / uint32_t(d.slabs);
    const Walk w = walk_of<VEC>(d, chunk, slab);
    if (w.steps == 0) return;
    constexpr int P = kPairs<VEC>;
    Two mu[P], a[P], b[P];
    auto scales = [&] {
        await_previous();
        float m1[2 * P], a1[2 * P], b1[2 * P];
        each_channel<VEC>(d, w, [&](int j, int c, int g) {
            m1[j] = -mean[n * d.G + g];
            a1[j] = rstd[n * d.G + g] * (weight ? weight[c] : 1.f);
            b1[j] = bias ? bias[c] : 0.f;
        });
        if (VEC == 1) m1[1] = a1[1] = b1[1] = 0.f;
#pragma unroll
        for (int j = 0; j < P; j++) {
            mu[j] = two(m1[2 * j], m1[2 * j + 1]);
            a[j] = two(a1[2 * j], a1[2 * j + 1]);
            b[j] = two(b1[2 * j], b1[2 * j + 1]);
        }
    };
    T* to = y + n * d.rows * d.C + w.base;
    walk_over<T, VEC, 1>(
            x + n * d.rows * d.C + w.base, static_cast<const T*>(nullptr),
            w.step, w.steps, ring, scales,
            [&](const Pack<T, VEC>& v, const Pack<T, VEC>&) {
                Two e[P];
                unpack<T, VEC>(v, e);
#pragma unroll
                for (int j = 0; j < P; j++)
                    e[j] = act2<ACT>(fma2(add2(e[j], mu[j]), a[j], b[j]));
                *reinterpret_cast<Pack<T, VEC>*>(to) = pack<T, VEC>(e);
                to += w.step;
            });
}

// ----------------------------------------------------------------- resident
//
// A slab of a sample that fits a block's shared memory (an item) stays there
// from the statistics to the result: one launch, one read, no exchange. Slots
// are each thread's own, and refilled for the block's next item as soon as the
// thread has used them. (Keeping larger samples in several blocks that exchange
// their sums and wait for one another was no faster than separate launches: 71
// us against 51 for 8x256x256x64 bf16, the sums' way through memory being 8 us
// of it each time.)

template <int BYTES>
__device__ __forceinline__ void copy_vector(void* to, const void* from) {
    if constexpr (BYTES == 16) {
        copy_16(to, from);
    } else if constexpr (BYTES == 4) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                             uint32_t(__cvta_generic_to_shared(to))),
                     "l"(from)
                     : "memory");
    } else {
        static_assert(BYTES == 2, "16, 4 or 2 bytes");
        *static_cast<uint16_t*>(to) = *static_cast<const uint16_t*>(from);
    }
}

// Calls fn(g, sum of a, sum of b) in one lane for each of `groups` groups, of
// add(g, e, &a, &b) over e = 0 .. parts - 1; all groups' lanes at once.
template <typename A, typename F>
__device__ __forceinline__ void sum_parts(int groups, uint32_t parts, A&& add,
                                          F&& fn) {
    const int lanes = lanes_for(groups), lane = threadIdx.x & (lanes - 1);
    for (int g0 = 0; g0 < groups; g0 += kGnThreads / lanes) {
        const int g = g0 + threadIdx.x / lanes;
        double a = 0.0, b = 0.0;
        if (g < groups)
            for (uint32_t e = lane; e < parts; e += lanes) add(g, e, &a, &b);
        a = lane_sum(a, lanes);
        b = lane_sum(b, lanes);
        if (g < groups && lane == 0) fn(g, a, b);
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads, kGnResident)
        k_gn_resident(GnDims d, uint32_t items, const T* __restrict__ x,
                      const float* __restrict__ weight,
                      const float* __restrict__ bias,
                      float* __restrict__ mean, float* __restrict__ rstd,
                      T* __restrict__ y) {
    using V = Pack<T, VEC>;
    constexpr int P = kPairs<VEC>;
    extern __shared__ __align__(16) char smem[];
    __shared__ uint32_t cnt[kGnThreads];
    V* const slot = reinterpret_cast<V*>(smem) + threadIdx.x;
    float2* const sm = reinterpret_cast<float2*>(
            smem + size_t(d.slots) * kGnThreads * sizeof(V));
    float2* const stat = sm + kGnThreads * (VEC / d.run);

    uint32_t i = blockIdx.x;
    uint64_t n = i / uint32_t(d.slabs);
    Walk w = walk_of<VEC>(d, 0, int(i % uint32_t(d.slabs)));
    {
        const T* p = x + n * d.rows * d.C + w.base;
        for (uint32_t k = 0; k < w.steps; k++, p += w.step)
            copy_vector<sizeof(V)>(slot + k * kGnThreads, p);
    }
    for (;;) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (w.steps > 0) {
            ThreadMoments<VEC> m;
            m.begin(*slot, true);
            for (uint32_t k = 1; k < w.steps; k++) m.add(slot[k * kGnThreads]);
            m.put(w.steps, d.run, sm);
        }
        cnt[threadIdx.x] = w.steps;
        __syncthreads();
        const int first = w.col0 / d.cpg, groups = w.cols / d.cpg;
        const double all = double(d.rows) * d.cpg;
        merge_block<VEC>(d, w, sm, cnt, [&](int g, double mu, double m2) {
            const float2 st = make_float2(
                    float(mu), float(1.0 / sqrt(m2 / all + d.eps)));
            stat[g] = st;
            if (mean) {
                mean[n * d.G + first + g] = st.x;
                rstd[n * d.G + first + g] = st.y;
            }
        });
        __syncthreads();
        Two mu[P], a[P], b[P];
        {
            float m1[2 * P], a1[2 * P], b1[2 * P];
            each_channel<VEC>(d, w, [&](int j, int c, int g) {
                const float2 st = stat[g - first];
                m1[j] = -st.x;
                a1[j] = st.y * (weight ? weight[c] : 1.f);
                b1[j] = bias ? bias[c] : 0.f;
            });
            if (VEC == 1) m1[1] = a1[1] = b1[1] = 0.f;
#pragma unroll
            for (int j = 0; j < P; j++) {
                mu[j] = two(m1[2 * j], m1[2 * j + 1]);
                a[j] = two(a1[2 * j], a1[2 * j + 1]);
                b[j] = two(b1[2 * j], b1[2 * j + 1]);
            }
        }
        i += gridDim.x;
        const bool more = i < items;
        T* to = y + n * d.rows * d.C + w.base;
        const uint32_t steps = w.steps;
        const uint64_t step = w.step;
        const T* p = nullptr;
        if (more) {
            n = i / uint32_t(d.slabs);
            w = walk_of<VEC>(d, 0, int(i % uint32_t(d.slabs)));
            p = x + n * d.rows * d.C + w.base;
        } else {
            w.steps = 0;
        }
        V* at = slot;
        for (uint32_t k = 0; k < steps; k++, at += kGnThreads, to += step) {
            Two e[P];
            unpack<T, VEC>(*at, e);
            if (k < w.steps) {
                copy_vector<sizeof(V)>(at, p);
                p += w.step;
            }
#pragma unroll
            for (int j = 0; j < P; j++)
                e[j] = act2<ACT>(fma2(add2(e[j], mu[j]), a[j], b[j]));
            *reinterpret_cast<V*>(to) = pack<T, VEC>(e);
        }
        for (uint32_t k = steps; k < w.steps; k++, at += kGnThreads) {
            copy_vector<sizeof(V)>(at, p);
            p += w.step;
        }
        if (!more) break;
    }
}

// ----------------------------------------------------------------- backward

// What a thread's channels are scaled by: -mean, rstd, rstd weight, bias. z is
// (x - mean) (rstd weight) + bias as in the forward pass, rounded alike: relu
// passes a gradient exactly where it passed a value.
template <int VEC>
struct Scales {
    Two mu[kPairs<VEC>], r[kPairs<VEC>], a[kPairs<VEC>], b[kPairs<VEC>];
};
template <int VEC>
__device__ __forceinline__ Scales<VEC> scales_of(const GnDims& d,
                                                 const Walk& w, uint64_t n,
                                                 const float* weight,
                                                 const float* bias,
                                                 const float* mean,
                                                 const float* rstd) {
    constexpr int P = kPairs<VEC>;
    float m1[2 * P], r1[2 * P], a1[2 * P], b1[2 * P];
    each_channel<VEC>(d, w, [&](int j, int c, int g) {
        m1[j] = -mean[n * d.G + g];
        r1[j] = rstd[n * d.G + g];
        a1[j] = r1[j] * (weight ? weight[c] : 1.f);
        b1[j] = bias ? bias[c] : 0.f;
    });
    if (VEC == 1) m1[1] = r1[1] = a1[1] = b1[1] = 0.f;
    Scales<VEC> s;
#pragma unroll
    for (int j = 0; j < P; j++) {
        s.mu[j] = two(m1[2 * j], m1[2 * j + 1]);
        s.r[j] = two(r1[2 * j], r1[2 * j + 1]);
        s.a[j] = two(a1[2 * j], a1[2 * j + 1]);
        s.b[j] = two(b1[2 * j], b1[2 * j + 1]);
    }
    return s;
}

// (x, dy) of a pair of values to (h, dz).
template <int ACT, int VEC>
__device__ __forceinline__ void terms(const Scales<VEC>& c, int j, Two* h,
                                      Two* g) {
    const Two e = add2(h[j], c.mu[j]);
    h[j] = mul2(e, c.r[j]);
    g[j] = act_grad2<ACT>(g[j], fma2(e, c.a[j], c.b[j]));
}

// part[n][chunk][c] = (sum dz, sum dz h) over the chunk's rows.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads)
        k_gn_grad_sums(GnDims d, const T* __restrict__ dy,
                       const T* __restrict__ x,
                       const float* __restrict__ weight,
                       const float* __restrict__ bias,
                       const float* __restrict__ mean,
                       const float* __restrict__ rstd,
                       float2* __restrict__ part) {
    extern __shared__ __align__(16) char ring[];
    const int slab = d.slabs == 1 ? 0 : int(blockIdx.x % uint32_t(d.slabs));
    const uint32_t chunk =
            d.slabs == 1 ? blockIdx.x : blockIdx.x / uint32_t(d.slabs);
    const uint64_t n = blockIdx.y;
    start_next();
    const Walk w = walk_of<VEC>(d, chunk, slab);
    constexpr int P = kPairs<VEC>;
    Two A[P], B[P];
    if (w.works) {
        Scales<VEC> c;
#pragma unroll
        for (int j = 0; j < P; j++) A[j] = B[j] = two(0.f);
        const uint64_t at = n * d.rows * d.C + w.base;
        walk_over<T, VEC, 2>(
                x + at, dy + at, w.step, w.steps, ring,
                [&] {
                    c = scales_of<VEC>(d, w, n, weight, bias, mean, rstd);
                },
                [&](const Pack<T, VEC>& v, const Pack<T, VEC>& e) {
                    Two h[P], g[P];
                    unpack<T, VEC>(v, h);
                    unpack<T, VEC>(e, g);
#pragma unroll
                    for (int j = 0; j < P; j++) {
                        terms<ACT>(c, j, h, g);
                        A[j] = add2(A[j], g[j]);
                        B[j] = fma2(g[j], h[j], B[j]);
                    }
                });
    }
    // the ring is free once every thread has left it
    __syncthreads();
    float2* const sm = reinterpret_cast<float2*>(ring);
    if (w.works) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float2 a = of_two(A[j / 2]), b = of_two(B[j / 2]);
            sm[threadIdx.x * VEC + j] =
                    j % 2 ? make_float2(a.y, b.y) : make_float2(a.x, b.x);
        }
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
    start_next();
    await_previous();
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
        k_gn_grad_apply(GnDims d, const T* __restrict__ dy,
                        const T* __restrict__ x,
                        const float* __restrict__ weight,
                        const float* __restrict__ bias,
                        const float* __restrict__ mean,
                        const float* __restrict__ rstd,
                        const float2* means,
                        T* __restrict__ dx) {
    extern __shared__ __align__(16) char ring[];
    const uint32_t i = gridDim.x - 1 - blockIdx.x;
    const uint64_t n = gridDim.y - 1 - blockIdx.y;
    const int slab = d.slabs == 1 ? 0 : int(i % uint32_t(d.slabs));
    const uint32_t chunk = d.slabs == 1 ? i : i / uint32_t(d.slabs);
    const Walk w = walk_of<VEC>(d, chunk, slab);
    if (w.steps == 0) return;
    constexpr int P = kPairs<VEC>;
    Scales<VEC> c;
    Two ma[P], mb[P];
    auto scales = [&] {
        c = scales_of<VEC>(d, w, n, weight, bias, mean, rstd);
        await_previous();
        float a1[2 * P], b1[2 * P];
        each_channel<VEC>(d, w, [&](int j, int, int g) {
            const float2 m = means[n * d.G + g];
            const float r = rstd[n * d.G + g];
            a1[j] = -m.x * r;
            b1[j] = -m.y * r;
        });
        if (VEC == 1) a1[1] = b1[1] = 0.f;
#pragma unroll
        for (int j = 0; j < P; j++) {
            ma[j] = two(a1[2 * j], a1[2 * j + 1]);
            mb[j] = two(b1[2 * j], b1[2 * j + 1]);
        }
    };
    const uint64_t at = n * d.rows * d.C + w.base;
    T* to = dx + at;
    walk_over<T, VEC, 2>(
            x + at, dy + at, w.step, w.steps, ring, scales,
            [&](const Pack<T, VEC>& v, const Pack<T, VEC>& e) {
                Two h[P], g[P];
                unpack<T, VEC>(v, h);
                unpack<T, VEC>(e, g);
#pragma unroll
                for (int j = 0; j < P; j++) {
                    terms<ACT>(c, j, h, g);
                    g[j] = fma2(c.a[j], g[j], fma2(h[j], mb[j], ma[j]));
                }
                *reinterpret_cast<Pack<T, VEC>*>(to) = pack<T, VEC>(g);
                to += w.step;
            });
}

// dx of an item that stays in shared memory, and sums[n][c] = (sum dz,
// sum dz h).
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kGnThreads, kGnResidentGrad)
        k_gn_resident_grad(GnDims d, uint32_t items, const T* __restrict__ dy,
                           const T* __restrict__ x,
                           const float* __restrict__ weight,
                           const float* __restrict__ bias,
                           const float* __restrict__ mean,
                           const float* __restrict__ rstd,
                           float2* __restrict__ sums, T* __restrict__ dx) {
    using V = Pack<T, VEC>;
    constexpr int P = kPairs<VEC>;
    extern __shared__ __align__(16) char smem[];
    // x and dy of a step side by side
    V* const slot = reinterpret_cast<V*>(smem) + threadIdx.x;
    float2* const sm = reinterpret_cast<float2*>(
            smem + size_t(d.slots) * 2 * kGnThreads * sizeof(V));
    float2* const stat = sm + kGnThreads * VEC;

    uint32_t i = blockIdx.x;
    uint64_t n = i / uint32_t(d.slabs);
    Walk w = walk_of<VEC>(d, 0, int(i % uint32_t(d.slabs)));
    {
        const uint64_t at = n * d.rows * d.C + w.base;
        for (uint32_t k = 0; k < w.steps; k++) {
            copy_vector<sizeof(V)>(slot + 2 * k * kGnThreads,
                                   x + at + k * w.step);
            copy_vector<sizeof(V)>(slot + (2 * k + 1) * kGnThreads,
                                   dy + at + k * w.step);
        }
    }
    for (;;) {
        Scales<VEC> c;
        if (w.works) c = scales_of<VEC>(d, w, n, weight, bias, mean, rstd);
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (w.works) {
            Two A[P], B[P];
#pragma unroll
            for (int j = 0; j < P; j++) A[j] = B[j] = two(0.f);
            for (uint32_t k = 0; k < w.steps; k++) {
                Two h[P], g[P];
                unpack<T, VEC>(slot[2 * k * kGnThreads], h);
                unpack<T, VEC>(slot[(2 * k + 1) * kGnThreads], g);
#pragma unroll
                for (int j = 0; j < P; j++) {
                    terms<ACT>(c, j, h, g);
                    A[j] = add2(A[j], g[j]);
                    B[j] = fma2(g[j], h[j], B[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float2 a = of_two(A[j / 2]), b = of_two(B[j / 2]);
                sm[threadIdx.x * VEC + j] =
                        j % 2 ? make_float2(a.y, b.y) : make_float2(a.x, b.x);
            }
        }
        __syncthreads();
        for (int q = threadIdx.x; q < w.cols; q += kGnThreads) {
            double a = 0.0, b = 0.0;
            for (int l = 0; l < w.lanes; l++) {
                a += sm[l * w.cols + q].x;
                b += sm[l * w.cols + q].y;
            }
            sums[n * d.C + w.col0 + q] = make_float2(float(a), float(b));
            // no other thread reads this column
            const double wt = weight ? weight[w.col0 + q] : 1.f;
            sm[q] = make_float2(float(a * wt), float(b * wt));
        }
        __syncthreads();
        const int first = w.col0 / d.cpg;
        const double share = 1.0 / (double(d.rows) * d.cpg);
        sum_parts(
                w.cols / d.cpg, d.cpg,
                [&](int g, uint32_t e, double* a, double* b) {
                    const float2 v = sm[g * d.cpg + e];
                    *a += v.x;
                    *b += v.y;
                },
                [&](int g, double a, double b) {
                    stat[g] = make_float2(float(a * share), float(b * share));
                });
        __syncthreads();
        Two ma[P], mb[P];
        {
            float a1[2 * P], b1[2 * P];
            each_channel<VEC>(d, w, [&](int j, int, int g) {
                const float2 m = stat[g - first];
                const float r = rstd[n * d.G + g];
                a1[j] = -m.x * r;
                b1[j] = -m.y * r;
            });
            if (VEC == 1) a1[1] = b1[1] = 0.f;
#pragma unroll
            for (int j = 0; j < P; j++) {
                ma[j] = two(a1[2 * j], a1[2 * j + 1]);
                mb[j] = two(b1[2 * j], b1[2 * j + 1]);
            }
        }
        i += gridDim.x;
        const bool more = i < items;
        T* to = dx + n * d.rows * d.C + w.base;
        const uint32_t steps = w.steps;
        const uint64_t step = w.step;
        uint64_t from = 0;
        if (more) {
            n = i / uint32_t(d.slabs);
            w = walk_of<VEC>(d, 0, int(i % uint32_t(d.slabs)));
            from = n * d.rows * d.C + w.base;
        } else {
            w.steps = 0;
        }
        V* at = slot;
        auto refill = [&] {
            copy_vector<sizeof(V)>(at, x + from);
            copy_vector<sizeof(V)>(at + kGnThreads, dy + from);
            from += w.step;
        };
        for (uint32_t k = 0; k < steps;
             k++, at += 2 * kGnThreads, to += step) {
            Two h[P], g[P];
            unpack<T, VEC>(*at, h);
            unpack<T, VEC>(at[kGnThreads], g);
            if (k < w.steps) refill();
#pragma unroll
            for (int j = 0; j < P; j++) {
                terms<ACT>(c, j, h, g);
                g[j] = fma2(c.a[j], g[j], fma2(h[j], mb[j], ma[j]));
            }
            *reinterpret_cast<V*>(to) = pack<T, VEC>(g);
        }
        for (uint32_t k = steps; k < w.steps; k++, at += 2 * kGnThreads)
            refill();
        if (!more) break;
    }
}

// dweight[c], dbias[c] = the sums over `rows` rows of sums[row][c], in an
// order that their number gives: 32 columns x 16 lanes a block.
__global__ void __launch_bounds__(512)
        k_gn_grad_affine(int C, uint64_t rows, const float2* sums,
                         float* __restrict__ dweight,
                         float* __restrict__ dbias) {
    __shared__ double sa[16][33], sb[16][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x / 32;
    const int c = blockIdx.x * 32 + lane;
    await_previous();
    double a = 0.0, b = 0.0;
    if (c < C) {
#pragma unroll 8
        for (uint64_t r = row; r < rows; r += 16) {
            const float2 v = sums[r * C + c];
            a += v.x;
            b += v.y;
        }
    }
    sa[row][lane] = a;
    sb[row][lane] = b;
    __syncthreads();
    if (row == 0 && c < C) {
        for (int k = 1; k < 16; k++) {
            a += sa[k][lane];
            b += sb[k][lane];
        }
        if (dbias) dbias[c] = float(a);
        if (dweight) dweight[c] = float(b);
    }
}

// --------------------------------------------------------------------- host

struct GnPlan {
    GnDims d;
    int vec;
    uint64_t batch;  // samples per round of launches
    uint32_t items;  // of a resident launch; 0: rounds of launches
    uint32_t grid;   // its blocks
    int smem;        // bytes of a resident block
};

// A round of launches covers as many samples as L2 (126 MB) about holds
// between its two passes. 256x256x64 bf16, us: 9 views forward 64 with rounds
// of 64 MiB at most and 49 with 128, 16 views 90 and 78, 8 views backward (two
// images) 73 and 64. Over 34 shapes of 28 MiB to 2 GiB, forward and backward,
// 128 MiB is never slower than 64 and takes up to 22% less. Above it no size
// wins throughout: 192, 256, 512 MiB or no limit take up to 17% less again (9
// views backward), 512 MiB also 29% more (300x64x64x128 bf16 backward, 430 us
// against 333).
constexpr uint64_t kGnRoundBytes = 128ull << 20;

bool aligned(const void* p, size_t a) {
    return p == nullptr || reinterpret_cast<uintptr_t>(p) % a == 0;
}

void split_rows(GnDims* d, uint64_t chunks, uint64_t row_unit) {
    d->chunk_rows = (d->rows + chunks - 1) / chunks;
    d->chunk_rows = (d->chunk_rows + row_unit - 1) / row_unit * row_unit;
    d->chunks = uint32_t((d->rows + d->chunk_rows - 1) / d->chunk_rows);
}

// Dynamic shared memory of a resident block where `each` share an SM.
constexpr uint64_t resident_bytes(int each) {
    return uint64_t(226 / each - 3) << 10;
}

GnPlan make_plan(const GroupNormArgs& a, std::initializer_list<const void*> ps,
                 bool grad, bool resident) {
    const int es = a.dtype == 0 ? 4 : 2;
    GnPlan p{};
    GnDims& d = p.d;
    d.rows = a.rows;
    d.C = a.C;
    d.G = a.G;
    d.cpg = a.C / a.G;
    d.eps = a.eps;
    d.pieces = 1;
    // vectors of 16 bytes, of 4 or of a value
    int vec = 16 / es;
    auto narrower = [&] { vec = vec * es > 4 ? 4 / es : 1; };
    const uint64_t sample = a.rows * uint64_t(a.C);
    auto fits = [&](int v) {
        for (const void* q : ps)
            if (!aligned(q, size_t(v) * es)) return false;
        return true;
    };
    // flat: vectors need only the sample's size to be a multiple of them
    while (vec > 1 && (sample % vec != 0 || !fits(vec))) narrower();
    const int cover = a.C / std::gcd(a.C, vec);  // threads of whole rows
    uint64_t row_unit = 1;  // rows a chunk is a multiple of
    uint64_t lanes;         // rows a step of a block covers
    if (cover <= kGnThreads) {
        d.slabs = 1;
        d.slab_cols = a.C;
        const uint64_t want =
                std::max<uint64_t>(1, (sample / vec + cover - 1) / cover);
        d.threads = cover * int(std::min<uint64_t>(kGnThreads / cover,
                                                   want));
        d.lanes = int(int64_t(d.threads) * vec / a.C);
        lanes = d.lanes;
        row_unit = vec / std::gcd(a.C, vec);
    } else {
        // slabs start at multiples of the vector in a row of such
        for (;; narrower()) {
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
        lanes = std::max(1, kGnThreads / (std::min(d.slab_cols, a.C) / vec));
    }
    p.vec = vec;
    d.run = vec;
    while (d.cpg % d.run != 0) d.run /= 2;

    // Resident: a slab of a sample in one block, several blocks an SM where
    // there are that many.
    const int images = grad ? 2 : 1;
    const uint64_t items = uint64_t(d.slabs) * a.n;
    const int groups = std::min(d.slab_cols, a.C) / d.cpg;
    const int side = kGnThreads * (grad ? vec : vec / d.run) * 8 + groups * 8;
    const int step_bytes = images * kGnThreads * vec * es;
    const uint64_t steps = (a.rows + lanes - 1) / lanes;
    const int most = grad ? kGnResidentGrad : kGnResident;
    if (resident && d.pieces == 1 && items < (1u << 30)) {
        for (int each = most; each >= 1; each /= 2) {
            const uint64_t bytes = steps * step_bytes + side;
            if (bytes > resident_bytes(each)) continue;
            if (each < most && items > uint64_t(kGnSms) * each) break;
            split_rows(&d, 1, row_unit);
            d.slots = int(steps);
            p.items = uint32_t(items);
            p.grid = uint32_t(
                    std::min<uint64_t>(items, uint64_t(kGnSms) * each));
            p.smem = int(bytes);
            return p;
        }
    }

    // Rounds of launches: one wave of blocks, 4 steps or more a thread.
    const uint64_t bytes = std::max<uint64_t>(1, sample * es * images);
    const uint64_t rounds = std::max<uint64_t>(
            (a.n + 65534) / 65535,
            (a.n - 1) / std::max<uint64_t>(1, kGnRoundBytes / bytes) + 1);
    p.batch = (a.n + rounds - 1) / rounds;
    auto chunks_of = [&](int blocks_per_sm) {
        return std::max<uint64_t>(
                1, uint64_t(kGnSms) * blocks_per_sm /
                           std::max<uint64_t>(1, p.batch * d.slabs));
    };
    uint64_t chunks = chunks_of(grad ? 2 : 4);
    // Half as many blocks where a thread would take under 8 steps and then
    // takes more: what a block does but once counts. Of 180 f16 images (1, 3 or
    // 8 samples of 16 to 384 channels, 2 to 48 MB) 36 meet this rule: 16 take 2
    // to 19% less (1x110x111x384: 20.3 us and 16.5), 3 take 2 to 9% more
    // (8x135x136x64: 20.7 and 22.5). With 8 steps or more, half the blocks take
    // up to 18% more (3x128x128x384: 31.1 and 36.6).
    if (!grad && a.rows < lanes * 8 * chunks &&
        a.rows >= lanes * 8 * chunks_of(2))
        chunks = chunks_of(2);
    chunks = std::min(chunks, std::max<uint64_t>(1, a.rows / (lanes * 4)));
    split_rows(&d, chunks, row_unit);
    return p;
}

struct GnWorkspace {
    double2* part;
    float2* sums_part;
    float* mean;
    float* rstd;
    float2* sums;
    float2* means;
    size_t bytes;
};

GnWorkspace carve(const GroupNormArgs& a, const GnPlan& p, bool grad,
                  char* base) {
    Arena ar;
    ar.base = base;
    ar.size = ~size_t(0);
    GnWorkspace w{};
    const size_t parts = size_t(p.d.chunks) * p.d.pieces;
    if (p.items) {
        if (grad) w.sums = ar.take<float2>(size_t(a.n) * a.C);
    } else if (grad) {
        w.sums_part = ar.take<float2>(size_t(p.batch) * p.d.chunks * a.C);
        w.sums = ar.take<float2>(size_t(a.n) * a.C);
        w.means = ar.take<float2>(size_t(a.n) * a.G);
    } else {
        w.part = ar.take<double2>(size_t(p.batch) * a.G * parts);
        w.mean = ar.take<float>(size_t(a.n) * a.G);
        w.rstd = ar.take<float>(size_t(a.n) * a.G);
    }
    w.bytes = ar.used;
    return w;
}

// Launches a kernel with `smem` bytes of dynamic shared memory; early: it may
// begin while the launch before still runs (which is one of this file). What a
// kernel may use is the kernel's own state, shared by all host threads, so it
// is always set to the same: the most of any call.
template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, int smem, bool early,
            cudaStream_t s, A... args) {
    if (smem > 40 << 10)  // 48 KB with a kernel's static tables need no leave
        DRESSI_CUDA(cudaFuncSetAttribute(
                kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                int(resident_bytes(1))));
    if (early) {
        launch_early(kernel, grid, kGnThreads, size_t(smem), s, args...);
        return;
    }
    kernel<<<grid, kGnThreads, smem, s>>>(args...);
    DRESSI_CUDA(cudaGetLastError());
}

template <typename T, int VEC>
void forward_t(const GnPlan& p, const GroupNormArgs& a, const void* x,
               const float* weight, const float* bias, void* y, float* mean,
               float* rstd, const GnWorkspace& w, cudaStream_t s) {
    if (p.items) {
        launch(a.act == 1   ? k_gn_resident<T, VEC, 1>
               : a.act == 2 ? k_gn_resident<T, VEC, 2>
                            : k_gn_resident<T, VEC, 0>,
               dim3(p.grid), p.smem, false, s, p.d, p.items,
               static_cast<const T*>(x), weight, bias, mean, rstd,
               static_cast<T*>(y));
        return;
    }
    if (!mean) {
        mean = w.mean;
        rstd = w.rstd;
    }
    const size_t sample = size_t(a.rows) * a.C;
    for (uint64_t n0 = 0; n0 < a.n; n0 += p.batch) {
        const uint64_t nb = std::min<uint64_t>(p.batch, a.n - n0);
        const dim3 grid(p.d.chunks * p.d.slabs, unsigned(nb));
        const T* xb = static_cast<const T*>(x) + n0 * sample;
        T* yb = static_cast<T*>(y) + n0 * sample;
        float* mb = mean + n0 * a.G;
        float* rb = rstd + n0 * a.G;
        constexpr int smem = ring_bytes<T, VEC>(1);
        launch(k_gn_stats<T, VEC>, grid, smem, false, s, p.d, xb, w.part);
        launch_early(k_gn_finish, dim3(unsigned((nb * a.G + 7) / 8)), 256, 0,
                     s, p.d, uint32_t(nb), static_cast<const double2*>(w.part),
                     mb, rb);
        launch(a.act == 1   ? k_gn_apply<T, VEC, 1>
               : a.act == 2 ? k_gn_apply<T, VEC, 2>
                            : k_gn_apply<T, VEC, 0>,
               grid, smem, true, s, p.d, xb, weight, bias,
               static_cast<const float*>(mb), static_cast<const float*>(rb),
               yb);
    }
}

template <typename T, int VEC, int ACT>
void backward_a(const GnPlan& p, const GroupNormArgs& a, const void* dy,
                const void* x, const float* weight, const float* bias,
                const float* mean, const float* rstd, void* dx,
                float* dweight, float* dbias, const GnWorkspace& w,
                cudaStream_t s) {
    auto affine = [&](uint64_t rows) {
        if (!dweight && !dbias) return;
        launch_early(k_gn_grad_affine, dim3(unsigned((a.C + 31) / 32)), 512, 0,
                     s, a.C, rows, static_cast<const float2*>(w.sums), dweight,
                     dbias);
    };
    if (p.items) {
        launch(k_gn_resident_grad<T, VEC, ACT>, dim3(p.grid), p.smem, false, s,
               p.d, p.items, static_cast<const T*>(dy),
               static_cast<const T*>(x), weight, bias, mean, rstd, w.sums,
               static_cast<T*>(dx));
        affine(a.n);
        return;
    }
    const size_t sample = size_t(a.rows) * a.C;
    const int bundle = std::min(32, std::max(1, 32 / p.d.cpg));
    const int bundles = (a.G + bundle - 1) / bundle;
    for (uint64_t n0 = 0; n0 < a.n; n0 += p.batch) {
        const uint64_t nb = std::min<uint64_t>(p.batch, a.n - n0);
        const dim3 grid(p.d.chunks * p.d.slabs, unsigned(nb));
        const T* xb = static_cast<const T*>(x) + n0 * sample;
        const T* gb = static_cast<const T*>(dy) + n0 * sample;
        const float* mb = mean + n0 * a.G;
        const float* rb = rstd + n0 * a.G;
        float2* means = w.means + n0 * a.G;
        constexpr int smem = ring_bytes<T, VEC>(2);
        launch(k_gn_grad_sums<T, VEC, ACT>, grid, smem, false, s, p.d, gb, xb,
               weight, bias, mb, rb, w.sums_part);
        launch_early(k_gn_grad_finish, dim3(unsigned(nb * bundles)), 512, 0, s,
                     p.d, bundle, static_cast<const float2*>(w.sums_part),
                     weight, w.sums + n0 * a.C, means);
        if (dx)
            launch(k_gn_grad_apply<T, VEC, ACT>, grid, smem, true, s, p.d, gb,
                   xb, weight, bias, mb, rb, static_cast<const float2*>(means),
                   static_cast<T*>(dx) + n0 * sample);
    }
    affine(a.n);
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

// Calls fn(T(), integral constant VEC) for the plan's type and width.
template <typename F>
void by_type(int dtype, int vec, F&& fn) {
    if (dtype == 0) {
        if (vec == 4) fn(float(), std::integral_constant<int, 4>());
        else fn(float(), std::integral_constant<int, 1>());
        return;
    }
    auto half = [&](auto t) {
        if (vec == 8) fn(t, std::integral_constant<int, 8>());
        else if (vec == 2) fn(t, std::integral_constant<int, 2>());
        else fn(t, std::integral_constant<int, 1>());
    };
    if (dtype == 1) half(__half());
    else half(__nv_bfloat16());
}

}  // namespace

size_t group_norm_workspace(const GroupNormArgs& a, bool grad) {
    if (a.n == 0 || a.rows == 0) return 256;
    // vectors get narrower with a pointer's alignment: the most of any
    size_t most = 256;
    for (int align = 16; align >= 1; align /= 2)
        for (bool resident : {false, true}) {
            const GnPlan p = make_plan(
                    a, {reinterpret_cast<const void*>(uintptr_t(align))}, grad,
                    resident);
            most = std::max(most, carve(a, p, grad, nullptr).bytes);
        }
    return most;
}

void group_norm_op(const GroupNormArgs& a, const void* x, const float* weight,
                   const float* bias, void* y, float* mean, float* rstd,
                   void* workspace, cudaStream_t s) {
    if (a.n == 0 || a.rows == 0) return;
    const GnPlan p = make_plan(a, {x, y}, false, true);
    const GnWorkspace w = carve(a, p, false, static_cast<char*>(workspace));
    ProfScope ps("group_norm", s);
    by_type(a.dtype, p.vec, [&](auto t, auto v) {
        forward_t<decltype(t), decltype(v)::value>(
                p, a, x, weight, bias, y, mean, rstd, w, s);
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
    const GnPlan p = make_plan(a, {dy, x, dx}, true, dx != nullptr);
    const GnWorkspace w = carve(a, p, true, static_cast<char*>(workspace));
    ProfScope ps("group_norm_grad", s);
    by_type(a.dtype, p.vec, [&](auto t, auto v) {
        backward_t<decltype(t), decltype(v)::value>(
                p, a, dy, x, weight, bias, mean, rstd, dx, dweight, dbias, w,
                s);
    });
}

}  // namespace dressi
