// AdamW over many tensors in one launch, its moments in 32 or in 8 bits, and
// the norm over many tensors that it clips by (an extension: the reference
// steps one image per in-graph Adam).
//
//   m = m b1 + g (1 - b1);  v = v b2 + g g (1 - b2);  t = t + 1
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// with g first scaled by min(1, max_norm / (norm + 1e-6)) when clipping, and p
// clamped last. Bound by memory: 28 bytes a value with f32 parameters and
// 32-bit moments (100.7M values: 418 us, 6.7 TB/s), 16 + 16/256 with 8-bit ones
// (260 us, 6.2 TB/s; 283 to 307 at the clock of a sustained load, since its 60
// instructions a value fill two thirds of the issue slots).
//
// The tensors' addresses travel as a kernel argument (no table to upload, so
// a step can be captured), the work is cut into blocks of 256 values of one
// tensor, a warp each, and every thread block takes an equal contiguous run of
// them. Step counters live on the device, one per tensor: the last thread
// block of a launch to finish adds one to each.
//
// 8-bit moments. Each block of 256 holds e4m3 codes of m and of r = sqrt(v)
// (v itself would need twice the exponent range) and a scale each, the
// largest |value| / 448. A moving average moves by far less than the half step
// of an 8-bit format in one step (0.05% against 6%), so rounding to the
// nearest would hold it where it is: values are rounded up or down with the
// probability of their place between the two neighbours. The 16 random bits
// for each come from Wang's hash of (seed, step, tensor, place), so a run
// repeats exactly. r > 0 is never rounded to 0: m / (0 + eps) would explode.
// (A root below 2^-63 counts as 0 where eps is 2^-40 or more.) What is not
// finite is stored as NaN and leaves the block's scale alone.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "exact.cuh"
#include "kernels.h"

namespace dressi {

namespace {

constexpr int kBlock = 256;    // values a warp takes, and that share a scale
constexpr int kLane = 8;       // values a lane takes
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCtasPerSm = 4;  // with 32-bit moments
// With codes: 5 blocks on their way to each warp. 100.7M f32 values take 282
// us with 3 thread blocks an SM and 3 blocks ahead, 301 with 4 and 3, 325 with
// 4 and 2, 264 with 2 and 4, 256 with 2 and 5 (and 14 blocks a warp, below).
constexpr int kCtasPerSm8 = 2;
constexpr int kStages = 5;
template <int BITS>
constexpr int ctas_per_sm() {
    return BITS == 8 ? kCtasPerSm8 : kCtasPerSm;
}
constexpr uint64_t kMostBlocks = 1ull << 31;  // of one launch

struct AdamWHyper {
    float b1, omb1, b2, omb2, eps, ln_b1, ln_b2;
    float lo, hi, max_norm;
    bool clamped, small_eps;
    double lr, wd;
    const float* lr_device;
    const float* norm;
    uint32_t seed;
    uint32_t* ticket;
};

// The tensors of a launch: 73 bytes each, 29 kB for 400 of the 32764 bytes that
// a kernel's arguments may take (a launch with that many takes 3 us longer than
// one with 4 kB: three sizes).
template <int CAP>
struct AdamWTable {
    void* p[CAP];
    const void* g[CAP];
    void* m[CAP];
    void* v[CAP];
    float* sm[CAP];
    float* sv[CAP];
    int32_t* step[CAP];
    uint64_t n[CAP];
    uint32_t first[CAP + 1];  // block that the tensor begins with
    uint32_t index[CAP];
    uint8_t wide[CAP];  // aligned for whole-lane loads and stores
    uint32_t count;
};

struct alignas(32) F8 {
    float v[8];
};

__device__ __forceinline__ void load8(const float* p, float* o) {
    const F8 a = *reinterpret_cast<const F8*>(p);
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] = a.v[j];
}
__device__ __forceinline__ void store8(float* p, const float* o) {
    F8 a;
#pragma unroll
    for (int j = 0; j < 8; j++) a.v[j] = o[j];
    *reinterpret_cast<F8*>(p) = a;
}
__device__ __forceinline__ void load8(const __half* p, float* o) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&a);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        o[2 * j] = __low2float(h[j]);
        o[2 * j + 1] = __high2float(h[j]);
    }
}
__device__ __forceinline__ void store8(__half* p, const float* o) {
    uint4 a;
    __half2* h = reinterpret_cast<__half2*>(&a);
#pragma unroll
    for (int j = 0; j < 4; j++)
        h[j] = __floats2half2_rn(o[2 * j], o[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = a;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* o) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t* h = reinterpret_cast<const uint32_t*>(&a);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        o[2 * j] = __uint_as_float(h[j] << 16);
        o[2 * j + 1] = __uint_as_float(h[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* o) {
    uint4 a;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
    for (int j = 0; j < 4; j++)
        h[j] = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
    *reinterpret_cast<uint4*>(p) = a;
}
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) {
    *p = __float2half_rn(v);
}
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
}

// The 8 values of a lane: consecutive ones where the block is whole and
// aligned, else those at lane + 32 j with j's bit of `mask` set.
template <typename T>
__device__ __forceinline__ void load_lane(const T* p, bool wide, uint32_t mask,
                                          int lane, float* o) {
    if (wide) {
        load8(p + lane * kLane, o);
    } else {
#pragma unroll
        for (int j = 0; j < kLane; j++)
            o[j] = mask >> j & 1 ? to_f(p[lane + 32 * j]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store_lane(T* p, bool wide, uint32_t mask,
                                           int lane, const float* o) {
    if (wide) {
        store8(p + lane * kLane, o);
    } else {
#pragma unroll
        for (int j = 0; j < kLane; j++)
            if (mask >> j & 1) put(p + lane + 32 * j, o[j]);
    }
}

// e4m3 codes of a lane's values lane + 32 j, packed, and what they stand for.
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, uint32_t mask,
                                            int lane) {
    uint32_t c[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < kLane; j++)
        if (mask >> j & 1)
            c[j / 4] |= uint32_t(p[lane + 32 * j]) << (j % 4 * 8);
    return make_uint2(c[0], c[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t mask,
                                            int lane, uint2 c) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int j = 0; j < kLane; j++)
        if (mask >> j & 1)
            p[lane + 32 * j] = uint8_t(w[j / 4] >> (j % 4 * 8));
}
__device__ __forceinline__ void decode(uint2 c, float* o) {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const __half2 h(__nv_cvt_fp8x2_to_halfraw2(
                __nv_fp8x2_storage_t(w[j / 2] >> (j % 2 * 16)), __NV_E4M3));
        o[2 * j] = __low2float(h);
        o[2 * j + 1] = __high2float(h);
    }
}

// Two 32-bit values in one register pair and one instruction.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
    Two d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ void of_two(Two d, float* o) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o[0]), "=f"(o[1]) : "l"(d));
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

// sqrt to 2^-23; the quick one takes numbers below 2^-126 for 0.
__device__ __forceinline__ float sqrt_quick(float v) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float sqrt_fast(float v) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// 1 / v to 2^-23, for v in [2^-126, 2^126] and 0.
__device__ __forceinline__ float rcp_fast(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// The largest |a|, |b|, |c|; NaN if one is.
__device__ __forceinline__ float largest(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;"
        : "=f"(d)
        : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
    return d;
}

// The largest finite |x| of the warp's block, 2^-100 at least (448 over it
// stays finite), and whether all of x is finite.
__device__ __forceinline__ float top_of(const float* x, bool* finite) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < kLane; j += 2) most = largest(most, x[j], x[j + 1]);
    uint32_t top = __reduce_max_sync(0xffffffffu,
                                     __float_as_uint(most) & 0x7fffffffu);
    *finite = top < 0x7f800000u;
    if (!*finite) {
        top = 0u;
#pragma unroll
        for (int j = 0; j < kLane; j++) {
            const uint32_t u = __float_as_uint(x[j]) & 0x7fffffffu;
            top = max(top, u < 0x7f800000u ? u : 0u);
        }
        top = __reduce_max_sync(0xffffffffu, top);
    }
    return fmaxf(__uint_as_float(top), 0x1p-100f);
}

// The highest bytes of four words, the first's lowest.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t* b) {
    return __byte_perm(__byte_perm(b[0], b[1], 0x0073),
                       __byte_perm(b[2], b[3], 0x0073), 0x5410);
}

// The codes of a lane's values x, top the block's largest, inv = 448 / top.
// ROOT: of values that are not negative and do not become 0 unless they are.
//
// 2^-120 |x| inv, as the bits of a float, is an e4m3 number with 20 more bits
// of fraction: the exponents of both then count from the same power of two,
// and below 2^-6 (there 2^-126) both are equally spaced. 16 random bits and a
// half are added to those 20 and what carries goes up: up with the probability
// of the value's place between its neighbours. (All of it is moved up by 4
// bits, which drops the sign: a code is then the highest byte.) inv and the
// product are rounded: the largest comes out below 448 + 8 * 2^-15 and never
// carries past 448.
template <bool ROOT>
__device__ __forceinline__ uint2 encode(const float* x, float top, bool finite,
                                        const uint32_t* bits) {
    const float inv = 448.f / top;
    uint32_t b[kLane];
    float z[kLane];
    // one product where inv 2^-120 is no denormal number
    const bool once = top < 0x1p14f;
    const Two first = two(once ? inv * 0x1p-120f : inv);
#pragma unroll
    for (int j = 0; j < kLane; j += 2)
        of_two(mul2(two(x[j], x[j + 1]), first), z + j);
    if (!once) {
#pragma unroll
        for (int j = 0; j < kLane; j++) z[j] = __fmul_rn(z[j], 0x1p-120f);
    }
#pragma unroll
    for (int j = 0; j < kLane; j++) {
        uint32_t c = __float_as_uint(z[j]);
        // the smallest code where x > 0; what is no root of 0 has more bits
        if (ROOT) c = max(c, min(__float_as_uint(x[j]), 1u << 20));
        const uint32_t r = __byte_perm(bits[j], 0x80u, ROOT ? 0x7324 : 0x7104);
        b[j] = c * 16u + r;
    }
    if (!finite) {
#pragma unroll
        for (int j = 0; j < kLane; j++)
            if ((__float_as_uint(x[j]) & 0x7f800000u) == 0x7f800000u)
                b[j] = 0x7f000000u;  // NaN
    }
    uint2 c = make_uint2(top_bytes(b), top_bytes(b + 4));
    if (!ROOT) {
        uint32_t sign[kLane];
#pragma unroll
        for (int j = 0; j < kLane; j++) sign[j] = __float_as_uint(x[j]);
        c.x |= top_bytes(sign) & 0x80808080u;
        c.y |= top_bytes(sign + 4) & 0x80808080u;
    }
    return c;
}

template <int BITS>
struct StateOf {
    using type = float;
};
template <>
struct StateOf<8> {
    using type = uint8_t;
};

// The tensor whose blocks block b is among.
template <typename Table>
__device__ __forceinline__ uint32_t tensor_of(const Table& t, uint32_t b) {
    uint32_t lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (t.first[mid] <= b) lo = mid;
        else hi = mid;
    }
    return lo;
}

// What a warp knows of the tensor it is in.
template <typename T, typename State>
struct Target {
    T* p;
    const T* g;
    State* m;
    State* v;
    float* sm;
    float* sv;
    uint64_t n;
    bool aligned;
    uint32_t key;      // of the random bits
    float size, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    float scale, decay;
};

// Which of a lane's values lane + 32 j a block with `left` values has.
__device__ __forceinline__ uint32_t lane_mask(uint64_t left, int lane) {
    uint32_t mask = 0u;
#pragma unroll
    for (int j = 0; j < kLane; j++)
        mask |= uint32_t(uint64_t(lane + 32 * j) < left) << j;
    return mask;
}

// The step of a lane's values. ROOT: v is left as its root.
template <bool ROOT, typename Tensor>
__device__ __forceinline__ void update(const Tensor& t, const AdamWHyper& h,
                                       float* p, const float* g, float* m,
                                       float* v) {
    float r[kLane];
#pragma unroll
    for (int j = 0; j < kLane; j += 2) {
        const Two gj = mul2(two(g[j], g[j + 1]), two(t.scale));
        of_two(fma2(two(m[j], m[j + 1]), two(h.b1), mul2(gj, two(h.omb1))),
               m + j);
        of_two(fma2(two(v[j], v[j + 1]), two(h.b2),
                    mul2(mul2(gj, gj), two(h.omb2))),
               v + j);
    }
#pragma unroll
    for (int j = 0; j < kLane; j++) r[j] = sqrt_quick(v[j]);
    if (h.small_eps) {  // where the roots of denormal numbers count
#pragma unroll
        for (int j = 0; j < kLane; j++) r[j] = sqrt_fast(v[j]);
    }
#pragma unroll
    for (int j = 0; j < kLane; j += 2) {
        float d[2];
        of_two(fma2(two(r[j], r[j + 1]), two(t.root), two(h.eps)), d);
        const Two u = mul2(two(m[j], m[j + 1]),
                           two(rcp_fast(d[0]), rcp_fast(d[1])));
        of_two(fma2(two(-t.size), u, mul2(two(p[j], p[j + 1]), two(t.decay))),
               p + j);
        if (ROOT) {
            v[j] = r[j];
            v[j + 1] = r[j + 1];
        }
    }
    if (h.clamped) {
#pragma unroll
        for (int j = 0; j < kLane; j++) {  // NaN stays
            p[j] = p[j] < h.lo ? h.lo : p[j];
            p[j] = p[j] > h.hi ? h.hi : p[j];
        }
    }
}

// Blocks q, q + kWarps, ... below stop of a tensor with 32-bit moments; the
// first one behind stop.
template <typename T>
__device__ __forceinline__ uint32_t blocks_32(const Target<T, float>& t,
                                              const AdamWHyper& h, uint32_t q,
                                              uint32_t stop, int lane) {
    for (; q < stop; q += kWarps) {
        const uint64_t at = uint64_t(q) * kBlock;
        const bool wide = t.aligned && t.n - at >= kBlock;
        const uint32_t mask = wide ? 0u : lane_mask(t.n - at, lane);
        float p[kLane], g[kLane], m[kLane], v[kLane];
        load_lane(t.g + at, wide, mask, lane, g);
        load_lane(static_cast<const T*>(t.p + at), wide, mask, lane, p);
        load_lane(static_cast<const float*>(t.m + at), wide, mask, lane, m);
        load_lane(static_cast<const float*>(t.v + at), wide, mask, lane, v);
        update<false>(t, h, p, g, m, v);
        store_lane(t.p + at, wide, mask, lane, p);
        store_lane(t.m + at, wide, mask, lane, m);
        store_lane(t.v + at, wide, mask, lane, v);
    }
    return q;
}

// A warp's coming block on its way to shared memory (8-bit moments), copied
// in 16 bytes a lane past L1.
template <typename T>
struct alignas(4 * sizeof(T)) Quad {
    T v[4];
};
template <typename T>
struct alignas(16) Stage {
    T g[kBlock], p[kBlock];
    uint8_t codes[2][kBlock];
    float scale[4];
};

__device__ __forceinline__ void copy_16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         uint32_t(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copy_4(void* to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                         uint32_t(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void fetch(const Target<T, uint8_t>& t, uint64_t at,
                                      int lane, Stage<T>* s) {
    constexpr int run = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < kBlock; k += 32 * run) {
        copy_16(s->g + k + lane * run, t.g + at + k + lane * run);
        copy_16(s->p + k + lane * run, t.p + at + k + lane * run);
    }
    copy_16(s->codes[0] + lane * 16,
            (lane < 16 ? t.m : t.v - kBlock) + at + lane * 16);
}

template <typename T>
__device__ __forceinline__ void quad_in(const Quad<T>& q, float* o) {
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = to_f(q.v[j]);
}
template <typename T>
__device__ __forceinline__ void quad_out(T* to, const float* o) {
    Quad<T> f;
#pragma unroll
    for (int j = 0; j < 4; j++) put(&f.v[j], o[j]);
    *reinterpret_cast<Quad<T>*>(to) = f;
}

// The same with 8-bit moments: codes are bound by arithmetic nearly as much as
// by memory, so coming blocks are fetched while one is computed.
template <typename T>
__device__ __forceinline__ uint32_t blocks_8(const Target<T, uint8_t>& t,
                                             const AdamWHyper& h, uint32_t q,
                                             uint32_t stop, int lane,
                                             Stage<T>* stage) {
    auto is_wide = [&](uint32_t b) {
        return t.aligned && t.n - uint64_t(b) * kBlock >= kBlock;
    };
    auto begin = [&](uint32_t b, Stage<T>* s) {
        if (b < stop) {
            if (is_wide(b)) fetch(t, uint64_t(b) * kBlock, lane, s);
            if (lane < 2) copy_4(&s->scale[lane], (lane ? t.sv : t.sm) + b);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int turn = 0;
#pragma unroll
    for (int k = 0; k < kStages; k++) begin(q + k * kWarps, &stage[k]);
    for (; q < stop; q += kWarps) {
        const uint64_t at = uint64_t(q) * kBlock;
        const bool wide = is_wide(q);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        Stage<T>& s = stage[turn];
        const float am = s.scale[0], av = s.scale[1];
        float p[kLane], g[kLane], m[kLane], v[kLane];
        uint2 cm, cv;
        uint32_t mask = 0u;
        if (wide) {  // two runs of 4 values
            auto quad = [&](const T* q, int k) {
                return *reinterpret_cast<const Quad<T>*>(q + k * 128 +
                                                         lane * 4);
            };
            auto word = [&](const uint8_t* q, int k) {
                return *reinterpret_cast<const uint32_t*>(q + k * 128 +
                                                          lane * 4);
            };
#pragma unroll
            for (int k = 0; k < 2; k++) {
                quad_in(quad(s.g, k), g + 4 * k);
                quad_in(quad(s.p, k), p + 4 * k);
            }
            cm = make_uint2(word(s.codes[0], 0), word(s.codes[0], 1));
            cv = make_uint2(word(s.codes[1], 0), word(s.codes[1], 1));
        } else {
            mask = lane_mask(t.n - at, lane);
            load_lane(t.g + at, false, mask, lane, g);
            load_lane(static_cast<const T*>(t.p + at), false, mask, lane, p);
            cm = load_codes(t.m + at, mask, lane);
            cv = load_codes(t.v + at, mask, lane);
        }
        // all lanes have theirs: the place is free for a later block
        __syncwarp();
        begin(q + kStages * kWarps, &s);
        if (++turn == kStages) turn = 0;
        decode(cm, m);
        decode(cv, v);
#pragma unroll
        for (int j = 0; j < kLane; j += 2) {
            of_two(mul2(two(m[j], m[j + 1]), two(am)), m + j);
            const Two r = mul2(two(v[j], v[j + 1]), two(av));
            of_two(mul2(r, r), v + j);
        }
        update<true>(t, h, p, g, m, v);
        bool fm, fv;
        const float tm = top_of(m, &fm), tv = top_of(v, &fv);
        uint32_t bits[kLane];
        const uint32_t place = t.key + uint32_t(at) + (wide ? 4 * lane : lane);
        const uint32_t next = wide ? 1u : 32u, half = 128u;
#pragma unroll
        for (int j = 0; j < kLane; j++)
            bits[j] = wang_hash(place + j % 4 * next + j / 4 * half);
        cm = encode<false>(m, tm, fm, bits);
        cv = encode<true>(v, tv, fv, bits);
        if (wide) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint64_t i = at + k * 128 + lane * 4;
                quad_out(t.p + i, p + 4 * k);
                *reinterpret_cast<uint32_t*>(t.m + i) = k ? cm.y : cm.x;
                *reinterpret_cast<uint32_t*>(t.v + i) = k ? cv.y : cv.x;
            }
        } else {
            store_lane(t.p + at, false, mask, lane, p);
            store_codes(t.m + at, mask, lane, cm);
            store_codes(t.v + at, mask, lane, cv);
        }
        if (lane == 0) {
            t.sm[q] = tm * (1.f / 448.f);
            t.sv[q] = tv * (1.f / 448.f);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    return q;
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<BITS>())
        k_adamw(const __grid_constant__ AdamWTable<CAP> t,
                const __grid_constant__ AdamWHyper h) {
    await_previous();  // the norm, where this launch began early
    using State = typename StateOf<BITS>::type;
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint64_t all = t.first[t.count];
    const uint32_t b_end = uint32_t(all * (blockIdx.x + 1) / gridDim.x);
    uint32_t b = uint32_t(all * blockIdx.x / gridDim.x) + warp;

    Target<T, State> w;
    w.scale = 1.f;
    if (h.norm) {
        const float c = h.max_norm / (*h.norm + 1e-6f);
        w.scale = c > 1.f ? 1.f : c;  // NaN stays
    }
    const double lr = h.lr_device ? double(*h.lr_device) : h.lr;
    w.decay = float(1.0 - lr * h.wd);

    uint32_t ti = b < b_end ? tensor_of(t, b) : 0u;
    while (b < b_end) {  // tensor after tensor
        while (b >= t.first[ti + 1]) ti++;
        const uint32_t first = t.first[ti];
        const uint32_t stop = min(b_end, t.first[ti + 1]) - first;
        const int32_t step = *t.step[ti] + 1;
        // 1 - b^t = -expm1(t ln b): exact to a few 2^-24, also where b^t is
        // next to 1
        w.size = float(lr / double(-expm1f(float(step) * h.ln_b1)));
        w.root = 1.f / sqrtf(-expm1f(float(step) * h.ln_b2));
        w.key = wang_hash(wang_hash(h.seed ^ wang_hash(uint32_t(step))) +
                          t.index[ti]);
        w.p = static_cast<T*>(t.p[ti]);
        w.g = static_cast<const T*>(t.g[ti]);
        w.m = static_cast<State*>(t.m[ti]);
        w.v = static_cast<State*>(t.v[ti]);
        w.sm = t.sm[ti];
        w.sv = t.sv[ti];
        w.n = t.n[ti];
        w.aligned = t.wide[ti];
        if constexpr (BITS == 32) {
            b = first + blocks_32(w, h, b - first, stop, lane);
        } else {
            extern __shared__ __align__(16) char stages[];
            b = first +
                blocks_8(w, h, b - first, stop, lane,
                         reinterpret_cast<Stage<T>*>(stages) + warp * kStages);
        }
    }
    // every block has read the counters once all have drawn a ticket
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(h.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (last) {
        for (uint32_t i = threadIdx.x; i < t.count; i += kThreads)
            *t.step[i] += 1;
        if (threadIdx.x == 0) *h.ticket = 0u;
    }
}

int sm_count() {
    int dev = 0, sms = 148;
    DRESSI_CUDA(cudaGetDevice(&dev));
    DRESSI_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount,
                                       dev));
    return sms;
}

bool aligned(const void* p, size_t a) {
    return reinterpret_cast<uintptr_t>(p) % a == 0;
}

template <typename T, int BITS, int CAP>
void launch_adamw(const AdamWArgs& a, const AdamWHyper& h, uint32_t i0,
                  uint32_t i1, bool early, cudaStream_t s) {
    AdamWTable<CAP> t;
    t.count = i1 - i0;
    uint64_t blocks = 0;
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t k = i - i0;
        t.p[k] = a.params[i];
        t.g[k] = a.grads[i];
        t.m[k] = a.exp_avg[i];
        t.v[k] = a.avg_sq[i];
        t.sm[k] = BITS == 8 ? a.exp_avg_scale[i] : nullptr;
        t.sv[k] = BITS == 8 ? a.avg_sq_scale[i] : nullptr;
        t.step[k] = a.steps[i];
        t.n[k] = a.numel[i];
        t.index[k] = a.index ? a.index[i] : i;
        const size_t run = BITS == 8 ? 16 : kLane * sizeof(T);
        const size_t st = BITS == 8 ? 16 : kLane * sizeof(float);
        t.wide[k] = aligned(t.p[k], run) && aligned(t.g[k], run) &&
                    aligned(t.m[k], st) && aligned(t.v[k], st);
        t.first[k] = uint32_t(blocks);
        blocks += (t.n[k] + kBlock - 1) / kBlock;
    }
    t.first[t.count] = uint32_t(blocks);
    // Whole waves of thread blocks, each a run of memory of its own: SMs
    // further from the memory take fewer of them, and all of them together
    // touch few pages at a time. Of 4 or more blocks a warp (100.7M f32
    // values, 32 bits: 472 us as one wave, 434 of 16, 424 of 8, 419 of 4 and
    // of 2, 442 of 1), of 14 with codes (278 of 8, 262 of 10, 256 of 14, 260
    // of 20, 266 of 32: there the fetch ahead starts anew in each).
    const uint64_t wave = uint64_t(sm_count()) * ctas_per_sm<BITS>();
    const uint64_t waves = std::max<uint64_t>(
            1, blocks / (wave * kWarps * (BITS == 8 ? 14 : 4)));
    const uint64_t grid = std::max<uint64_t>(
            1, std::min<uint64_t>((blocks + kWarps - 1) / kWarps,
                                  wave * waves));
    const int smem = BITS == 8 ? kWarps * kStages * sizeof(Stage<T>) : 0;
    if (smem > 48 << 10)
        DRESSI_CUDA(cudaFuncSetAttribute(
                k_adamw<T, BITS, CAP>,
                cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (early) {
        launch_early(k_adamw<T, BITS, CAP>, dim3(unsigned(grid)), kThreads,
                     smem, s, t, h);
    } else {
        k_adamw<T, BITS, CAP><<<unsigned(grid), kThreads, smem, s>>>(t, h);
        DRESSI_CUDA(cudaGetLastError());
    }
}

template <typename T, int BITS>
void adamw_t(const AdamWArgs& a, const AdamWHyper& h, cudaStream_t s) {
    constexpr uint32_t kFew = 32, kSome = 192, kMany = 400;
    for (uint32_t i0 = 0; i0 < a.n_tensors;) {
        // behind the norm's launch, which lets it
        const bool early = h.norm && i0 == 0;
        uint32_t i1 = i0;
        uint64_t blocks = 0;
        while (i1 < a.n_tensors && i1 - i0 < kMany) {
            const uint64_t more = (a.numel[i1] + kBlock - 1) / kBlock;
            if (i1 > i0 && blocks + more > kMostBlocks) break;
            blocks += more;
            i1++;
        }
        if (i1 - i0 <= kFew)
            launch_adamw<T, BITS, kFew>(a, h, i0, i1, early, s);
        else if (i1 - i0 <= kSome)
            launch_adamw<T, BITS, kSome>(a, h, i0, i1, early, s);
        else
            launch_adamw<T, BITS, kMany>(a, h, i0, i1, early, s);
        i0 = i1;
    }
}

// --------------------------------------------------------------------- norm

constexpr int kNormUnit = kThreads * kLane;  // values a thread block takes
constexpr int kNormCtasPerSm = 4;  // one wave: more blocks were slower
constexpr int kNormMost = 1024;    // thread blocks (partial sums)

// A launch takes longer the more arguments it has (2.8 us with 4 kB, 4.9 with
// 21 kB), so tables come in three sizes.
template <int CAP>
struct NormTable {
    const void* p[CAP];
    uint64_t n[CAP];
    uint32_t first[CAP + 1];
    uint8_t type[CAP];
    uint32_t count;
};

// Squares are summed in 64 bits from the first on: no overflow, and an order
// that the sizes, the alignments and the number of SMs give. Units q .. stop - 1 of a
// tensor, four loads under way together.
template <typename T>
__device__ __forceinline__ double squares(const T* p, uint64_t n, uint32_t q,
                                          uint32_t stop) {
    double s = 0.0;
    auto add = [&](const float* x) {
#pragma unroll
        for (int j = 0; j < kLane; j++) s += double(x[j]) * double(x[j]);
    };
    if (reinterpret_cast<uintptr_t>(p) % (kLane * sizeof(T)) == 0) {
        const uint32_t whole = uint32_t(min(uint64_t(stop), n / kNormUnit));
        const T* at = p + uint64_t(q) * kNormUnit + threadIdx.x * kLane;
        for (; q + 4 <= whole; q += 4, at += 4 * kNormUnit) {
            float x[4][kLane];
#pragma unroll
            for (int k = 0; k < 4; k++) load8(at + k * kNormUnit, x[k]);
#pragma unroll
            for (int k = 0; k < 4; k++) add(x[k]);
        }
        for (; q < whole; q++, at += kNormUnit) {
            float x[kLane];
            load8(at, x);
            add(x);
        }
    }
    for (; q < stop; q++) {
        const T* at = p + uint64_t(q) * kNormUnit;
        const uint64_t left = n - uint64_t(q) * kNormUnit;
        float x[kLane];
#pragma unroll
        for (int j = 0; j < kLane; j++) {
            const uint32_t i = threadIdx.x + kThreads * j;
            x[j] = i < left ? to_f(at[i]) : 0.f;
        }
        add(x);
    }
    return s;
}

__device__ __forceinline__ double block_sum(double s) {
    __shared__ double red[kWarps];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = s;
    __syncthreads();
    s = 0.0;
    for (int k = 0; k < kWarps; k++) s += red[k];
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kNormCtasPerSm)
        k_norm_parts(const __grid_constant__ NormTable<CAP> t, double* part,
                     int add) {
    start_next();
    const uint64_t all = t.first[t.count];
    const uint32_t end = uint32_t(all * (blockIdx.x + 1) / gridDim.x);
    uint32_t b = uint32_t(all * blockIdx.x / gridDim.x);
    double s = 0.0;
    uint32_t ti = b < end ? tensor_of(t, b) : 0u;
    while (b < end) {
        while (b >= t.first[ti + 1]) ti++;
        const uint32_t first = t.first[ti];
        const uint32_t stop = min(end, t.first[ti + 1]);
        const uint64_t n = t.n[ti];
        if (t.type[ti] == 0)
            s += squares(static_cast<const float*>(t.p[ti]), n, b - first,
                         stop - first);
        else if (t.type[ti] == 1)
            s += squares(static_cast<const __half*>(t.p[ti]), n, b - first,
                         stop - first);
        else
            s += squares(static_cast<const __nv_bfloat16*>(t.p[ti]), n,
                         b - first, stop - first);
        b = stop;
    }
    s = block_sum(s);
    if (threadIdx.x == 0)
        part[blockIdx.x] = add ? part[blockIdx.x] + s : s;
}

__global__ void __launch_bounds__(kThreads)
        k_norm_finish(const double* part, int n, float* out) {
    start_next();
    await_previous();
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) s += part[i];
    s = block_sum(s);
    if (threadIdx.x == 0) out[0] = float(sqrt(s));
}

}  // namespace

void adamw_op(const AdamWArgs& a, cudaStream_t s) {
    if (a.n_tensors == 0) return;
    AdamWHyper h{};
    h.b1 = float(a.beta1);
    h.omb1 = float(1.0 - a.beta1);
    h.b2 = float(a.beta2);
    h.omb2 = float(1.0 - a.beta2);
    h.eps = float(a.eps);
    h.ln_b1 = float(std::log(a.beta1));
    h.ln_b2 = float(std::log(a.beta2));
    h.lo = a.clamp_lo;
    h.hi = a.clamp_hi;
    h.clamped = a.clamp_lo > -INFINITY || a.clamp_hi < INFINITY;
    h.max_norm = float(a.max_norm);
    // the root of 2^-126 is 2^-63: nothing next to an eps of 2^-40
    h.small_eps = h.eps < 0x1p-40f;
    h.lr = a.lr;
    h.wd = a.weight_decay;
    h.lr_device = a.lr_device;
    h.norm = a.max_norm > 0.0 ? a.grad_norm : nullptr;
    h.seed = a.seed;
    h.ticket = a.ticket;
    ProfScope ps("adamw", s);
    auto by_bits = [&](auto t) {
        using T = decltype(t);
        if (a.state_bits == 8) adamw_t<T, 8>(a, h, s);
        else adamw_t<T, 32>(a, h, s);
    };
    if (a.dtype == 0) by_bits(float());
    else if (a.dtype == 1) by_bits(__half());
    else by_bits(__nv_bfloat16());
}

size_t grad_norm_workspace() { return kNormMost * sizeof(double); }

void grad_norm_op(uint32_t n_tensors, const void* const* tensors,
                  const uint64_t* numel, const int32_t* dtypes, float* out,
                  void* workspace, cudaStream_t s) {
    double* part = static_cast<double*>(workspace);
    auto units = [&](uint32_t i) {
        return (numel[i] + kNormUnit - 1) / kNormUnit;
    };
    uint64_t all = 0;
    for (uint32_t i = 0; i < n_tensors; i++) all += units(i);
    const int grid = int(std::max<uint64_t>(
            1, std::min<uint64_t>(
                       all, std::min(kNormMost, sm_count() * kNormCtasPerSm))));
    ProfScope ps("grad_norm", s);
    uint32_t i = 0;
    int add = 0;
    auto run = [&](auto cap) {
        constexpr uint32_t kCap = decltype(cap)::value;
        NormTable<kCap> t;
        uint64_t blocks = 0;
        uint32_t k = 0;
        for (; i < n_tensors && k < kCap; i++, k++) {
            if (k > 0 && blocks + units(i) > kMostBlocks) break;
            t.p[k] = tensors[i];
            t.n[k] = numel[i];
            t.type[k] = uint8_t(dtypes[i]);
            t.first[k] = uint32_t(blocks);
            blocks += units(i);
        }
        t.first[k] = uint32_t(blocks);
        t.count = k;
        k_norm_parts<kCap><<<grid, kThreads, 0, s>>>(t, part, add);
        DRESSI_CUDA(cudaGetLastError());
        add = 1;
    };
    do {
        const uint32_t left = n_tensors - i;
        if (left <= 32) run(std::integral_constant<uint32_t, 32>());
        else if (left <= 192) run(std::integral_constant<uint32_t, 192>());
        else run(std::integral_constant<uint32_t, 1000>());
    } while (i < n_tensors);
    launch_early(k_norm_finish, dim3(1), kThreads, 0, s,
                 static_cast<const double*>(part), grid, out);
}

}  // namespace dressi
