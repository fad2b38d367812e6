// Rotary positions with several axes, and the per-head RMS norm of q and k with that rotation
// in the same pass.
//
//   angle(token, pair p) = position(token, axis of p) * frequency(p); every axis has a slice of
//   d_axis / 2 pairs, the slices follow one another.
//   (a, b) -> (a cos - b sin, b cos + a sin) for pair p's two values: neighbours 2p, 2p + 1
//   ("interleaved") or p, p + R/2 ("halves"), R = sum of d_axis; values from R on stay.
//   With the norm: a, b are first x * rsqrt(mean(x^2) + eps) * weight over the head's dim.
//   Everything in fp32 (the angle in fp64 up to the fraction of its last turn, so that far positions
//   keep their phase), one rounding at the store.
//
// Bound: HBM (each value is read once and written once; about 3 to 7 operations a value), with the
// issue rate close behind: the first form, 19 instructions a value, took 380 us for 14 x 4096 tokens
// of 24 + 24 heads of 128 where 218 us move the bytes.
// Split: a warp takes one token (and a run of its heads) at a time.  The lanes that share a head hold
// 8 of its values each.  A token's cosines and sines are evaluated once, each pair's by one lane,
// handed round through shared memory, and (with the norm) multiplied by the weights once, so that a
// pair costs four products two at a time (f32x2), the norm's factor two more.  The sum of squares is
// a shuffle inside the lanes of a head.  kBatch heads are loaded before the first is used, the
// token's first ones before its angles.
// Measured on B200: 14 x 4096 tokens of 24 + 24 heads of 128, norm and rotation, 245 us (5.75 TB/s, 0.89 of
// the measured copy rate; 251 us back to back, at the 1 kW cap); 32760 tokens of 24 heads, rotation, 63 us
// (6.4 TB/s, 0.98); one token 2.9 us.
// A second batch of heads on its way while one is turned took registers that cost more (306 us).
#include <cmath>
#include <type_traits>

#include "device_common.cuh"
#include "host_common.h"

namespace lithe {
namespace ra {

constexpr int kMaxPairs = LITHE_MAX_HEAD_DIM / 2;
constexpr int kMostHeads = 1 << 30;            // the heads' arithmetic stays inside 32 bits
// heads a lane group loads before it uses the first: 64 bytes a lane (four heads of fp32 spill: 2767 x 4 tokens
// of 4 heads of 64, norm and rotation, 11.4 us, 8.4 us with two)
template <typename T, bool kVec>
constexpr int kBatch = sizeof(T) == 4 || !kVec ? 2 : 4;
constexpr int kMinBlocks = 4;      // CTAs that have to fit an SM (64 registers a thread)
constexpr int kWarps = 8;          // warps of a CTA

struct Heads {
    const void* in;
    void* out;
    const void* weight;            // (dim) or nullptr
    int64_t in_sample, in_token, in_head;      // strides, in elements
    int64_t out_sample, out_token, out_head;
    int32_t heads;
    int32_t per_unit;              // heads of one unit
    int32_t weight_f32;            // weight is fp32 (else the activations' type)
};

struct Params {
    Heads t[2];
    const void* positions;         // (tokens, axes) or (batch, tokens, axes)
    int64_t pos_sample;            // elements between samples' positions (0: shared)
    int32_t pos_type;              // LITHE_POS_*
    int32_t axes;
    int32_t tensors;
    int32_t tokens, dim, rotated;  // rotated = R
    int32_t chunks;                // units a token is split into
    int32_t group;                 // lanes that share a head
    int64_t units;                 // batch * tokens * chunks
    float eps, inv_dim;
    uint8_t axis[kMaxPairs];
    double turn[kMaxPairs];        // revolutions per unit of position
};

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 zero() { return __ushort_as_bfloat16(0); }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half zero() { return __ushort_as_half(0); }
};
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float zero() { return 0.0f; }
};

// A lane's 8 values in their stored type and order: interleaved, value 2i and 2i + 1 are pair i's; halves,
// values i and 4 + i.
template <typename T>
struct alignas(16) Eight {
    T v[8];
};

// Two fp32 values that one instruction computes on.
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float a, float b) {
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    }
    __device__ __forceinline__ void split(float& a, float& b) const {
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    }
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}

// The first and second values of a lane's four pairs, two pairs to an F2; and back, rounded.
template <typename T, bool kHalves>
__device__ __forceinline__ void unpack(const Eight<T>& e, F2 (&a)[2], F2 (&b)[2]) {
    float x[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = Elem<T>::get(e.v[i]);
    } else {
        constexpr bool kF16 = std::is_same<T, __half>::value;
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&e);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = Act<kF16>::lo(w[i]), x[2 * i + 1] = Act<kF16>::hi(w[i]);
    }
    constexpr int kStep = kHalves ? 1 : 2, kSecond = kHalves ? 4 : 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        a[i] = F2(x[2 * i * kStep], x[(2 * i + 1) * kStep]);
        b[i] = F2(x[2 * i * kStep + kSecond], x[(2 * i + 1) * kStep + kSecond]);
    }
}
template <typename T, bool kHalves>
__device__ __forceinline__ void pack(const F2 (&a)[2], const F2 (&b)[2], Eight<T>& e) {
    constexpr int kStep = kHalves ? 1 : 2, kSecond = kHalves ? 4 : 1;
    float x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        a[i].split(x[2 * i * kStep], x[(2 * i + 1) * kStep]);
        b[i].split(x[2 * i * kStep + kSecond], x[(2 * i + 1) * kStep + kSecond]);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e.v[i] = x[i];
    } else {
        constexpr bool kF16 = std::is_same<T, __half>::value;
        uint32_t* w = reinterpret_cast<uint32_t*>(&e);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = Act<kF16>::pack(x[2 * i], x[2 * i + 1]);
    }
}

// Offset inside a head of the first and second value of pair p (p < dim / 2).  Pairs from R/2 on
// are the values that stay, taken two and two.
template <bool kHalves>
__device__ __forceinline__ int first_of(const Params& p, int pair) {
    if (!kHalves) return 2 * pair;
    const int h = p.rotated >> 1;
    return pair < h ? pair : pair + h;
}
template <bool kHalves>
__device__ __forceinline__ int second_of(const Params& p, int pair) {
    if (!kHalves) return 2 * pair + 1;
    const int h = p.rotated >> 1;
    return pair < h ? pair + h : pair + (p.dim >> 1);
}

// kVec: the lane's values come as whole 16-byte (interleaved) or 8- / 16-byte (halves) pieces, at first
// and (halves) second, and its pairs are neighbours; else one by one, for strides, bases or slices that are
// not aligned to them, and its pairs are as many apart as lanes share the head, so that the lanes' values
// are neighbours (5 x 5295 tokens of 32 heads of 32 in fp32, halves of 9: 62 us; 281 us with neighbouring
// pairs and 32 lanes to every head).
template <bool kVec, int kGroup>
__device__ __forceinline__ int pair_of(int lane, int i) {
    return kVec ? 4 * lane + i : lane + kGroup * i;
}

template <typename T, bool kHalves, bool kVec, int kGroup>
__device__ __forceinline__ void load8(const Params& p, const T* head, int lane, int first, int second, Eight<T>& e) {
    if constexpr (kVec && !kHalves) {
        const uint4* s = reinterpret_cast<const uint4*>(head + first);
        uint4* d = reinterpret_cast<uint4*>(&e);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) d[i] = s[i];
    } else if constexpr (kVec) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; };
        reinterpret_cast<Four*>(&e)[0] = *reinterpret_cast<const Four*>(head + first);
        reinterpret_cast<Four*>(&e)[1] = *reinterpret_cast<const Four*>(head + second);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pair = pair_of<kVec, kGroup>(lane, i);
            const bool in = pair < (p.dim >> 1);
            e.v[kHalves ? i : 2 * i] = in ? head[first_of<kHalves>(p, pair)] : Elem<T>::zero();
            e.v[kHalves ? 4 + i : 2 * i + 1] = in ? head[second_of<kHalves>(p, pair)] : Elem<T>::zero();
        }
    }
}

template <typename T, bool kHalves, bool kVec, int kGroup>
__device__ __forceinline__ void store8(const Params& p, T* head, int lane, int first, int second, const Eight<T>& e) {
    if constexpr (kVec && !kHalves) {
        uint4* d = reinterpret_cast<uint4*>(head + first);
        const uint4* s = reinterpret_cast<const uint4*>(&e);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) d[i] = s[i];
    } else if constexpr (kVec) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; };
        *reinterpret_cast<Four*>(head + first) = reinterpret_cast<const Four*>(&e)[0];
        *reinterpret_cast<Four*>(head + second) = reinterpret_cast<const Four*>(&e)[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pair = pair_of<kVec, kGroup>(lane, i);
            if (pair < (p.dim >> 1)) {
                head[first_of<kHalves>(p, pair)] = e.v[kHalves ? i : 2 * i];
                head[second_of<kHalves>(p, pair)] = e.v[kHalves ? 4 + i : 2 * i + 1];
            }
        }
    }
}

__device__ __forceinline__ double position_of(const Params& p, int64_t at) {
    if (p.pos_type == LITHE_POS_I32) return static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
    if (p.pos_type == LITHE_POS_I64) return static_cast<double>(static_cast<const int64_t*>(p.positions)[at]);
    return static_cast<double>(static_cast<const float*>(p.positions)[at]);
}

// The matrix of each of a lane's pairs, (a, b) -> (aa a - ab b, bb b + ba a): cosine and sine, and with
// the norm the weights of its two values, whose products are taken once per token.
struct Turn {
    F2 aa[2], ab[2], bb[2], ba[2];             // (ab negated)
    uint32_t stay;                             // bit i: no axis turns the lane's pair i
};

// With whole pieces of halves a lane's pairs all stay or all turn (R / 2 is a multiple of 4).
template <bool kHalves, bool kVec>
__device__ __forceinline__ bool stays(uint32_t stay, int i) {
    return kHalves && kVec ? (stay & 1) != 0 : (stay >> i & 1) != 0;
}

// A lane's part of the heads that a warp has loaded: kBatch heads, 32 / kGroup apart, from the lane's own on.
// live: how many heads there are from it on (none for a lane without pairs); the others load zeros and store
// nothing, but take part in the norm's shuffles.
template <typename T, bool kVec>
struct Batch {
    Eight<T> e[kBatch<T, kVec>];
};

template <typename T, bool kHalves, bool kVec, int kGroup>
__device__ __forceinline__ void load_batch(const Params& p, const T* in, int64_t step, int lane, int first, int second,
                                           int live, Batch<T, kVec>& b) {
    const int per_iter = 32 / kGroup;
#pragma unroll
    for (int j = 0; j < kBatch<T, kVec>; ++j) {
        if (j * per_iter < live)
            load8<T, kHalves, kVec, kGroup>(p, in + j * step, lane, first, second, b.e[j]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) b.e[j].v[i] = Elem<T>::zero();
    }
}

// kWhole: every value of a head is turned; else the values that stay never meet an angle.
template <typename T, bool kHalves, bool kVec, bool kNorm, bool kWhole, int kGroup>
__device__ __forceinline__ void turn_batch(const Params& p, T* out, int64_t step, int lane, int first, int second,
                                           int live, const Turn& m, Batch<T, kVec>& b) {
    const int per_iter = 32 / kGroup;
#pragma unroll
    for (int j = 0; j < kBatch<T, kVec>; ++j) {
        F2 x[2], y[2];
        unpack<T, kHalves>(b.e[j], x, y);
        float r = 1.0f;
        if constexpr (kNorm) {
            F2 sum2 = mul2(x[0], x[0]);
            sum2 = fma2(x[1], x[1], sum2);
            sum2 = fma2(y[0], y[0], sum2);
            sum2 = fma2(y[1], y[1], sum2);
            float s0, s1;
            sum2.split(s0, s1);
            float sum = s0 + s1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
                if (o < kGroup) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float mean = fmaf(sum, p.inv_dim, p.eps);
            r = rsqrtf(mean);
        }
        const F2 rr(r, r);
        F2 u[2], v[2], xc[2] = {x[0], x[1]}, yc[2] = {y[0], y[1]};
        if constexpr (!kWhole) {
            // pairs that stay: their values do not meet (a product with a zero sine would carry a NaN or an
            // infinity across)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float a0, a1, b0, b1;
                xc[i].split(a0, a1), yc[i].split(b0, b1);
                const bool s0 = stays<kHalves, kVec>(m.stay, 2 * i), s1 = stays<kHalves, kVec>(m.stay, 2 * i + 1);
                xc[i] = F2(s0 ? 0.0f : a0, s1 ? 0.0f : a1), yc[i] = F2(s0 ? 0.0f : b0, s1 ? 0.0f : b1);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u[i] = fma2(x[i], m.aa[i], mul2(yc[i], m.ab[i]));
            v[i] = fma2(y[i], m.bb[i], mul2(xc[i], m.ba[i]));
            if constexpr (kNorm) u[i] = mul2(u[i], rr), v[i] = mul2(v[i], rr);
        }
        if constexpr (kWhole || kNorm) {
            pack<T, kHalves>(u, v, b.e[j]);
        } else {
            // (without the norm not touched at all)
            Eight<T> turned;
            pack<T, kHalves>(u, v, turned);
            constexpr int kA = kHalves ? 1 : 2, kB = kHalves ? 4 : 1;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!stays<kHalves, kVec>(m.stay, i)) {
                    b.e[j].v[kA * i] = turned.v[kA * i];
                    b.e[j].v[kA * i + kB] = turned.v[kA * i + kB];
                }
        }
        if (j * per_iter < live) store8<T, kHalves, kVec, kGroup>(p, out + j * step, lane, first, second, b.e[j]);
    }
}

// What every unit needs, laid out by pair once per CTA: revolutions per unit of position and axis, the
// norms' weights of the pair's two values, and a warp's cosines and sines of its token.
struct alignas(16) Tables {
    double turn[kMaxPairs];
    float weight[2][2][kMaxPairs];             // [tensor][first, second][pair]
    float2 angle[kWarps][kMaxPairs];
    int32_t axis[kMaxPairs];
};

template <typename T, bool kHalves, bool kNorm>
__device__ __forceinline__ void fill_tables(const Params& p, Tables& tab) {
    for (int pair = threadIdx.x; pair < kMaxPairs; pair += 32 * kWarps) {
        const bool turned = pair < (p.rotated >> 1), in = pair < (p.dim >> 1);
        tab.turn[pair] = turned ? p.turn[pair] : 0.0;
        tab.axis[pair] = turned ? p.axis[pair] : 0;
        if constexpr (kNorm) {
            for (int t = 0; t < p.tensors; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v = 1.0f;
                    if (p.t[t].weight && in) {
                        const int at = e ? second_of<kHalves>(p, pair) : first_of<kHalves>(p, pair);
                        v = p.t[t].weight_f32 ? __ldg(static_cast<const float*>(p.t[t].weight) + at)
                                              : Elem<T>::get(__ldg(static_cast<const T*>(p.t[t].weight) + at));
                    }
                    tab.weight[t][e][pair] = v;
                }
        }
    }
    __syncthreads();
}

template <typename T, bool kHalves, bool kVec, bool kNorm, bool kWhole, int kGroup>
__global__ void __launch_bounds__(32 * kWarps, kMinBlocks) rotate_kernel(const __grid_constant__ Params p) {
    const int lane = threadIdx.x & 31, part = lane & (kGroup - 1), sub = lane / kGroup;
    const int pair0 = pair_of<kVec, kGroup>(part, 0);
    const bool has_pairs = pair0 < (p.dim >> 1);
    const int first = has_pairs ? first_of<kHalves>(p, pair0) : 0, second = has_pairs ? second_of<kHalves>(p, pair0) : 0;
    const int per_iter = 32 / kGroup;
    __shared__ Tables tab;
    fill_tables<T, kHalves, kNorm>(p, tab);
    float2* angle = tab.angle[threadIdx.x >> 5];
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); u < p.units; u += warps) {
        const int64_t row = u / p.chunks;
        const int chunk = static_cast<int>(u - row * p.chunks);
        const int64_t sample = row / p.tokens, token = row - sample * p.tokens;
        Batch<T, kVec> b;
        int h = chunk * p.t[0].per_unit;
        {
            const Heads& t = p.t[0];
            const int live = has_pairs ? min(h + t.per_unit, t.heads) - h - sub : 0;
            load_batch<T, kHalves, kVec, kGroup>(
                p, static_cast<const T*>(t.in) + sample * t.in_sample + token * t.in_token + (h + sub) * t.in_head,
                per_iter * t.in_head, part, first, second, live, b);
        }
        // revolutions in fp64; their fraction f, in half turns, as an fp32 number and what is left of it, an angle
        // of at most 2^-25 pi whose sine and cosine are itself and 1 (to 1e-14): the values are within 1.5 units in
        // their last place, near zero too, where f alone in fp32 would leave 2^-26 pi.  Each pair's by one lane
        __syncwarp();
        for (int pair = lane; pair < (4 * kGroup); pair += 32) {
            float2 a = make_float2(1.0f, 0.0f);
            if (pair < (p.rotated >> 1)) {
                const double r =
                    position_of(p, sample * p.pos_sample + token * p.axes + tab.axis[pair]) * tab.turn[pair];
                const double f = 2.0 * (r - rint(r));
                const float near = static_cast<float>(f);
                const float rest = static_cast<float>(f - near) * 3.14159265f;
                float s, c;
                sincospif(near, &s, &c);
                a = make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
            }
            angle[pair] = a;
        }
        __syncwarp();
        float cs[4], sn[4];
        if constexpr (kVec) {
            const float4 a01 = *reinterpret_cast<const float4*>(&angle[pair0]);
            const float4 a23 = *reinterpret_cast<const float4*>(&angle[pair0 + 2]);
            cs[0] = a01.x, cs[1] = a01.z, cs[2] = a23.x, cs[3] = a23.z;
            sn[0] = a01.y, sn[1] = a01.w, sn[2] = a23.y, sn[3] = a23.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) cs[i] = angle[pair_of<kVec, kGroup>(part, i)].x, sn[i] = angle[pair_of<kVec, kGroup>(part, i)].y;
        }
        uint32_t stay = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) stay |= (pair_of<kVec, kGroup>(part, i) >= (p.rotated >> 1) ? 1u : 0u) << i;
#pragma unroll 1
        for (int k = 0; k < p.tensors; ++k) {
            const Heads& t = p.t[k];
            Turn m;
            m.stay = stay;
            float w[2][4] = {{1.0f, 1.0f, 1.0f, 1.0f}, {1.0f, 1.0f, 1.0f, 1.0f}};
            if constexpr (kNorm && kVec) {
                *reinterpret_cast<float4*>(w[0]) = *reinterpret_cast<const float4*>(&tab.weight[k][0][pair0]);
                *reinterpret_cast<float4*>(w[1]) = *reinterpret_cast<const float4*>(&tab.weight[k][1][pair0]);
            } else if constexpr (kNorm) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[0][i] = tab.weight[k][0][pair_of<kVec, kGroup>(part, i)], w[1][i] = tab.weight[k][1][pair_of<kVec, kGroup>(part, i)];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = 2 * i;
                m.aa[i] = F2(cs[j] * w[0][j], cs[j + 1] * w[0][j + 1]), m.ab[i] = F2(-sn[j] * w[1][j], -sn[j + 1] * w[1][j + 1]);
                m.bb[i] = F2(cs[j] * w[1][j], cs[j + 1] * w[1][j + 1]), m.ba[i] = F2(sn[j] * w[0][j], sn[j + 1] * w[0][j + 1]);
            }
            h = chunk * t.per_unit;
            const int end = min(h + t.per_unit, t.heads);
            const T* in = static_cast<const T*>(t.in) + sample * t.in_sample + token * t.in_token + (h + sub) * t.in_head;
            T* out = static_cast<T*>(t.out) + sample * t.out_sample + token * t.out_token + (h + sub) * t.out_head;
            for (; h < end; h += per_iter * kBatch<T, kVec>) {
                const int live = has_pairs ? end - h - sub : 0;
                if (k > 0 || h > chunk * t.per_unit)
                    load_batch<T, kHalves, kVec, kGroup>(p, in, per_iter * t.in_head, part, first, second, live, b);
                turn_batch<T, kHalves, kVec, kNorm, kWhole, kGroup>(p, out, per_iter * t.out_head, part, first, second, live, m, b);
                in += kBatch<T, kVec> * per_iter * t.in_head;
                out += kBatch<T, kVec> * per_iter * t.out_head;
            }
        }
    }
}

template <typename T, bool kHalves, bool kVec, bool kNorm, bool kWhole, int kGroup>
int32_t launch(const Params& p, int sms, cudaStream_t st) {
    const int64_t blocks = (p.units + kWarps - 1) / kWarps;
    // (the rotation alone: four CTAs to a place, 126 us against 144 us for 14 x 4608 tokens; with the norm, whose
    // tables a CTA lays out at its start, one: 246 us against 249 us for 14 x 4096)
    const int64_t most = static_cast<int64_t>(sms) * kMinBlocks * (kNorm ? 1 : 4);
    rotate_kernel<T, kHalves, kVec, kNorm, kWhole, kGroup>
        <<<static_cast<int>(blocks < most ? blocks : most), 32 * kWarps, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LITHE_OK : fail_cuda(e, "rotate_kernel launch");
}

// The lanes of a head are a compile-time number: 8, 16 or 32 (with the norm 252 us for 14 x 4096 tokens against
// 276 us with a run-time one, both at the power cap).
template <typename T, bool kHalves, bool kVec, bool kNorm, bool kWhole>
int32_t launch_group(const Params& p, int sms, cudaStream_t st) {
    if (p.group == 8) return launch<T, kHalves, kVec, kNorm, kWhole, 8>(p, sms, st);
    if (p.group == 16) return launch<T, kHalves, kVec, kNorm, kWhole, 16>(p, sms, st);
    return launch<T, kHalves, kVec, kNorm, kWhole, 32>(p, sms, st);
}

template <typename T, bool kNorm, bool kHalves>
int32_t launch_vec(const Params& p, bool vec, int sms, cudaStream_t st) {
    if (!vec) return launch_group<T, kHalves, false, kNorm, false>(p, sms, st);
    return p.rotated == p.dim ? launch_group<T, kHalves, true, kNorm, true>(p, sms, st)
                              : launch_group<T, kHalves, true, kNorm, false>(p, sms, st);
}

template <typename T, bool kNorm>
int32_t launch_layout(const Params& p, bool halves, bool vec, int sms, cudaStream_t st) {
    return halves ? launch_vec<T, kNorm, true>(p, vec, sms, st) : launch_vec<T, kNorm, false>(p, vec, sms, st);
}

// Whether a tensor's heads can be read and written in whole 16-byte pieces.
bool aligned(const Heads& t, int size) {
    const int64_t s = t.in_sample | t.in_token | t.in_head | t.out_sample | t.out_token | t.out_head;
    return reinterpret_cast<uintptr_t>(t.in) % 16 == 0 && reinterpret_cast<uintptr_t>(t.out) % 16 == 0 &&
           (s * size) % 16 == 0;
}

int32_t check_heads(const lithe_heads_view& v, const char* name) {
    if (v.heads <= 0) return fail_arg("%s: heads must be positive, got %d", name, v.heads);
    if (v.heads > kMostHeads) return fail_unsupported("%s: %d heads above %d", name, v.heads, kMostHeads);
    if (!v.base) return fail_arg("%s must be non-NULL", name);
    if (v.sample_stride < 0 || v.token_stride < 0 || v.head_stride < 0)
        return fail_arg("%s: strides must not be negative", name);
    return LITHE_OK;
}

int32_t run(const lithe_heads_view* in, const lithe_heads_view* out, const void* const* weight, int tensors,
            bool norm, float eps, int32_t weight_dtype, int32_t dtype, int32_t batch, int32_t tokens, int32_t dim,
            const void* positions, int32_t pos_type, int32_t per_sample, const int32_t* axis_dims, int32_t n_axes,
            const double* frequencies, int32_t pairing, void* stream) {
    clear_error();
    if (dtype != LITHE_DTYPE_BF16 && dtype != LITHE_DTYPE_F16 && dtype != LITHE_DTYPE_F32)
        return fail_arg("dtype must be LITHE_DTYPE_BF16, _F16 or _F32, got %d", dtype);
    if (batch < 0 || tokens < 0) return fail_arg("batch and tokens must be >= 0 (%d, %d)", batch, tokens);
    if (dim <= 0 || dim % 2) return fail_arg("the head dim must be positive and even, got %d", dim);
    if (dim > LITHE_MAX_HEAD_DIM) return fail_unsupported("head dim %d above %d", dim, LITHE_MAX_HEAD_DIM);
    if (n_axes < 1 || n_axes > LITHE_MAX_AXES) return fail_arg("1 to %d axes, got %d", LITHE_MAX_AXES, n_axes);
    if (!axis_dims || !frequencies) return fail_arg("axis_dims and frequencies must be non-NULL");
    if (pairing != LITHE_PAIR_INTERLEAVED && pairing != LITHE_PAIR_HALVES)
        return fail_arg("pairing must be LITHE_PAIR_INTERLEAVED or LITHE_PAIR_HALVES, got %d", pairing);
    if (pos_type != LITHE_POS_I32 && pos_type != LITHE_POS_I64 && pos_type != LITHE_POS_F32)
        return fail_arg("pos_type must be LITHE_POS_I32, _I64 or _F32, got %d", pos_type);
    if (norm && !(eps >= 0.0f)) return fail_arg("eps must be >= 0");
    if (norm && weight_dtype != dtype && weight_dtype != LITHE_DTYPE_F32)
        return fail_arg("the norms' weights have the activations' type or fp32");
    Params p{};
    int rotated = 0;
    const double two_pi = 6.283185307179586476925286766559;
    for (int a = 0; a < n_axes; ++a) {
        const int d = axis_dims[a];
        if (d < 0 || d % 2 || d > dim - rotated)
            return fail_arg("the axes' dims must be even, not negative and sum to at most the head dim %d (axis %d: %d)",
                            dim, a, d);
        for (int i = 0; i < d / 2; ++i) {
            p.axis[rotated / 2 + i] = static_cast<uint8_t>(a);
            const double f = frequencies[rotated / 2 + i];
            if (!std::isfinite(f)) return fail_arg("frequency %d is not finite", rotated / 2 + i);
            p.turn[rotated / 2 + i] = f / two_pi;
        }
        rotated += d;
    }
    const int size = dtype == LITHE_DTYPE_F32 ? 4 : 2;
    p.tensors = tensors;
    // Pieces of 16 bytes need every stride, base and (pairs half a head apart) slice aligned to
    // them; the other form loads value by value.
    bool vec = dim % 8 == 0 && (pairing == LITHE_PAIR_INTERLEAVED || rotated % 8 == 0);
    int most_heads = 0;
    if (batch == 0 || tokens == 0) return LITHE_OK;
    if (!positions) return fail_arg("positions must be non-NULL");
    for (int i = 0; i < tensors; ++i) {
        int32_t rc = check_heads(in[i], i ? "k" : "x");
        if (rc == LITHE_OK) rc = check_heads(out[i], i ? "out_k" : "out");
        if (rc != LITHE_OK) return rc;
        if (in[i].heads != out[i].heads) return fail_arg("an output's heads differ from its input's");
        Heads& t = p.t[i];
        t.in = in[i].base;
        t.out = const_cast<void*>(out[i].base);
        t.weight = weight ? weight[i] : nullptr;
        t.weight_f32 = weight_dtype == LITHE_DTYPE_F32;
        t.in_sample = in[i].sample_stride, t.in_token = in[i].token_stride, t.in_head = in[i].head_stride;
        t.out_sample = out[i].sample_stride, t.out_token = out[i].token_stride, t.out_head = out[i].head_stride;
        t.heads = in[i].heads;
        if (reinterpret_cast<uintptr_t>(t.in) % size || reinterpret_cast<uintptr_t>(t.out) % size)
            return fail_arg("a tensor is not aligned to its element size");
        vec = vec && aligned(t, size);
        most_heads = t.heads > most_heads ? t.heads : most_heads;
    }
    int device = 0, sms = 0;
    const int32_t rc = current_device_sms(&device, &sms);
    if (rc != LITHE_OK) return rc;
    p.positions = positions;
    p.pos_type = pos_type;
    p.axes = n_axes;
    p.pos_sample = per_sample ? static_cast<int64_t>(tokens) * n_axes : 0;
    p.tokens = tokens;
    p.dim = dim;
    p.rotated = rotated;
    p.eps = eps;
    p.inv_dim = 1.0f / static_cast<float>(dim);
    // A token's heads are split over warps while that leaves the SMs room: more units than resident
    // warps pay their angles for nothing (1024 tokens of 24 heads: 5.9 us on 4 chunks, 13 us on 8).
    // Lanes that share a head: 4 pairs each, a power of two for the norm's shuffles.
    p.group = dim > 128 ? 32 : dim > 64 ? 16 : 8;
    const int per_iter = 32 / p.group;
    const int most_chunks = (most_heads + per_iter - 1) / per_iter;
    const int64_t rows = static_cast<int64_t>(batch) * tokens;
    int chunks = 1;
    while (chunks < most_chunks && rows * chunks * 2 <= static_cast<int64_t>(sms) * kMinBlocks * kWarps) chunks *= 2;
    chunks = chunks < most_chunks ? chunks : most_chunks;
    for (int i = 0; i < tensors; ++i) {
        const int per = (p.t[i].heads + chunks - 1) / chunks;
        p.t[i].per_unit = (per + per_iter - 1) / per_iter * per_iter;
    }
    p.chunks = chunks;
    p.units = rows * chunks;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool halves = pairing == LITHE_PAIR_HALVES;
    if (norm) {
        if (dtype == LITHE_DTYPE_BF16) return launch_layout<__nv_bfloat16, true>(p, halves, vec, sms, st);
        if (dtype == LITHE_DTYPE_F16) return launch_layout<__half, true>(p, halves, vec, sms, st);
        return launch_layout<float, true>(p, halves, vec, sms, st);
    }
    if (dtype == LITHE_DTYPE_BF16) return launch_layout<__nv_bfloat16, false>(p, halves, vec, sms, st);
    if (dtype == LITHE_DTYPE_F16) return launch_layout<__half, false>(p, halves, vec, sms, st);
    return launch_layout<float, false>(p, halves, vec, sms, st);
}

}  // namespace ra
}  // namespace lithe

extern "C" int32_t lithe_rotate_axes(const lithe_heads_view* x, const lithe_heads_view* out, int32_t dtype,
                                     int32_t batch, int32_t tokens, int32_t dim, const void* positions,
                                     int32_t pos_type, int32_t per_sample, const int32_t* axis_dims, int32_t n_axes,
                                     const double* frequencies, int32_t pairing, void* stream) {
    if (!x || !out) return lithe::fail_arg("x and out must be non-NULL");
    return lithe::ra::run(x, out, nullptr, 1, false, 0.0f, LITHE_DTYPE_F32, dtype, batch, tokens, dim, positions,
                          pos_type, per_sample, axis_dims, n_axes, frequencies, pairing, stream);
}

extern "C" int32_t lithe_qk_norm_rotate(const lithe_heads_view* q, const lithe_heads_view* k,
                                        const lithe_heads_view* out_q, const lithe_heads_view* out_k,
                                        const void* weight_q, const void* weight_k, int32_t weight_dtype, float eps,
                                        int32_t dtype, int32_t batch, int32_t tokens, int32_t dim,
                                        const void* positions, int32_t pos_type, int32_t per_sample,
                                        const int32_t* axis_dims, int32_t n_axes, const double* frequencies,
                                        int32_t pairing, void* stream) {
    if (!q || !k || !out_q || !out_k) return lithe::fail_arg("q, k, out_q and out_k must be non-NULL");
    const lithe_heads_view in[2] = {*q, *k}, out[2] = {*out_q, *out_k};
    const void* weight[2] = {weight_q, weight_k};
    return lithe::ra::run(in, out, weight, 2, true, eps, weight_dtype, dtype, batch, tokens, dim, positions, pos_type,
                          per_sample, axis_dims, n_axes, frequencies, pairing, stream);
}
