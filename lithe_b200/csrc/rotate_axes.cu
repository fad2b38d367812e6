// Rotary positions with several axes, and the per-head RMS norm of q and k with that rotation
// in the same pass.
//
//   angle(token, pair p) = position(token, axis of p) * theta^(-2 i / d_axis),  i = p's index
//   inside its axis's slice of d_axis / 2 pairs; the axes' slices follow one another.
//   (a, b) -> (a cos - b sin, b cos + a sin) for pair p's two values: neighbours 2p, 2p + 1
//   ("interleaved") or p, p + R/2 ("halves"), R = sum of d_axis; values from R on stay.
//   With the norm: a, b are first x * rsqrt(mean(x^2) + eps) * weight over the head's dim.
//   Everything in fp32 (the angle's revolution count in fp64, so that far positions keep their
//   phase), one rounding at the store.
//
// Bound: HBM (each value read once and written once; about 3 to 10 operations a value).
// Split: a warp takes one token (and a run of its heads) at a time.  The lanes that share a
// head hold 8 of its values each, and hold the cosines and sines of their 4 pairs for all of
// the token's heads, so the angles cost one evaluation per token and not one per head; the
// sum of squares is a shuffle inside the lanes of a head.  kBatch heads are loaded before the
// first is used.
#include <cmath>

#include "device_common.cuh"
#include "host_common.h"

namespace lithe {
namespace ra {

constexpr int kMaxPairs = LITHE_MAX_HEAD_DIM / 2;
constexpr int kBatch = 4;          // heads a lane group loads before it uses the first
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
    int32_t group_log2;            // lanes that share a head
    int64_t units;                 // batch * tokens * chunks
    float eps;
    uint8_t axis[kMaxPairs];
    double turn[kMaxPairs];        // revolutions per unit of position
};

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};

// A lane's 8 values in their stored type: value 2i and 2i + 1 are pair i's.
template <typename T>
struct alignas(16) Eight {
    T v[8];
};

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

// kVec: the lane's values come as whole 16-byte (interleaved) or 8- / 16-byte (halves) pieces;
// else one by one, for strides, bases or slices that are not aligned to them.
template <typename T, bool kHalves, bool kVec>
__device__ __forceinline__ void load8(const Params& p, const T* head, int pair0, Eight<T>& e) {
    if constexpr (kVec && !kHalves) {
        const uint4* s = reinterpret_cast<const uint4*>(head + 2 * pair0);
        uint4* d = reinterpret_cast<uint4*>(&e);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) d[i] = s[i];
    } else if constexpr (kVec) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; };
        const Four a = *reinterpret_cast<const Four*>(head + first_of<true>(p, pair0));
        const Four b = *reinterpret_cast<const Four*>(head + second_of<true>(p, pair0));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e.v[2 * i] = a.v[i];
            e.v[2 * i + 1] = b.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = pair0 + i < (p.dim >> 1);
            e.v[2 * i] = in ? head[first_of<kHalves>(p, pair0 + i)] : Elem<T>::put(0.0f);
            e.v[2 * i + 1] = in ? head[second_of<kHalves>(p, pair0 + i)] : Elem<T>::put(0.0f);
        }
    }
}

template <typename T, bool kHalves, bool kVec>
__device__ __forceinline__ void store8(const Params& p, T* head, int pair0, const Eight<T>& e) {
    if constexpr (kVec && !kHalves) {
        uint4* d = reinterpret_cast<uint4*>(head + 2 * pair0);
        const uint4* s = reinterpret_cast<const uint4*>(&e);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) d[i] = s[i];
    } else if constexpr (kVec) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; };
        Four a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a.v[i] = e.v[2 * i];
            b.v[i] = e.v[2 * i + 1];
        }
        *reinterpret_cast<Four*>(head + first_of<true>(p, pair0)) = a;
        *reinterpret_cast<Four*>(head + second_of<true>(p, pair0)) = b;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (pair0 + i < (p.dim >> 1)) {
                head[first_of<kHalves>(p, pair0 + i)] = e.v[2 * i];
                head[second_of<kHalves>(p, pair0 + i)] = e.v[2 * i + 1];
            }
        }
    }
}

__device__ __forceinline__ double position_of(const Params& p, int64_t at) {
    if (p.pos_type == LITHE_POS_I32) return static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
    if (p.pos_type == LITHE_POS_I64) return static_cast<double>(static_cast<const int64_t*>(p.positions)[at]);
    return static_cast<double>(static_cast<const float*>(p.positions)[at]);
}

// One tensor's heads [h0, h1) of one token.  Every lane of the warp runs every iteration (the
// norm's shuffles need them); lanes without a head or without pairs load and store nothing.
template <typename T, bool kHalves, bool kVec, bool kNorm>
__device__ __forceinline__ void token_heads(const Params& p, const Heads& t, int64_t sample, int64_t token, int h0,
                                            int h1, int lane, int pair0, const float (&cs)[4], const float (&sn)[4],
                                            const float (&w)[8]) {
    const int group = 1 << p.group_log2;
    const int per_iter = 32 >> p.group_log2;
    const bool has_pairs = pair0 < (p.dim >> 1);
    const T* in = static_cast<const T*>(t.in) + sample * t.in_sample + token * t.in_token;
    T* out = static_cast<T*>(t.out) + sample * t.out_sample + token * t.out_token;
    const float inv_dim = 1.0f / static_cast<float>(p.dim);
    for (int h = h0 + (lane >> p.group_log2); __any_sync(0xffffffffu, h < h1); h += per_iter * kBatch) {
        Eight<T> e[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int hj = h + j * per_iter;
            if (has_pairs && hj < h1)
                load8<T, kHalves, kVec>(p, in + hj * t.in_head, pair0, e[j]);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) e[j].v[i] = Elem<T>::put(0.0f);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = Elem<T>::get(e[j].v[i]);
            if constexpr (kNorm) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
                for (int o = group >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float r = rsqrtf(fmaf(sum, inv_dim, p.eps));
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = x[2 * i], b = x[2 * i + 1];
                const bool turned = pair0 + i < (p.rotated >> 1);     // values that stay never meet the angle
                e[j].v[2 * i] = Elem<T>::put(turned ? a * cs[i] - b * sn[i] : a);
                e[j].v[2 * i + 1] = Elem<T>::put(turned ? b * cs[i] + a * sn[i] : b);
            }
            const int hj = h + j * per_iter;
            if (has_pairs && hj < h1) store8<T, kHalves, kVec>(p, out + hj * t.out_head, pair0, e[j]);
        }
    }
}

template <typename T, bool kHalves>
__device__ __forceinline__ void load_weight(const Params& p, const Heads& t, int pair0, float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float v = 1.0f;
            if (t.weight && pair0 + i < (p.dim >> 1)) {
                const int at = s ? second_of<kHalves>(p, pair0 + i) : first_of<kHalves>(p, pair0 + i);
                v = t.weight_f32 ? static_cast<const float*>(t.weight)[at]
                                 : Elem<T>::get(static_cast<const T*>(t.weight)[at]);
            }
            w[2 * i + s] = v;
        }
    }
}

template <typename T, bool kHalves, bool kVec, bool kNorm>
__global__ void __launch_bounds__(32 * kWarps) rotate_kernel(const __grid_constant__ Params p) {
    const int lane = threadIdx.x & 31;
    const int pair0 = 4 * (lane & ((1 << p.group_log2) - 1));
    double turn[4];
    int axis[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = pair0 + i < (p.rotated >> 1);
        turn[i] = in ? p.turn[pair0 + i] : 0.0;
        axis[i] = in ? p.axis[pair0 + i] : 0;
    }
    float w0[8], w1[8];
    if constexpr (kNorm) {
        load_weight<T, kHalves>(p, p.t[0], pair0, w0);
        load_weight<T, kHalves>(p, p.t[1], pair0, w1);
    }
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); u < p.units; u += warps) {
        const int64_t row = u / p.chunks;
        const int chunk = static_cast<int>(u - row * p.chunks);
        const int64_t sample = row / p.tokens, token = row - sample * p.tokens;
        float cs[4], sn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // revolutions in fp64, their fraction (at most half a turn) in fp32
            const double r = position_of(p, sample * p.pos_sample + token * p.axes + axis[i]) * turn[i];
            sincospif(static_cast<float>(2.0 * (r - rint(r))), &sn[i], &cs[i]);
        }
        int h0 = chunk * p.t[0].per_unit;
        token_heads<T, kHalves, kVec, kNorm>(p, p.t[0], sample, token, h0, min(h0 + p.t[0].per_unit, p.t[0].heads),
                                             lane, pair0, cs, sn, w0);
        if (p.tensors > 1) {
            h0 = chunk * p.t[1].per_unit;
            token_heads<T, kHalves, kVec, kNorm>(p, p.t[1], sample, token, h0,
                                                 min(h0 + p.t[1].per_unit, p.t[1].heads), lane, pair0, cs, sn, w1);
        }
    }
}

template <typename T, bool kHalves, bool kVec, bool kNorm>
int32_t launch(const Params& p, int sms, cudaStream_t st) {
    const int64_t blocks = (p.units + kWarps - 1) / kWarps;
    const int64_t most = static_cast<int64_t>(sms) * 8;
    rotate_kernel<T, kHalves, kVec, kNorm><<<static_cast<int>(blocks < most ? blocks : most), 32 * kWarps, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LITHE_OK : fail_cuda(e, "rotate_kernel launch");
}

template <typename T, bool kNorm>
int32_t launch_layout(const Params& p, bool halves, bool vec, int sms, cudaStream_t st) {
    if (halves) return vec ? launch<T, true, true, kNorm>(p, sms, st) : launch<T, true, false, kNorm>(p, sms, st);
    return vec ? launch<T, false, true, kNorm>(p, sms, st) : launch<T, false, false, kNorm>(p, sms, st);
}

// Whether a tensor's heads can be read and written in whole 16-byte pieces.
bool aligned(const Heads& t, int size) {
    const int64_t s = t.in_sample | t.in_token | t.in_head | t.out_sample | t.out_token | t.out_head;
    return reinterpret_cast<uintptr_t>(t.in) % 16 == 0 && reinterpret_cast<uintptr_t>(t.out) % 16 == 0 &&
           (s * size) % 16 == 0;
}

int32_t check_heads(const lithe_heads_view& v, const char* name, int32_t batch, int32_t tokens, int64_t* elements) {
    if (v.heads <= 0) return fail_arg("%s: heads must be positive, got %d", name, v.heads);
    if (!v.base) return fail_arg("%s must be non-NULL", name);
    if (v.sample_stride < 0 || v.token_stride < 0 || v.head_stride < 0)
        return fail_arg("%s: strides must not be negative", name);
    *elements = static_cast<int64_t>(batch) * tokens * v.heads;
    return LITHE_OK;
}

int32_t run(const lithe_heads_view* in, const lithe_heads_view* out, const void* const* weight, int tensors,
            bool norm, float eps, int32_t weight_dtype, int32_t dtype, int32_t batch, int32_t tokens, int32_t dim,
            const void* positions, int32_t pos_type, int32_t per_sample, const int32_t* axis_dims, int32_t n_axes,
            double theta, int32_t pairing, void* stream) {
    clear_error();
    if (dtype != LITHE_DTYPE_BF16 && dtype != LITHE_DTYPE_F16 && dtype != LITHE_DTYPE_F32)
        return fail_arg("dtype must be LITHE_DTYPE_BF16, _F16 or _F32, got %d", dtype);
    if (batch < 0 || tokens < 0) return fail_arg("batch and tokens must be >= 0 (%d, %d)", batch, tokens);
    if (dim <= 0 || dim % 2) return fail_arg("the head dim must be positive and even, got %d", dim);
    if (dim > LITHE_MAX_HEAD_DIM) return fail_unsupported("head dim %d above %d", dim, LITHE_MAX_HEAD_DIM);
    if (n_axes < 1 || n_axes > LITHE_MAX_AXES) return fail_arg("1 to %d axes, got %d", LITHE_MAX_AXES, n_axes);
    if (!axis_dims) return fail_arg("axis_dims must be non-NULL");
    if (!(theta > 0.0) || !std::isfinite(theta)) return fail_arg("theta must be positive and finite");
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
            p.turn[rotated / 2 + i] = std::pow(theta, -2.0 * i / d) / two_pi;
        }
        rotated += d;
    }
    const int size = dtype == LITHE_DTYPE_F32 ? 4 : 2;
    // Lanes that share a head: 4 pairs each, a power of two for the norm's shuffles.
    int lg = 0;
    while ((4 << lg) < dim / 2) ++lg;
    p.group_log2 = lg;
    p.tensors = tensors;
    // Pieces of 16 bytes need every stride, base and (pairs half a head apart) slice aligned to
    // them; the other form loads value by value.
    bool vec = dim % 8 == 0 && (pairing == LITHE_PAIR_INTERLEAVED || rotated % 8 == 0);
    int most_heads = 0;
    if (batch == 0 || tokens == 0) return LITHE_OK;
    if (!positions) return fail_arg("positions must be non-NULL");
    for (int i = 0; i < tensors; ++i) {
        int64_t n;
        int32_t rc = check_heads(in[i], i ? "k" : "x", batch, tokens, &n);
        if (rc == LITHE_OK) rc = check_heads(out[i], i ? "out_k" : "out", batch, tokens, &n);
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
    // A token's heads are split over warps while there are too few tokens to fill the SMs.
    const int per_iter = 32 >> lg;
    const int most_chunks = (most_heads + per_iter - 1) / per_iter;
    const int64_t rows = static_cast<int64_t>(batch) * tokens;
    int chunks = 1;
    while (chunks < most_chunks && rows * chunks < static_cast<int64_t>(sms) * 32) chunks *= 2;
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
                                     double theta, int32_t pairing, void* stream) {
    if (!x || !out) return lithe::fail_arg("x and out must be non-NULL");
    return lithe::ra::run(x, out, nullptr, 1, false, 0.0f, LITHE_DTYPE_F32, dtype, batch, tokens, dim, positions,
                          pos_type, per_sample, axis_dims, n_axes, theta, pairing, stream);
}

extern "C" int32_t lithe_qk_norm_rotate(const lithe_heads_view* q, const lithe_heads_view* k,
                                        const lithe_heads_view* out_q, const lithe_heads_view* out_k,
                                        const void* weight_q, const void* weight_k, int32_t weight_dtype, float eps,
                                        int32_t dtype, int32_t batch, int32_t tokens, int32_t dim,
                                        const void* positions, int32_t pos_type, int32_t per_sample,
                                        const int32_t* axis_dims, int32_t n_axes, double theta, int32_t pairing,
                                        void* stream) {
    if (!q || !k || !out_q || !out_k) return lithe::fail_arg("q, k, out_q and out_k must be non-NULL");
    const lithe_heads_view in[2] = {*q, *k}, out[2] = {*out_q, *out_k};
    const void* weight[2] = {weight_q, weight_k};
    return lithe::ra::run(in, out, weight, 2, true, eps, weight_dtype, dtype, batch, tokens, dim, positions, pos_type,
                          per_sample, axis_dims, n_axes, theta, pairing, stream);
}
