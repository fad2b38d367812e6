// 8-bit integer linear: activations quantised per token, weights per output channel, the
// adapters' rank-16 expand added before the one rounding.
//
//   s_r = max_k |x[r, k]| / 127,  q[r, k] = x[r, k] * 127 / max_k |x[r, k]| to the nearest whole
//   number, ties to even                                              (lithe_quantize_rows)
//   out[r, n] = (sum_k q[r, k] w[n, k]) s_r s_n + bias[n] + sum_j h[r, j] b_dec[sample(r), n, j]
//                                                                     (lithe_int8_linear)
//   The products are summed exactly in int32 (k <= 131072), everything after in fp32.
#include "device_common.cuh"
#include "host_common.h"
#include "tcgen05.cuh"

namespace lithe {
namespace i8 {

constexpr int kRank = 16;              // rank of the fused expand
constexpr int kMaxK = 131072;          // 127 * 127 * kMaxK < 2^31
constexpr int kMostRows = 0x7fffffff - 1024;   // rows and channels of whole tiles stay inside 32 bits

// ------------------------------------------------------------------------------------------
// lithe_quantize_rows
//
// q is the exact quotient's rounding: with r = 127 / max and t = x r in fp32, t is within
// 2^-23 |t| of x 127 / max.  The quotient of two values of at most 11 bits is either exactly
// halfway between two whole numbers or at least 2^-19 |t| away from it (its distance is a whole
// number over 2 max's mantissa, 254 of x's mantissa times smaller than |t| at most).  So a t
// within 2^-21 |t| of halfway is a tie, which goes to the even number, and any other t rounds
// as the quotient does.
//
// Bound: HBM (x read once, a byte a value written).  kWarps warps take a row, each lane up to kPieces
// 8-value pieces of it, which stay in registers between the maximum and the rounding: one warp where
// there are many rows (57344 x 3072: 80 us, 6.6 TB/s; four a row 102 us), four where there are few and
// their latency counts (one row 1.8 us; 3.0 us).  A longer row is read twice, the second time from L2
// (20000 x 18432: 216 us, 5.1 TB/s).  Rows that do not start on 16-byte boundaries are put together out of
// aligned pieces (15488 x 5591: 77 us, 102 us with both granules of a piece loaded by its lane; 20000 x 1001:
// 18 us, value by value 29 us; 1237 x 1898: 4.0 and 6.1 us).
// The quotients of a piece are checked for nearness to halfway together, with a bound (2^-13) above every
// 2^-21 |t|; the few pieces it stops are done value by value.
// ------------------------------------------------------------------------------------------
constexpr int kThreadsQ = 128;

template <bool kF16>
__device__ __forceinline__ float value_of(uint32_t bits) {
    if (kF16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
    return __uint_as_float(bits << 16);
}

constexpr float kMagic = 12582912.0f;          // 1.5 * 2^23: adding it rounds to a whole number, ties to even

// Low byte: q of the value x of a row with r = 127 / max (x and r both scaled to keep r finite).
__device__ __forceinline__ uint32_t quantize(float x, float r) {
    const float t = x * r;
    const float s = t + kMagic;
    const float d = fabsf(t - (s - kMagic));
    if (d > fmaf(fabsf(t), -0x1p-21f, 0.5f)) return 2u * __float_as_uint(fmaf(t, 0.5f, kMagic));
    return __float_as_uint(s);
}

// The row's scale (written by one thread) and the two factors of a value's quotient.  A row with
// an infinity or NaN gets scale NaN (its outputs are NaN) and zeros.
template <bool kF16>
__device__ __forceinline__ void row_factors(uint32_t max_bits, bool write, float* scale, float& pre, float& r) {
    const float most = value_of<kF16>(max_bits);
    const bool finite = max_bits < (kF16 ? 0x7c00u : 0x7f80u);
    pre = 1.0f;
    r = 0.0f;
    if (finite && most > 0.0f) {
        if (most < 0x1p-64f) pre = 0x1p+64f;          // keeps 127 / max finite
        r = __fdiv_rn(127.0f, most * pre);
    }
    if (write) *scale = finite ? __fdiv_rn(most, 127.0f) : __uint_as_float(0x7fffffffu);
    if (!finite) pre = 0.0f;
}

struct QuantParams {
    const uint16_t* x;
    int8_t* q;
    float* scale;
    int64_t x_stride, q_stride;
    int32_t rows, k;
};

// Eight values to eight bytes.
template <bool kF16>
__device__ __forceinline__ uint2 quantize8(const uint4& v, float pre, float r) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t b[8];
    float near = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = value_of<kF16>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu) * r;
        const float s = t + kMagic;
        near = fmaxf(near, fabsf(t - (s - kMagic)));
        b[i] = __float_as_uint(s);
    }
    if (near > 0.5f - 0x1p-13f || pre != 1.0f) {       // (pre: rows of values below 2^-64)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            b[i] = quantize(value_of<kF16>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu) * pre, r);
    }
    const uint32_t a0 = __byte_perm(b[0], b[1], 0x0040), a1 = __byte_perm(b[2], b[3], 0x0040);
    const uint32_t a2 = __byte_perm(b[4], b[5], 0x0040), a3 = __byte_perm(b[6], b[7], 0x0040);
    return make_uint2(__byte_perm(a0, a1, 0x5410), __byte_perm(a2, a3, 0x5410));
}

__device__ __forceinline__ uint32_t max_of(uint32_t m, const uint4& v) {
    return __vmaxu2(__vmaxu2(m, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)),
                    __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
}

// A lane's kPieces pieces of a row of k values, piece `at` being the values 8 at to 8 at + 7, zeros from k on.
// kWhole: rows are whole pieces on 16-byte boundaries.  Else a piece is shifted together out of two of the
// 16-byte granules that the row lies in, one the lane's own and one its neighbour's: a warp holds 32 kPieces
// granules in a row and the one behind them (lane 31).  The granules that reach beyond the row are read value
// by value, after the others have been loaded.
template <bool kWhole, int kPieces>
struct Pieces {
    uint4 g[kPieces];
    uint4 behind;
    int shift;

    // The lane's piece c: row pieces `first` on, kLanes lanes side by side.
    template <int kLanes>
    static __device__ __forceinline__ int at(int first, int c) {
        if constexpr (kWhole) return first + c * kLanes + static_cast<int>(threadIdx.x) % kLanes;
        const int t = static_cast<int>(threadIdx.x) % kLanes;
        return first + (t / 32 * kPieces + c) * 32 + t % 32;
    }

    static __device__ __forceinline__ uint4 edge(const uint16_t* row, int value, int k) {
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = value + i >= 0 && value + i < k ? __ldg(row + value + i) : 0u;
        return make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
    }

    template <int kLanes>
    __device__ __forceinline__ void load(const uint16_t* row, int first, int k) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        shift = kWhole ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 7;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int value = 8 * at<kLanes>(first, c) - shift;
            g[c] = value >= 0 && value + 8 <= k ? __ldg(reinterpret_cast<const uint4*>(row + value)) : zero;
        }
        if constexpr (!kWhole) {
            const int next = 8 * (at<kLanes>(first, kPieces - 1) + 1) - shift;
            const bool last = (threadIdx.x & 31) == 31;
            behind = last && next >= 0 && next + 8 <= k ? __ldg(reinterpret_cast<const uint4*>(row + next)) : zero;
#pragma unroll
            for (int c = 0; c < kPieces; ++c) {
                const int value = 8 * at<kLanes>(first, c) - shift;
                if (value < k && (value < 0 || value + 8 > k)) g[c] = edge(row, value, k);
            }
            if (last && next < k && next + 8 > k) behind = edge(row, next, k);
        }
    }

    __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
        for (int c = 0; c < kPieces; ++c) m = max_of(m, g[c]);
        return kWhole ? m : max_of(m, behind);
    }

    // The lane's piece c, in the order of c; every lane of the warp takes part.
    __device__ __forceinline__ uint4 piece(int c) {
        if constexpr (kWhole) return g[c];
        const int lane = threadIdx.x & 31;
        // lane 31's neighbour is lane 0's next granule, and behind the last the one that lane 31 holds
        const uint4 wrap = c + 1 < kPieces ? g[c + 1 < kPieces ? c + 1 : 0] : behind;
        const bool hand_on = c + 1 < kPieces && lane == 0;
        uint32_t w[8] = {g[c].x, g[c].y, g[c].z, g[c].w, hand_on ? wrap.x : g[c].x, hand_on ? wrap.y : g[c].y,
                         hand_on ? wrap.z : g[c].z, hand_on ? wrap.w : g[c].w};
#pragma unroll
        for (int i = 4; i < 8; ++i) w[i] = __shfl_sync(0xffffffffu, w[i], (lane + 1) & 31);
        if (c + 1 == kPieces && lane == 31) w[4] = behind.x, w[5] = behind.y, w[6] = behind.z, w[7] = behind.w;
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = shift & 4 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = shift & 2 ? w[i + 1] : w[i];
        const int half = 16 * (shift & 1);
        return make_uint4(__funnelshift_r(w[0], w[1], half), __funnelshift_r(w[1], w[2], half),
                          __funnelshift_r(w[2], w[3], half), __funnelshift_r(w[3], w[4], half));
    }
};

// Its bytes to q's row (which starts on a 16-byte boundary); those from k on are left as they are.
template <bool kWhole>
__device__ __forceinline__ void store_piece(int8_t* row, int at, int k, const uint2& b) {
    if (kWhole || 8 * at + 8 <= k) {
        reinterpret_cast<uint2*>(row)[at] = b;
    } else {
        for (int i = 0; 8 * at + i < k; ++i)
            row[8 * at + i] = static_cast<int8_t>(((i < 4 ? b.x : b.y) >> (8 * (i & 3))) & 0xffu);
    }
}

template <bool kF16, bool kWhole, int kWarps, int kPieces>
__global__ void __launch_bounds__(kThreadsQ) quantize_kernel(const QuantParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int kLanes = 32 * kWarps, kRowsCta = kThreadsQ / kLanes;
    __shared__ uint32_t part[kThreadsQ / 32];
    const int warp = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsCta + threadIdx.x / kLanes;
    const bool live = row < p.rows;
    const int k = live ? p.k : 0, pieces = (k + 7) >> 3;
    Pieces<kWhole, kPieces> v;
    v.template load<kLanes>(p.x + row * p.x_stride, 0, k);
    uint32_t m = v.most(0);
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
    if constexpr (kWarps > 1) {
        if ((threadIdx.x & 31) == 0) part[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWarps; ++i) m = max(m, part[warp / kWarps * kWarps + i]);
    }
    if (!live) return;                         // (whole warps: they share a row)
    float pre, r;
    row_factors<kF16>(m, threadIdx.x % kLanes == 0, p.scale + row, pre, r);
    int8_t* q = p.q + row * p.q_stride;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
        const int at = v.template at<kLanes>(0, c);
        const uint4 x = v.piece(c);
        if (at < pieces)
            store_piece<kWhole>(q, at, p.k, pre == 0.0f ? make_uint2(0, 0) : quantize8<kF16>(x, pre, r));
    }
}

// Short rows that start anywhere: a warp a row, value by value, each lane kShort of them (20000 x 100: 6.0 us
// by 4 a lane, 7.4 us by 12, 10.2 us by pieces; x 301: 10.7 and 13.1 us; x 500: 14.5 by 16 and 11.7 us).
constexpr int kShortMost = 12;
template <bool kF16, int kShort>
__global__ void __launch_bounds__(kThreadsQ) quantize_short_kernel(const QuantParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreadsQ / 32) + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const uint16_t* x = p.x + row * p.x_stride;
    uint32_t v[kShort], m = 0;
#pragma unroll
    for (int c = 0; c < kShort; ++c) v[c] = 32 * c + lane < p.k ? __ldg(x + 32 * c + lane) : 0u;
#pragma unroll
    for (int c = 0; c < kShort; ++c) m = max(m, v[c] & 0x7fffu);
    m = __reduce_max_sync(0xffffffffu, m);
    float pre, r;
    row_factors<kF16>(m, lane == 0, p.scale + row, pre, r);
    int8_t* q = p.q + row * p.q_stride;
#pragma unroll
    for (int c = 0; c < kShort; ++c)
        if (32 * c + lane < p.k)
            q[32 * c + lane] = pre == 0.0f ? 0 : static_cast<int8_t>(quantize(value_of<kF16>(v[c]) * pre, r) & 0xffu);
}

// Rows that registers do not hold: a CTA a row, read twice.
template <bool kF16, bool kWhole>
__global__ void __launch_bounds__(kThreadsQ) quantize_long_kernel(const QuantParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ uint32_t part[kThreadsQ / 32];
    const int64_t row = blockIdx.x;
    const uint16_t* x = p.x + row * p.x_stride;
    int8_t* q = p.q + row * p.q_stride;
    constexpr int kPieces = 4;
    const int pieces = (p.k + 7) >> 3;
    uint32_t m = 0;
    Pieces<kWhole, kPieces> v;
    // (every warp goes round as often: the pieces are put together across its lanes)
    for (int first = 0; first < pieces; first += kPieces * kThreadsQ) {
        v.template load<kThreadsQ>(x, first, p.k);
        m = v.most(m);
    }
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreadsQ / 32; ++i) m = max(m, part[i]);
    float pre, r;
    row_factors<kF16>(m, threadIdx.x == 0, p.scale + row, pre, r);
    for (int first = 0; first < pieces; first += kPieces * kThreadsQ) {
        v.template load<kThreadsQ>(x, first, p.k);
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
            const int at = v.template at<kThreadsQ>(first, c);
            const uint4 piece = v.piece(c);
            if (at < pieces)
                store_piece<kWhole>(q, at, p.k, pre == 0.0f ? make_uint2(0, 0) : quantize8<kF16>(piece, pre, r));
        }
    }
}

// ------------------------------------------------------------------------------------------
// lithe_int8_linear
// ------------------------------------------------------------------------------------------
struct Params {
    const int8_t* q;               // (rows, k), row stride q_stride; or nullptr, and
    const uint16_t* x;             // the activations themselves (direct_row)
    const int8_t* w;               // (n, k), row stride w_stride
    const float* x_scale;          // (rows)
    const float* w_scale;          // (n)
    const uint16_t* bias;          // (n) or nullptr
    uint16_t* out;                 // (rows, n)
    const __nv_bfloat16* h;        // (rows, 16) or nullptr
    const __nv_bfloat16* b_dec;    // (rows / rows_per_sample, n, 16)
    int32_t* err;
    int64_t q_stride, w_stride;
    int32_t rows, n, k;
    int32_t rows_per_sample;
};

// D(16 x 8, int32) += A(16 x 32, int8, row) * B(32 x 8, int8, col)
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row at k0; bytes from k on are zeros.  kWeights: read once and kept out of L1, as memory that
// nobody writes while the kernel runs.  The activations are read by ordinary loads: their quantisation may
// still be writing them when the kernel starts (see grid_dependency_wait).
template <bool kWeights>
__device__ __forceinline__ uint4 load16(const int8_t* row, int k0, int k) {
    if (k0 + 16 <= k) {
        if (!kWeights) return *reinterpret_cast<const uint4*>(row + k0);
        uint4 v;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(row + k0));
        return v;
    }
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; k0 + i < k && i < 16; ++i)
        w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k0 + i])) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// y + the expand of one output.
__device__ __forceinline__ float expand_of(const Params& p, int r, int n, float y) {
    const uint32_t* hr = reinterpret_cast<const uint32_t*>(p.h + static_cast<int64_t>(r) * kRank);
    const int64_t at = static_cast<int64_t>(r / p.rows_per_sample) * p.n + n;
    const uint32_t* br = reinterpret_cast<const uint32_t*>(p.b_dec + at * kRank);
#pragma unroll
    for (int j = 0; j < kRank / 2; ++j) {
        const uint32_t hv = __ldg(hr + j), bv = __ldg(br + j);
        y = fmaf(bf16lo_to_f32(hv), bf16lo_to_f32(bv), y);
        y = fmaf(bf16hi_to_f32(hv), bf16hi_to_f32(bv), y);
    }
    return y;
}

// The linear's kernels may start while the quantisation of their activations runs (it lets them at its
// start): they wait here before they read what it writes.  What ran before it has completed by then,
// since it was launched in stream order.  Returns at once in a launch that depends on nothing so.
// q and x_scale are read by ordinary loads behind it: they are written in the kernel's lifetime, which the
// loads of __ldg (ld.global.nc) rule out and which would let the compiler move them over the wait.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Launch {
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute attrs[2];
    Launch(int grid, int threads, size_t smem, cudaStream_t st) {
        config.gridDim = dim3(grid);
        config.blockDim = dim3(threads);
        config.dynamicSmemBytes = smem;
        config.stream = st;
        config.attrs = attrs;
    }
    Launch(const Launch&) = delete;
    void after_last() {
        attrs[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    void clusters_of(int n) {
        attrs[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[config.numAttrs].val.clusterDim.x = n;
        attrs[config.numAttrs].val.clusterDim.y = 1;
        attrs[config.numAttrs++].val.clusterDim.z = 1;
    }
};

// Few rows (at most 16): the weights' bytes are the work.  A CTA takes 16 output channels and all the
// rows (8 kTiles); its warps take turns at pieces of 128 k's and add their int32 sums at the end.
// Inside a piece a lane reads 16 contiguous bytes of a row and uses its four words as the k's of
// two MMAs: the same bijection of k for weights and activations, so the sums stand.  Both halves of
// a 128-byte line are one warp's (64-byte pieces: 15% slower).  As many warps share a channel tile
// as fill the SMs once, 32 a SM of 64 registers: one wave, all of it loading from the start.
// Measured: 14 x 3072 -> 18432 13.4 us (4.2 TB/s), 3 x 15360 -> 3072 12.6 us, 3072 -> 3072 4.7 us (fixed costs).
// Rings of cp.async and activations held in registers or shared memory by persistent CTAs were
// no faster (14 to 22 us).
constexpr int kMaxSplit = 16;                  // warps that share a channel tile
constexpr int kRowWarps = 32;                  // per SM
constexpr int kUnroll = 2;                     // 64-byte pieces a warp loads before it uses the first

// kDirect: a single row, quantised here instead of in a launch of its own: every CTA needs it, and reads it
// from L2 while its first weights come from HBM (3072 -> 3072: 5.2 us, 6.7 us in two launches; two rows of
// 3072 -> 18432 are slower so, 15.2 us and 14.2 us).
constexpr int kDirectMost = 16384;             // values of the row

// p's row (k a multiple of 8, on a 16-byte boundary) as int8, zeros up to the next 16, in shared memory, and
// its scale; every thread of the CTA takes part.
template <bool kF16>
__device__ __forceinline__ void quantize_here(const Params& p, int8_t* q, float* scale, uint32_t* part) {
    const uint4* x = reinterpret_cast<const uint4*>(p.x);
    uint32_t m = 0;
    for (int at = threadIdx.x; at < p.k >> 3; at += blockDim.x) {
        const uint4 v = __ldg(x + at);
        m = __vmaxu2(__vmaxu2(m, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)),
                     __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    }
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) m = max(m, part[i]);
    float pre, r;
    row_factors<kF16>(m, threadIdx.x == 0, scale, pre, r);
    for (int at = threadIdx.x; at < (p.k + 15) / 16 * 2; at += blockDim.x)
        *reinterpret_cast<uint2*>(q + 8 * at) =
            at < p.k >> 3 && pre != 0.0f ? quantize8<kF16>(__ldg(x + at), pre, r) : make_uint2(0, 0);
    __syncthreads();
}

template <bool kF16, int kTiles, bool kDirect>
__global__ void __launch_bounds__(32 * kMaxSplit, 2) int8_rows_kernel(const Params p) {
    extern __shared__ __align__(16) int part_raw[];          // (kDirect reads its row from it in 16-byte pieces)
    __shared__ float scale;
    __shared__ uint32_t row_max[kMaxSplit];
    int(*part)[8 * kTiles][17] = reinterpret_cast<int(*)[8 * kTiles][17]>(part_raw);   // [warp][row][channel]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, kq = 16 * (lane & 3);
    const int split = blockDim.x >> 5, n0 = blockIdx.x * 16;
    int8_t* here = reinterpret_cast<int8_t*>(part + split);                            // kDirect: the row's q
    const int8_t* w0 = p.w + static_cast<int64_t>(n0 + g) * p.w_stride;
    const int8_t* w1 = w0 + 8 * p.w_stride;
    const bool in0 = n0 + g < p.n, in1 = n0 + g + 8 < p.n;
    int acc[kTiles][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 a0[kUnroll], a1[kUnroll], b[kUnroll][kTiles];
    const auto load_weights = [&](int k0) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int k = k0 + 64 * u + kq;
            a0[u] = in0 && k < p.k ? load16<true>(w0, k, p.k) : zero;
            a1[u] = in1 && k < p.k ? load16<true>(w1, k, p.k) : zero;
        }
    };
    load_weights(128 * warp);                  // on their way while the rows are quantised
    if constexpr (kDirect) quantize_here<kF16>(p, here, &scale, row_max);
    else grid_dependency_wait();
    for (int k0 = 128 * warp; k0 < p.k; k0 += 128 * split) {
        if (k0 > 128 * warp) load_weights(k0);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int k = k0 + 64 * u + kq;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int r = 8 * t + g;
                b[u][t] = zero;
                if (r < p.rows && k < p.k)
                    b[u][t] = kDirect ? *reinterpret_cast<const uint4*>(here + k)
                                      : load16<false>(p.q + r * p.q_stride, k, p.k);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                mma_s8(acc[t], a0[u].x, a1[u].x, a0[u].y, a1[u].y, b[u][t].x, b[u][t].y);
                mma_s8(acc[t], a0[u].z, a1[u].z, a0[u].w, a1[u].w, b[u][t].z, b[u][t].w);
            }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)        // element i: channel g + 8 (i / 2), row 2 (lane % 4) + i % 2
            part[warp][8 * t + 2 * (lane & 3) + (i & 1)][g + 8 * (i >> 1)] = acc[t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * 8 * kTiles; e += blockDim.x) {
        const int r = e >> 4, n = n0 + (e & 15);
        if (r >= p.rows || n >= p.n) continue;
        int sum = 0;
        for (int i = 0; i < split; ++i) sum += part[i][r][e & 15];
        const float sx = kDirect ? scale : p.x_scale[r];
        float y = fmaf(static_cast<float>(sum) * sx, p.w_scale[n], p.bias ? value_of<kF16>(p.bias[n]) : 0.0f);
        if (p.h) y = expand_of(p, r, n, y);
        p.out[static_cast<int64_t>(r) * p.n + n] = static_cast<uint16_t>(Act<kF16>::pack(y, 0.0f) & 0xffffu);
    }
}

// Whether p's activations are quantised by the few-row kernel itself.
bool direct_row(const Params& p) {
    return p.rows == 1 && p.k <= kDirectMost && p.k % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
}

template <bool kF16, int kTiles, bool kDirect>
int32_t launch_rows(const Params& p, int sms, bool after_quantize, cudaStream_t st) {
    const int tiles = (p.n + 15) / 16, pairs = (p.k + 127) / 128;
    int split = static_cast<int>(static_cast<int64_t>(sms) * kRowWarps / tiles);
    split = split < 1 ? 1 : split > kMaxSplit ? kMaxSplit : split;
    split = split < pairs ? split : pairs;
    const int share = (pairs + split - 1) / split;
    split = (pairs + share - 1) / share;           // no more warps than their share of the pieces needs
    const int sums = split * 8 * kTiles * 17 * static_cast<int>(sizeof(int));
    static_assert(8 * kTiles * 17 * sizeof(int) % 16 == 0, "the row behind the sums stays aligned");
    Launch l(tiles, 32 * split, sums + (kDirect ? (p.k + 15) / 16 * 16 : 0), st);
    if (after_quantize) l.after_last();
    const cudaError_t e = cudaLaunchKernelEx(&l.config, int8_rows_kernel<kF16, kTiles, kDirect>, p);
    return e == cudaSuccess ? LITHE_OK : fail_cuda(e, "int8_rows_kernel launch");
}

// Many rows: a persistent tcgen05 GEMM (kind::i8, int32 accumulators in TMEM).  kPair: a cluster of
// two CTAs computes 256 x 256 tiles with cta_group::2 (M256 N256 K32); else one CTA computes
// 128 x 128 tiles.  Either way a CTA streams 128 rows of q and 128 rows of w, 128 bytes of k each,
// per stage (two 16 KB TMA boxes, 128-byte swizzle; rows, channels and k's past the ends come as
// zeros), kStages deep, and keeps two accumulators so that a tile's epilogue runs under the next
// tile's products.
//   warp 0       TMA producer          warp 1   TMEM allocation, MMA issue (the pair's leader only)
//   warps 2..9   epilogue: each 32 accumulator rows and half of the columns, 64 at a time
//   warp 10      (kExpandTmem) issues the expand
// The epilogue reads the accumulator in the 16 x 256-bit shape, the register layout of a warp MMA's
// result: a lane holds column pairs of four rows, so a column's scale and bias are read once for
// all of them, and two neighbouring results make one staged word.
//
// The expand h . b_dec^T (an int32 accumulator cannot take its fp32 sums):
//   kExpandMma    one m16n8k16 warp MMA per 128 outputs on top of the scaled sums, any rows per sample.
//                 The factors' k runs through the same bijection in h and b_dec, so that a lane reads
//                 8 contiguous bytes of each.
//   kExpandTmem   (pairs, samples of whole tiles) the epilogue writes the scaled sums, now fp32, back into
//                 TMEM in place of the int32 ones; one tcgen05.mma (kind::f16, K = 16) adds the expand
//                 of the whole tile there, issued by a warp of its own (polled for by the products'
//                 issuer it cost 10%), and the epilogue reads the result.  Warp MMAs share the
//                 tensor pipe with tcgen05.mma and slow it: 57344 x 3072 -> 12288 takes 1.42 ms
//                 this way, 1.69 ms with them and 1.38 ms without an expand, calls 30 ms apart; with
//                 the quantisation and in a row, under the 1 kW cap, 1.75, 2.01 and 1.67 ms.
// Measured without an expand: 14336 x 3072 -> 12288 2.8 POP/s, x 768 -> 12288 130 us (an epilogue of 4
// warps with a TMA store of 64-byte rows: 257 us).  In a tile the stages' bytes (64 KB a pair and
// 128 k's) keep shared memory as busy as the products keep the tensor pipe.
// Too few 128 x 128 tiles for the SMs: a cluster of `split` CTAs takes one, each a run of its k's.  Their
// int32 sums go through shared memory, where each CTA adds the others' for its share of the rows (an
// exact sum, so the split does not show in the result) and finishes them.  A CTA takes in about 60
// bytes a cycle, 0.3 us a stage of a 128 x 128 tile, and the exchange costs 4 us; clusters of 8 took 4 us more
// to start.  From 24 stages on a cluster was as fast as a single CTA or faster at every size tried (us, clusters
// and single CTAs: 32 x 12288 -> 3072 14.7 and 30.8; at 24 stages, -> 3072, 128 rows 11.8 and 11.8, 32 rows 9.3
// and 11.4, 256 rows -> 1024 10.9 and 11.5; at 16 stages 11.2 and 9.7, 8.6 and 9.3, 10.0 and 9.2; at 8 10.4 and
// 7.4, 7.5 and 6.9, 8.9 and 6.5).
// Every mbarrier wait is bounded (4 s, LITHE_DEVERR_TIMEOUT, shared abort flag).
enum Expand { kExpandNone, kExpandMma, kExpandTmem };

constexpr int kBK = 128;                       // bytes of k per stage
constexpr int kRows = 128;                     // rows of q and of w a CTA loads per stage
constexpr int kBox = kRows * kBK;              // 16 KB
constexpr int kStages = 6;
constexpr int kEpiWarps = 8;                   // two for each 32 accumulator rows
constexpr int kEpiChunk = 16 * 64 * 2;         // a warp's staged output: 16 rows x 64 columns
template <int kExpand>
constexpr int kThreads = 32 * (2 + kEpiWarps + (kExpand == kExpandTmem ? 1 : 0));
constexpr int kGroupN = 8;                     // tile order: groups of 8 column tiles, row tiles inside a group
constexpr int kHBytes = kRows * kRank * 2;     // 4 KB: a CTA's rows of h
constexpr int kExpandBytes = 2 * kHBytes;      // and 4 KB: its half of the tile's columns of b_dec


struct Barriers {
    uint64_t full[kStages], empty[kStages];
    uint64_t tfull[2], tempty[2];
    uint64_t cfull, cempty;                    // the tile's columns staged / done with
    uint64_t lfull[2], lempty[2];              // kExpandTmem: h and b_dec of a tile
    uint64_t ereq, efull;                      // scaled sums back in TMEM / expand added to them
    uint64_t done, edone;                      // every product / every expand issued has completed
    uint32_t tmem_base;
    int abort;
};

// What the epilogue needs of a tile's columns, staged once per tile: scale, bias and (kExpandMma) the
// decoded B factors of the sample of the CTA's first row; rows of other samples read theirs from
// global memory.
template <int kSize, int kExpand>
struct Columns {
    float scale[kSize];
    uint16_t bias[kSize];
    uint4 factors[kExpand == kExpandMma ? kSize : 1][2];
};

// Shared memory: stages, h and b_dec (two tiles), staged output, columns, barriers.
template <int kSize, int kExpand>
struct Layout {
    static constexpr int kExpandAt = kStages * 2 * kBox;
    static constexpr int kOutAt = kExpandAt + (kExpand == kExpandTmem ? 2 * kExpandBytes : 0);
    static constexpr int kColumnsAt = kOutAt + kEpiWarps * kEpiChunk;
    static constexpr int kBarriersAt = kColumnsAt + static_cast<int>(sizeof(Columns<kSize, kExpand>));
    static constexpr int kBytes = kBarriersAt + static_cast<int>(sizeof(Barriers)) + 1024;   // + alignment slack
    static_assert(kBytes <= 232448, "shared memory of the tile kernel");
    static_assert(kColumnsAt % 16 == 0 && kBarriersAt % 16 == 0, "alignment");
};

struct TileParams {
    Params p;
    int32_t m_tiles, n_tiles, total_tiles;
    int32_t out16;                 // the result's rows are 16-byte aligned
    int32_t split;                 // single CTAs: CTAs of a cluster that share a tile's k
};

// Instruction descriptor of tcgen05.mma kind::i8: int32 accumulator (bits 4-5 = 2), signed A and B
// (bits 7-9, 10-12 = 1), both K-major, N >> 3 in bits 17-22, M >> 4 in bits 24-28.
template <bool kPair>
constexpr uint32_t kIdesc = (2u << 4) | (1u << 7) | (1u << 10) |
                            (static_cast<uint32_t>((kPair ? 256 : 128) >> 3) << 17) |
                            (static_cast<uint32_t>((kPair ? 256 : 128) >> 4) << 24);
// The expand's, kind::f16: fp32 accumulator, bf16 A and B, M256 N256.
constexpr uint32_t kIdescExpand = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(256 >> 3) << 17) |
                                  (static_cast<uint32_t>(256 >> 4) << 24);

template <bool kPair>
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(kIdesc<true>), "r"(accumulate));
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(kIdesc<false>), "r"(accumulate));
}

__device__ __forceinline__ void umma_expand(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.eq.b32 p, 0, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(kIdescExpand));
}

// 16 accumulator rows x 64 columns: r[4 j + i] is row lane / 4 + 8 (i / 2), column
// 8 j + 2 (lane % 4) + i % 2, once tcgen05.wait::ld has returned.
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_16x64(uint32_t taddr, const float (&y)[8][4]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "f"(y[0][0]), "f"(y[0][1]), "f"(y[0][2]), "f"(y[0][3]), "f"(y[1][0]), "f"(y[1][1]), "f"(y[1][2]),
        "f"(y[1][3]), "f"(y[2][0]), "f"(y[2][1]), "f"(y[2][2]), "f"(y[2][3]), "f"(y[3][0]), "f"(y[3][1]),
        "f"(y[3][2]), "f"(y[3][3]), "f"(y[4][0]), "f"(y[4][1]), "f"(y[4][2]), "f"(y[4][3]), "f"(y[5][0]),
        "f"(y[5][1]), "f"(y[5][2]), "f"(y[5][3]), "f"(y[6][0]), "f"(y[6][1]), "f"(y[6][2]), "f"(y[6][3]),
        "f"(y[7][0]), "f"(y[7][1]), "f"(y[7][2]), "f"(y[7][3])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tile_of(const TileParams& tp, int t, int size, int& m0, int& n0) {
    const int per_group = kGroupN * tp.m_tiles;
    const int g = t / per_group;
    const int in = t - g * per_group;
    const int width = min(kGroupN, tp.n_tiles - g * kGroupN);
    m0 = (in / width) * size;
    n0 = (g * kGroupN + in % width) * size;
}

// One epilogue thread's part of a tile's columns, on its way from global memory: loaded while the
// tile before is finished, so that no epilogue waits for it.
template <int kSize, int kExpand>
struct ColumnRegs {
    uint4 f[2];
    float scale;
    uint16_t bias;

    __device__ __forceinline__ void load(const Params& p, int row, int n0, int thread) {
        if (thread >= kSize) return;
        const int n = min(n0 + thread, p.n - 1);
        scale = __ldg(p.w_scale + n);
        bias = p.bias ? __ldg(p.bias + n) : static_cast<uint16_t>(0);
        if constexpr (kExpand == kExpandMma) {
            const int sample = min(row, p.rows - 1) / p.rows_per_sample;
            const uint4* b = reinterpret_cast<const uint4*>(p.b_dec + (static_cast<int64_t>(sample) * p.n + n) * kRank);
            f[0] = __ldg(b);
            f[1] = __ldg(b + 1);
        }
    }
    __device__ __forceinline__ void store(Columns<kSize, kExpand>* c, int thread) const {
        if (thread >= kSize) return;
        c->scale[thread] = scale;
        c->bias[thread] = bias;
        if constexpr (kExpand == kExpandMma) {
            c->factors[thread][0] = f[0];
            c->factors[thread][1] = f[1];
        }
    }
};

// What the epilogue needs of a lane's rows row0 + lane / 4 + 8 i.
template <int kExpand>
struct RowRegs {
    float sx[4];
    uint2 h[4];
    int sample[4];

    __device__ __forceinline__ void load(const Params& p, int row0, int lane) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row0 + (lane >> 2) + 8 * i;
            const bool in = r < p.rows;
            sx[i] = in ? p.x_scale[r] : 0.0f;
            if constexpr (kExpand == kExpandMma) {
                h[i] = in ? __ldg(reinterpret_cast<const uint2*>(p.h + static_cast<int64_t>(r) * kRank) + (lane & 3))
                          : make_uint2(0, 0);
                sample[i] = min(r, p.rows - 1) / p.rows_per_sample;
            }
        }
    }
};

// The sums of 32 rows x 64 columns (c0 .. of the tile), scaled, with the bias: y[half][j][i] is row
// 16 half + lane / 4 + 8 (i / 2), column 8 j + 2 (lane % 4) + i % 2.
template <bool kF16, int kSize, int kExpand>
__device__ __forceinline__ void scaled_sums(uint32_t tmem_acc, int c0, const RowRegs<kExpand>& rows,
                                            const Columns<kSize, kExpand>* cols, float (&y)[2][8][4]) {
    const int q = threadIdx.x & 3;
    uint32_t acc[2][32];
    tmem_ld_16x64(tmem_acc + c0, acc[0]);
    tmem_ld_16x64(tmem_acc + (16u << 16) + c0, acc[1]);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 s = *reinterpret_cast<const float2*>(&cols->scale[c0 + 8 * j + 2 * q]);
        const uint32_t b = *reinterpret_cast<const uint32_t*>(&cols->bias[c0 + 8 * j + 2 * q]);
        const float b0 = Act<kF16>::lo(b), b1 = Act<kF16>::hi(b);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[half][j][i] = fmaf(static_cast<float>(static_cast<int>(acc[half][4 * j + i])) * rows.sx[2 * half + (i >> 1)],
                                     i & 1 ? s.y : s.x, i & 1 ? b1 : b0);
    }
}

// 16 rows x 64 columns rounded into the warp's staging buffer (16 rows of 128 bytes, 16-byte unit u of
// row r at u ^ (r & 7): no bank conflicts either way) and from there to global memory in whole
// 128-byte lines.
template <bool kF16>
__device__ __forceinline__ void store_rows(const TileParams& tp, const float (&y)[8][4], int row0, int col0,
                                           uint8_t* buf) {
    const Params& p = tp.p;
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint32_t*>(buf + (g + 8 * i) * 128 + ((j ^ g) << 4) + 4 * q) =
                Act<kF16>::pack(y[j][2 * i], y[j][2 * i + 1]);
    __syncwarp();
    if (tp.out16) {
        const int col = col0 + 8 * (lane & 7);
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int in = 4 * i + (lane >> 3);
            v[i] = *reinterpret_cast<const uint4*>(buf + in * 128 + (((lane & 7) ^ (in & 7)) << 4));
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row0 + 4 * i + (lane >> 3);
            if (r < p.rows && col < p.n)
                *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(r) * p.n + col) = v[i];
        }
    } else {
        // rows off the 16-byte boundaries: a column a lane, 64 bytes of a row at a time
#pragma unroll 4
        for (int in = 0; in < 16; ++in) {
            uint16_t* out = p.out + static_cast<int64_t>(row0 + in) * p.n + col0;
#pragma unroll
            for (int c = lane; c < 64; c += 32) {
                const uint16_t v = *reinterpret_cast<const uint16_t*>(buf + in * 128 + (((c >> 3) ^ (in & 7)) << 4) + 2 * (c & 7));
                if (row0 + in < p.rows && col0 + c < p.n) out[c] = v;
            }
        }
        __syncwarp();
    }
}

// kExpandMma: the expand of 32 rows x 64 columns onto y.
template <int kSize>
__device__ __forceinline__ void add_expand(const Params& p, int n0, int c0, int staged,
                                           const RowRegs<kExpandMma>& rows, const Columns<kSize, kExpandMma>* cols,
                                           float (&y)[2][8][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const uint2* factors = reinterpret_cast<const uint2*>(cols->factors);
    // whether all 32 rows are the staged sample's
    if (__all_sync(0xffffffffu, rows.sample[0] == staged && rows.sample[3] == staged)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint2 b = factors[(c0 + 8 * j + g) * 4 + q];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t a[4] = {rows.h[2 * half].x, rows.h[2 * half + 1].x, rows.h[2 * half].y,
                                       rows.h[2 * half + 1].y};
                mma_bf16_16816(y[half][j], a, b.x, b.y, y[half][j]);
            }
        }
        return;
    }
    // sample s's factors of channel block j
    const auto factors_of = [&](int s, int j) {
        if (s == staged) return factors[(c0 + 8 * j + g) * 4 + q];
        const int n = min(n0 + c0 + 8 * j + g, p.n - 1);
        return __ldg(reinterpret_cast<const uint2*>(p.b_dec + (static_cast<int64_t>(s) * p.n + n) * kRank) + q);
    };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int first = __shfl_sync(0xffffffffu, rows.sample[2 * half], 0);
        const int last = __shfl_sync(0xffffffffu, rows.sample[2 * half + 1], 31);
        const uint32_t a[4] = {rows.h[2 * half].x, rows.h[2 * half + 1].x, rows.h[2 * half].y, rows.h[2 * half + 1].y};
        if (first == last) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint2 b = factors_of(first, j);
                mma_bf16_16816(y[half][j], a, b.x, b.y, y[half][j]);
            }
            continue;
        }
        // the samples of the 16 rows, one after the other; a row takes the sum with its own sample's factors
        // (zeros in place of the other rows' h would not do: times a factor that is not finite they are NaN)
#pragma unroll 1
        for (int s = first; s <= last; ++s) {
            const bool lo = rows.sample[2 * half] == s, hi = rows.sample[2 * half + 1] == s;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint2 b = factors_of(s, j);
                float sum[4];
                mma_bf16_16816(sum, a, b.x, b.y, y[half][j]);
                if (lo) y[half][j][0] = sum[0], y[half][j][1] = sum[1];
                if (hi) y[half][j][2] = sum[2], y[half][j][3] = sum[3];
            }
        }
    }
}

constexpr int kSumPitch = 132;                 // ints between the rows of a tile's sums in shared memory

// A warp's 32 rows x 64 columns of a split tile's sums to shared memory (the stages' place: every load
// and every product of the tile has completed).
__device__ __forceinline__ void keep_sums(uint32_t tmem_acc, int* sums) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t acc[32];
        tmem_ld_16x64(tmem_acc + (static_cast<uint32_t>(16 * half) << 16), acc);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *reinterpret_cast<uint2*>(sums + (16 * half + g + 8 * i) * kSumPitch + 8 * j + 2 * q) =
                    make_uint2(acc[4 * j + 2 * i], acc[4 * j + 2 * i + 1]);
    }
}

__device__ __forceinline__ uint4 ld_cluster(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// This CTA's share of the tile's rows, the cluster's sums of them added and finished: 8 columns a
// thread at a time.
constexpr int kSplits = 4;                     // most CTAs of a cluster
constexpr int kSplitStages = 24;               // fewest stages of a tile that is split
template <bool kF16, int kSize, int kExpand>
__device__ __forceinline__ void finish_sums(const TileParams& tp, const uint8_t* smem,
                                            const Columns<kSize, kExpand>* cols, int part, int m0, int n0) {
    const Params& p = tp.p;
    const int tasks = min(kSize, p.rows - m0) * (kSize / 8);
    const int end = tasks * (part + 1) / tp.split;
    for (int e = tasks * part / tp.split + threadIdx.x; e < end; e += blockDim.x) {
        const int in = e / (kSize / 8), c = 8 * (e % (kSize / 8));             // row of the tile, first column
        const int r = m0 + in, n = n0 + c;
        if (n >= p.n) continue;
        const float sx = p.x_scale[r];
        uint4 a[kSplits][2];
#pragma unroll
        for (int s = 0; s < kSplits; ++s) {
            const uint32_t at = map_to_rank(smem + (in * kSumPitch + c) * 4, s < tp.split ? s : 0);
            a[s][0] = s < tp.split ? ld_cluster(at) : make_uint4(0, 0, 0, 0);
            a[s][1] = s < tp.split ? ld_cluster(at + 16) : make_uint4(0, 0, 0, 0);
        }
        uint32_t sum[8] = {};
#pragma unroll
        for (int s = 0; s < kSplits; ++s) {
            sum[0] += a[s][0].x, sum[1] += a[s][0].y, sum[2] += a[s][0].z, sum[3] += a[s][0].w;
            sum[4] += a[s][1].x, sum[5] += a[s][1].y, sum[6] += a[s][1].z, sum[7] += a[s][1].w;
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = fmaf(static_cast<float>(static_cast<int>(sum[i])) * sx, cols->scale[c + i], value_of<kF16>(cols->bias[c + i]));
            if (kExpand == kExpandMma) y[i] = expand_of(p, r, min(n + i, p.n - 1), y[i]);
        }
        const uint4 v = make_uint4(Act<kF16>::pack(y[0], y[1]), Act<kF16>::pack(y[2], y[3]),
                                   Act<kF16>::pack(y[4], y[5]), Act<kF16>::pack(y[6], y[7]));
        uint16_t* out = p.out + static_cast<int64_t>(r) * p.n + n;
        if (tp.out16) {
            *reinterpret_cast<uint4*>(out) = v;
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (n + i < p.n) out[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

template <bool kPair, bool kF16, int kExpand>
__device__ __forceinline__ void tile_kernel_body(const CUtensorMap& tm_q, const CUtensorMap& tm_w,
                                                 const CUtensorMap& tm_h, const CUtensorMap& tm_bd,
                                                 const TileParams& tp) {
    static_assert(kPair || kExpand != kExpandTmem, "the expand in TMEM is the pairs'");
    constexpr int kSize = kPair ? 256 : 128;               // rows and columns of a tile
    constexpr uint32_t kCols = 2 * kSize;                  // TMEM columns: two accumulators
    using L = Layout<kSize, kExpand>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* expand_base = smem + L::kExpandAt;
    Columns<kSize, kExpand>* cols = reinterpret_cast<Columns<kSize, kExpand>*>(smem + L::kColumnsAt);
    Barriers* bars = reinterpret_cast<Barriers*>(smem + L::kBarriersAt);
    volatile int* abort = &bars->abort;
    int32_t* err = tp.p.err;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kPair ? static_cast<int>(cluster_rank()) : 0;
    const bool leader = rank == 0;
    const int group = kPair ? 2 : tp.split;                // CTAs of a tile
    const int first = blockIdx.x / group, step = gridDim.x / group;
    // this CTA's stages of a tile
    const int stages = (tp.p.k + kBK - 1) / kBK, part = kPair || group == 1 ? 0 : static_cast<int>(cluster_rank());
    const int kb0 = kPair ? 0 : stages * part / group, nk = kPair ? stages : stages * (part + 1) / group - kb0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bars->tfull[a], 1);
            mbar_init(&bars->tempty[a], (kPair ? 2 : 1) * kEpiWarps);
            mbar_init(&bars->lfull[a], 1);
            mbar_init(&bars->lempty[a], 1);
        }
        mbar_init(&bars->ereq, 2 * kEpiWarps);
        mbar_init(&bars->efull, 1);
        mbar_init(&bars->cfull, kEpiWarps);
        mbar_init(&bars->cempty, kEpiWarps);
        mbar_init(&bars->done, 1);
        mbar_init(&bars->edone, 1);
        bars->abort = 0;
        fence_mbar_init();
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_w);
        if constexpr (kExpand == kExpandTmem) {
            prefetch_tmap(&tm_h);
            prefetch_tmap(&tm_bd);
        }
    }
    if (warp == 1) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(&bars->tmem_base)),
                         "r"(kCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(&bars->tmem_base)),
                         "r"(kCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    tc_fence_before();
    if constexpr (kPair) cluster_sync();                   // both CTAs' barriers initialised, TMEM allocated
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        if (lane == 0) {
            grid_dependency_wait();
            uint32_t it = 0, tile = 0;
            for (int t = first; t < tp.total_tiles && !*abort; t += step, ++tile) {
                int m0, n0;
                tile_of(tp, t, kSize, m0, n0);
                if constexpr (kExpand == kExpandTmem) {
                    const uint32_t b = tile & 1u, ph = (tile >> 1) & 1u;
                    if (!mbar_wait(&bars->lempty[b], ph ^ 1u, abort, err)) break;
                    if (leader) mbar_arrive_expect_tx(&bars->lfull[b], 2 * kExpandBytes);
                    const uint32_t fb = map_to_rank(&bars->lfull[b], 0);
                    uint8_t* l = expand_base + b * kExpandBytes;
                    tma_load_2d_pair(l, &tm_h, fb, 0, m0 + kRows * rank);
                    tma_load_2d_pair(l + kHBytes, &tm_bd, fb, 0,
                                     m0 / tp.p.rows_per_sample * tp.p.n + n0 + kRows * rank);
                }
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const uint32_t s = it % kStages, ph = (it / kStages) & 1u;
                    if (!mbar_wait(&bars->empty[s], ph ^ 1u, abort, err)) break;
                    uint8_t* a = smem + s * 2 * kBox;
                    if constexpr (kPair) {
                        if (leader) mbar_arrive_expect_tx(&bars->full[s], 4 * kBox);
                        const uint32_t fb = map_to_rank(&bars->full[s], 0);
                        tma_load_2d_pair(a, &tm_q, fb, kb * kBK, m0 + kRows * rank);
                        tma_load_2d_pair(a + kBox, &tm_w, fb, kb * kBK, n0 + kRows * rank);
                    } else {
                        mbar_arrive_expect_tx(&bars->full[s], 2 * kBox);
                        tma_load_2d(a, &tm_q, &bars->full[s], (kb0 + kb) * kBK, m0);
                        tma_load_2d(a + kBox, &tm_w, &bars->full[s], (kb0 + kb) * kBK, n0);
                    }
                }
            }
            if (*abort) drain_pause();
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        if (leader && lane == 0) {
            uint32_t s = 0, ph = 0, tile = 0;
            const uint64_t base = desc_k_major(smem_u32(smem), 128, 2);
            for (int t = first; t < tp.total_tiles && !*abort; t += step, ++tile) {
                const uint32_t acc = tile & 1u, aph = (tile >> 1) & 1u;
                if (!mbar_wait(&bars->tempty[acc], aph ^ 1u, abort, err)) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * kSize;
                bool ok = true;
                for (int kb = 0; kb < nk; ++kb) {
                    if (!mbar_wait(&bars->full[s], ph, abort, err)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = base + s * (2 * kBox >> 4), bd = ad + (kBox >> 4);
#pragma unroll
                    for (int kk = 0; kk < kBK / 32; ++kk)  // +32 bytes along k inside the 128-byte swizzle atom
                        umma_i8<kPair>(d, ad + 2 * kk, bd + 2 * kk, (kb | kk) != 0);
                    if constexpr (kPair) umma_commit_pair(&bars->empty[s]);
                    else umma_commit(&bars->empty[s]);
                    if (++s == kStages) s = 0, ph ^= 1u;
                }
                if (!ok) break;
                if constexpr (kPair) umma_commit_pair(&bars->tfull[acc]);
                else umma_commit(&bars->tfull[acc]);
            }
            if constexpr (kPair) umma_commit_pair_local(&bars->done);
            else umma_commit(&bars->done);                 // arrives once every MMA above has completed
        }
    } else if (kExpand == kExpandTmem && warp == 2 + kEpiWarps) {
        // ---------------------------------------------------------------- expand issuer
        if (leader && lane == 0) {
            uint32_t tile = 0;
            for (int t = first; t < tp.total_tiles && !*abort; t += step, ++tile) {
                const uint32_t b = tile & 1u, ph = (tile >> 1) & 1u;
                if (!mbar_wait(&bars->lfull[b], ph, abort, err)) break;
                if (!mbar_wait(&bars->ereq, tile & 1u, abort, err)) break;
                tc_fence_after();
                const uint32_t l = smem_u32(expand_base + b * kExpandBytes);
                umma_expand(tmem + b * kSize, desc_k_major(l, 32, 6), desc_k_major(l + kHBytes, 32, 6));
                umma_commit_pair(&bars->efull);
                umma_commit_pair(&bars->lempty[b]);
            }
            umma_commit_pair_local(&bars->edone);
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        grid_dependency_wait();
        const int quarter = warp & 3;                      // TMEM lanes 32 * quarter .. + 31
        const int side = (warp - 2) >> 2;                  // which half of the columns
        uint8_t* buf = smem + L::kOutAt + (warp - 2) * kEpiChunk;
        uint32_t tempty[2] = {0, 0}, ereq = 0;
        if constexpr (kPair) {
            tempty[0] = map_to_rank(&bars->tempty[0], 0);
            tempty[1] = map_to_rank(&bars->tempty[1], 0);
            ereq = map_to_rank(&bars->ereq, 0);
        }
        const int thread = threadIdx.x - 64, row_in = kRows * rank + 32 * quarter;
        uint32_t tile = 0;
        ColumnRegs<kSize, kExpand> next;
        int m0 = 0, n0 = 0;
        if (first < tp.total_tiles) {
            tile_of(tp, first, kSize, m0, n0);
            next.load(tp.p, m0 + kRows * rank, n0, thread);
        }
        for (int t = first; t < tp.total_tiles && !*abort; t += step, ++tile) {
            const uint32_t acc = tile & 1u, aph = (tile >> 1) & 1u;
            RowRegs<kExpand> rows;
            rows.load(tp.p, m0 + row_in, lane);
            const int staged =
                kExpand == kExpandMma ? min(m0 + kRows * rank, tp.p.rows - 1) / tp.p.rows_per_sample : 0;
            // every epilogue warp is done with the tile before's columns; then this one's are in place
            if (!mbar_wait(&bars->cempty, (tile & 1u) ^ 1u, abort, err)) break;
            next.store(cols, thread);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->cfull);
            const int row0 = m0 + row_in, col0 = n0;
            if (t + step < tp.total_tiles) {
                tile_of(tp, t + step, kSize, m0, n0);
                next.load(tp.p, m0 + kRows * rank, n0, thread);
            }
            if (!mbar_wait(&bars->cfull, tile & 1u, abort, err)) break;
            if (!mbar_wait(&bars->tfull[acc], aph, abort, err)) break;
            tc_fence_after();
            const uint32_t tmem_acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kSize;
            const int c_first = kSize / 2 * side;
            if (!kPair && group > 1) {
                keep_sums(tmem_acc + c_first, reinterpret_cast<int*>(smem) + (32 * quarter) * kSumPitch + c_first);
                break;                                     // (one tile a cluster)
            }
            if constexpr (kExpand == kExpandTmem) {
                // (every warp takes part, those behind the last column too; the rows are whole tiles)
#pragma unroll 1
                for (int c0 = c_first; c0 < c_first + kSize / 2; c0 += 64) {
                    float y[2][8][4];
                    scaled_sums<kF16, kSize, kExpand>(tmem_acc, c0, rows, cols, y);
                    tmem_st_16x64(tmem_acc + c0, y[0]);
                    tmem_st_16x64(tmem_acc + (16u << 16) + c0, y[1]);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                // (relaxed: wait::st and the fences, this one and the issuer's, order the sums before its product)
                if (lane == 0) mbar_arrive_remote_relaxed(ereq);
                if (!mbar_wait(&bars->efull, tile & 1u, abort, err)) break;
                tc_fence_after();
            }
#pragma unroll 1
            for (int c0 = c_first; c0 < c_first + kSize / 2; c0 += 64) {
                if (row0 >= tp.p.rows || col0 + c0 >= tp.p.n) break;
                float y[2][8][4];
                if constexpr (kExpand == kExpandTmem) {
                    uint32_t e[2][32];
                    tmem_ld_16x64(tmem_acc + c0, e[0]);
                    tmem_ld_16x64(tmem_acc + (16u << 16) + c0, e[1]);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 64; ++j) y[j >> 5][(j >> 2) & 7][j & 3] = __uint_as_float(e[j >> 5][j & 31]);
                } else {
                    scaled_sums<kF16, kSize, kExpand>(tmem_acc, c0, rows, cols, y);
                }
                if constexpr (kExpand == kExpandMma) add_expand<kSize>(tp.p, col0, c0, staged, rows, cols, y);
#pragma unroll
                for (int half = 0; half < 2; ++half) store_rows<kF16>(tp, y[half], row0 + 16 * half, col0 + c0, buf);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bars->cempty);
                if constexpr (kPair) mbar_arrive_remote_relaxed(tempty[acc]);
                else mbar_arrive(&bars->tempty[acc]);
            }
        }
    }

    __syncthreads();
    if (!kPair && group > 1) {
        cluster_sync();                                    // every CTA's sums are in place
        int m0, n0;
        tile_of(tp, first, kSize, m0, n0);
        finish_sums<kF16, kSize, kExpand>(tp, smem, cols, part, m0, n0);
        cluster_sync();                                    // no CTA leaves while its sums are read
    }
    if (leader && warp == 1 && lane == 0) {
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(&bars->done, 0) && global_timer_ns() - t0 < 100000000ull) {
        }
        if constexpr (kExpand == kExpandTmem)
            while (!mbar_try_wait(&bars->edone, 0) && global_timer_ns() - t0 < 100000000ull) {
            }
    }
    tc_fence_before();
    if constexpr (kPair) cluster_sync();                   // the pair's MMAs are done before either CTA frees anything
    else __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        if constexpr (kPair)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
    }
}

template <bool kF16, int kExpand>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads<kExpand>, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_h, const __grid_constant__ CUtensorMap tm_bd,
                     const __grid_constant__ TileParams tp) {
    tile_kernel_body<true, kF16, kExpand>(tm_q, tm_w, tm_h, tm_bd, tp);
}

template <bool kF16, int kExpand>
__global__ void __launch_bounds__(kThreads<kExpand>, 1)
    int8_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ TileParams tp) {
    tile_kernel_body<false, kF16, kExpand>(tm_q, tm_w, tm_q, tm_q, tp);
}

template <bool kPair, bool kF16, int kExpand>
int32_t launch_tiles(const Params& p, int device, int sms, bool after_quantize, cudaStream_t st) {
    constexpr int kSize = kPair ? 256 : 128;
    constexpr int kBytes = Layout<kSize, kExpand>::kBytes;
    CUtensorMap tm_q, tm_w, tm_h, tm_bd;
    int32_t rc = encode_u8_2d(&tm_q, p.q, p.k, p.rows, p.q_stride, kBK, kRows);
    if (rc != LITHE_OK) return rc;
    if ((rc = encode_u8_2d(&tm_w, p.w, p.k, p.n, p.w_stride, kBK, kRows)) != LITHE_OK) return rc;
    if constexpr (kExpand == kExpandTmem) {
        if ((rc = encode_bf16_2d(&tm_h, p.h, kRank, p.rows, kRank, kRows, 32)) != LITHE_OK) return rc;
        if ((rc = encode_bf16_2d(&tm_bd, p.b_dec, kRank, static_cast<uint64_t>(p.rows / p.rows_per_sample) * p.n, kRank,
                                 kRows, 32)) != LITHE_OK)
            return rc;
    }
    TileParams tp{};
    tp.p = p;
    tp.out16 = p.n % 8 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    tp.m_tiles = (p.rows + kSize - 1) / kSize;
    tp.n_tiles = (p.n + kSize - 1) / kSize;
    const int64_t tiles = static_cast<int64_t>(tp.m_tiles) * tp.n_tiles;
    if (tiles > 0x7fffffffLL - 0x10000) return fail_arg("too many tiles");
    tp.total_tiles = static_cast<int32_t>(tiles);
    const auto kernel = [] {
        if constexpr (kPair) return int8_pair_kernel<kF16, kExpand>;
        else return int8_tile_kernel<kF16, kExpand>;
    }();
    static bool configured[64] = {false};
    if (!configured[device]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != cudaSuccess) return fail_cuda(e, "cudaFuncSetAttribute(int8 tile kernel)");
        configured[device] = true;
    }
    tp.split = 1;
    int grid = 0;
    if constexpr (kPair) {
        grid = 2 * static_cast<int>(tiles < sms / 2 ? tiles : sms / 2);
    } else {
        // CTAs a tile, while they find SMs, where the stages that this saves outweigh the exchange
        const int stages = (p.k + kBK - 1) / kBK;
        while (stages >= kSplitStages && tp.split < kSplits && tiles * tp.split * 2 <= sms) tp.split *= 2;
        grid = static_cast<int>(tiles * tp.split < sms ? tiles * tp.split : sms);
    }
    Launch l(grid, kThreads<kExpand>, kBytes, st);
    if (after_quantize) l.after_last();
    if (tp.split > 1) l.clusters_of(tp.split);
    cudaError_t e;
    if constexpr (kPair) e = cudaLaunchKernelEx(&l.config, kernel, tm_q, tm_w, tm_h, tm_bd, tp);
    else e = cudaLaunchKernelEx(&l.config, kernel, tm_q, tm_w, tp);
    return e == cudaSuccess ? LITHE_OK : fail_cuda(e, "int8 tile kernel launch");
}

// b_dec's rows are TMA coordinates, 32-bit.
inline bool factor_rows_fit(const Params& p) {
    return static_cast<int64_t>(p.rows / p.rows_per_sample) * p.n < 0x7fffffffLL - 256;
}

template <bool kF16>
int32_t launch_linear(const Params& p, bool after_quantize, cudaStream_t st) {
    int device = 0, sms = 0;
    const int32_t rc = current_device_sms(&device, &sms);
    if (rc != LITHE_OK) return rc;
    // (14 x 3072 -> 18432: 13.4 us, 18.4 us on the tile kernel; 32 x 3072 -> 18432: 21.7 us and 18.4 us)
    if (!p.q) return launch_rows<kF16, 1, true>(p, sms, false, st);
    if (p.rows <= 8) return launch_rows<kF16, 1, false>(p, sms, after_quantize, st);
    if (p.rows <= 16) return launch_rows<kF16, 2, false>(p, sms, after_quantize, st);
    // A stage takes both kernels equally long, so pairs where their 256 x 256 tiles take fewer passes over the
    // GPU (us, pairs and 128 x 128 tiles: 1024 x 12288 -> 3072, one pass and two, 44 and 68; 1024 x 3072 -> 3072
    // 16.9 and 22.5; 600 x 1000 -> 4000 11.1 and 13.2), and the smaller tiles, whose epilogue is shorter and
    // which use more SMs, where they take as many (512 x 3072 -> 3072 15.4 and 14.3; 1237 x 1898 -> 1091 18.4
    // and 15.9).
    const int64_t pair_tiles = static_cast<int64_t>((p.rows + 255) / 256) * ((p.n + 255) / 256);
    const int64_t tiles = static_cast<int64_t>((p.rows + 127) / 128) * ((p.n + 127) / 128);
    const bool pair = (pair_tiles + sms / 2 - 1) / (sms / 2) < (tiles + sms - 1) / sms;
    if constexpr (!kF16) {
        if (p.h && pair && p.rows_per_sample % 256 == 0 && factor_rows_fit(p))
            return launch_tiles<true, kF16, kExpandTmem>(p, device, sms, after_quantize, st);
        if (p.h) return pair ? launch_tiles<true, kF16, kExpandMma>(p, device, sms, after_quantize, st)
                             : launch_tiles<false, kF16, kExpandMma>(p, device, sms, after_quantize, st);
    }
    return pair ? launch_tiles<true, kF16, kExpandNone>(p, device, sms, after_quantize, st)
                : launch_tiles<false, kF16, kExpandNone>(p, device, sms, after_quantize, st);
}

template <bool kF16, bool kWhole, int kWarps, int kPieces>
void launch_quantize_rows(const QuantParams& p, cudaStream_t st) {
    constexpr int kRowsCta = kThreadsQ / (32 * kWarps);
    const int64_t ctas = (static_cast<int64_t>(p.rows) + kRowsCta - 1) / kRowsCta;
    quantize_kernel<kF16, kWhole, kWarps, kPieces><<<static_cast<int>(ctas), kThreadsQ, 0, st>>>(p);
}

template <bool kF16, bool kWhole>
int32_t launch_quantize(const QuantParams& p, cudaStream_t st) {
    const int pieces = (p.k + 7) / 8;
    const int short_ctas = static_cast<int>((static_cast<int64_t>(p.rows) + kThreadsQ / 32 - 1) / (kThreadsQ / 32));
    // Four warps a row where there are few: up to 2048 rows, up to 1024 of at most 1024 values (us, four warps and
    // one: 256 x 3072 2.3 and 3.4, 2048 x 3072 6.3 and 6.9, 4096 x 3072 9.6 and 9.5, 8192 x 3072 16.8 and 14.9;
    // 2048 x 1536 4.2 and 4.5, 4096 x 1536 6.5 and 6.1; 512 x 1001 2.5 and 2.8, 1024 x 1001 3.1 and 3.0,
    // 2048 x 1001 5.3 and 4.3; 1024 x 576 2.2 and 2.2, 2048 x 576 2.9 and 2.6).
    const bool few = p.rows <= (pieces > 128 ? 2048 : 1024) && pieces > 32 * 2;
    if (!kWhole && p.k <= 32 * 4) quantize_short_kernel<kF16, 4><<<short_ctas, kThreadsQ, 0, st>>>(p);
    else if (!kWhole && p.k <= 32 * kShortMost) quantize_short_kernel<kF16, kShortMost><<<short_ctas, kThreadsQ, 0, st>>>(p);
    else if (few && pieces <= 128 * 2) launch_quantize_rows<kF16, kWhole, 4, 2>(p, st);
    else if (few && pieces <= 128 * 4) launch_quantize_rows<kF16, kWhole, 4, 4>(p, st);
    else if (pieces <= 32 * 2) launch_quantize_rows<kF16, kWhole, 1, 2>(p, st);
    else if (pieces <= 32 * 4) launch_quantize_rows<kF16, kWhole, 1, 4>(p, st);
    else if (pieces <= 32 * 8) launch_quantize_rows<kF16, kWhole, 1, 8>(p, st);
    else if (kWhole && pieces <= 32 * 12) launch_quantize_rows<kF16, kWhole, 1, 12>(p, st);
    else if (pieces <= 64 * 8) launch_quantize_rows<kF16, kWhole, 2, 8>(p, st);
    else if (kWhole && pieces <= 64 * 12) launch_quantize_rows<kF16, kWhole, 2, 12>(p, st);
    else if (pieces <= 128 * 8) launch_quantize_rows<kF16, kWhole, 4, 8>(p, st);
    else if (kWhole && pieces <= 128 * 12) launch_quantize_rows<kF16, kWhole, 4, 12>(p, st);
    else if (kWhole && pieces <= 128 * 16) launch_quantize_rows<kF16, kWhole, 4, 16>(p, st);
    else quantize_long_kernel<kF16, kWhole><<<p.rows, kThreadsQ, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LITHE_OK : fail_cuda(e, "quantize_kernel launch");
}

int32_t check_size(int32_t dtype, int32_t rows, int32_t n, int32_t k) {
    if (dtype != LITHE_DTYPE_BF16 && dtype != LITHE_DTYPE_F16)
        return fail_arg("dtype must be LITHE_DTYPE_BF16 or _F16, got %d", dtype);
    if (rows < 0 || n <= 0 || k <= 0) return fail_arg("rows must be >= 0 and n, k > 0 (rows %d, n %d, k %d)", rows, n, k);
    if (k > kMaxK) return fail_unsupported("k %d above %d: the int32 sums could overflow", k, kMaxK);
    if (rows > kMostRows || n > kMostRows) return fail_unsupported("rows %d or n %d above %d", rows, n, kMostRows);
    return LITHE_OK;
}

int32_t check_bytes(const void* base, int64_t stride, int32_t k, const char* name) {
    if (!base) return fail_arg("%s must be non-NULL", name);
    if (reinterpret_cast<uintptr_t>(base) % 16 || stride % 16 || stride < k)
        return fail_arg("%s: rows must start on 16-byte boundaries, a stride of at least k apart (stride %lld, k %d)",
                        name, static_cast<long long>(stride), k);
    return LITHE_OK;
}

int32_t check_x(const void* x, int64_t x_stride) {
    if (!x || reinterpret_cast<uintptr_t>(x) % 2) return fail_arg("x must be non-NULL and aligned to its elements");
    if (x_stride < 0) return fail_arg("x_stride must be >= 0");
    return LITHE_OK;
}

// The checks of a linear's operands other than its activations; fills p.
int32_t linear_params(Params* p, const void* w, int64_t w_stride, const float* w_scale, const void* bias, void* out,
                      int32_t dtype, int32_t rows, int32_t n, int32_t k, const void* h, const void* b_dec,
                      int32_t rows_per_sample, int32_t rank, int32_t* err_flag) {
    int32_t rc = check_size(dtype, rows, n, k);
    if (rc != LITHE_OK) return rc;
    if (h) {
        if (!b_dec) return fail_arg("b_dec is NULL while h is given");
        if (dtype != LITHE_DTYPE_BF16) return fail_unsupported("the fused expand is bf16");
        if (rank != kRank) return fail_unsupported("the fused expand supports rank %d, got %d", kRank, rank);
        if (rows_per_sample <= 0 || rows % rows_per_sample)
            return fail_arg("rows per sample (%d) must be positive and divide rows (%d)", rows_per_sample, rows);
        if (reinterpret_cast<uintptr_t>(h) % 16 || reinterpret_cast<uintptr_t>(b_dec) % 16)
            return fail_arg("h and b_dec must be 16-byte aligned");
    }
    if (rows == 0) return LITHE_OK;
    if ((rc = check_bytes(w, w_stride, k, "w")) != LITHE_OK) return rc;
    if (!w_scale || !out) return fail_arg("w_scale and out must be non-NULL");
    if (reinterpret_cast<uintptr_t>(w_scale) % 4 || reinterpret_cast<uintptr_t>(out) % 2 ||
        reinterpret_cast<uintptr_t>(bias) % 2)
        return fail_arg("w_scale, bias and out must be aligned to their elements");
    p->w = static_cast<const int8_t*>(w);
    p->w_scale = w_scale;
    p->bias = static_cast<const uint16_t*>(bias);
    p->out = static_cast<uint16_t*>(out);
    p->h = static_cast<const __nv_bfloat16*>(h);
    p->b_dec = static_cast<const __nv_bfloat16*>(b_dec);
    p->err = err_flag;
    p->w_stride = w_stride;
    p->rows = rows;
    p->n = n;
    p->k = k;
    p->rows_per_sample = rows_per_sample;
    return LITHE_OK;
}

int32_t quantize(const QuantParams& p, int32_t dtype, cudaStream_t st) {
    // whole 16-byte pieces of x to whole 8-byte pieces of q
    const bool whole = p.k % 8 == 0 && p.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
    if (dtype == LITHE_DTYPE_F16) return whole ? launch_quantize<true, true>(p, st) : launch_quantize<true, false>(p, st);
    return whole ? launch_quantize<false, true>(p, st) : launch_quantize<false, false>(p, st);
}

// after_quantize: the stream's last launch is the quantisation of these activations.
int32_t linear(const Params& p, int32_t dtype, bool after_quantize, cudaStream_t st) {
    return dtype == LITHE_DTYPE_F16 ? launch_linear<true>(p, after_quantize, st)
                                    : launch_linear<false>(p, after_quantize, st);
}

}  // namespace i8
}  // namespace lithe

extern "C" int32_t lithe_quantize_rows(const void* x, int32_t dtype, int32_t rows, int32_t k, int64_t x_stride,
                                       void* q, int64_t q_stride, float* scale, void* stream) {
    using namespace lithe;
    using namespace lithe::i8;
    clear_error();
    int32_t rc = check_size(dtype, rows, 1, k);
    if (rc != LITHE_OK) return rc;
    if (rows == 0) return LITHE_OK;
    if ((rc = check_x(x, x_stride)) != LITHE_OK) return rc;
    if (!scale || reinterpret_cast<uintptr_t>(scale) % 4)
        return fail_arg("scale must be non-NULL and aligned to its elements");
    if ((rc = check_bytes(q, q_stride, k, "q")) != LITHE_OK) return rc;
    const QuantParams p{static_cast<const uint16_t*>(x), static_cast<int8_t*>(q), scale, x_stride, q_stride, rows, k};
    return quantize(p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int32_t lithe_int8_linear(const void* q, int64_t q_stride, const float* x_scale, const void* w,
                                     int64_t w_stride, const float* w_scale, const void* bias, void* out,
                                     int32_t dtype, int32_t rows, int32_t n, int32_t k, const void* h,
                                     const void* b_dec, int32_t rows_per_sample, int32_t rank, int32_t* err_flag,
                                     void* stream) {
    using namespace lithe;
    using namespace lithe::i8;
    clear_error();
    Params p{};
    int32_t rc = linear_params(&p, w, w_stride, w_scale, bias, out, dtype, rows, n, k, h, b_dec, rows_per_sample, rank,
                               err_flag);
    if (rc != LITHE_OK || rows == 0) return rc;
    if ((rc = check_bytes(q, q_stride, k, "q")) != LITHE_OK) return rc;
    if (!x_scale || reinterpret_cast<uintptr_t>(x_scale) % 4)
        return fail_arg("x_scale must be non-NULL and aligned to its elements");
    p.q = static_cast<const int8_t*>(q);
    p.q_stride = q_stride;
    p.x_scale = x_scale;
    return linear(p, dtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t lithe_int8_workspace_bytes(int32_t rows, int32_t k) {
    if (rows <= 0 || k <= 0) return 0;
    return static_cast<int64_t>(rows) * ((static_cast<int64_t>(k) + 15) / 16 * 16 + 4);
}

extern "C" int32_t lithe_int8_linear_dynamic(const void* x, int64_t x_stride, const void* w, int64_t w_stride,
                                             const float* w_scale, const void* bias, void* out, int32_t dtype,
                                             int32_t rows, int32_t n, int32_t k, const void* h, const void* b_dec,
                                             int32_t rows_per_sample, int32_t rank, int32_t* err_flag,
                                             void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace lithe;
    using namespace lithe::i8;
    clear_error();
    Params p{};
    int32_t rc = linear_params(&p, w, w_stride, w_scale, bias, out, dtype, rows, n, k, h, b_dec, rows_per_sample, rank,
                               err_flag);
    if (rc != LITHE_OK || rows == 0) return rc;
    if ((rc = check_x(x, x_stride)) != LITHE_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    p.x = static_cast<const uint16_t*>(x);
    if (direct_row(p)) return linear(p, dtype, false, st);
    const int64_t need = lithe_int8_workspace_bytes(rows, k);
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need)
        return fail_arg("workspace must be 16-byte aligned and hold %lld bytes, got %lld", static_cast<long long>(need),
                        static_cast<long long>(workspace_bytes));
    const int64_t q_stride = (static_cast<int64_t>(k) + 15) / 16 * 16;
    int8_t* q = static_cast<int8_t*>(workspace);
    float* scale = reinterpret_cast<float*>(q + rows * q_stride);
    rc = quantize(QuantParams{static_cast<const uint16_t*>(x), q, scale, x_stride, q_stride, rows, k}, dtype, st);
    if (rc != LITHE_OK) return rc;
    p.q = q;
    p.q_stride = q_stride;
    p.x_scale = scale;
    return linear(p, dtype, true, st);
}
