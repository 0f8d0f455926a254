// Dropout of a series from a counter-based generator, with an optional residual:
//   y_k = residual_k + keep * scale * x_k   for every plane k, one mask for all planes.
// The mask is never stored: element i (row-major) is kept when word i % 4 of
// Philox4x32-10(counter = (i / 4, offset), key = seed) is at least `threshold`, so the backward
// (y with the gradient as x) forms it again.  Philox4x32-10: J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011.
// A dropped element is 0 whatever x holds there (NaN and infinities included).  scale * x + residual
// is formed in float (double for float64 planes) and rounded once, when it is stored.
#include <algorithm>

#include "pk_vec.cuh"

namespace pk {

struct DropoutParams {
    const void* x[PK_MAX_PLANES];
    const void* residual[PK_MAX_PLANES];
    void* y[PK_MAX_PLANES];
    int np, nx, nr;          // planes of y, x and the residual (missing ones are zero)
    int64_t n;               // elements of a plane
    uint64_t seed, offset;
    uint32_t threshold;      // (a threshold of 2^32 drops everything: nx is 0 then)
    double scale;
};

// Philox4x32-10 of the counter (i, offset), i of 64 or (HIGH false) of 32 bits.  The second product of the first
// round, and with 32-bit i the first of the second, are the same for all threads of a launch.
template <bool HIGH>
__device__ __forceinline__ uint4 philox4x32_10(uint64_t i, uint64_t offset, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(i), c1 = HIGH ? static_cast<uint32_t>(i >> 32) : 0u;
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0, b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Planes whose bases lie on no 16-byte boundary, and more than 2^34 elements: one thread per counter (four consecutive
// elements); 8192 x 4096 degree 0 one element past such a boundary: float32 85 us, bfloat16 69 (53 and 45 on one).
template <typename T>
__global__ void __launch_bounds__(256) dropout_scalar_kernel(const DropoutParams p) {
    using C = typename Compute<T>::type;
    const C scale = C(p.scale);
    const int64_t groups = (p.n + 3) / 4;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < groups;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const uint4 words = philox4x32_10<true>(static_cast<uint64_t>(i), p.offset, p.seed);
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
        for (int k = 0; k < p.np; ++k) {
            for (int u = 0; u < 4; ++u) {
                const int64_t e = 4 * i + u;
                if (e >= p.n) break;
                C v = C(0);
                if (k < p.nx && word[u] >= p.threshold) v = to_c<C>(static_cast<const T*>(p.x[k])[e]) * scale;
                if (k < p.nr) v += to_c<C>(static_cast<const T*>(p.residual[k])[e]);
                static_cast<T*>(p.y[k])[e] = from_c<T>(v);
            }
        }
    }
}

// Elements of a thread: whole counters, and vectors of 16 bytes.
template <typename T>
constexpr int dropout_unit() { return sizeof(T) == 2 ? 8 : 4; }

// Vector form: a thread asks for its 16-byte vectors of every plane of x and the residual, forms their counters'
// words while they are on the way (twenty 32 x 32 -> 64-bit products for four elements, whatever the
// degree), and writes.  Measured on B200, device time, without a residual: 8192 x 4096 float32 degree 3 159 us
// = 6.8 TB/s and float64 degree 0 80 us = 6.7 TB/s, the rate of a copy; bfloat16 degree 3 84 us = 6.4 TB/s.  At
// degree 0 the instructions are the limit for 16-bit planes: 46 us = 2.9 TB/s, where the bytes alone would take
// 21 us (74 % of the issue slots, the integer pipe 47 %, the multiplier's 38 %; of 237 instructions per eight elements
// the generator has about 90, the rest is conversion, masking and addresses).
template <typename T, int NP>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const __grid_constant__ DropoutParams p) {
    using C = typename Compute<T>::type;
    constexpr int UNIT = dropout_unit<T>(), VEC = 16 / sizeof(T), PARTS = UNIT / VEC, WORDS = UNIT / 4;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t first = i * UNIT;
    if (first >= p.n) return;
    const bool whole = first + UNIT <= p.n;
    Raw<T, VEC> x[NP][PARTS], r[NP][PARTS];
    if (whole) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
#pragma unroll
            for (int v = 0; v < PARTS; ++v) {
                if (k < p.nx) x[k][v] = *reinterpret_cast<const Raw<T, VEC>*>(static_cast<const T*>(p.x[k]) + first + v * VEC);
                if (k < p.nr) r[k][v] = *reinterpret_cast<const Raw<T, VEC>*>(static_cast<const T*>(p.residual[k]) + first + v * VEC);
            }
        }
    }
    uint32_t word[UNIT];
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        const uint4 q = philox4x32_10<false>(static_cast<uint64_t>(i) * WORDS + w, p.offset, p.seed);
        word[4 * w] = q.x;
        word[4 * w + 1] = q.y;
        word[4 * w + 2] = q.z;
        word[4 * w + 3] = q.w;
    }
    const C scale = C(p.scale);
    if (!whole) {                     // the last elements
        for (int k = 0; k < p.np; ++k) {
#pragma unroll
            for (int u = 0; u < UNIT; ++u) {
                if (first + u >= p.n) break;
                C v = C(0);
                if (k < p.nx && word[u] >= p.threshold) v = to_c<C>(static_cast<const T*>(p.x[k])[first + u]) * scale;
                if (k < p.nr) v += to_c<C>(static_cast<const T*>(p.residual[k])[first + u]);
                static_cast<T*>(p.y[k])[first + u] = from_c<T>(v);
            }
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        if (NP > 6 && k >= p.np) continue;
#pragma unroll
        for (int v = 0; v < PARTS; ++v) {
            Raw<T, VEC> out;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                C a = C(0), b = C(0), c = C(0), d = C(0);
                if (k < p.nx) x[k][v].get(j).get(a, b);
                if (k < p.nr) r[k][v].get(j).get(c, d);
                a = word[v * VEC + 2 * j] >= p.threshold ? a : C(0);
                b = word[v * VEC + 2 * j + 1] >= p.threshold ? b : C(0);
                out.set(j, fma2(Two<C>(a, b), Two<C>(scale), Two<C>(c, d)));
            }
            *reinterpret_cast<Raw<T, VEC>*>(static_cast<T*>(p.y[k]) + first + v * VEC) = out;
        }
    }
}

template <typename T, int NP>
static void launch_dropout_vec(const DropoutParams& p, cudaStream_t s) {
    const int64_t blocks = ceil_div(ceil_div(p.n, dropout_unit<T>()), 256);
    PK_LAUNCHED(dropout_vec_kernel<T, NP><<<static_cast<unsigned>(blocks), 256, 0, s>>>(p));
}

template <typename T>
static void launch_dropout(const DropoutParams& p, cudaStream_t s) {
    const bool aligned = planes_aligned(p.x, p.nx, 16) && planes_aligned(p.residual, p.nr, 16) && planes_aligned(p.y, p.np, 16);
    if (!aligned || p.n > (1ll << 34)) {
        const int64_t groups = ceil_div(p.n, 4);
        const int grid = static_cast<int>(std::min<int64_t>(ceil_div(groups, 256), static_cast<int64_t>(num_sms()) * 32));
        PK_LAUNCHED(dropout_scalar_kernel<T><<<grid, 256, 0, s>>>(p));
        return;
    }
    switch (p.np) {
        case 1: launch_dropout_vec<T, 1>(p, s); break;
        case 2: launch_dropout_vec<T, 2>(p, s); break;
        case 3: launch_dropout_vec<T, 3>(p, s); break;
        case 4: launch_dropout_vec<T, 4>(p, s); break;
        case 5: launch_dropout_vec<T, 5>(p, s); break;
        case 6: launch_dropout_vec<T, 6>(p, s); break;
        case 7: case 8: case 9: launch_dropout_vec<T, 9>(p, s); break;
        default: launch_dropout_vec<T, 16>(p, s); break;
    }
}

}  // namespace pk

using namespace pk;

extern "C" int pk_dropout(int dtype, int degree, int64_t n, const void* const* x, int x_planes,
                          const void* const* residual, int residual_planes, uint64_t threshold, double scale,
                          uint64_t seed, uint64_t offset, void* const* y, void* stream) {
    if (dtype != PK_F32 && dtype != PK_F64 && dtype != PK_BF16 && dtype != PK_F16)
        return fail(PK_ERR_UNSUPPORTED, "pk_dropout: unsupported dtype");
    if (degree < 0 || degree >= PK_MAX_PLANES) return fail(PK_ERR_UNSUPPORTED, "pk_dropout: degree out of range");
    if (n < 0) return fail(PK_ERR_ARG, "pk_dropout: negative extent");
    if (threshold > (1ull << 32)) return fail(PK_ERR_ARG, "pk_dropout: threshold beyond 2^32");
    DropoutParams p{};
    p.np = degree + 1;
    if (x_planes < 1 || x_planes > p.np || residual_planes < 0 || residual_planes > p.np)
        return fail(PK_ERR_ARG, "pk_dropout: bad plane count");
    if (!x || !y || (residual_planes && !residual)) return fail(PK_ERR_ARG, "pk_dropout: null plane array");
    if (n == 0) return PK_OK;
    p.nx = threshold >> 32 ? 0 : x_planes;
    p.nr = residual_planes;
    p.n = n;
    p.seed = seed;
    p.offset = offset;
    p.threshold = static_cast<uint32_t>(threshold);
    p.scale = scale;
    for (int k = 0; k < p.np; ++k) {
        if (k < p.nx) p.x[k] = x[k];
        if (k < p.nr) p.residual[k] = residual[k];
        p.y[k] = y[k];
        if ((k < p.nx && !p.x[k]) || (k < p.nr && !p.residual[k]) || !p.y[k])
            return fail(PK_ERR_ARG, "pk_dropout: null plane");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* tok;
    prof_begin("dropout", s, &tok);
    switch (dtype) {
        case PK_F32: launch_dropout<float>(p, s); break;
        case PK_F64: launch_dropout<double>(p, s); break;
        case PK_BF16: launch_dropout<__nv_bfloat16>(p, s); break;
        default: launch_dropout<__half>(p, s); break;
    }
    prof_end("dropout", s, tok);
    PK_CHECK_LAUNCH("pk_dropout");
    return PK_OK;
}
