// Dropout of a series from a counter-based generator, with an optional residual:
//   y_k = residual_k + keep * scale * x_k   for every plane k, one mask for all planes.
// The mask is never stored: element i (row-major) is kept when word i % 4 of
// Philox4x32-10(counter = (i / 4, offset), key = seed) is at least `threshold`, so the backward
// (y with the gradient as x) forms it again.  Philox4x32-10: J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011.
// A dropped element is 0 whatever x holds there (NaN and infinities included).  scale * x + residual
// is formed in float (double for float64 planes) and rounded once, when it is stored.
#include <algorithm>

#include "pk_rows.cuh"

namespace pk {

struct DropoutParams {
    const void* x[PK_MAX_PLANES];
    const void* residual[PK_MAX_PLANES];
    void* y[PK_MAX_PLANES];
    int np, nx, nr;          // planes of y, x and the residual (missing ones are zero)
    int64_t n;               // elements of a plane
    uint64_t seed, offset;
    uint64_t threshold;      // 0 .. 2^32
    double scale;
};

__device__ __forceinline__ uint4 philox4x32_10(uint64_t counter, uint64_t offset, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32);
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

// One thread per counter (four consecutive elements) and step, all planes.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutParams p) {
    using C = typename Compute<T>::type;
    const C scale = C(p.scale);
    const int64_t groups = (p.n + 3) / 4;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < groups;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const uint4 words = philox4x32_10(static_cast<uint64_t>(i), p.offset, p.seed);
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

template <typename T>
static void launch_dropout(const DropoutParams& p, cudaStream_t s) {
    const int64_t groups = ceil_div(p.n, 4);
    const int grid = static_cast<int>(std::min<int64_t>(ceil_div(groups, 256), static_cast<int64_t>(num_sms()) * 32));
    PK_LAUNCHED(dropout_kernel<T><<<grid, 256, 0, s>>>(p));
}

}  // namespace pk

using namespace pk;

extern "C" int pk_dropout(int dtype, int degree, int64_t n, const void* const* x, int x_planes,
                          const void* const* residual, int residual_planes, uint64_t threshold, double scale,
                          uint64_t seed, uint64_t offset, void* const* y, void* stream) {
    if (degree < 0 || degree >= PK_MAX_PLANES) return fail(PK_ERR_UNSUPPORTED, "pk_dropout: degree out of range");
    if (n < 0) return fail(PK_ERR_ARG, "pk_dropout: negative extent");
    if (threshold > (1ull << 32)) return fail(PK_ERR_ARG, "pk_dropout: threshold beyond 2^32");
    DropoutParams p{};
    p.np = degree + 1;
    if (x_planes < 1 || x_planes > p.np || residual_planes < 0 || residual_planes > p.np)
        return fail(PK_ERR_ARG, "pk_dropout: bad plane count");
    if (!x || !y || (residual_planes && !residual)) return fail(PK_ERR_ARG, "pk_dropout: null plane array");
    if (n == 0) return PK_OK;
    p.nx = x_planes;
    p.nr = residual_planes;
    p.n = n;
    p.seed = seed;
    p.offset = offset;
    p.threshold = threshold;
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
        case PK_F16: launch_dropout<__half>(p, s); break;
        default: return fail(PK_ERR_UNSUPPORTED, "pk_dropout: unsupported dtype");
    }
    prof_end("dropout", s, tok);
    PK_CHECK_LAUNCH("pk_dropout");
    return PK_OK;
}
