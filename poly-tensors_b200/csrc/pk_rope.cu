// Per-head RMS norm of queries and keys with the position rotation in the same pass.
//
// One row is one head of one token, D features, n+1 planes; (*) is the truncated series product:
//   s = mean(x (*) x) + eps,  r = s^(-1/2),  v = x (*) r (*) w,  y = R(position) v.
// R turns the pairs of the first `rotary` features (feature j with j + rotary/2, or the adjacent
// features 2j and 2j+1) by the angle whose cosine and sine the caller's tables hold for that
// position; the other features pass.  R acts on every plane alike, its transpose is its inverse.
// Backward, with g' = R^T g, gy = g' (*) w and c = mean(x (*) gy):
//   dx = gy (*) r - x (*) (r (*) r (*) r (*) c),   dw = sum over rows of g' (*) (x (*) r).
// x is [batch][token][head][feature] with unit feature stride, y is [batch][head][token][feature]:
// what attention reads next, so that no copy stands between the two.
//
// Sums, means and the series r are held in float (double for float64 planes); y, dx and dw are
// rounded once, when they are stored.
#include <algorithm>

#include "pk_rows.cuh"

namespace pk {

struct HeadSet {                        // the queries or the keys
    const void* x[PK_MAX_PLANES];       // forward input
    const void* g[PK_MAX_PLANES];       // gradient of y (backward)
    const void* w[PK_MAX_PLANES];       // feature weights, nw planes (0: no weight)
    void* out[PK_MAX_PLANES];           // y [b][h][t][d] (forward) or dx [b][t][h][d] (backward)
    int64_t bs, ts, hs;                 // strides of x
    int64_t g_bs, g_hs, g_ts;           // strides of g
    int64_t heads;
    int nw;
    void* partial;                      // backward: [blocks][nw][D] weight-gradient sums, or null
};

struct RopeParams {
    HeadSet set[2];                     // queries, keys
    int np;
    int64_t batch, len, dim;
    int rotary, interleaved;
    const void* cos_t;                  // [table_rows][rotary / 2], compute type
    const void* sin_t;
    int64_t table_rows;
    const int64_t* positions;           // [b * pos_bs + t], or null: position t
    int64_t pos_bs;
    double eps;
};

// The two features of slot i: rotated pairs first, then the passing features two by two (the second
// one missing at the end of an odd count: hi = -1).
__device__ __forceinline__ void slot_features(const RopeParams& p, int i, int& lo, int& hi, bool& turned) {
    const int pairs = p.rotary / 2;
    turned = i < pairs;
    if (turned) {
        lo = p.interleaved ? 2 * i : i;
        hi = p.interleaved ? 2 * i + 1 : i + pairs;
    } else {
        lo = p.rotary + 2 * (i - pairs);
        hi = lo + 1 < p.dim ? lo + 1 : -1;
    }
}

// Angle of slot i at table row `pos`; a position outside the table gives NaN (never another row's angle).
template <typename C>
__device__ __forceinline__ void slot_angle(const RopeParams& p, int64_t pos, int i, bool turned, C& c, C& s) {
    c = C(1);
    s = C(0);
    if (pos < 0 || pos >= p.table_rows) {
        c = s = C(NAN);
    } else if (turned) {
        c = static_cast<const C*>(p.cos_t)[pos * (p.rotary / 2) + i];
        s = static_cast<const C*>(p.sin_t)[pos * (p.rotary / 2) + i];
    }
}

template <int NP, typename T, typename C>
__device__ __forceinline__ void load_series(const void* const* planes, int np, int64_t off, bool valid, C (&x)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) x[k] = (valid && k < np) ? to_c<C>(static_cast<const T*>(planes[k])[off]) : C(0);
}

template <int NP, typename C>
__device__ __forceinline__ void warp_sum(C (&v)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
}

// Where row `row` of the flat (batch, token, head) order lies: the query heads of a token come first.
struct RowAt {
    int which;
    int64_t b, t, h;
};
__device__ __forceinline__ RowAt row_at(const RopeParams& p, int64_t row) {
    const int64_t all = p.set[0].heads + p.set[1].heads;
    const int64_t token = row / all;
    int64_t h = row - token * all;
    const int which = h >= p.set[0].heads ? 1 : 0;
    if (which) h -= p.set[0].heads;
    return {which, token / p.len, token % p.len, h};
}

__device__ __forceinline__ int64_t position_of(const RopeParams& p, int64_t b, int64_t t) {
    return p.positions ? p.positions[b * p.pos_bs + t] : t;
}

// One warp per row, one pair of features per lane and step, the row read twice.
template <typename T, int NP>
__global__ void __launch_bounds__(256) qk_norm_rope_fwd_kernel(const RopeParams p) {
    using C = typename Compute<T>::type;
    const int lane = threadIdx.x & 31;
    const int64_t rows = p.batch * p.len * (p.set[0].heads + p.set[1].heads);
    const int slots = p.rotary / 2 + static_cast<int>((p.dim - p.rotary + 1) / 2);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); row < rows;
         row += static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5)) {
        const RowAt at = row_at(p, row);
        const HeadSet& set = p.set[at.which];
        const int64_t xb = at.b * set.bs + at.t * set.ts + at.h * set.hs;
        const int64_t yb = ((at.b * set.heads + at.h) * p.len + at.t) * p.dim;
        const int64_t pos = position_of(p, at.b, at.t);
        C cross[NP] = {}, diag[NP] = {};
        for (int i = lane; i < slots; i += 32) {
            int lo, hi;
            bool turned;
            slot_features(p, i, lo, hi, turned);
            C x[NP];
            load_series<NP, T, C>(set.x, p.np, xb + lo, true, x);
            s_square_acc<NP, C>(x, cross, diag);
            load_series<NP, T, C>(set.x, p.np, xb + hi, hi >= 0, x);
            s_square_acc<NP, C>(x, cross, diag);
        }
        C s[NP], r[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) s[k] = C(2) * cross[k] + diag[k];
        warp_sum<NP, C>(s);
#pragma unroll
        for (int k = 0; k < NP; ++k) s[k] /= C(p.dim);
        s[0] += C(p.eps);
        s_rsqrt<NP, C>(s, r);
        for (int i = lane; i < slots; i += 32) {
            int lo, hi;
            bool turned;
            slot_features(p, i, lo, hi, turned);
            C a[NP], b[NP], w[NP], c, sn;
            load_series<NP, T, C>(set.x, p.np, xb + lo, true, a);
            load_series<NP, T, C>(set.x, p.np, xb + hi, hi >= 0, b);
            s_mul<NP, C>(a, r, a);
            s_mul<NP, C>(b, r, b);
            if (set.nw) {
                load_series<NP, T, C>(set.w, set.nw, lo, true, w);
                s_mul<NP, C>(a, w, a);
                load_series<NP, T, C>(set.w, set.nw, hi, hi >= 0, w);
                s_mul<NP, C>(b, w, b);
            }
            slot_angle<C>(p, pos, i, turned, c, sn);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if (k >= p.np) continue;
                T* y = static_cast<T*>(set.out[k]) + yb;
                y[lo] = from_c<T>(a[k] * c - b[k] * sn);
                if (hi >= 0) y[hi] = from_c<T>(b[k] * c + a[k] * sn);
            }
        }
    }
}

// The gradient of slot i turned back: (ga, gb) = R^T (g_lo, g_hi).
template <int NP, typename T, typename C>
__device__ __forceinline__ void load_turned_back(const RopeParams& p, const HeadSet& set, int64_t gb, int64_t pos, int i,
                                                 int lo, int hi, bool turned, C (&a)[NP], C (&b)[NP]) {
    C c, s;
    load_series<NP, T, C>(set.g, p.np, gb + lo, true, a);
    load_series<NP, T, C>(set.g, p.np, gb + hi, hi >= 0, b);
    slot_angle<C>(p, pos, i, turned, c, s);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const C u = a[k] * c + b[k] * s, v = b[k] * c - a[k] * s;
        a[k] = u;
        b[k] = v;
    }
}

// One warp per row of the queries (the first q_blocks blocks) or of the keys.  The weight gradient is
// summed over a warp's rows in its own shared-memory planes, over the block's warps at the end, and
// over the blocks by the kernel below: a fixed order, so that runs agree bit for bit.
template <typename T, int NP>
__global__ void __launch_bounds__(256) qk_norm_rope_bwd_kernel(const RopeParams p, int q_blocks) {
    using C = typename Compute<T>::type;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int which = static_cast<int>(blockIdx.x) >= q_blocks ? 1 : 0;
    const HeadSet& set = p.set[which];
    const int64_t block = which ? blockIdx.x - q_blocks : blockIdx.x;
    const int64_t blocks = which ? gridDim.x - q_blocks : q_blocks;
    const int dim = static_cast<int>(p.dim);
    const int64_t rows = p.batch * p.len * set.heads;
    const int slots = p.rotary / 2 + (dim - p.rotary + 1) / 2;
    C* sums = reinterpret_cast<C*>(smem) + static_cast<int64_t>(warp) * set.nw * dim;
    if (set.partial)
        for (int i = lane; i < set.nw * dim; i += 32) sums[i] = C(0);
    __syncwarp();
    for (int64_t row = block * warps + warp; row < rows; row += blocks * warps) {
        const int64_t token = row / set.heads, h = row - token * set.heads, b = token / p.len, t = token % p.len;
        const int64_t xb = b * set.bs + t * set.ts + h * set.hs;
        const int64_t gb = b * set.g_bs + h * set.g_hs + t * set.g_ts;
        const int64_t ob = row * dim;
        const int64_t pos = position_of(p, b, t);
        C cross[NP] = {}, diag[NP] = {}, m[NP] = {};
        for (int i = lane; i < slots; i += 32) {
            int lo, hi;
            bool turned;
            slot_features(p, i, lo, hi, turned);
            C ga[NP], gv[NP], x[NP], w[NP];
            load_turned_back<NP, T, C>(p, set, gb, pos, i, lo, hi, turned, ga, gv);
            load_series<NP, T, C>(set.x, p.np, xb + lo, true, x);
            s_square_acc<NP, C>(x, cross, diag);
            if (set.nw) {
                load_series<NP, T, C>(set.w, set.nw, lo, true, w);
                s_mul<NP, C>(ga, w, ga);
            }
            s_mul_acc<NP, C>(x, ga, m);
            load_series<NP, T, C>(set.x, p.np, xb + hi, hi >= 0, x);
            s_square_acc<NP, C>(x, cross, diag);
            if (set.nw) {
                load_series<NP, T, C>(set.w, set.nw, hi, hi >= 0, w);
                s_mul<NP, C>(gv, w, gv);
            }
            s_mul_acc<NP, C>(x, gv, m);
        }
        C s[NP], r[NP], q[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) s[k] = C(2) * cross[k] + diag[k];
        warp_sum<NP, C>(s);
        warp_sum<NP, C>(m);
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            s[k] /= C(dim);
            m[k] /= C(dim);
        }
        s[0] += C(p.eps);
        s_rsqrt<NP, C>(s, r);
        s_mul<NP, C>(r, r, q);
        s_mul<NP, C>(q, r, q);
        s_mul<NP, C>(q, m, q);
        for (int i = lane; i < slots; i += 32) {
            int lo, hi;
            bool turned;
            slot_features(p, i, lo, hi, turned);
            C ga[2][NP];
            load_turned_back<NP, T, C>(p, set, gb, pos, i, lo, hi, turned, ga[0], ga[1]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int f = half ? hi : lo;
                if (f < 0) continue;
                C x[NP], u[NP], w[NP];
                load_series<NP, T, C>(set.x, p.np, xb + f, true, x);
                if (set.partial) {
                    s_mul<NP, C>(x, r, u);
                    s_mul<NP, C>(ga[half], u, u);
#pragma unroll
                    for (int k = 0; k < NP; ++k)
                        if (k < set.nw) sums[k * dim + f] += u[k];
                }
                if (set.nw) {
                    load_series<NP, T, C>(set.w, set.nw, f, true, w);
                    s_mul<NP, C>(ga[half], w, ga[half]);
                }
                s_mul<NP, C>(ga[half], r, u);
                s_sub_mul<NP, C>(u, x, q, u);
#pragma unroll
                for (int k = 0; k < NP; ++k)
                    if (k < p.np) static_cast<T*>(set.out[k])[ob + f] = from_c<T>(u[k]);
            }
        }
    }
    if (set.partial) {
        __syncthreads();
        const C* all = reinterpret_cast<const C*>(smem);
        for (int i = threadIdx.x; i < set.nw * dim; i += blockDim.x) {
            C acc = C(0);
            for (int v = 0; v < warps; ++v) acc += all[static_cast<int64_t>(v) * set.nw * dim + i];
            static_cast<C*>(set.partial)[block * set.nw * dim + i] = acc;
        }
    }
}

struct WeightSumParams {
    const void* partial;   // [blocks][nw][D]
    void* dw[PK_MAX_PLANES];
    int64_t blocks;
    int nw, dim;
};

template <typename T>
__global__ void __launch_bounds__(256) qk_weight_sum_kernel(const WeightSumParams p) {
    using C = typename Compute<T>::type;
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= p.nw * p.dim) return;
    C acc = C(0);
    for (int64_t b = 0; b < p.blocks; ++b) acc += static_cast<const C*>(p.partial)[b * p.nw * p.dim + i];
    static_cast<T*>(p.dw[i / p.dim])[i % p.dim] = from_c<T>(acc);
}

constexpr int ROPE_MAX_DIM = 1024;

static int compute_bytes(int dtype) { return dtype == PK_F64 ? 8 : 4; }

// Backward launch shape: warps per block so that their weight-gradient planes fit in shared memory,
// and the blocks of the queries and of the keys in proportion to their rows.
struct BwdShape {
    int warps, q_blocks, k_blocks;
    size_t smem;
};
static BwdShape bwd_shape(int dtype, int64_t q_rows, int64_t k_rows, int64_t dim, int planes) {
    BwdShape s{};
    const size_t per_warp = static_cast<size_t>(planes) * dim * compute_bytes(dtype);
    s.warps = 8;
    while (s.warps > 1 && s.warps * per_warp > 96 * 1024) s.warps /= 2;
    s.smem = s.warps * per_warp;
    const int64_t room = static_cast<int64_t>(num_sms()) * 4;
    const auto blocks = [&](int64_t rows) {
        if (rows == 0) return static_cast<int64_t>(0);
        const int64_t share = std::max<int64_t>(1, room * rows / (q_rows + k_rows));
        return std::min<int64_t>(share, ceil_div(rows, s.warps));
    };
    s.q_blocks = static_cast<int>(blocks(q_rows));
    s.k_blocks = static_cast<int>(blocks(k_rows));
    return s;
}

template <typename T, int NP>
static void launch_rope_fwd(const RopeParams& p, cudaStream_t s) {
    const int64_t rows = p.batch * p.len * (p.set[0].heads + p.set[1].heads);
    const int grid = static_cast<int>(std::min<int64_t>(ceil_div(rows, 8), static_cast<int64_t>(num_sms()) * 32));
    PK_LAUNCHED(qk_norm_rope_fwd_kernel<T, NP><<<grid, 256, 0, s>>>(p));
}

template <typename T, int NP>
static void launch_rope_bwd(const RopeParams& p, const BwdShape& shape, cudaStream_t s) {
    if (shape.smem > 48 * 1024)
        cudaFuncSetAttribute(qk_norm_rope_bwd_kernel<T, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(shape.smem));
    PK_LAUNCHED(qk_norm_rope_bwd_kernel<T, NP>
                <<<shape.q_blocks + shape.k_blocks, shape.warps * 32, shape.smem, s>>>(p, shape.q_blocks));
}

template <typename T>
static void launch_rope(const RopeParams& p, const BwdShape* shape, cudaStream_t s) {
#define PK_ROPE_CASE(NP) \
    if (shape) launch_rope_bwd<T, NP>(p, *shape, s); \
    else launch_rope_fwd<T, NP>(p, s); \
    break
    switch (p.np) {
        case 1: PK_ROPE_CASE(1);
        case 2: PK_ROPE_CASE(2);
        case 3: PK_ROPE_CASE(3);
        case 4: PK_ROPE_CASE(4);
        case 5: PK_ROPE_CASE(5);
        case 6: PK_ROPE_CASE(6);
        case 7: case 8: case 9: PK_ROPE_CASE(9);
        default: PK_ROPE_CASE(16);
    }
#undef PK_ROPE_CASE
}

static int launch_rope_dtype(int dtype, const RopeParams& p, const BwdShape* shape, cudaStream_t s, const char* what) {
    switch (dtype) {
        case PK_F32: launch_rope<float>(p, shape, s); break;
        case PK_F64: launch_rope<double>(p, shape, s); break;
        case PK_BF16: launch_rope<__nv_bfloat16>(p, shape, s); break;
        case PK_F16: launch_rope<__half>(p, shape, s); break;
        default: return fail(PK_ERR_UNSUPPORTED, std::string(what) + ": unsupported dtype");
    }
    return PK_OK;
}

static int check_planes(const void* const* planes, int n, const char* what) {
    if (!planes) return fail(PK_ERR_ARG, std::string(what) + ": null plane array");
    for (int k = 0; k < n; ++k)
        if (!planes[k]) return fail(PK_ERR_ARG, std::string(what) + ": null plane");
    return PK_OK;
}

static int check_rope(int dtype, int degree, int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads, int64_t dim,
                      int64_t rotary, const void* cos_t, const void* sin_t, int64_t table_rows, const char* what) {
    const std::string w(what);
    if (dtype != PK_F32 && dtype != PK_F64 && dtype != PK_BF16 && dtype != PK_F16)
        return fail(PK_ERR_UNSUPPORTED, w + ": unsupported dtype");
    if (degree < 0 || degree >= PK_MAX_PLANES) return fail(PK_ERR_UNSUPPORTED, w + ": degree out of range");
    if (batch < 0 || len < 0 || q_heads < 0 || k_heads < 0) return fail(PK_ERR_ARG, w + ": negative extent");
    if (dim < 1 || dim > ROPE_MAX_DIM) return fail(PK_ERR_UNSUPPORTED, w + ": head dimension out of range");
    if (rotary < 0 || rotary > dim || rotary % 2) return fail(PK_ERR_ARG, w + ": bad rotary dimension");
    if (table_rows < 0 || (rotary > 0 && table_rows > 0 && (!cos_t || !sin_t)))
        return fail(PK_ERR_ARG, w + ": null angle table");
    return PK_OK;
}

}  // namespace pk

using namespace pk;

extern "C" {

int pk_qk_norm_rope_fwd(int dtype, int degree, int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads,
                        int64_t dim, int64_t rotary, int interleaved, const void* const* q, int64_t q_bs,
                        int64_t q_ts, int64_t q_hs, const void* const* k, int64_t k_bs, int64_t k_ts, int64_t k_hs,
                        const void* const* qw, int qw_planes, const void* const* kw, int kw_planes,
                        const void* cos_t, const void* sin_t, int64_t table_rows, const int64_t* positions,
                        int64_t pos_bs, double eps, void* const* q_out, void* const* k_out, void* stream) {
    const char* what = "pk_qk_norm_rope_fwd";
    if (int rc = check_rope(dtype, degree, batch, len, q_heads, k_heads, dim, rotary, cos_t, sin_t, table_rows, what))
        return rc;
    const int np = degree + 1;
    if (qw_planes < 0 || qw_planes > np || kw_planes < 0 || kw_planes > np)
        return fail(PK_ERR_ARG, "pk_qk_norm_rope_fwd: bad weight plane count");
    if (batch == 0 || len == 0 || q_heads + k_heads == 0) return PK_OK;
    RopeParams p{};
    p.np = np;
    p.batch = batch;
    p.len = len;
    p.dim = dim;
    p.rotary = static_cast<int>(rotary);
    p.interleaved = interleaved != 0;
    p.cos_t = cos_t;
    p.sin_t = sin_t;
    p.table_rows = table_rows;
    p.positions = positions;
    p.pos_bs = pos_bs;
    p.eps = eps;
    const void* const* x[2] = {q, k};
    const void* const* w[2] = {qw, kw};
    void* const* out[2] = {q_out, k_out};
    const int nw[2] = {qw_planes, kw_planes};
    const int64_t heads[2] = {q_heads, k_heads};
    const int64_t strides[2][3] = {{q_bs, q_ts, q_hs}, {k_bs, k_ts, k_hs}};
    for (int i = 0; i < 2; ++i) {
        HeadSet& s = p.set[i];
        s.heads = heads[i];
        if (heads[i] == 0) continue;
        if (int rc = check_planes(x[i], np, what)) return rc;
        if (int rc = check_planes(out[i], np, what)) return rc;
        if (nw[i])
            if (int rc = check_planes(w[i], nw[i], what)) return rc;
        s.bs = strides[i][0];
        s.ts = strides[i][1];
        s.hs = strides[i][2];
        s.nw = nw[i];
        for (int j = 0; j < np; ++j) {
            s.x[j] = x[i][j];
            s.out[j] = out[i][j];
        }
        for (int j = 0; j < nw[i]; ++j) s.w[j] = w[i][j];
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* tok;
    prof_begin("qk_norm_rope_fwd", s, &tok);
    const int rc = launch_rope_dtype(dtype, p, nullptr, s, what);
    prof_end("qk_norm_rope_fwd", s, tok);
    if (rc) return rc;
    PK_CHECK_LAUNCH(what);
    return PK_OK;
}

size_t pk_qk_norm_rope_bwd_workspace_size(int dtype, int degree, int64_t batch, int64_t len, int64_t q_heads,
                                          int64_t k_heads, int64_t dim, int dqw_planes, int dkw_planes) {
    if (check_rope(dtype, degree, batch, len, q_heads, k_heads, dim, 0, nullptr, nullptr, 0,
                   "pk_qk_norm_rope_bwd_workspace_size"))
        return 0;
    if (dqw_planes < 0 || dqw_planes > degree + 1 || dkw_planes < 0 || dkw_planes > degree + 1) return 0;
    const BwdShape s = bwd_shape(dtype, batch * len * q_heads, batch * len * k_heads, dim,
                                 std::max(dqw_planes, dkw_planes));
    return static_cast<size_t>(s.q_blocks * dqw_planes + s.k_blocks * dkw_planes) * dim * compute_bytes(dtype);
}

int pk_qk_norm_rope_bwd(int dtype, int degree, int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads,
                        int64_t dim, int64_t rotary, int interleaved, const void* const* q, int64_t q_bs,
                        int64_t q_ts, int64_t q_hs, const void* const* k, int64_t k_bs, int64_t k_ts, int64_t k_hs,
                        const void* const* qw, int qw_planes, const void* const* kw, int kw_planes,
                        const void* cos_t, const void* sin_t, int64_t table_rows, const int64_t* positions,
                        int64_t pos_bs, double eps, const void* const* gq, int64_t gq_bs, int64_t gq_hs,
                        int64_t gq_ts, const void* const* gk, int64_t gk_bs, int64_t gk_hs, int64_t gk_ts,
                        void* const* dq, void* const* dk, void* const* dqw, void* const* dkw, void* workspace,
                        size_t workspace_bytes, void* stream) {
    const char* what = "pk_qk_norm_rope_bwd";
    if (int rc = check_rope(dtype, degree, batch, len, q_heads, k_heads, dim, rotary, cos_t, sin_t, table_rows, what))
        return rc;
    const int np = degree + 1;
    if (qw_planes < 0 || qw_planes > np || kw_planes < 0 || kw_planes > np)
        return fail(PK_ERR_ARG, "pk_qk_norm_rope_bwd: bad weight plane count");
    RopeParams p{};
    p.np = np;
    p.batch = batch;
    p.len = len;
    p.dim = dim;
    p.rotary = static_cast<int>(rotary);
    p.interleaved = interleaved != 0;
    p.cos_t = cos_t;
    p.sin_t = sin_t;
    p.table_rows = table_rows;
    p.positions = positions;
    p.pos_bs = pos_bs;
    p.eps = eps;
    const void* const* x[2] = {q, k};
    const void* const* w[2] = {qw, kw};
    const void* const* g[2] = {gq, gk};
    void* const* out[2] = {dq, dk};
    void* const* dw[2] = {dqw, dkw};
    const int nw[2] = {qw_planes, kw_planes};
    const int64_t heads[2] = {q_heads, k_heads};
    const int64_t strides[2][6] = {{q_bs, q_ts, q_hs, gq_bs, gq_hs, gq_ts}, {k_bs, k_ts, k_hs, gk_bs, gk_hs, gk_ts}};
    const int sums[2] = {dqw ? qw_planes : 0, dkw ? kw_planes : 0};
    const BwdShape shape = bwd_shape(dtype, batch * len * q_heads, batch * len * k_heads, dim,
                                     std::max(sums[0], sums[1]));
    const int64_t blocks[2] = {shape.q_blocks, shape.k_blocks};
    const size_t need = pk_qk_norm_rope_bwd_workspace_size(dtype, degree, batch, len, q_heads, k_heads, dim, sums[0],
                                                           sums[1]);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(PK_ERR_WORKSPACE, "pk_qk_norm_rope_bwd: workspace missing or too small");
    size_t used = 0;
    for (int i = 0; i < 2; ++i) {
        HeadSet& s = p.set[i];
        s.heads = heads[i];
        if (sums[i])
            if (int rc = check_planes(reinterpret_cast<const void* const*>(dw[i]), sums[i], what)) return rc;
        if (batch * len * heads[i] == 0) continue;
        if (int rc = check_planes(x[i], np, what)) return rc;
        if (int rc = check_planes(g[i], np, what)) return rc;
        if (int rc = check_planes(out[i], np, what)) return rc;
        if (nw[i])
            if (int rc = check_planes(w[i], nw[i], what)) return rc;
        s.bs = strides[i][0];
        s.ts = strides[i][1];
        s.hs = strides[i][2];
        s.g_bs = strides[i][3];
        s.g_hs = strides[i][4];
        s.g_ts = strides[i][5];
        s.nw = nw[i];
        for (int j = 0; j < np; ++j) {
            s.x[j] = x[i][j];
            s.g[j] = g[i][j];
            s.out[j] = out[i][j];
        }
        for (int j = 0; j < nw[i]; ++j) s.w[j] = w[i][j];
        if (sums[i]) {
            s.partial = static_cast<unsigned char*>(workspace) + used;
            used += static_cast<size_t>(blocks[i]) * sums[i] * dim * compute_bytes(dtype);
        }
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* tok;
    prof_begin("qk_norm_rope_bwd", s, &tok);
    int rc = PK_OK;
    if (shape.q_blocks + shape.k_blocks > 0) rc = launch_rope_dtype(dtype, p, &shape, s, what);
    for (int i = 0; i < 2 && rc == PK_OK; ++i) {
        if (!sums[i]) continue;
        WeightSumParams q2{};
        q2.partial = p.set[i].partial;
        q2.blocks = blocks[i];
        q2.nw = sums[i];
        q2.dim = static_cast<int>(dim);
        for (int j = 0; j < sums[i]; ++j) q2.dw[j] = dw[i][j];
        const int grid = static_cast<int>(ceil_div(sums[i] * dim, 256));
        switch (dtype) {
            case PK_F32: PK_LAUNCHED(qk_weight_sum_kernel<float><<<grid, 256, 0, s>>>(q2)); break;
            case PK_F64: PK_LAUNCHED(qk_weight_sum_kernel<double><<<grid, 256, 0, s>>>(q2)); break;
            case PK_BF16: PK_LAUNCHED(qk_weight_sum_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(q2)); break;
            default: PK_LAUNCHED(qk_weight_sum_kernel<__half><<<grid, 256, 0, s>>>(q2)); break;
        }
    }
    prof_end("qk_norm_rope_bwd", s, tok);
    if (rc) return rc;
    PK_CHECK_LAUNCH(what);
    return PK_OK;
}

}  // extern "C"
