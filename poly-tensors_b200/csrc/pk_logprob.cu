// Log probabilities of given tokens, entropy and top alternatives of a row of logits, and their
// gradient.  A row has V logits x of n+1 planes; z = scale * x (scale = 1 / temperature), (*) is the
// truncated series product.  With m = max z_0 and w_i = exp(z_i - m) (a series):
//   S = sum_i w_i,  L = log S,  logp_i = (z_i - m) - L,  H = L - (sum_i w_i (*) (z_i - m)) / S.
// L lies in [0, log V] and both terms of H are nonnegative at plane 0, so nothing cancels however large
// the logits are.  Backward, with p_i = exp(logp_i), upstream series a (token), b (entropy), c_j
// (alternative j) and A = a + sum_j c_j:
//   dx_i = scale ( a [i = token] + sum_j c_j [i = top_j] - p_i (*) (A + b (*) (logp_i + H)) ).
// A logit whose constant plane is -inf is masked: it takes no part whatever its other planes hold, its
// log probability is the constant -inf (no direction, no gradient).  A row with no open logit has
// entropy 0 and log probabilities -inf.  A NaN, or +inf, makes the row's results NaN.
//
// Sums, maxima and the row series are held in float (double for float64 logits); the results have that
// type, and the gradient is rounded once to the logits' type when it is stored.
#include <algorithm>

#include "pk_rows.cuh"

namespace pk {

struct LogProbParams {
    const void* x[PK_MAX_PLANES];        // logits
    void* logp[PK_MAX_PLANES];           // forward results, compute type
    void* entropy[PK_MAX_PLANES];
    void* top_logp[PK_MAX_PLANES];       // [rows][top]
    const void* h[PK_MAX_PLANES];        // backward: the forward's entropy
    const void* ga[PK_MAX_PLANES];       // upstream of logp, entropy, top_logp (null: none)
    const void* gb[PK_MAX_PLANES];
    const void* gc[PK_MAX_PLANES];
    void* dx[PK_MAX_PLANES];
    int np, top;
    int has_a, has_b, has_c;
    int64_t rows, cols, x_rs, dx_rs;
    const int64_t* tokens;
    int64_t ignore_index;
    double scale;
    int64_t* top_tokens;                 // [rows][top]
    void* stats;                         // [rows][np + 1]: m, L_0 .. L_n
    const int64_t* top_at;               // backward: the forward's top_tokens and stats
    const void* stats_in;
};

constexpr int LP_MAX_TOP = 32;

// Running state of a part of a row: the largest z_0 seen, S and T = sum w (*) (z - m) below it.
template <int NP, typename C>
struct LogSum {
    C m;
    C S[NP], T[NP];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NP; ++k) S[k] = T[k] = C(0);
    }
    // The same sums below a larger maximum.
    __device__ __forceinline__ void raise(C to) {
        if (m == -INFINITY) {
            m = to;
            return;
        }
        const C f = c_exp(m - to), d = m - to;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            T[k] = f == C(0) ? C(0) : f * (T[k] + d * S[k]);
            S[k] = f == C(0) ? C(0) : f * S[k];
        }
        m = to;
    }
    __device__ __forceinline__ void add(const C (&z)[NP]) {
        if (z[0] == -INFINITY) return;
        if (!(z[0] <= m)) raise(z[0]);
        const C d = z[0] - m, w = c_exp(d);
        if (w == C(0)) return;
        // e = exp(directions) and q = e (*) directions from the same products u_i e_{k-i}
        C e[NP], q[NP];
        e[0] = C(1);
        q[0] = C(0);
#pragma unroll
        for (int k = 1; k < NP; ++k) {
            C t = C(0), v = C(0);
#pragma unroll
            for (int i = 1; i <= k; ++i) {
                const C o = z[i] * e[k - i];
                t += C(i) * o;
                v += o;
            }
            e[k] = t * inv_int<C>(k);
            q[k] = v;
        }
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            S[k] += w * e[k];
            T[k] += w * (q[k] + d * e[k]);
        }
    }
    __device__ __forceinline__ void join(const LogSum& o) {
        if (o.m == -INFINITY) return;
        if (!(o.m <= m)) {
            const C om = o.m;
            raise(om);
        }
        LogSum b = o;
        b.raise(m);
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            S[k] += b.S[k];
            T[k] += b.T[k];
        }
    }
};

template <int NP, typename T, typename C>
__device__ __forceinline__ void load_logit(const LogProbParams& p, int64_t row, int64_t col, C (&z)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k)
        z[k] = k < p.np ? to_c<C>(static_cast<const T*>(p.x[k])[row * p.x_rs + col]) * C(p.scale) : C(0);
}

// log probability series of one logit
template <int NP, typename C>
__device__ __forceinline__ void log_prob(const C (&z)[NP], C m, const C (&L)[NP], C (&out)[NP]) {
    const bool masked = z[0] == -INFINITY;
    out[0] = masked ? C(-INFINITY) : (z[0] - m) - L[0];
#pragma unroll
    for (int k = 1; k < NP; ++k) out[k] = masked ? C(0) : z[k] - L[k];
}

// A value as an unsigned integer in the same order, NaN above everything, -0 as +0.
__device__ __forceinline__ uint64_t order_key(float v) {
    if (v != v) return ~0ull;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? static_cast<uint32_t>(~b) : static_cast<uint64_t>(b | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return ~0ull;
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return b >> 63 ? ~b : b | (1ull << 63);
}

// One block per row.
template <typename T, int NP>
__global__ void __launch_bounds__(256) token_log_probs_fwd_kernel(const LogProbParams p) {
    using C = typename Compute<T>::type;
    __shared__ LogSum<NP, C> part[8];
    __shared__ uint64_t best_key[8];
    __shared__ int64_t best_at[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t token = p.tokens[row];
        if (token == p.ignore_index) {   // not read: zeros, and no alternatives
            if (threadIdx.x == 0) {
                for (int k = 0; k < p.np; ++k) {
                    static_cast<C*>(p.logp[k])[row] = static_cast<C*>(p.entropy[k])[row] = C(0);
                    for (int j = 0; j < p.top; ++j) static_cast<C*>(p.top_logp[k])[row * p.top + j] = C(0);
                }
                for (int j = 0; j < p.top; ++j) p.top_tokens[row * p.top + j] = -1;
                for (int k = 0; k <= p.np; ++k) static_cast<C*>(p.stats)[row * (p.np + 1) + k] = C(0);
            }
            continue;
        }
        LogSum<NP, C> sum;
        sum.clear();
        for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
            C z[NP];
            load_logit<NP, T, C>(p, row, i, z);
            sum.add(z);
        }
        for (int off = 16; off > 0; off >>= 1) {
            LogSum<NP, C> o;
            o.m = __shfl_xor_sync(0xffffffffu, sum.m, off);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                o.S[k] = __shfl_xor_sync(0xffffffffu, sum.S[k], off);
                o.T[k] = __shfl_xor_sync(0xffffffffu, sum.T[k], off);
            }
            sum.join(o);
        }
        __syncthreads();
        if (lane == 0) part[warp] = sum;
        __syncthreads();
        C L[NP];
        sum = part[0];
        for (int w = 1; w < warps; ++w) sum.join(part[w]);
        if (sum.m != -INFINITY) {
            s_log<NP, C>(sum.S, L);
        } else {
#pragma unroll
            for (int k = 0; k < NP; ++k) L[k] = C(0);
        }
        if (threadIdx.x == 0) {
            C z[NP], v[NP], H[NP];
            const bool inside = token >= 0 && token < p.cols;
            if (inside) {
                load_logit<NP, T, C>(p, row, token, z);
                log_prob<NP, C>(z, sum.m, L, v);
            }
            if (sum.m != -INFINITY) s_div<NP, C>(sum.T, sum.S, H);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if (k >= p.np) continue;
                static_cast<C*>(p.logp[k])[row] = inside ? v[k] : C(NAN);
                static_cast<C*>(p.entropy[k])[row] = sum.m != -INFINITY ? L[k] - H[k] : C(0);
                static_cast<C*>(p.stats)[row * (p.np + 1) + 1 + k] = L[k];
            }
            static_cast<C*>(p.stats)[row * (p.np + 1)] = sum.m;
        }
        // the alternatives, one pass each: the best logit below the last one in (value, index) order
        uint64_t last_key = ~0ull;
        int64_t last_at = -1;
        for (int j = 0; j < p.top; ++j) {
            uint64_t key = 0;
            int64_t at = p.cols;
            for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
                const uint64_t q = order_key(to_c<C>(static_cast<const T*>(p.x[0])[row * p.x_rs + i]));
                if (j > 0 && (q > last_key || (q == last_key && i <= last_at))) continue;
                if (at == p.cols || q > key) {
                    key = q;
                    at = i;
                }
            }
            for (int off = 16; off > 0; off >>= 1) {
                const uint64_t k2 = __shfl_xor_sync(0xffffffffu, key, off);
                const int64_t a2 = __shfl_xor_sync(0xffffffffu, at, off);
                if (a2 < p.cols && (at == p.cols || k2 > key || (k2 == key && a2 < at))) {
                    key = k2;
                    at = a2;
                }
            }
            __syncthreads();
            if (lane == 0) {
                best_key[warp] = key;
                best_at[warp] = at;
            }
            __syncthreads();
            key = best_key[0];
            at = best_at[0];
            for (int w = 1; w < warps; ++w) {
                const uint64_t k2 = best_key[w];
                const int64_t a2 = best_at[w];
                if (a2 < p.cols && (at == p.cols || k2 > key || (k2 == key && a2 < at))) {
                    key = k2;
                    at = a2;
                }
            }
            last_key = key;
            last_at = at;
            if (threadIdx.x == 0) {
                C z[NP], v[NP];
                load_logit<NP, T, C>(p, row, at, z);
                log_prob<NP, C>(z, sum.m, L, v);
                p.top_tokens[row * p.top + j] = at;
#pragma unroll
                for (int k = 0; k < NP; ++k)
                    if (k < p.np) static_cast<C*>(p.top_logp[k])[row * p.top + j] = v[k];
            }
        }
    }
}

template <typename T, int NP>
__global__ void __launch_bounds__(256) token_log_probs_bwd_kernel(const LogProbParams p) {
    using C = typename Compute<T>::type;
    const C scale = C(p.scale);
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t token = p.tokens[row];
        const C m = static_cast<const C*>(p.stats_in)[row * (p.np + 1)];
        if (token == p.ignore_index || m == -INFINITY) {
            for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x)
                for (int k = 0; k < p.np; ++k) static_cast<T*>(p.dx[k])[row * p.dx_rs + i] = from_c<T>(C(0));
            continue;
        }
        C L[NP], a[NP], b[NP], A[NP], H[NP], z[NP];
        const bool inside = token >= 0 && token < p.cols;
        bool open = false;
        if (inside && p.has_a) {
            load_logit<NP, T, C>(p, row, token, z);
            open = z[0] != -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const bool live = k < p.np;
            L[k] = live ? static_cast<const C*>(p.stats_in)[row * (p.np + 1) + 1 + k] : C(0);
            H[k] = live ? static_cast<const C*>(p.h[k])[row] : C(0);
            a[k] = !live || !p.has_a ? C(0) : !inside ? C(NAN) : open ? static_cast<const C*>(p.ga[k])[row] : C(0);
            b[k] = live && p.has_b ? static_cast<const C*>(p.gb[k])[row] : C(0);
            A[k] = a[k];
        }
        for (int j = 0; j < (p.has_c ? p.top : 0); ++j) {
            load_logit<NP, T, C>(p, row, p.top_at[row * p.top + j], z);
            if (z[0] == -INFINITY) continue;
#pragma unroll
            for (int k = 0; k < NP; ++k)
                if (k < p.np) A[k] += static_cast<const C*>(p.gc[k])[row * p.top + j];
        }
        for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
            C lp[NP], P[NP], q[NP], r[NP];
            load_logit<NP, T, C>(p, row, i, z);
            const bool masked = z[0] == -INFINITY;
            log_prob<NP, C>(z, m, L, lp);
            s_exp<NP, C>(lp, P);
            if (P[0] == C(0)) {
#pragma unroll
                for (int k = 0; k < NP; ++k) r[k] = C(0);
            } else {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    lp[k] += H[k];
                    q[k] = A[k];
                }
                s_mul_acc<NP, C>(b, lp, q);
                s_mul<NP, C>(P, q, r);
#pragma unroll
                for (int k = 0; k < NP; ++k) r[k] = -r[k];
            }
            if (!masked) {
                if (i == token) {
#pragma unroll
                    for (int k = 0; k < NP; ++k) r[k] += a[k];
                }
                for (int j = 0; j < (p.has_c ? p.top : 0); ++j)
                    if (p.top_at[row * p.top + j] == i) {
#pragma unroll
                        for (int k = 0; k < NP; ++k)
                            if (k < p.np) r[k] += static_cast<const C*>(p.gc[k])[row * p.top + j];
                    }
            }
#pragma unroll
            for (int k = 0; k < NP; ++k)
                if (k < p.np) static_cast<T*>(p.dx[k])[row * p.dx_rs + i] = from_c<T>(r[k] * scale);
        }
    }
}

template <typename T, int NP>
static void launch_log_probs(const LogProbParams& p, bool backward, cudaStream_t s) {
    const int grid = static_cast<int>(std::min<int64_t>(p.rows, static_cast<int64_t>(num_sms()) * 16));
    if (backward) PK_LAUNCHED(token_log_probs_bwd_kernel<T, NP><<<grid, 256, 0, s>>>(p));
    else PK_LAUNCHED(token_log_probs_fwd_kernel<T, NP><<<grid, 256, 0, s>>>(p));
}

template <typename T>
static void launch_log_probs_np(const LogProbParams& p, bool backward, cudaStream_t s) {
    switch (p.np) {
        case 1: launch_log_probs<T, 1>(p, backward, s); break;
        case 2: launch_log_probs<T, 2>(p, backward, s); break;
        case 3: launch_log_probs<T, 3>(p, backward, s); break;
        case 4: launch_log_probs<T, 4>(p, backward, s); break;
        case 5: launch_log_probs<T, 5>(p, backward, s); break;
        case 6: launch_log_probs<T, 6>(p, backward, s); break;
        case 7: case 8: case 9: launch_log_probs<T, 9>(p, backward, s); break;
        default: launch_log_probs<T, 16>(p, backward, s); break;
    }
}

static int run_log_probs(int dtype, const LogProbParams& p, bool backward, void* stream, const char* name) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* tok;
    prof_begin(name, s, &tok);
    switch (dtype) {
        case PK_F32: launch_log_probs_np<float>(p, backward, s); break;
        case PK_F64: launch_log_probs_np<double>(p, backward, s); break;
        case PK_BF16: launch_log_probs_np<__nv_bfloat16>(p, backward, s); break;
        default: launch_log_probs_np<__half>(p, backward, s); break;
    }
    prof_end(name, s, tok);
    PK_CHECK_LAUNCH(name);
    return PK_OK;
}

static int check_log_probs(int dtype, int degree, int64_t rows, int64_t cols, int top, const void* const* x,
                           const void* tokens, const void* stats, const void* top_tokens, const std::string& what) {
    if (dtype != PK_F32 && dtype != PK_F64 && dtype != PK_BF16 && dtype != PK_F16)
        return fail(PK_ERR_UNSUPPORTED, what + ": unsupported dtype");
    if (degree < 0 || degree >= PK_MAX_PLANES) return fail(PK_ERR_UNSUPPORTED, what + ": degree out of range");
    if (rows < 0 || cols < 1 || cols > 0x7fffffff) return fail(PK_ERR_ARG, what + ": bad extent");
    if (top < 0 || top > LP_MAX_TOP || top > cols) return fail(PK_ERR_ARG, what + ": bad number of alternatives");
    if (rows == 0) return PK_OK;
    if (!x || !tokens || !stats || (top && !top_tokens)) return fail(PK_ERR_ARG, what + ": null pointer");
    for (int k = 0; k <= degree; ++k)
        if (!x[k]) return fail(PK_ERR_ARG, what + ": null plane");
    return PK_OK;
}

// Copies n plane pointers; false when one is missing.
template <typename To, typename From>
static bool take_planes(To* to, From* from, int n) {
    if (!from) return false;
    for (int k = 0; k < n; ++k) {
        if (!from[k]) return false;
        to[k] = from[k];
    }
    return true;
}

}  // namespace pk

using namespace pk;

extern "C" {

int pk_token_log_probs_fwd(int dtype, int degree, int64_t rows, int64_t cols, const void* const* logits,
                           int64_t logits_rs, const int64_t* tokens, int64_t ignore_index, double scale, int top,
                           void* const* log_probs, void* const* entropy, void* const* top_log_probs,
                           int64_t* top_tokens, void* stats, void* stream) {
    const char* what = "pk_token_log_probs_fwd";
    if (int rc = check_log_probs(dtype, degree, rows, cols, top, logits, tokens, stats, top_tokens, what)) return rc;
    if (rows == 0) return PK_OK;
    LogProbParams p{};
    p.np = degree + 1;
    if (!take_planes(p.x, logits, p.np) || !take_planes(p.logp, log_probs, p.np) ||
        !take_planes(p.entropy, entropy, p.np) || (top && !take_planes(p.top_logp, top_log_probs, p.np)))
        return fail(PK_ERR_ARG, "pk_token_log_probs_fwd: null plane");
    p.top = top;
    p.rows = rows;
    p.cols = cols;
    p.x_rs = logits_rs;
    p.tokens = tokens;
    p.ignore_index = ignore_index;
    p.scale = scale;
    p.top_tokens = top_tokens;
    p.stats = stats;
    return run_log_probs(dtype, p, false, stream, "token_log_probs_fwd");
}

int pk_token_log_probs_bwd(int dtype, int degree, int64_t rows, int64_t cols, const void* const* logits,
                           int64_t logits_rs, const int64_t* tokens, int64_t ignore_index, double scale, int top,
                           const void* stats, const void* const* entropy, const int64_t* top_tokens,
                           const void* const* g_log_probs, const void* const* g_entropy,
                           const void* const* g_top_log_probs, void* const* dlogits, int64_t dlogits_rs,
                           void* stream) {
    const char* what = "pk_token_log_probs_bwd";
    if (int rc = check_log_probs(dtype, degree, rows, cols, top, logits, tokens, stats, top_tokens, what)) return rc;
    if (rows == 0) return PK_OK;
    LogProbParams p{};
    p.np = degree + 1;
    p.has_a = g_log_probs != nullptr;
    p.has_b = g_entropy != nullptr;
    p.has_c = top > 0 && g_top_log_probs != nullptr;
    if (!take_planes(p.x, logits, p.np) || !take_planes(p.dx, dlogits, p.np) ||
        !take_planes(p.h, entropy, p.np) || (p.has_a && !take_planes(p.ga, g_log_probs, p.np)) ||
        (p.has_b && !take_planes(p.gb, g_entropy, p.np)) || (p.has_c && !take_planes(p.gc, g_top_log_probs, p.np)))
        return fail(PK_ERR_ARG, "pk_token_log_probs_bwd: null plane");
    p.top = top;
    p.rows = rows;
    p.cols = cols;
    p.x_rs = logits_rs;
    p.dx_rs = dlogits_rs;
    p.tokens = tokens;
    p.ignore_index = ignore_index;
    p.scale = scale;
    p.top_at = top_tokens;
    p.stats_in = stats;
    return run_log_probs(dtype, p, true, stream, "token_log_probs_bwd");
}

}  // extern "C"
