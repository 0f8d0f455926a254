// Log probabilities of given tokens, entropy and top alternatives of a row of logits, and their
// gradient.  A row has V logits x of n+1 planes; z = scale * x (scale = 1 / temperature), (*) is the
// truncated series product.  With m = max z_0 and w_i = exp(z_i - m) (a series):
//   S = sum_i w_i,  L = log S,  logp_i = (z_i - m) - L,  H = L - (sum_i w_i (*) (z_i - m)) / S.
// At plane 0 the largest logit's weight is exactly 1, L lies between 0 and log V and the mean of z - m is of the
// size of H: nothing cancels, however large the logits are or however much of the row one word holds.
// Backward, with p_i = exp(logp_i), upstream series a (token), b (entropy), c_j (alternative j) and
// A = a + sum_j c_j:
//   dx_i = scale ( a [i = token] + sum_j c_j [i = top_j] - p_i (*) (A + b (*) (logp_i + H)) ).
// A logit whose constant plane is -inf is masked: it takes no part whatever its other planes hold, its
// log probability is the constant -inf (no direction, no gradient).  A row with no open logit has
// entropy 0 and log probabilities -inf.  A NaN, or +inf, makes the row's results NaN.
//
// Sums, maxima and the row series are held in float (double for float64 logits); the results have that
// type, and the gradient is rounded once to the logits' type when it is stored.
//
// Each direction reads the logits once (the forward writes a few numbers per row, the backward the
// gradient), so memory traffic is the floor.  Measured on B200, device time: 2048 x 32000 float32 degree 3
// forward 182 us = 5.8 TB/s, backward 337 us = 6.2 TB/s; 8192 rows forward 666 us = 6.3 TB/s.  16-bit logits at
// degree 0 and 1 and 64-bit ones are held up by their instructions: 8192 x 32000 bfloat16 forward 114 us = 4.6 TB/s at
// degree 0 (68 % of the issue slots, the exponentials' pipe 50 %, the integer pipe 48 %), 236 us = 4.5 TB/s at
// degree 1; five alternatives add 53 us to the former (a search and a merge per row behind two block barriers, with
// none of the next row's loads under way); 1024 x 32000 float64 degree 2 forward 189 us = 4.2 TB/s (58 % of the issue
// slots, the double-precision pipe 40 %, 22 % of the warps active: waits between dependent operations), backward 290 us =
// 5.4 TB/s; 300 x 8191 45 and 30 us, where the bytes alone would take 9 and 18.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstring>

#include "pk_vec.cuh"

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
    int aligned;                         // every plane's base lies alike within 16 bytes
    int64_t rows, cols, x_rs, dx_rs;
    const int64_t* tokens;
    int64_t ignore_index;
    double scale;
    int64_t* top_tokens;                 // [rows][top]
    void* stats;                         // [rows][np + 1]: m, L_0 .. L_n
    const int64_t* top_at;               // backward: the forward's top_tokens and stats
    const void* stats_in;
};

constexpr int LP_MAX_TOP = 32;       // a warp's lanes
constexpr int LP_MAX_SHARE = 8;      // blocks of a row's cluster (the portable limit)

// Largest value, NaN when there is one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a != a ? a : b != b ? b : fmax(a, b); }

// exp of two values in hardware, 2^(d log2 e).  (The difference z - m comes first and is scaled to base 2 after:
// folding log2 e into the difference would round m log2 e, which shows when logits are large.)
// The product's rounding moves a weight by |d| 2^-24.  That is the size of a logit's own rounding, but the
// directions' sums take powers of it apart (degree 4: 1.6e-6 in log p's last plane).  float32 logits are bound by
// memory and take the library's exponential; for 16-bit ones with directions EXP_CAREFUL returns the error: the
// fused multiply-add gives the product's error r exactly (TwoProduct of Ogita, Rump and Oishi, "Accurate sum and
// dot product", 2005), and 2^(a + r) = 2^a (1 + r log 2) to first order.
enum { EXP_PLAIN, EXP_CAREFUL, EXP_LIBRARY };
template <int HOW>
__device__ __forceinline__ void exp_both(Two<float> d, float& w0, float& w1) {
    if constexpr (HOW == EXP_LIBRARY) {
        float x, y;
        d.get(x, y);
        w0 = expf(x);
        w1 = expf(y);
        return;
    }
    constexpr float LOG2E = 1.4426950408889634f, LOG2 = 0.6931471805599453f;
    const Two<float> minus = d * Two<float>(-LOG2E);
    float a, b;
    minus.get(a, b);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w0) : "f"(-a));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w1) : "f"(-b));
    if constexpr (HOW == EXP_CAREFUL) {
        const Two<float> w(w0, w1), r = fma2(d, Two<float>(LOG2E), minus);
        fma2(w, r * Two<float>(LOG2), w).get(w0, w1);
    }
}
template <int HOW>
__device__ __forceinline__ void exp_both(Two<double> d, double& w0, double& w1) {
    w0 = exp(d.lo);
    w1 = exp(d.hi);
}
// The same with subnormal results (a gradient of 1e-38 is one; a weight of 1e-38 beside a sum of 1 is not): 2^32
// times the result stays normal down to the smallest of them.
__device__ __forceinline__ void exp_small_both(Two<float> d, float& w0, float& w1) {
    float a, b;
    fma2(d, Two<float>(1.4426950408889634f), Two<float>(32.0f)).get(a, b);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(a));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(b));
    w0 = a * 0x1p-32f;
    w1 = b * 0x1p-32f;
}
__device__ __forceinline__ void exp_small_both(Two<double> d, double& w0, double& w1) { exp_both<EXP_PLAIN>(d, w0, w1); }

// The largest of a vector's elements (16-bit ones are compared in pairs as they are stored).
template <typename T, int VEC, typename C>
__device__ __forceinline__ C largest_of(const Raw<T, VEC>& v) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&v.w[0]);
#pragma unroll
        for (int i = 1; i < VEC / 2; ++i) t = __hmax2_nan(t, *reinterpret_cast<const __nv_bfloat162*>(&v.w[i]));
        return max_nan(__low2float(t), __high2float(t));
    } else if constexpr (std::is_same<T, __half>::value) {
        __half2 t = *reinterpret_cast<const __half2*>(&v.w[0]);
#pragma unroll
        for (int i = 1; i < VEC / 2; ++i) t = __hmax2_nan(t, *reinterpret_cast<const __half2*>(&v.w[i]));
        return max_nan(__low2float(t), __high2float(t));
    } else {
        C top = -INFINITY;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            C a, b;
            v.get(i).get(a, b);
            top = max_nan(top, max_nan(a, b));
        }
        return top;
    }
}

// Elements of a 16-byte vector.
template <typename T>
constexpr int lp_vec() { return 16 / sizeof(T); }

// A row as groups of one vector: group g holds elements g * VEC - skew ..; the first group starts at the
// 16-byte boundary at or before the row, so that whole groups are aligned whatever the row's offset.
struct RowGroups {
    int skew, count;
    int full, last;          // groups full .. last - 1 lie within the row and are aligned
    template <typename T>
    __device__ __forceinline__ void set(const void* row, int64_t cols, bool aligned) {
        constexpr int VEC = lp_vec<T>();
        skew = aligned ? static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T)) : 0;
        count = static_cast<int>((cols + skew + VEC - 1) / VEC);
        full = skew ? 1 : 0;
        last = aligned ? static_cast<int>((cols + skew) / VEC) : 0;
    }
    __device__ __forceinline__ bool whole(int g) const { return g >= full && g < last; }
};

// One group of every plane; elements outside the row read as masked (-inf, no direction).
template <int NP, typename T>
struct Group {
    static constexpr int VEC = lp_vec<T>();
    Raw<T, VEC> v[NP];

    __device__ __forceinline__ void load(const LogProbParams& p, int64_t row_at, const RowGroups& row, int g) {
        if (row.whole(g)) {
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if constexpr (NP > 6) v[k] = Raw<T, VEC>{};
                if (NP <= 6 || k < p.np)
                    v[k] = reinterpret_cast<const Raw<T, VEC>*>(static_cast<const T*>(p.x[k]) + (row_at - row.skew))[g];
            }
        } else {
            const int64_t first = static_cast<int64_t>(g) * VEC - row.skew;
#pragma unroll
            for (int k = 0; k < NP; ++k) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const bool in = first + j >= 0 && first + j < p.cols && (NP <= 6 || k < p.np);
                    const T e = in ? static_cast<const T*>(p.x[k])[row_at + first + j]
                                   : from_c<T>(k ? typename Compute<T>::type(0) : typename Compute<T>::type(-INFINITY));
                    uint64_t bits = 0;
                    memcpy(&bits, &e, sizeof(T));
                    v[k].set_bits(j, bits);
                }
            }
        }
    }
};

// The largest of a warp's values, NaN left out.
template <typename C>
__device__ __forceinline__ C warp_largest(C v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}

// What a sum leaves behind when its weight underflows: nothing, unless a NaN logit is in it.
template <typename C>
__device__ __forceinline__ C nan_or_zero(C v) { return v == v ? C(0) : v; }

// Running state of a part of a row below a reference m: S = sum w and T = sum w (*) (z - m), w = exp(z - m).  m is
// the largest z_0 that the thread's warp has seen, the same in all its lanes: raised by a vote of the warp, three or
// four times in a row's thirty steps, where a reference per lane is raised in some lane in nearly every step of the
// warp (8192 x 32000 bfloat16, device time: 113 us, 127 so).  Raising it later, when a logit lies some distance above,
// saves no more than 3 % and costs digits: log S and T / S are then of that distance and nearly cancel in a row
// that one word holds (up to 8 above the rest of 400 rows of two words: error of the entropy 7.9e-7, 6.2e-8 so; of its
// gradient, relative, 2.3e-4, 3.2e-7 so).  Two sums of each run side by side (even and odd elements) and are
// joined at the end.
template <int NP, typename C, int HOW>
struct LogSum {
    C m;
    Two<C> S[NP], T[NP];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NP; ++k) S[k] = T[k] = Two<C>(C(0));
    }
    // The same sums below a larger m.
    __device__ __forceinline__ void raise(C to) {
        to = fmax(to, m);
        const C d = m - to, f = m == -INFINITY ? C(0) : c_exp(d);
        if (f == C(0)) {
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                C a, b;
                S[k].get(a, b);
                S[k] = Two<C>(nan_or_zero(a), nan_or_zero(b));
                T[k] = Two<C>(C(0));
            }
        } else {
            const Two<C> ff(f), dd(d);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                T[k] = ff * fma2(dd, S[k], T[k]);
                S[k] = ff * S[k];
            }
        }
        m = to;
    }
    // Two elements into the sums gs, gt of their group (FIRST: which starts with them).  x holds the constant planes
    // unscaled, u the directions scaled (u[0] unused).  Group sums first, one addition of them to S and T after:
    // a quarter or half of the roundings against the running sums, which at degree 3 and 4 show in the entropy's
    // last planes (2.0e-6 without, 1.1e-6 so) for 1.5 to 4 % of the time.
    template <bool FIRST>
    __device__ __forceinline__ void add(Two<C> x, C scale, Two<C> (&u)[NP], Two<C> (&gs)[NP], Two<C> (&gt)[NP]) {
        Two<C> d = fma2(x, Two<C>(scale), Two<C>(m == -INFINITY ? C(0) : -m));
        C w0, w1;
        d.get(w0, w1);
        d = Two<C>(max_nan(w0, C(-1000)), max_nan(w1, C(-1000)));     // masked logits: finite, with a weight of 0
        exp_both<HOW>(d, w0, w1);
        if (NP > 1 && (w0 == C(0) || w1 == C(0))) {
            // masked, or too far below the reference to count: its directions do not enter either
#pragma unroll
            for (int k = 1; k < NP; ++k) {
                C a, b;
                u[k].get(a, b);
                u[k] = Two<C>(w0 == C(0) ? C(0) : a, w1 == C(0) ? C(0) : b);
            }
        }
        const Two<C> w(w0, w1);
        // e = exp(directions) and q = e (*) directions from the same products u_i e_(k-i)
        Two<C> e[NP];
        gs[0] = FIRST ? w : gs[0] + w;
        gt[0] = FIRST ? w * d : fma2(w, d, gt[0]);
        e[0] = Two<C>(C(1));
#pragma unroll
        for (int k = 1; k < NP; ++k) {
            Two<C> t = u[k], v = u[k];                       // i = k: e_0 = 1
#pragma unroll
            for (int i = 1; i < k; ++i) {
                const Two<C> o = u[i] * e[k - i];
                t = fma2(o, Two<C>(C(i) / C(k)), t);
                v = v + o;
            }
            e[k] = t;
            gs[k] = FIRST ? w * t : fma2(w, t, gs[k]);
            gt[k] = FIRST ? w * fma2(d, t, v) : fma2(w, fma2(d, t, v), gt[k]);
        }
    }
};

// The joined sums of many threads' parts.
template <int NP, typename C>
struct RowSum {
    C m, S[NP], T[NP];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NP; ++k) S[k] = T[k] = C(0);
    }
    // All lanes of the warp: every lane gets the total.  The largest maximum first, then plain sums.
    __device__ __forceinline__ void join_warp() {
        C top = m;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, off));
        const C d = m - top, f = m == -INFINITY ? C(0) : c_exp(d);
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            T[k] = f == C(0) ? C(0) : f * (T[k] + d * S[k]);
            S[k] = f == C(0) ? nan_or_zero(S[k]) : f * S[k];
        }
        m = top;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) {
                S[k] += __shfl_xor_sync(0xffffffffu, S[k], off);
                T[k] += __shfl_xor_sync(0xffffffffu, T[k], off);
            }
        }
    }
};

// One logit: the constant plane as stored, the directions scaled.
template <int NP, typename T, typename C>
__device__ __forceinline__ void load_logit(const LogProbParams& p, int64_t row, int64_t col, C (&x)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        x[k] = k < p.np ? to_c<C>(static_cast<const T*>(p.x[k])[row * p.x_rs + col]) : C(0);
        if (k) x[k] *= C(p.scale);
    }
}

// Log probability series of one logit.  z - m is one rounding of scale * x - m, as in the sums and the gradient: a
// product rounded by itself would stand in full (2e-6 at |z| = 40) in a log probability near 0.
template <int NP, typename C>
__device__ __forceinline__ void log_prob(const C (&x)[NP], C scale, C m, const C (&L)[NP], C (&out)[NP]) {
    const bool masked = x[0] * scale == -INFINITY;
    out[0] = masked ? C(-INFINITY) : fma(x[0], scale, -m) - L[0];
#pragma unroll
    for (int k = 1; k < NP; ++k) out[k] = masked ? C(0) : x[k] - L[k];
}

// A logit and its index as one key: a larger key is a larger logit, or the same with a lower index.  NaN
// stands above every number, -0 with +0; the all-zero key is below every logit.
template <typename C> struct Key;
template <> struct Key<float> {
    uint64_t k;
    __device__ __forceinline__ static Key make(float v, int at) {
        const uint32_t b = __float_as_uint(v + 0.0f);
        const uint32_t o = v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
        return {static_cast<uint64_t>(o) << 32 | ~static_cast<uint32_t>(at)};
    }
    __device__ __forceinline__ bool above(Key o) const { return k > o.k; }
    __device__ __forceinline__ int at() const { return static_cast<int>(~static_cast<uint32_t>(k)); }
    __device__ __forceinline__ bool none() const { return k == 0; }
    __device__ __forceinline__ float value() const {
        const uint32_t o = static_cast<uint32_t>(k >> 32);
        return o == 0xffffffffu ? NAN : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
    }
    __device__ __forceinline__ Key from(int lane) const { return {__shfl_sync(0xffffffffu, k, lane)}; }
    __device__ __forceinline__ Key across(int mask) const { return {__shfl_xor_sync(0xffffffffu, k, mask)}; }
};
template <> struct Key<double> {
    uint64_t k;
    uint32_t i;
    __device__ __forceinline__ static Key make(double v, int at) {
        const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
        return {v != v ? ~0ull : b >> 63 ? ~b : b | (1ull << 63), ~static_cast<uint32_t>(at)};
    }
    __device__ __forceinline__ bool above(Key o) const { return k > o.k || (k == o.k && i > o.i); }
    __device__ __forceinline__ int at() const { return static_cast<int>(~i); }
    __device__ __forceinline__ bool none() const { return k == 0; }
    __device__ __forceinline__ double value() const {
        return k == ~0ull ? NAN : __longlong_as_double(static_cast<long long>(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
    }
    __device__ __forceinline__ Key from(int lane) const { return {__shfl_sync(0xffffffffu, k, lane), __shfl_sync(0xffffffffu, i, lane)}; }
    __device__ __forceinline__ Key across(int mask) const {
        return {__shfl_xor_sync(0xffffffffu, k, mask), __shfl_xor_sync(0xffffffffu, i, mask)};
    }
};

// A warp's best logits so far, lane j holding the (j + 1)-th.  Logits that reach `bar` (no more than the
// top-th best) wait in shared memory until 32 have come, which are then sorted and merged in a bitonic
// network: 21 exchanges for 32 candidates.
template <typename C>
struct Best {
    Key<C> mine, last;       // last: the list's top-th (nothing while it is not full)
    Key<C>* waiting;         // 64 places of this warp
    int count;
    bool sorted;             // `mine` holds something
    C bar;
    __device__ __forceinline__ void clear(Key<C>* place) {
        mine = last = Key<C>{};
        waiting = place;
        count = 0;
        sorted = false;
        bar = -INFINITY;
    }
    static __device__ __forceinline__ void exchange(Key<C>& k, int mask, bool keep_larger) {
        const Key<C> o = k.across(mask);
        if (o.above(k) == keep_larger) k = o;
    }
    // Both lists fall from lane 0: the larger of k_j and other_(31 - j) are the best 32 of both, in bitonic order.
    __device__ __forceinline__ void merge(Key<C> other) {
        const int lane = threadIdx.x & 31;
        other = other.across(31);
        if (other.above(mine)) mine = other;
#pragma unroll
        for (int mask = 16; mask > 0; mask >>= 1) exchange(mine, mask, (lane & mask) == 0);
    }
    // The bar from the largest logit of every thread of the block: with j = ceil(top / warps), the
    // ceil(top / j)-th largest of the warps' j-th largest has at least `top` logits at or above it.
    __device__ __forceinline__ void start(C lane_top, int top, Key<C>* of_warps) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        const int j = (top + warps - 1) / warps, want = (top + j - 1) / j - 1;
        Key<C> k = Key<C>::make(lane_top, threadIdx.x);
        if (j == 1) {
#pragma unroll
            for (int mask = 16; mask > 0; mask >>= 1) exchange(k, mask, true);
        } else {
            sort(k);
        }
        if (lane == j - 1) of_warps[warp] = k;
        __syncthreads();
        k = lane < warps ? of_warps[lane] : Key<C>{};
        int rank = lane < warps ? 0 : -1;
        if (rank == 0)
            for (int w = 0; w < warps; ++w) rank += of_warps[w].above(k) ? 1 : 0;
        bar = k.from(__ffs(__ballot_sync(0xffffffffu, rank == want)) - 1).value();
    }
    static __device__ __forceinline__ void sort(Key<C>& k) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
            for (int mask = size >> 1; mask > 0; mask >>= 1) exchange(k, mask, ((lane & size) == 0) == ((lane & mask) == 0));
        }
    }
    __device__ __forceinline__ void flush(int top) {
        const int lane = threadIdx.x & 31;
        Key<C> k = lane < count ? waiting[lane] : Key<C>{};
        const Key<C> rest = lane + 32 < count ? waiting[lane + 32] : Key<C>{};
        __syncwarp();
        waiting[lane] = rest;
        count = max(count - 32, 0);
        __syncwarp();
        sort(k);
        merge(k);
        sorted = true;
        last = mine.from(top - 1);
        if (!last.none()) bar = max_nan(bar, last.value());
    }
    // One candidate of every lane with `offer`; the whole warp takes part.
    __device__ __forceinline__ void add(bool offer, C value, int index, int top) {
        const Key<C> k = Key<C>::make(value, index);
        offer = offer && k.above(last);
        const unsigned who = __ballot_sync(0xffffffffu, offer);
        if (offer) waiting[count + __popc(who & ((1u << (threadIdx.x & 31)) - 1u))] = k;
        count += __popc(who);
        __syncwarp();
        if (count >= 32) flush(top);
    }
};

template <int NP, typename C, bool TOP>
struct FwdShared {
    RowSum<NP, C> part[16];
    RowSum<NP, C> block;
    Key<C> first[TOP ? 16 : 1];        // a value of each warp for the first bar
    Key<C> best[TOP ? 16 : 1][64];     // a warp's waiting candidates
    Key<C> list[TOP ? 16 : 1][32];     // its sorted list, where it has one
    int waiting[TOP ? 16 : 1], sorted[TOP ? 16 : 1];
};

// Groups of a thread that are in flight while as many are worked on: enough bytes to cover the latency of
// memory at low degrees, what the registers allow at high ones.
template <typename T, int NP, bool TOP>
constexpr int lp_depth() { return NP == 1 || (NP == 2 && sizeof(T) == 4 && !TOP) ? 2 : 1; }

// Most threads of a forward block.
template <int NP>
constexpr int lp_threads() { return NP > 3 ? 256 : 512; }

// Blocks per SM that the registers have to leave room for, where the compiler would take more than pays: 64 or
// 80 registers a thread (1511 x 50021 bfloat16, degree 1, masked words, four alternatives: 120 us unasked, 102 so;
// 2048 x 32000 float32, degree 3: 198 and 182 us).
template <typename T, int NP, bool TOP>
constexpr int lp_blocks() {
    if (sizeof(T) == 8) return 1;
    if (NP == 4) return 3;
    return NP <= 3 && TOP ? 2 : 1;
}

// One pass over the logits: the blocks of a cluster (gridDim.x of them, one or more) share a row, each
// thread keeps the running sums of its groups of 16 bytes per plane, and the parts are joined in the warp,
// in the block and through distributed shared memory in the cluster's first block.
template <typename T, int NP, bool TOP>
__global__ void __launch_bounds__(lp_threads<NP>(), lp_blocks<T, NP, TOP>())
token_log_probs_fwd_kernel(const __grid_constant__ LogProbParams p) {
    using C = typename Compute<T>::type;
    constexpr int VEC = lp_vec<T>(), DEPTH = lp_depth<T, NP, TOP>();
    __shared__ FwdShared<NP, C, TOP> sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t row = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
    if (row >= p.rows) return;               // the whole cluster
    const int64_t row_at = row * p.x_rs;
    const bool aligned = p.aligned != 0;
    RowGroups groups{};
    groups.set<T>(static_cast<const T*>(p.x[0]) + row_at, p.cols, aligned);
    // this block's groups, and every thread of a warp the same number of steps
    const int per_block = (groups.count + gridDim.x - 1) / gridDim.x;
    const int begin = blockIdx.x * per_block, end = min(begin + per_block, groups.count);
    const int stride = blockDim.x;
    Group<NP, T> now[DEPTH], next[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
        const int g = begin + static_cast<int>(threadIdx.x) + d * stride;
        if (g < end) next[d].load(p, row_at, groups, g);
    }
    const int64_t token = p.tokens[row];
    const bool first_block = blockIdx.x == 0;
    if (token == p.ignore_index) {           // zeros, and no alternatives
        if (first_block) {
            for (int i = threadIdx.x; i < p.np; i += blockDim.x) static_cast<C*>(p.logp[i])[row] = static_cast<C*>(p.entropy[i])[row] = C(0);
            for (int i = threadIdx.x; i <= p.np; i += blockDim.x) static_cast<C*>(p.stats)[row * (p.np + 1) + i] = C(0);
            for (int i = threadIdx.x; i < p.top; i += blockDim.x) {
                p.top_tokens[row * p.top + i] = -1;
                for (int k = 0; k < p.np; ++k) static_cast<C*>(p.top_logp[k])[row * p.top + i] = C(0);
            }
        }
        return;                              // the whole cluster
    }
    const bool inside = token >= 0 && token < p.cols;
    C chosen[NP];                            // the token's logit, asked for now, used at the end
    if (first_block && threadIdx.x == 0 && inside) load_logit<NP, T, C>(p, row, token, chosen);
    const C scale = C(p.scale);
    LogSum<NP, C, (sizeof(T) == 4 ? EXP_LIBRARY : NP > 1 ? EXP_CAREFUL : EXP_PLAIN)> sum;
    sum.clear();
    C largest = -INFINITY, second = -INFINITY;      // of the thread's groups (NaN above all), and
    int where = begin + threadIdx.x;                // the group of the first
    for (int base = begin + warp * 32; base < end; base += DEPTH * stride) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) now[d] = next[d];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int g = base + lane + (DEPTH + d) * stride;
            if (g < end) next[d].load(p, row_at, groups, g);
        }
        C tops[DEPTH], step_top = -INFINITY;
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            tops[d] = base + lane + d * stride < end ? largest_of<T, VEC, C>(now[d].v[0]) : C(-INFINITY);
            step_top = fmax(step_top, tops[d]);
        }
        if (__any_sync(0xffffffffu, step_top * scale > sum.m)) sum.raise(warp_largest(step_top * scale));
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int g = base + lane + d * stride;
            const bool live = g < end;
            const C top = tops[d];
            if (live) {
                Two<C> gs[NP], gt[NP];
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    Two<C> u[NP];
#pragma unroll
                    for (int k = 1; k < NP; ++k) u[k] = now[d].v[k].get(i);
                    if (scale != C(1)) {
#pragma unroll
                        for (int k = 1; k < NP; ++k) u[k] = u[k] * Two<C>(scale);
                    }
                    if (i == 0) sum.template add<true>(now[d].v[0].get(i), scale, u, gs, gt);
                    else sum.template add<false>(now[d].v[0].get(i), scale, u, gs, gt);
                }
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    sum.S[k] = sum.S[k] + gs[k];
                    sum.T[k] = sum.T[k] + gt[k];
                }
            }
            if constexpr (TOP) {
                const bool up = top > largest || top != top;
                second = max_nan(second, up ? largest : top);
                where = up ? g : where;
                largest = max_nan(largest, top);
            }
        }
    }
    RowSum<NP, C> all;
    all.m = sum.m;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        C a, b;
        sum.S[k].get(a, b);
        all.S[k] = a + b;
        sum.T[k].get(a, b);
        all.T[k] = a + b;
    }
    all.join_warp();
    if (lane == 0) sh.part[warp] = all;
    Best<C> best;
    if constexpr (TOP) {
        // Only threads whose largest logit reaches the bar can hold an alternative (a few of the block).  They
        // read that logit's group again, and the rest of theirs only where the second largest reaches it too.
        best.clear(sh.best[warp]);
        best.start(largest, p.top, sh.first);
        const bool look = !(largest < best.bar), everywhere = look && !(second < best.bar);
        if (__any_sync(0xffffffffu, look)) {
            const auto examine = [&](bool here, int g) {
                Group<1, T> again;
                unsigned open = 0;
                if (here) {
                    again.load(p, row_at, groups, g);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        C a, b;
                        again.v[0].get(i / 2).get(a, b);
                        const int index = g * VEC - groups.skew + i;
                        open |= (index >= 0 && index < p.cols && !((i % 2 ? b : a) < best.bar) ? 1u : 0u) << i;
                    }
                }
                while (__any_sync(0xffffffffu, open != 0)) {
                    const int i = __ffs(open) - 1;
                    C value = C(0);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        C a, b;
                        again.v[0].get(j / 2).get(a, b);
                        if (j == i) value = j % 2 ? b : a;
                    }
                    best.add(open != 0, value, g * VEC - groups.skew + i, p.top);
                    open &= open - 1;
                }
            };
            const bool mine = begin + static_cast<int>(threadIdx.x) < end;
            examine(look && mine, where);
            if (__any_sync(0xffffffffu, everywhere))
                for (int base = begin + warp * 32; base < end; base += stride) {
                    const int g = base + lane;
                    examine(everywhere && g < end && g != where, g);
                }
        }
        if (best.sorted) sh.list[warp][lane] = best.mine;
        if (lane == 0) {
            sh.waiting[warp] = best.count;
            sh.sorted[warp] = best.sorted;
        }
    }
    __syncthreads();
    if constexpr (TOP) {
        // the first warp takes what all have: the waiting candidates 32 at a time, and the others' lists
        if (warp == 0) {
            int count = 0;
            for (int w = 0; w < warps; ++w) count += sh.waiting[w];
            for (int base = 0; base < count; base += 32) {
                int at = base + lane;
                Key<C> k{};
                for (int w = 0; w < warps; ++w) {
                    if (at >= 0 && at < sh.waiting[w]) k = sh.best[w][at];
                    at -= sh.waiting[w];
                }
                Best<C>::sort(k);
                best.merge(k);
            }
            for (int w = 1; w < warps; ++w)
                if (sh.sorted[w]) best.merge(sh.list[w][lane]);
        }
    }
    if (warp == 0) {
        if (lane < warps) all = sh.part[lane];
        else all.clear();
        all.join_warp();
    }
    if (gridDim.x > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) sh.block = all;
        if (TOP && warp == 0) sh.list[0][lane] = best.mine;
        cluster.sync();
        if (first_block && warp == 0) {
            if (lane < static_cast<int>(gridDim.x)) all = *cluster.map_shared_rank(&sh.block, lane);
            else all.clear();
            all.join_warp();
            if constexpr (TOP) {
                Key<C> other[LP_MAX_SHARE];
#pragma unroll
                for (int o = 1; o < LP_MAX_SHARE; ++o)
                    if (o < static_cast<int>(gridDim.x)) other[o] = cluster.map_shared_rank(&sh, o)->list[0][lane];
#pragma unroll
                for (int o = 1; o < LP_MAX_SHARE; ++o)
                    if (o < static_cast<int>(gridDim.x)) best.merge(other[o]);
            }
        }
        cluster.sync();                      // the others' shared memory stays until it has been read
    }
    if (!first_block || warp != 0) return;
    // the same in every lane: the normaliser's logarithm; then lane j writes alternative j, lane 0 the rest
    C L[NP];
    // a part with open logits has m > -inf; NaN sums without any (all NaN) count as open
    const bool empty = all.m == -INFINITY && all.S[0] == C(0);
    const C m = all.m == -INFINITY && !empty ? C(NAN) : all.m;
    if (empty) {
#pragma unroll
        for (int k = 0; k < NP; ++k) L[k] = C(0);
    } else {
        s_log<NP, C>(all.S, L);
    }
    if (TOP && lane < p.top) {
        C z[NP], v[NP];
        load_logit<NP, T, C>(p, row, best.mine.at(), z);
        log_prob<NP, C>(z, scale, m, L, v);
        p.top_tokens[row * p.top + lane] = best.mine.at();
#pragma unroll
        for (int k = 0; k < NP; ++k)
            if (k < p.np) static_cast<C*>(p.top_logp[k])[row * p.top + lane] = v[k];
    }
    if (lane == 0) {
        C v[NP], E[NP];
        if (inside) log_prob<NP, C>(chosen, scale, m, L, v);
        s_div<NP, C>(all.T, all.S, E);
        C* stats = static_cast<C*>(p.stats) + row * (p.np + 1);
        stats[0] = m;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if (k >= p.np) continue;
            static_cast<C*>(p.logp[k])[row] = inside ? v[k] : C(NAN);
            static_cast<C*>(p.entropy[k])[row] = empty ? C(0) : L[k] - E[k];
            stats[1 + k] = L[k];
        }
    }
}

// The gradient of a part of a row: blockIdx.x takes its share of the row's groups.  Everything that the row
// has in common is folded into two series first: with d_i = logp_i,
//   dx_i = p_i (*) (B (*) d_i + G) + scale (a [i = token] + sum_j c_j [i = top_j]),
//   B = -scale b,  G = -scale (A + b (*) H).
// The token and the alternatives are written again at the end, in full, by a thread each.
template <int NP, typename C>
struct RowGrad {
    C m, L[NP], B[NP], G[NP];
};

template <int NP, typename T, typename C>
__device__ __forceinline__ void grad_of(const RowGrad<NP, C>& r, C scale, bool has_b, const C (&x)[NP], C (&out)[NP]) {
    C d[NP], P[NP], q[NP];
    log_prob<NP, C>(x, scale, r.m, r.L, d);
    const C p0 = d[0] == -INFINITY ? C(0) : c_exp(d[0]);
    s_exp_dir<NP, C>(d, P);
#pragma unroll
    for (int k = 0; k < NP; ++k) q[k] = r.G[k];
    if (has_b) s_mul_acc<NP, C>(r.B, d, q);
    s_mul<NP, C>(P, q, out);
#pragma unroll
    for (int k = 0; k < NP; ++k) out[k] = p0 == C(0) ? C(0) : p0 * out[k];
}

// The blocks of a row share its groups, up to about eight a thread: enough loads in flight, and few enough blocks
// that reading the row's own numbers (a dozen) costs little.  There is nothing to join.
template <typename T, int NP>
__global__ void __launch_bounds__(256) token_log_probs_bwd_kernel(const __grid_constant__ LogProbParams p) {
    using C = typename Compute<T>::type;
    constexpr int VEC = lp_vec<T>();
    const int64_t row = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
    if (row >= p.rows) return;
    const int64_t token = p.tokens[row], x_at = row * p.x_rs, dx_at = row * p.dx_rs;
    const C* stats = static_cast<const C*>(p.stats_in) + row * (p.np + 1);
    const C scale = C(p.scale);
    RowGrad<NP, C> r;
    r.m = stats[0];
    const bool dead = token == p.ignore_index || r.m == -INFINITY;      // no gradient at all
    RowGroups groups{};
    const T* row0 = static_cast<const T*>(p.x[0]) + x_at;
    bool aligned = p.aligned != 0;
    if (aligned && reinterpret_cast<uintptr_t>(row0) % 16 != reinterpret_cast<uintptr_t>(static_cast<const T*>(p.dx[0]) + dx_at) % 16)
        aligned = false;                                                // the two rows start apart
    groups.set<T>(row0, p.cols, aligned);
    const int per_block = (groups.count + gridDim.x - 1) / gridDim.x;
    const int begin = blockIdx.x * per_block, end = min(begin + per_block, groups.count);
    C a[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) a[k] = r.L[k] = r.B[k] = r.G[k] = C(0);
    if (!dead) {
        C A[NP], b[NP], H[NP], z[NP];
        const bool inside = token >= 0 && token < p.cols;
        bool open = false;
        if (inside && p.has_a) open = to_c<C>(row0[token]) * scale != -INFINITY;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const bool live = k < p.np;
            r.L[k] = live ? stats[1 + k] : C(0);
            H[k] = live ? static_cast<const C*>(p.h[k])[row] : C(0);
            a[k] = !live || !p.has_a ? C(0) : !inside ? C(NAN) : open ? static_cast<const C*>(p.ga[k])[row] : C(0);
            b[k] = live && p.has_b ? static_cast<const C*>(p.gb[k])[row] : C(0);
            A[k] = a[k];
        }
        for (int j = 0; j < (p.has_c ? p.top : 0); ++j) {
            const int64_t at = p.top_at[row * p.top + j];
            if (at < 0 || at >= p.cols || to_c<C>(row0[at]) * scale == -INFINITY) continue;
#pragma unroll
            for (int k = 0; k < NP; ++k)
                if (k < p.np) A[k] += static_cast<const C*>(p.gc[k])[row * p.top + j];
        }
        if (p.has_b) s_mul_acc<NP, C>(b, H, A);
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            r.G[k] = -scale * A[k];
            r.B[k] = -scale * b[k];
        }
    }
    Two<C> L[NP], B[NP], G[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        L[k] = Two<C>(-r.L[k]);
        B[k] = Two<C>(r.B[k]);
        G[k] = Two<C>(r.G[k]);
    }
    for (int g = begin + threadIdx.x; g < end; g += blockDim.x) {
        Group<NP, T> x;
        if (!dead) x.load(p, x_at, groups, g);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            Two<C> d[NP], e[NP], q[NP], o[NP];
            if (dead) {
#pragma unroll
                for (int k = 0; k < NP; ++k) x.v[k].set(i, Two<C>(C(0)));
                continue;
            }
            d[0] = fma2(x.v[0].get(i), Two<C>(scale), Two<C>(-r.m)) + L[0];
#pragma unroll
            for (int k = 1; k < NP; ++k) d[k] = fma2(x.v[k].get(i), Two<C>(scale), L[k]);
            C d0, d1;
            d[0].get(d0, d1);
            C p0, p1;
            if constexpr (sizeof(T) == 4) exp_both<EXP_LIBRARY>(d[0], p0, p1);
            else exp_small_both(d[0], p0, p1);
            if constexpr (NP == 1) d[0] = Two<C>(fmax(d0, C(-1000)), fmax(d1, C(-1000)));   // masked: the weight is 0
            e[0] = Two<C>(C(1));
#pragma unroll
            for (int k = 1; k < NP; ++k) {
                Two<C> t = d[k];
#pragma unroll
                for (int j = 1; j < k; ++j) t = fma2(d[j] * e[k - j], Two<C>(C(j) / C(k)), t);
                e[k] = t;
            }
#pragma unroll
            for (int k = 0; k < NP; ++k) q[k] = G[k];
            if (p.has_b) pair_mul_acc<NP, C>(B, d, q);
            pair_mul<NP, C>(e, q, o);
            const Two<C> w(p0, p1);
#pragma unroll
            for (int k = 0; k < NP; ++k) o[k] = o[k] * w;
            if (NP > 1 && (p0 == C(0) || p1 == C(0))) {      // masked: 0 whatever the directions hold
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    C u, v;
                    o[k].get(u, v);
                    o[k] = Two<C>(p0 == C(0) ? C(0) : u, p1 == C(0) ? C(0) : v);
                }
            }
#pragma unroll
            for (int k = 0; k < NP; ++k) x.v[k].set(i, o[k]);
        }
        const int64_t first = static_cast<int64_t>(g) * VEC - groups.skew;
        if (groups.whole(g)) {
#pragma unroll
            for (int k = 0; k < NP; ++k)
                if (NP <= 6 || k < p.np) *reinterpret_cast<Raw<T, VEC>*>(static_cast<T*>(p.dx[k]) + dx_at + first) = x.v[k];
        } else {
#pragma unroll
            for (int k = 0; k < NP; ++k) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (first + j >= 0 && first + j < p.cols && (NP <= 6 || k < p.np)) {
                        const uint64_t bits = x.v[k].bits(j);
                        memcpy(static_cast<T*>(p.dx[k]) + dx_at + first + j, &bits, sizeof(T));
                    }
            }
        }
    }
    if (dead) return;
    __syncthreads();
    const int specials = 1 + (p.has_c ? p.top : 0);
    if (static_cast<int>(threadIdx.x) >= specials) return;
    const int64_t at = threadIdx.x == 0 ? token : p.top_at[row * p.top + threadIdx.x - 1];
    const int64_t low = static_cast<int64_t>(begin) * VEC - groups.skew, high = static_cast<int64_t>(end) * VEC - groups.skew;
    if (at < 0 || at >= p.cols || at < low || at >= high) return;
    C z[NP], o[NP];
    load_logit<NP, T, C>(p, row, at, z);
    if (z[0] * scale == -INFINITY) return;       // masked: the 0 stands
    grad_of<NP, T, C>(r, scale, p.has_b != 0, z, o);
    if (at == token) {
#pragma unroll
        for (int k = 0; k < NP; ++k) o[k] += scale * a[k];
    }
    for (int j = 0; j < (p.has_c ? p.top : 0); ++j)
        if (p.top_at[row * p.top + j] == at) {
#pragma unroll
            for (int k = 0; k < NP; ++k)
                if (k < p.np) o[k] += scale * static_cast<const C*>(p.gc[k])[row * p.top + j];
        }
#pragma unroll
    for (int k = 0; k < NP; ++k)
        if (k < p.np) static_cast<T*>(p.dx[k])[dx_at + at] = from_c<T>(o[k]);
}

// Rows over the grid's y and z (65535 blocks at most along each).
static dim3 row_grid(int64_t rows, int64_t per_row) {
    const int64_t y = std::min<int64_t>(rows, 65535);
    return dim3(static_cast<unsigned>(per_row), static_cast<unsigned>(y), static_cast<unsigned>(ceil_div(rows, y)));
}

template <typename T, int NP>
static cudaError_t launch_log_probs(const LogProbParams& p, bool backward, cudaStream_t s) {
    const int64_t groups = ceil_div(p.cols, lp_vec<T>()) + 1;
    if (backward) {
        // about eight groups a thread (4096 x 32000 bfloat16 degree 3: 345 us, with four 369 us: each thread reads the
        // row's own numbers first), fewer while the blocks would not fill the GPU (16 rows: 22 us with eight)
        const int64_t threads = groups >= 256 ? 256 : 128;
        int64_t each = 8, per_row = 1;
        for (;; each /= 2) {
            per_row = std::max<int64_t>(1, groups / (each * threads));
            if (each == 1 || p.rows * per_row >= 8 * num_sms()) break;
        }
        PK_LAUNCHED(token_log_probs_bwd_kernel<T, NP><<<row_grid(p.rows, per_row), static_cast<int>(threads), 0, s>>>(p));
        return cudaSuccess;
    }
    // a row is shared by more blocks while the blocks do not fill the GPU and each keeps a group a thread
    int share = 1;
    while (share < LP_MAX_SHARE && p.rows * share < num_sms() && groups / (2 * share) >= 256) share *= 2;
    int threads = share > 1 && groups / share >= 1024 ? lp_threads<NP>() : groups >= 512 ? 256 : 128;
    // many rows: about sixteen groups a thread, so that a row's join is not most of its work (20000 x 16000
    // bfloat16 degree 1: 291 us, with at least four 330 us); few rows: more threads, for their latency
    if (p.rows >= 8 * num_sms())
        while (threads > 32 && groups < 16 * threads) threads /= 2;
    cudaLaunchConfig_t config{};
    config.gridDim = row_grid(p.rows, share);
    config.blockDim = dim3(threads);
    config.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = share;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = share > 1 ? 1 : 0;
    const cudaError_t e = p.top ? cudaLaunchKernelEx(&config, token_log_probs_fwd_kernel<T, NP, true>, p)
                                : cudaLaunchKernelEx(&config, token_log_probs_fwd_kernel<T, NP, false>, p);
    note_launch();
    return e;
}

template <typename T>
static cudaError_t launch_log_probs_np(const LogProbParams& p, bool backward, cudaStream_t s) {
    switch (p.np) {
        case 1: return launch_log_probs<T, 1>(p, backward, s);
        case 2: return launch_log_probs<T, 2>(p, backward, s);
        case 3: return launch_log_probs<T, 3>(p, backward, s);
        case 4: return launch_log_probs<T, 4>(p, backward, s);
        case 5: return launch_log_probs<T, 5>(p, backward, s);
        case 6: return launch_log_probs<T, 6>(p, backward, s);
        case 7: case 8: case 9: return launch_log_probs<T, 9>(p, backward, s);
        default: return launch_log_probs<T, 16>(p, backward, s);
    }
}

static int run_log_probs(int dtype, LogProbParams& p, bool backward, void* stream, const char* name) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // whole groups are aligned in every plane when all bases lie alike within 16 bytes
    p.aligned = 1;
    for (int k = 1; k < p.np; ++k)
        if (reinterpret_cast<uintptr_t>(p.x[k]) % 16 != reinterpret_cast<uintptr_t>(p.x[0]) % 16 ||
            (backward && reinterpret_cast<uintptr_t>(p.dx[k]) % 16 != reinterpret_cast<uintptr_t>(p.dx[0]) % 16))
            p.aligned = 0;
    void* tok;
    cudaError_t e = cudaSuccess;
    prof_begin(name, s, &tok);
    switch (dtype) {
        case PK_F32: e = launch_log_probs_np<float>(p, backward, s); break;
        case PK_F64: e = launch_log_probs_np<double>(p, backward, s); break;
        case PK_BF16: e = launch_log_probs_np<__nv_bfloat16>(p, backward, s); break;
        default: e = launch_log_probs_np<__half>(p, backward, s); break;
    }
    prof_end(name, s, tok);
    if (e != cudaSuccess) return cuda_fail(e, name);
    PK_CHECK_LAUNCH(name);
    return PK_OK;
}

static int check_log_probs(int dtype, int degree, int64_t rows, int64_t cols, int top, const void* const* x,
                           const void* tokens, const void* stats, const void* top_tokens, const std::string& what) {
    if (dtype != PK_F32 && dtype != PK_F64 && dtype != PK_BF16 && dtype != PK_F16)
        return fail(PK_ERR_UNSUPPORTED, what + ": unsupported dtype");
    if (degree < 0 || degree >= PK_MAX_PLANES) return fail(PK_ERR_UNSUPPORTED, what + ": degree out of range");
    if (rows < 0 || cols < 1 || cols > 0x7fffff00) return fail(PK_ERR_ARG, what + ": bad extent");
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
