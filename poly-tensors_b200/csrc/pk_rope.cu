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

#include "pk_vec.cuh"

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
    int stage_at;                       // backward: where the stages begin in shared memory
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

// ---------------------------------------------------------------------------------------------
// Vector form: a row lives in the registers of `lanes` threads (a power of two up to 32; several rows
// share a warp), each holding one slot: V feature pairs, all planes, read once.  With half-split pairs
// a slot is two V-element vectors rotary/2 apart, with adjacent pairs 2V consecutive elements, so both
// members of a pair are in one thread and the rotation needs no exchange; features past `rotary` form
// slots of 2V consecutive elements with angle 0.  The planes stay in their storage type until they are
// worked on (16-bit planes take half the registers), and two neighbouring pairs go through packed float
// arithmetic together: the neighbours of a loaded vector already share a register pair, and so do their
// angles.  The feature weights wait in shared memory in slot order.
struct RowShape {
    int v = 0, lanes = 0, slots = 0;    // v == 0: the scalar form
    Divisor by_heads[2], by_len;
};

template <int V>
struct SlotAt {
    int a, b;           // first features of the slot's two vectors
    int angle;          // first pair, or -1: not turned
    __device__ __forceinline__ SlotAt(const RopeParams& p, int slot) {
        const int turned = p.rotary / (2 * V);
        if (slot >= turned) {
            a = p.rotary + 2 * V * (slot - turned);
            b = a + V;
            angle = -1;
        } else {
            a = p.interleaved ? 2 * V * slot : V * slot;
            b = p.interleaved ? a + V : a + p.rotary / 2;
            angle = V * slot;
        }
    }
    // feature of the first (m == 0) or second member of pair j
    __device__ __forceinline__ int feature(bool interleaved, int j, int m) const {
        if (interleaved) return a + 2 * j + m;
        return (m ? b : a) + j;
    }
};

// Degrees up to 5 have kernels of their own, the higher ones share one with planes to spare.
template <int NP>
__device__ __forceinline__ bool plane_live(int k, int np) {
    return NP <= 6 || k < np;
}

// The V pairs of a slot, all planes: first members in lo, second members in hi.
template <int NP, typename T, int V>
struct Slot {
    using C = typename Compute<T>::type;
    Raw<T, V> lo[NP], hi[NP];

    // All loads are issued before anything reads them: a test between two planes' loads makes the second
    // wait for the first (an early build, without copies ahead: 837 instead of 403 us at 4 x 2048 tokens, 2 x 16
    // heads of 128, degree 3, float32 backward).
    __device__ __forceinline__ void load(const void* const* planes, int np, int64_t off, const SlotAt<V>& at) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if constexpr (NP > 6) lo[k] = hi[k] = Raw<T, V>{};
            if (plane_live<NP>(k, np)) {
                const T* src = static_cast<const T*>(planes[k]) + off;
                lo[k] = *reinterpret_cast<const Raw<T, V>*>(src + at.a);
                hi[k] = *reinterpret_cast<const Raw<T, V>*>(src + at.b);
            }
        }
    }
    __device__ __forceinline__ void store(void* const* planes, int np, int64_t off, const SlotAt<V>& at) const {
#pragma unroll
        for (int k = 0; k < NP; ++k)
            if (plane_live<NP>(k, np)) {
                T* dst = static_cast<T*>(planes[k]) + off;
                *reinterpret_cast<Raw<T, V>*>(dst + at.a) = lo[k];
                *reinterpret_cast<Raw<T, V>*>(dst + at.b) = hi[k];
            }
    }
    // 2V consecutive elements into pairs of neighbours, and back
    __device__ __forceinline__ void part() {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const Raw<T, V> c = lo[k], d = hi[k];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                lo[k].set_bits(j, 2 * j < V ? c.bits((2 * j) % V) : d.bits((2 * j) % V));
                hi[k].set_bits(j, 2 * j + 1 < V ? c.bits((2 * j + 1) % V) : d.bits((2 * j + 1) % V));
            }
        }
    }
    __device__ __forceinline__ void join() {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const Raw<T, V> c = lo[k], d = hi[k];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                lo[k].set_bits(j, j % 2 ? d.bits(j / 2) : c.bits(j / 2));
                hi[k].set_bits(j, (V + j) % 2 ? d.bits((V + j) / 2) : c.bits((V + j) / 2));
            }
        }
    }
    // neighbours 2i and 2i + 1 of the first / second members as a series
    __device__ __forceinline__ void firsts(int i, Two<C> (&x)[NP]) const {
#pragma unroll
        for (int k = 0; k < NP; ++k) x[k] = lo[k].get(i);
    }
    __device__ __forceinline__ void seconds(int i, Two<C> (&x)[NP]) const {
#pragma unroll
        for (int k = 0; k < NP; ++k) x[k] = hi[k].get(i);
    }
    __device__ __forceinline__ void set(int i, const Two<C> (&a)[NP], const Two<C> (&b)[NP]) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            lo[k].set(i, a[k]);
            hi[k].set(i, b[k]);
        }
    }
};

// The angles of a slot's pairs, two neighbours at a time.
template <int V, typename C>
struct Angles {
    Two<C> c[V / 2], s[V / 2];
    __device__ __forceinline__ void load(const RopeParams& p, int64_t pos, int angle) {
        if (pos < 0 || pos >= p.table_rows) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) c[i] = s[i] = Two<C>(C(NAN));
        } else if (angle < 0) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                c[i] = Two<C>(C(1));
                s[i] = Two<C>(C(0));
            }
        } else {
            const int64_t at = pos * (p.rotary / 2) + angle;
            C u[V], v[V];
            load_vec<C, V, C>(static_cast<const C*>(p.cos_t) + at, u);
            load_vec<C, V, C>(static_cast<const C*>(p.sin_t) + at, v);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                c[i] = Two<C>(u[2 * i], u[2 * i + 1]);
                s[i] = Two<C>(v[2 * i], v[2 * i + 1]);
            }
        }
    }
    // (a, b) turned by the angles of pair neighbours i, on every plane; `back` the other way
    template <int NP>
    __device__ __forceinline__ void turn(int i, bool back, Two<C> (&a)[NP], Two<C> (&b)[NP]) const {
        const Two<C> minus = s[i] * Two<C>(C(-1));
        const Two<C> up = back ? minus : s[i], down = back ? s[i] : minus;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const Two<C> u = fma2(b[k], down, a[k] * c[i]);
            b[k] = fma2(a[k], up, b[k] * c[i]);
            a[k] = u;
        }
    }
};

// Weights of a slot's pair neighbours: first members, second members (16 bytes is what shared memory is declared with).
template <typename C>
struct alignas(16) Weight {
    Two<C> lo, hi;
};

// Feature weights in slot order, [plane][neighbours i][slot]; planes past nw are zero.
template <int NP, typename T, int V, typename C>
__device__ __forceinline__ void stage_weights(const RopeParams& p, const HeadSet& set, int slots, Weight<C>* to) {
    if (set.nw == 0) return;
    for (int i = threadIdx.x; i < NP * (V / 2) * slots; i += blockDim.x) {
        const int slot = i % slots, j = i / slots % (V / 2), k = i / (slots * (V / 2));
        const SlotAt<V> at(p, slot);
        const T* w = static_cast<const T*>(set.w[k < set.nw ? k : 0]);
        const auto value = [&](int pair, int m) {
            return k < set.nw ? to_c<C>(w[at.feature(p.interleaved, pair, m)]) : C(0);
        };
        to[i].lo = Two<C>(value(2 * j, 0), value(2 * j + 1, 0));
        to[i].hi = Two<C>(value(2 * j, 1), value(2 * j + 1, 1));
    }
}

// (a, b) (*) w for pair neighbours i of a slot; a weight without directions scales every plane.
template <int NP, int V, typename C>
__device__ __forceinline__ void weigh(const Weight<C>* w, int nw, int slots, int slot, int i, Two<C> (&a)[NP], Two<C> (&b)[NP]) {
    if (nw == 1) {
        const Weight<C> f = w[i * slots + slot];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            a[k] = a[k] * f.lo;
            b[k] = b[k] * f.hi;
        }
    } else if (nw > 1) {
        Two<C> f[NP], g[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const Weight<C> t = w[(k * (V / 2) + i) * slots + slot];
            f[k] = t.lo;
            g[k] = t.hi;
        }
        pair_mul<NP, C>(a, f, a);
        pair_mul<NP, C>(b, g, b);
    }
}

template <int NP, typename C>
__device__ __forceinline__ void group_sum(int lanes, C (&v)[NP]) {
    for (int off = lanes >> 1; off > 0; off >>= 1) {
#pragma unroll
        for (int k = 0; k < NP; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    }
}

// cross += sum over i < k - i of x_i x_(k-i), diag += x_(k/2)^2: x (*) x = 2 cross + diag
template <int NP, typename C>
__device__ __forceinline__ void pair_square_acc(const Two<C> (&x)[NP], Two<C> (&cross)[NP], Two<C> (&diag)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int i = 0; 2 * i < k; ++i) cross[k] = fma2(x[i], x[k - i], cross[k]);
        if (k % 2 == 0) diag[k] = fma2(x[k / 2], x[k / 2], diag[k]);
    }
}

// The mean of x (*) x over the row, and its r.
template <int NP, typename C>
__device__ __forceinline__ void row_rsqrt(const RopeParams& p, int lanes, const Two<C> (&cross)[NP], const Two<C> (&diag)[NP], C (&r)[NP]) {
    C s[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        C a, b;
        fma2(cross[k], Two<C>(C(2)), diag[k]).get(a, b);
        s[k] = a + b;
    }
    group_sum<NP, C>(lanes, s);
    const C inv = C(1) / C(p.dim);
#pragma unroll
    for (int k = 0; k < NP; ++k) s[k] *= inv;
    s[0] += C(p.eps);
    s_rsqrt<NP, C>(s, r);
}

constexpr int ROPE_THREADS = 128;

// Where a block's rows are: the blocks below q_blocks take the queries' rows, the others the keys', in
// strides of all their blocks, so that plane pointers and weights are the same for a whole block.
struct BlockRows {
    int which;
    uint32_t first, stride, rows, heads;
    __device__ __forceinline__ BlockRows(const RopeParams& p, int q_blocks, int lanes) {
        which = static_cast<int>(blockIdx.x) >= q_blocks ? 1 : 0;
        heads = static_cast<uint32_t>(p.set[which].heads);
        rows = static_cast<uint32_t>(p.batch * p.len) * heads;
        first = (blockIdx.x - (which ? q_blocks : 0)) * (ROPE_THREADS / lanes);
        stride = (which ? gridDim.x - q_blocks : q_blocks) * (ROPE_THREADS / lanes);
    }
};

// Persistent: the weights are staged once per block.
template <typename T, int NP, int V>
__global__ void __launch_bounds__(ROPE_THREADS) qk_norm_rope_fwd_vec_kernel(const __grid_constant__ RopeParams p, const RowShape shape, int q_blocks) {
    using C = typename Compute<T>::type;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lanes = shape.lanes, slots = shape.slots;
    const BlockRows mine(p, q_blocks, lanes);
    const HeadSet& set = p.set[mine.which];
    Weight<C>* weights = reinterpret_cast<Weight<C>*>(smem);
    stage_weights<NP, T, V, C>(p, set, slots, weights);
    __syncthreads();
    const uint32_t len = static_cast<uint32_t>(p.len);
    const int sub = threadIdx.x & (lanes - 1);
    const SlotAt<V> at(p, sub);
    const bool inter = p.interleaved != 0;
    // every thread of a warp takes the same number of steps (the sums below need the whole warp)
    for (uint32_t first = mine.first; first < mine.rows; first += mine.stride) {
        const uint32_t row = first + threadIdx.x / lanes;
        const bool live = sub < slots && row < mine.rows;
        const uint32_t token = shape.by_heads[mine.which].divide(row), h = row - token * mine.heads;
        const uint32_t b = shape.by_len.divide(token), t = token - b * len;
        Slot<NP, T, V> x;
        Angles<V, C> angles;
        Two<C> cross[NP], diag[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) cross[k] = diag[k] = Two<C>(C(0));
        if (live) {
            x.load(set.x, p.np, b * set.bs + t * set.ts + h * set.hs, at);
            angles.load(p, position_of(p, b, t), at.angle);
            if (inter) x.part();
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                Two<C> e[NP];
                x.firsts(i, e);
                pair_square_acc<NP, C>(e, cross, diag);
                x.seconds(i, e);
                pair_square_acc<NP, C>(e, cross, diag);
            }
        }
        C r[NP];
        row_rsqrt<NP, C>(p, lanes, cross, diag, r);
        if (!live) continue;
        Two<C> rr[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) rr[k] = Two<C>(r[k]);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            Two<C> e[NP], f[NP];
            x.firsts(i, e);
            x.seconds(i, f);
            pair_mul<NP, C>(e, rr, e);
            pair_mul<NP, C>(f, rr, f);
            weigh<NP, V, C>(weights, set.nw, slots, sub, i, e, f);
            angles.turn(i, false, e, f);
            x.set(i, e, f);
        }
        if (inter) x.join();
        x.store(set.out, p.np, ((b * set.heads + h) * p.len + t) * p.dim, at);
    }
}

// What a thread has under way for its next row: its slot of every plane of x and of the gradient and its angles,
// copied to places in shared memory that only it reads, so that its own wait for the copies is all that
// orders them.
template <typename T, int NP, int V>
struct Stage {
    using C = typename Compute<T>::type;
    static constexpr int VB = V * sizeof(T), AB = V * sizeof(C);
    static constexpr int BYTES = ROPE_THREADS * (4 * NP * VB + 2 * AB);
    unsigned char* at;

    __device__ __forceinline__ explicit Stage(unsigned char* base) : at(base) {}
    __device__ __forceinline__ unsigned char* place(int i) const { return at + (i * ROPE_THREADS + threadIdx.x) * VB; }
    __device__ __forceinline__ C* angle(int i) const {
        return reinterpret_cast<C*>(at + ROPE_THREADS * 4 * NP * VB + (i * ROPE_THREADS + threadIdx.x) * AB);
    }
    template <int BYTES_>
    static __device__ __forceinline__ void copy(void* to, const void* from) {
        if constexpr (BYTES_ == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES_) : "memory");
    }
    __device__ __forceinline__ void fetch(int first, const void* const* planes, int np, int64_t off, const SlotAt<V>& slot) const {
#pragma unroll
        for (int k = 0; k < NP; ++k)
            if (plane_live<NP>(k, np)) {
                const T* src = static_cast<const T*>(planes[k]) + off;
                copy<VB>(place(first + 2 * k), src + slot.a);
                copy<VB>(place(first + 2 * k + 1), src + slot.b);
            }
    }
    __device__ __forceinline__ void fetch_angles(const RopeParams& p, int64_t pos, int pair) const {
        const bool inside = pos >= 0 && pos < p.table_rows;
        if (inside && pair >= 0) {
            const int64_t from = pos * (p.rotary / 2) + pair;
#pragma unroll
            for (int v = 0; v < AB; v += 16) {
                constexpr int PIECE = AB < 16 ? AB : 16;
                copy<PIECE>(reinterpret_cast<unsigned char*>(angle(0)) + v, reinterpret_cast<const unsigned char*>(static_cast<const C*>(p.cos_t) + from) + v);
                copy<PIECE>(reinterpret_cast<unsigned char*>(angle(1)) + v, reinterpret_cast<const unsigned char*>(static_cast<const C*>(p.sin_t) + from) + v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                angle(0)[j] = inside ? C(1) : C(NAN);
                angle(1)[j] = inside ? C(0) : C(NAN);
            }
        }
    }
    __device__ __forceinline__ void read(int first, int np, Slot<NP, T, V>& s, bool inter) const {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if constexpr (NP > 6) s.lo[k] = s.hi[k] = Raw<T, V>{};
            if (plane_live<NP>(k, np)) {
                s.lo[k] = *reinterpret_cast<const Raw<T, V>*>(place(first + 2 * k));
                s.hi[k] = *reinterpret_cast<const Raw<T, V>*>(place(first + 2 * k + 1));
            }
        }
        if (inter) s.part();
    }
    __device__ __forceinline__ void read_angles(Angles<V, C>& a) const {
        C u[V], v[V];
        load_vec<C, V, C>(angle(0), u);
        load_vec<C, V, C>(angle(1), v);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            a.c[i] = Two<C>(u[2 * i], u[2 * i + 1]);
            a.s[i] = Two<C>(v[2 * i], v[2 * i + 1]);
        }
    }
};

// A thread keeps its slot from row to row, so the weight gradient is summed in registers; groups of a
// warp are joined by shuffles, warps in turn through shared memory, blocks by the weight-sum kernel,
// always in the same order.  The next row is on its way into shared memory while one is worked on: with the
// sums in registers too few warps fit an SM to cover the loads by themselves (bfloat16 degree 3 below: 256 us
// with loads straight into registers, then 241 us), and a row is read from there a second time after its sums.
//
// Measured on B200 (4 x 2048 tokens, 2 x 16 heads of 128; bytes are the planes read and written once):
// forward float32 degree 3 172 us = 6.2 TB/s, bfloat16 degree 3 106 us = 5.1 TB/s; backward 292 us =
// 5.5 TB/s and 241 us = 3.3 TB/s.  float32 runs near the rate of a copy.  The 16-bit backward is held up by latency:
// at 152 registers 17 % of the warps are active, and no pipe is near full (issue slots 54 %, L1 50 %, FMA 45 %).
// At degree 0 the angles are most of what a row reads, again for each of a token's heads: forward 40 us = 3.4 TB/s
// (issue 66 %, L1 58 %), backward 75 us = 2.7 TB/s (L1 68 %, waits for shared memory).  Degree 3 asks for three
// blocks per SM (float32 300 us with the two that its registers would allow; bfloat16 at 4 x 4096 tokens, 32 + 8
// heads 561, 549 so); more, or the same at other degrees, spills and loses.
template <typename T, int NP, int V>
__global__ void __launch_bounds__(ROPE_THREADS, NP == 4 ? 3 : 1) qk_norm_rope_bwd_vec_kernel(const __grid_constant__ RopeParams p, const RowShape shape, int q_blocks) {
    using C = typename Compute<T>::type;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lanes = shape.lanes, slots = shape.slots;
    const BlockRows mine(p, q_blocks, lanes);
    const HeadSet& set = p.set[mine.which];
    Weight<C>* weights = reinterpret_cast<Weight<C>*>(smem);
    stage_weights<NP, T, V, C>(p, set, slots, weights);
    __syncthreads();
    const uint32_t len = static_cast<uint32_t>(p.len);
    const int sub = threadIdx.x & (lanes - 1);
    const SlotAt<V> at(p, sub);
    const bool inter = p.interleaved != 0;
    const int nsum = set.partial ? set.nw : 0;
    Two<C> acc[NP][V / 2][2];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) acc[k][i][0] = acc[k][i][1] = Two<C>(C(0));
    }
    using S = Stage<T, NP, V>;
    unsigned char* stages = smem + p.stage_at;
    const bool mine_slot = sub < slots;
    const auto fetch = [&](uint32_t row, int stage) {
        if (mine_slot && row < mine.rows) {
            const uint32_t token = shape.by_heads[mine.which].divide(row), h = row - token * mine.heads;
            const uint32_t b = shape.by_len.divide(token), t = token - b * len;
            const S s(stages + stage * S::BYTES);
            s.fetch(0, set.x, p.np, b * set.bs + t * set.ts + h * set.hs, at);
            s.fetch(2 * NP, set.g, p.np, b * set.g_bs + h * set.g_hs + t * set.g_ts, at);
            s.fetch_angles(p, position_of(p, b, t), at.angle);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int stage = 0;
    fetch(mine.first + threadIdx.x / lanes, 0);
    for (uint32_t first = mine.first; first < mine.rows; first += mine.stride, stage ^= 1) {
        const uint32_t row = first + threadIdx.x / lanes;
        const bool live = mine_slot && row < mine.rows;
        fetch(row + mine.stride, stage ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        const S here(stages + stage * S::BYTES);
        Slot<NP, T, V> x, g;
        Angles<V, C> angles;
        Two<C> cross[NP], diag[NP], mean[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) cross[k] = diag[k] = mean[k] = Two<C>(C(0));
        if (live) {
            here.read(0, p.np, x, inter);
            here.read(2 * NP, p.np, g, inter);
            here.read_angles(angles);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                Two<C> e[NP], f[NP], u[NP];
                g.firsts(i, e);
                g.seconds(i, f);
                angles.turn(i, true, e, f);
                weigh<NP, V, C>(weights, set.nw, slots, sub, i, e, f);
                x.firsts(i, u);
                pair_square_acc<NP, C>(u, cross, diag);
                pair_mul_acc<NP, C>(u, e, mean);
                x.seconds(i, u);
                pair_square_acc<NP, C>(u, cross, diag);
                pair_mul_acc<NP, C>(u, f, mean);
            }
        }
        C m[NP], r[NP], q[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            C u, v;
            mean[k].get(u, v);
            m[k] = u + v;
        }
        group_sum<NP, C>(lanes, m);
        row_rsqrt<NP, C>(p, lanes, cross, diag, r);
        if (!live) continue;
        s_mul<NP, C>(r, r, q);
        s_mul<NP, C>(q, r, q);
        s_mul<NP, C>(q, m, q);
        Two<C> rr[NP], qq[NP];
        const C minus = C(-1) / C(p.dim);
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            rr[k] = Two<C>(r[k]);
            qq[k] = Two<C>(q[k] * minus);       // -(r (*) r (*) r (*) mean)
        }
        // read again: what the sums above left no registers for
        asm volatile("" ::: "memory");
        here.read(0, p.np, x, inter);
        here.read(2 * NP, p.np, g, inter);
        here.read_angles(angles);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            Two<C> e[2][NP], f[2][NP];
            x.firsts(i, e[0]);
            x.seconds(i, e[1]);
            g.firsts(i, f[0]);
            g.seconds(i, f[1]);
            angles.turn(i, true, f[0], f[1]);
#pragma unroll
            for (int m2 = 0; m2 < 2; ++m2) {
                pair_mul<NP, C>(f[m2], rr, f[m2]);          // g' (*) r
                if (nsum > 1) {                             // (g' (*) r) (*) x
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
#pragma unroll
                        for (int j = 0; j <= k; ++j) acc[k][i][m2] = fma2(f[m2][j], e[m2][k - j], acc[k][i][m2]);
                    }
                } else if (nsum == 1) {
                    acc[0][i][m2] = fma2(f[m2][0], e[m2][0], acc[0][i][m2]);
                }
            }
            weigh<NP, V, C>(weights, set.nw, slots, sub, i, f[0], f[1]);
            pair_mul_acc<NP, C>(e[0], qq, f[0]);
            pair_mul_acc<NP, C>(e[1], qq, f[1]);
            x.set(i, f[0], f[1]);
        }
        if (inter) x.join();
        x.store(set.out, p.np, static_cast<int64_t>(row) * p.dim, at);
    }
    if (nsum == 0) return;
    __syncthreads();                            // the weights are done with: their place takes the sums
    C* sums = reinterpret_cast<C*>(smem);
    const int lane = threadIdx.x & 31, dim = static_cast<int>(p.dim);
    for (int of = 0; of < ROPE_THREADS / 32; ++of) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if (k >= nsum) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {       // first members, then second members
                C u, v;
                acc[k][i / 2][i % 2].get(u, v);
                for (int off = lanes; off < 32; off <<= 1) {
                    u += __shfl_xor_sync(0xffffffffu, u, off);
                    v += __shfl_xor_sync(0xffffffffu, v, off);
                }
                if (static_cast<int>(threadIdx.x >> 5) == of && lane < slots) {
                    C* to = sums + k * dim;
                    const int a = at.feature(inter, i / 2 * 2, i % 2), b = at.feature(inter, i / 2 * 2 + 1, i % 2);
                    to[a] = of ? to[a] + u : u;
                    to[b] = of ? to[b] + v : v;
                }
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < nsum * dim; i += ROPE_THREADS)
        static_cast<C*>(set.partial)[static_cast<int64_t>(blockIdx.x - (mine.which ? q_blocks : 0)) * nsum * dim + i] = sums[i];
}

struct WeightSum {
    const void* partial;   // [blocks][nw][D]
    void* dw[PK_MAX_PLANES];
    int blocks, nw;
};
struct WeightSumParams {
    WeightSum set[2];
    int dim;
};

// dw = the sum of the blocks' partial sums: 32 values per block, eight threads for each, which take every
// eighth partial and are joined in order.
template <typename T>
__global__ void __launch_bounds__(256) qk_weight_sum_kernel(const WeightSumParams p) {
    using C = typename Compute<T>::type;
    __shared__ C part[8][32];
    const WeightSum& set = p.set[blockIdx.y];
    const int count = set.nw * p.dim;
    const int i = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    C acc = C(0);
    if (i < count) {
#pragma unroll 8
        for (int b = g; b < set.blocks; b += 8) acc += static_cast<const C*>(set.partial)[static_cast<int64_t>(b) * count + i];
    }
    part[g][threadIdx.x & 31] = acc;
    __syncthreads();
    if (g == 0 && i < count) {
        for (int j = 1; j < 8; ++j) acc += part[j][threadIdx.x];
        static_cast<T*>(set.dw[i / p.dim])[i % p.dim] = from_c<T>(acc);
    }
}

constexpr int ROPE_MAX_DIM = 1024;

// Whether the register form with NP planes and V-element vectors is built: the planes of a slot take `held`
// registers, and the backward holds the input's, the gradient's and the weight sums.  Past these
// limits the compiler spills (degree 3: 16-byte vectors forward and backward for float32, float64; 8-byte
// ones backward for the 16-bit types).
constexpr bool vec_built(int np, int v, int compute_bytes, bool backward) {
    const int held = np * 2 * v * compute_bytes / 4;
    return v >= 2 && held <= (backward ? 48 : 80);
}

// Vectors of 16 bytes, else of 8 or 4 (two elements at least), where that form is built, no pair or passing feature
// is cut, every base and stride is a multiple of the vector, and a row fits a warp; otherwise the scalar form, which
// reads each row twice, element by element (2 x 2048 tokens, 2 x 16 heads of 128, backward: float32 degree 9, where no
// vector form is built, 2860 us; bfloat16 degree 7 with 4-byte vectors 523 us).
template <typename T, int NP>
static RowShape row_shape(const RopeParams& p, bool backward) {
    RowShape s;
    constexpr int cb = sizeof(typename Compute<T>::type);
    const int64_t rows = p.batch * p.len * (p.set[0].heads + p.set[1].heads);
    for (int bytes = 16; bytes >= 2 * static_cast<int>(sizeof(T)) && bytes >= 4; bytes /= 2) {
        const int v = bytes / static_cast<int>(sizeof(T));
        if (!vec_built(NP, v, cb, backward) || p.rotary % (2 * v) || (p.dim - p.rotary) % (2 * v) || p.dim / (2 * v) > 32)
            continue;
        const int table = std::min(16, v * cb);
        bool ok = rows * 32 < (1ll << 32) && planes_aligned(&p.cos_t, 1, table) && planes_aligned(&p.sin_t, 1, table);
        for (const HeadSet& set : p.set) {
            if (set.heads == 0) continue;
            ok = ok && planes_aligned(set.x, p.np, bytes) && planes_aligned(set.out, p.np, bytes) &&
                 planes_aligned(set.w, set.nw, bytes) && set.bs % v == 0 && set.ts % v == 0 && set.hs % v == 0;
            if (backward)
                ok = ok && planes_aligned(set.g, p.np, bytes) && set.g_bs % v == 0 && set.g_hs % v == 0 && set.g_ts % v == 0;
        }
        if (!ok) continue;
        s.v = v;
        s.slots = static_cast<int>(p.dim) / (2 * v);
        s.lanes = 1;
        while (s.lanes < s.slots) s.lanes *= 2;
        for (int i = 0; i < 2; ++i) s.by_heads[i] = Divisor(static_cast<uint32_t>(std::max<int64_t>(1, p.set[i].heads)));
        s.by_len = Divisor(static_cast<uint32_t>(p.len));
        return s;
    }
    return s;
}

// The backward runs as many blocks as the GPU holds at a time (more would only add partial weight sums), at
// most ROPE_SUM_BLOCKS per SM, which is what the workspace has room for.
constexpr int ROPE_SUM_BLOCKS = 16;

// Blocks of the queries and of the keys, in proportion to their rows: at most `room` (about) together, and
// no more than have a row.
struct BlockShare {
    int q = 0, k = 0;
    BlockShare() = default;
    BlockShare(const RopeParams& p, int64_t room, int64_t rows_per_block) {
        const int64_t q_rows = p.batch * p.len * p.set[0].heads, k_rows = p.batch * p.len * p.set[1].heads;
        const auto share = [&](int64_t rows) {
            if (rows == 0) return 0;
            return static_cast<int>(std::min(std::max<int64_t>(1, room * rows / (q_rows + k_rows)), ceil_div(rows, rows_per_block)));
        };
        q = share(q_rows);
        k = share(k_rows);
    }
};

struct BwdLaunch {
    int sums[2];            // planes of the weight gradients wanted
    void* workspace;
    BlockShare blocks;

    template <typename C>
    void plan(RopeParams& p, int resident, int64_t rows_per_block) {
        blocks = BlockShare(p, static_cast<int64_t>(std::min(resident, ROPE_SUM_BLOCKS)) * num_sms(), rows_per_block);
        C* at = static_cast<C*>(workspace);
        p.set[0].partial = sums[0] ? at : nullptr;
        p.set[1].partial = sums[1] ? at + static_cast<int64_t>(blocks.q) * sums[0] * p.dim : nullptr;
    }
};

template <typename K>
static int resident_blocks(K kernel, int threads, size_t smem) {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) == cudaSuccess && n > 0 ? n : 1;
}

template <typename T, int NP, int V>
static bool launch_rope_vec(RopeParams& p, const RowShape& row, BwdLaunch* bwd, cudaStream_t s) {
    using C = typename Compute<T>::type;
    if (row.v != V) return false;
    const size_t weights = static_cast<size_t>(NP) * (V / 2) * row.slots * sizeof(Weight<C>);
    const int64_t rows_per_block = ROPE_THREADS / row.lanes;
    if (bwd) {
        if constexpr (vec_built(NP, V, sizeof(C), true)) {
            const auto kernel = qk_norm_rope_bwd_vec_kernel<T, NP, V>;
            // the weights' place also takes the sums at the end
            p.stage_at = static_cast<int>(round_up(std::max<int64_t>(weights, static_cast<int64_t>(std::max(bwd->sums[0], bwd->sums[1])) * p.dim * sizeof(C)), 16));
            const size_t smem = p.stage_at + 2 * static_cast<size_t>(Stage<T, NP, V>::BYTES);
            if (smem > 48 * 1024)
                cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            bwd->plan<C>(p, resident_blocks(kernel, ROPE_THREADS, smem), rows_per_block);
            PK_LAUNCHED(kernel<<<bwd->blocks.q + bwd->blocks.k, ROPE_THREADS, smem, s>>>(p, row, bwd->blocks.q));
        }
    } else {
        if constexpr (vec_built(NP, V, sizeof(C), false)) {
            const auto kernel = qk_norm_rope_fwd_vec_kernel<T, NP, V>;
            const BlockShare blocks(p, static_cast<int64_t>(num_sms()) * resident_blocks(kernel, ROPE_THREADS, weights), rows_per_block);
            PK_LAUNCHED(kernel<<<blocks.q + blocks.k, ROPE_THREADS, weights, s>>>(p, row, blocks.q));
        }
    }
    return true;
}

template <typename T, int NP>
static void launch_rope_np(RopeParams& p, BwdLaunch* bwd, cudaStream_t s) {
    using C = typename Compute<T>::type;
    const RowShape row = row_shape<T, NP>(p, bwd != nullptr);
    if (launch_rope_vec<T, NP, 16 / sizeof(T)>(p, row, bwd, s)) return;
    if constexpr (sizeof(T) <= 4) {
        if (launch_rope_vec<T, NP, 8 / sizeof(T)>(p, row, bwd, s)) return;
    }
    if constexpr (sizeof(T) == 2) {
        if (launch_rope_vec<T, NP, 2>(p, row, bwd, s)) return;
    }
    if (bwd) {
        // as many warps as have room for their weight sums in shared memory
        const size_t per_warp = static_cast<size_t>(std::max(bwd->sums[0], bwd->sums[1])) * p.dim * sizeof(C);
        int warps = 8;
        while (warps > 1 && warps * per_warp > 96 * 1024) warps /= 2;
        const size_t smem = warps * per_warp;
        const auto kernel = qk_norm_rope_bwd_kernel<T, NP>;
        if (smem > 48 * 1024)
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        bwd->plan<C>(p, resident_blocks(kernel, warps * 32, smem), warps);
        PK_LAUNCHED(kernel<<<bwd->blocks.q + bwd->blocks.k, warps * 32, smem, s>>>(p, bwd->blocks.q));
    } else {
        const int64_t rows = p.batch * p.len * (p.set[0].heads + p.set[1].heads);
        const int grid = static_cast<int>(std::min<int64_t>(ceil_div(rows, 8), static_cast<int64_t>(num_sms()) * 32));
        PK_LAUNCHED(qk_norm_rope_fwd_kernel<T, NP><<<grid, 256, 0, s>>>(p));
    }
}

template <typename T>
static void launch_rope(RopeParams& p, BwdLaunch* bwd, cudaStream_t s) {
    switch (p.np) {
        case 1: launch_rope_np<T, 1>(p, bwd, s); break;
        case 2: launch_rope_np<T, 2>(p, bwd, s); break;
        case 3: launch_rope_np<T, 3>(p, bwd, s); break;
        case 4: launch_rope_np<T, 4>(p, bwd, s); break;
        case 5: launch_rope_np<T, 5>(p, bwd, s); break;
        case 6: launch_rope_np<T, 6>(p, bwd, s); break;
        case 7: case 8: case 9: launch_rope_np<T, 9>(p, bwd, s); break;
        default: launch_rope_np<T, 16>(p, bwd, s); break;
    }
}

static void launch_rope_dtype(int dtype, RopeParams& p, BwdLaunch* bwd, cudaStream_t s) {
    switch (dtype) {
        case PK_F32: launch_rope<float>(p, bwd, s); break;
        case PK_F64: launch_rope<double>(p, bwd, s); break;
        case PK_BF16: launch_rope<__nv_bfloat16>(p, bwd, s); break;
        default: launch_rope<__half>(p, bwd, s); break;
    }
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
    launch_rope_dtype(dtype, p, nullptr, s);
    prof_end("qk_norm_rope_fwd", s, tok);
    PK_CHECK_LAUNCH(what);
    return PK_OK;
}

size_t pk_qk_norm_rope_bwd_workspace_size(int dtype, int degree, int64_t batch, int64_t len, int64_t q_heads,
                                          int64_t k_heads, int64_t dim, int dqw_planes, int dkw_planes) {
    if (check_rope(dtype, degree, batch, len, q_heads, k_heads, dim, 0, nullptr, nullptr, 0,
                   "pk_qk_norm_rope_bwd_workspace_size"))
        return 0;
    if (dqw_planes < 0 || dqw_planes > degree + 1 || dkw_planes < 0 || dkw_planes > degree + 1) return 0;
    return static_cast<size_t>(num_sms()) * ROPE_SUM_BLOCKS * std::max(dqw_planes, dkw_planes) * dim *
           (dtype == PK_F64 ? 8 : 4) + 2 * static_cast<size_t>(dqw_planes + dkw_planes) * dim * 8;
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
    const size_t need = pk_qk_norm_rope_bwd_workspace_size(dtype, degree, batch, len, q_heads, k_heads, dim, sums[0],
                                                           sums[1]);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(PK_ERR_WORKSPACE, "pk_qk_norm_rope_bwd: workspace missing or too small");
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
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    void* tok;
    prof_begin("qk_norm_rope_bwd", s, &tok);
    BwdLaunch bwd{{sums[0], sums[1]}, workspace, {}};
    if (batch * len * (q_heads + k_heads) > 0) launch_rope_dtype(dtype, p, &bwd, s);
    if (sums[0] + sums[1] > 0) {
        const int blocks[2] = {bwd.blocks.q, bwd.blocks.k};
        WeightSumParams total{};
        total.dim = static_cast<int>(dim);
        for (int i = 0; i < 2; ++i) {
            total.set[i].partial = p.set[i].partial;
            total.set[i].blocks = blocks[i];
            total.set[i].nw = sums[i];
            for (int j = 0; j < sums[i]; ++j) total.set[i].dw[j] = dw[i][j];
        }
        const dim3 grid(static_cast<unsigned>(ceil_div(std::max(sums[0], sums[1]) * dim, 32)), 2);
        switch (dtype) {
            case PK_F32: PK_LAUNCHED(qk_weight_sum_kernel<float><<<grid, 256, 0, s>>>(total)); break;
            case PK_F64: PK_LAUNCHED(qk_weight_sum_kernel<double><<<grid, 256, 0, s>>>(total)); break;
            case PK_BF16: PK_LAUNCHED(qk_weight_sum_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(total)); break;
            default: PK_LAUNCHED(qk_weight_sum_kernel<__half><<<grid, 256, 0, s>>>(total)); break;
        }
    }
    prof_end("qk_norm_rope_bwd", s, tok);
    PK_CHECK_LAUNCH(what);
    return PK_OK;
}

}  // extern "C"
