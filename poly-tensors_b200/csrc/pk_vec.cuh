// Aligned vectors of a storage type in registers, and loads and stores of them in pieces of 16 bytes at most.
#pragma once

#include <type_traits>

#include "pk_series.cuh"

namespace pk {

// A vector asks for its own size, for no more than 16 bytes though: longer ones are loaded in pieces, since callers
// check and lay out memory by 16 bytes (a type's alignment is the compiler's leave to use one wide access).
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vec {
    T e[V];
};

template <typename T, int V, typename C>
__device__ __forceinline__ void load_vec(const T* p, C (&v)[V]) {
    const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_c<C>(t.e[j]);
}

// Whether `bytes`-wide accesses fit every plane's base.
inline bool planes_aligned(const void* const* planes, int n, int bytes) {
    for (int k = 0; k < n; ++k)
        if (reinterpret_cast<uintptr_t>(planes[k]) % bytes) return false;
    return true;
}

}  // namespace pk

namespace pk {

// Two values that go through the same arithmetic.  For float they share one 64-bit register pair and every
// operation is one packed instruction (add / mul / fma .f32x2, round to nearest, the same result as
// two scalar ones): the series products of the row kernels issue half the instructions.
template <typename C> struct Two;

template <> struct Two<float> {
    unsigned long long v;
    Two() = default;
    __device__ __forceinline__ Two(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ explicit Two(float both) : Two(both, both) {}
    __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ Two<float> operator+(Two<float> a, Two<float> b) {
    Two<float> r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two<float> operator*(Two<float> a, Two<float> b) {
    Two<float> r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two<float> fma2(Two<float> a, Two<float> b, Two<float> c) {
    Two<float> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

template <> struct Two<double> {
    double lo, hi;
    Two() = default;
    __device__ __forceinline__ Two(double a, double b) : lo(a), hi(b) {}
    __device__ __forceinline__ explicit Two(double both) : lo(both), hi(both) {}
    __device__ __forceinline__ void get(double& a, double& b) const { a = lo; b = hi; }
};
__device__ __forceinline__ Two<double> operator+(Two<double> a, Two<double> b) { return {a.lo + b.lo, a.hi + b.hi}; }
__device__ __forceinline__ Two<double> operator*(Two<double> a, Two<double> b) { return {a.lo * b.lo, a.hi * b.hi}; }
__device__ __forceinline__ Two<double> fma2(Two<double> a, Two<double> b, Two<double> c) {
    return {fma(a.lo, b.lo, c.lo), fma(a.hi, b.hi, c.hi)};
}

// acc += a (*) b, truncated, on pairs
template <int NP, typename C>
__device__ __forceinline__ void pair_mul_acc(const Two<C> (&a)[NP], const Two<C> (&b)[NP], Two<C> (&acc)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int i = 0; i <= k; ++i) acc[k] = fma2(a[i], b[k - i], acc[k]);
    }
}

// out = a (*) b, truncated, on pairs (out may be a or b)
template <int NP, typename C>
__device__ __forceinline__ void pair_mul(const Two<C> (&a)[NP], const Two<C> (&b)[NP], Two<C> (&out)[NP]) {
    Two<C> r[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        r[k] = a[0] * b[k];
#pragma unroll
        for (int i = 1; i <= k; ++i) r[k] = fma2(a[i], b[k - i], r[k]);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) out[k] = r[k];
}

// V elements of a storage type as loaded, read and written two neighbours at a time in compute type.
template <typename T, int V>
struct alignas(sizeof(T) * V) Raw {
    uint32_t w[V * sizeof(T) / 4];

    __device__ __forceinline__ Two<typename Compute<T>::type> get(int i) const {
        if constexpr (std::is_same<T, float>::value) {
            return {__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])};
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            return {__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)};
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            return {f.x, f.y};
        } else {
            return {__hiloint2double(w[4 * i + 1], w[4 * i]), __hiloint2double(w[4 * i + 3], w[4 * i + 2])};
        }
    }
    __device__ __forceinline__ void set(int i, Two<typename Compute<T>::type> v) {
        typename Compute<T>::type a, b;
        v.get(a, b);
        if constexpr (std::is_same<T, float>::value) {
            w[2 * i] = __float_as_uint(a);
            w[2 * i + 1] = __float_as_uint(b);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            *reinterpret_cast<__nv_bfloat162*>(&w[i]) = __floats2bfloat162_rn(a, b);
        } else if constexpr (std::is_same<T, __half>::value) {
            *reinterpret_cast<__half2*>(&w[i]) = __floats2half2_rn(a, b);
        } else {
            w[4 * i] = __double2loint(a);
            w[4 * i + 1] = __double2hiint(a);
            w[4 * i + 2] = __double2loint(b);
            w[4 * i + 3] = __double2hiint(b);
        }
    }
    // element j of a row of raw words, for moving elements without converting them
    __device__ __forceinline__ uint64_t bits(int j) const {
        if constexpr (sizeof(T) == 2) return (w[j / 2] >> (16 * (j % 2))) & 0xffffu;
        else if constexpr (sizeof(T) == 4) return w[j];
        else return static_cast<uint64_t>(w[2 * j + 1]) << 32 | w[2 * j];
    }
    __device__ __forceinline__ void set_bits(int j, uint64_t v) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t other = j % 2 ? w[j / 2] & 0xffffu : w[j / 2] & 0xffff0000u;
            w[j / 2] = other | static_cast<uint32_t>(v) << (16 * (j % 2));
        } else if constexpr (sizeof(T) == 4) {
            w[j] = static_cast<uint32_t>(v);
        } else {
            w[2 * j] = static_cast<uint32_t>(v);
            w[2 * j + 1] = static_cast<uint32_t>(v >> 32);
        }
    }
};

// 32-bit division by a divisor known at launch: q = (t + (n - t) / 2) >> (l - 1) with t = high(m n),
// 2^(l-1) < d <= 2^l, m = floor(2^32 (2^l - d) / d) + 1 (Granlund and Montgomery, "Division by invariant
// integers using multiplication", PLDI 1994).
struct Divisor {
    uint32_t d, m;
    int shift;
    Divisor() = default;
    explicit Divisor(uint32_t div) : d(div), m(0), shift(0) {
        int l = 0;
        while (l < 32 && (1ull << l) < div) ++l;
        m = static_cast<uint32_t>(((1ull << 32) * ((1ull << l) - div)) / div + 1);
        shift = l - 1;
    }
    __device__ __forceinline__ uint32_t divide(uint32_t n) const {
        if (shift < 0) return n;
        const uint32_t t = __umulhi(m, n);
        return (t + ((n - t) >> 1)) >> shift;
    }
};

}  // namespace pk
