// Selection over a row of logits by one workgroup (top logits and sampling).
//
// The order of a row is (value descending, index ascending) with -0 equal to +0 and NaN after
// minus infinity. A prefix of that order is named by a key t and a count c: every value with a
// larger key, and the c of lowest index among those with key t. The functions here find (t, c)
// for a prefix of a given length or mass, digit by digit of the key.
#pragma once

#include "pcu_logits.hpp"

#pragma clang fp contract(off)

namespace pcu {

// ---------------------------------------------------------------------- keys

template <typename T> struct KeyOf { using K = uint32_t; };
template <> struct KeyOf<double> { using K = uint64_t; };

// Unsigned keys in the order of the values; 0 for NaN.
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t b = __float_as_uint(v);
    if (v != v)
        return 0u;
    if (v == 0.0f)
        return 0x80000000u;
    return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    if (v != v)
        return 0ull;
    if (v == 0.0)
        return 0x8000000000000000ull;
    return (int64_t)b < 0 ? ~b : b | 0x8000000000000000ull;
}
// The value of a key that is not 0.
__device__ __forceinline__ float value_of(uint32_t k)
{
    return __uint_as_float((int32_t)k < 0 ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ double value_of(uint64_t k)
{
    return __longlong_as_double((long long)((int64_t)k < 0 ? k & 0x7fffffffffffffffull : ~k));
}

template <typename K> struct Prefix {
    K t;
    uint32_t c;
};

// ------------------------------------------------------------------- scans of a wave

template <typename T> __device__ __forceinline__ T wave_inclusive_sum(T v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const T o = __shfl_up(v, off, 64);
        if (lane >= off)
            v += o;
    }
    return v;
}

// --------------------------------------------------------------------- the row

// Calls f(values, first index, count of real ones) for every vector of the row, each thread its
// own ones, four loads in flight.
template <typename S, int NT, typename F>
__device__ __forceinline__ void each_vec(const S *row, uint32_t n, F f)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>;
    constexpr int U = 4;
    const uint32_t vecs = (n + N - 1) / N;
    for (uint32_t i = threadIdx.x; i < vecs; i += NT * U) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            raw[u] = load_vec(row, i + u * NT, n);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t at = (i + u * NT) * N;
            if (at < n) {
                T v[N];
                unpack<S>(raw[u], v);
                f(v, at, n - at < N ? n - at : N);
            }
        }
    }
}

// The same for a wave's own run of vectors [first, last), in order: f(values, index, count) for
// 64 consecutive vectors a step on all lanes (count 0 past the end); stops where f returns true.
template <typename S, typename F>
__device__ __forceinline__ void wave_run(const S *row, uint32_t n, uint32_t first, uint32_t last, F f)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>;
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t i = first; i < last; i += 64) {
        const uint32_t at = (i + lane) * N;
        const bool in = i + lane < last && at < n;
        T v[N];
        unpack<S>(in ? load_vec(row, i + lane, n) : minus_infinities<S>(), v);
        if (f(v, at, in ? (n - at < N ? n - at : N) : 0u))
            return;
    }
}

// ---------------------------------------------------------------- digit by digit

// Among 256 bins, from the highest down: the bin in which the running sum reaches `need`
// (1 <= need <= the sum of all), and what of `need` is left before it. Whole workgroup.
template <typename H> struct Digit {
    uint32_t digit;
    H left;
};
template <typename H> __device__ __forceinline__ Digit<H> find_digit(const H *bins, H need, Digit<H> *out)
{
    __syncthreads(); // the bins are counted
    if (threadIdx.x < 64) {
        const int top = 255 - 4 * (int)threadIdx.x;
        H b[4], own = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            b[i] = bins[top - i];
            own += b[i];
        }
        const H upto = wave_inclusive_sum(own);
        H before = upto - own;
        if (before < need && need <= upto) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (before < need && need <= before + b[i])
                    *out = Digit<H>{(uint32_t)(top - i), need - before};
                before += b[i];
            }
        }
    }
    __syncthreads();
    return *out;
}

// The prefix of `k` values (1 <= k <= n).
template <typename S, int NT>
__device__ __forceinline__ Prefix<typename KeyOf<typename StatOf<S>::T>::K>
select_count(const S *row, uint32_t n, uint32_t k, uint32_t *bins, Digit<uint32_t> *found)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    K prefix = 0;
    for (int shift = (int)sizeof(K) * 8 - 8; shift >= 0; shift -= 8) {
        for (uint32_t b = threadIdx.x; b < 256; b += NT)
            bins[b] = 0;
        __syncthreads();
        each_vec<S, NT>(row, n, [&](const T *v, uint32_t, uint32_t count) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                const K key = key_of(v[i]);
                if (i < count && ((key ^ prefix) >> shift) < 256)
                    atomicAdd(&bins[(uint32_t)(key >> shift) & 255u], 1u);
            }
        });
        const Digit<uint32_t> d = find_digit(bins, k, found);
        prefix |= (K)d.digit << shift;
        k = d.left;
    }
    return {prefix, k};
}

} // namespace pcu
