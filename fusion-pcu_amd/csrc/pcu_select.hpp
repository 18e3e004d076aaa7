// Selection over a row of logits by one workgroup (top logits and sampling).
//
// The order of a row is (value descending, index ascending) with -0 equal to +0 and NaN after
// minus infinity. The usual way to a prefix of that order is a short list: a bound that at least
// as many values reach as are wanted and few more, the values that reach it gathered in LDS
// and sorted there. The bound comes from the largest values of groups of the row: k groups whose
// largest value reaches t mean k values that reach t, and where large values do not lie
// side by side few others do (k = 64 of 256 groups over 32000 normal values: 74 on average).
// Where the list overflows (long runs of equal values, large ones side by side), the prefix is found
// digit by digit of the key over the whole row instead, as a key t and a count c: every value
// with a larger key, and the c of lowest index among those with key t.
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

template <typename T> __device__ __forceinline__ T wave_inclusive_sum(T v) { return wave_upto(v, OpSum(), (T)0); }

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

// ------------------------------------------------------------------ a row at hand

// The row as one workgroup walks it: whole vectors tid + r * NT of thread tid, r < R held in
// registers (R = 0: read anew at every walk), then the n % N values after the last whole vector,
// one a lane from lane 0.
template <typename S, int NT, int R> struct Row {
    using T = typename StatOf<S>::T;
    static constexpr uint32_t N = kVec<S>;
    const S *s;
    uint32_t n, whole;
    T extra;
    bool has_extra;
    u32x4 raw[R ? R : 1];

    __device__ __forceinline__ Row(const S *row, uint32_t count) : s(row), n(count), whole(count / N)
    {
        const uint32_t rest = whole * N + threadIdx.x;
        has_extra = rest < n;
#pragma unroll
        for (int r = 0; r < R; r++)
            raw[r] = threadIdx.x + r * NT < whole ? load_held(s, r * NT, threadIdx.x) : minus_infinities<S>();
        extra = has_extra ? (T)s[rest] : (T)-INFINITY;
    }
    __device__ __forceinline__ uint32_t extra_at() const { return whole * N + threadIdx.x; }

    // f(values, index of the first, step) for each vector; held vectors past the row's end are
    // walked too, as minus infinities. The extra value is the caller's.
    template <typename F> __device__ __forceinline__ void walk(F f) const
    {
        const Pass pass = Pass::fresh();
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                T v[N];
                unpack<S>(raw[r], v, pass);
                f(v, (threadIdx.x + r * NT) * N, r);
                one_at_a_time();
            }
        } else {
            constexpr int U = 4;
            for (uint32_t i = threadIdx.x; i < whole; i += NT * U) {
                u32x4 in[U];
#pragma unroll
                for (int u = 0; u < U; u++)
                    in[u] = i + u * NT < whole ? load_whole(s, i + u * NT) : minus_infinities<S>();
#pragma unroll
                for (int u = 0; u < U; u++) {
                    T v[N];
                    unpack<S>(in[u], v, pass);
                    f(v, (i + u * NT) * N, u);
                }
            }
        }
    }
};

// ------------------------------------------------------------------- a short list

template <typename K, int CAP> struct List {
    __attribute__((aligned(16))) K key[CAP];
    __attribute__((aligned(16))) uint32_t at[CAP];
    uint32_t count; // may pass CAP: then the list is not whole

    __device__ __forceinline__ void add(K k, uint32_t i)
    {
        const uint32_t j = atomicAdd(&count, 1u);
        if (j < CAP) {
            key[j] = k;
            at[j] = i;
        }
    }
};

// Sorts the list's first n entries by key descending, index ascending (n <= CAP, a power of two);
// whole workgroup, ends with a barrier.
template <int NT, typename K, int CAP> __device__ __forceinline__ void sort_list(List<K, CAP> &l, uint32_t n)
{
    // Few entries: each finds its place by counting those before it.
    if (n <= 256 && n <= NT) {
        constexpr uint32_t kAtOnce = 8; // reads in flight
        if (threadIdx.x < kAtOnce) {
            l.key[n + threadIdx.x] = 0;
            l.at[n + threadIdx.x] = 0xffffffffu;
        }
        __syncthreads();
        K k = 0;
        uint32_t i = 0, place = 0;
        if (threadIdx.x < n) {
            k = l.key[threadIdx.x];
            i = l.at[threadIdx.x];
            for (uint32_t j = 0; j < n; j += kAtOnce) {
                K o[kAtOnce];
                uint32_t a[kAtOnce];
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; u++) {
                    o[u] = l.key[j + u];
                    a[u] = l.at[j + u];
                }
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; u++)
                    place += o[u] > k || (o[u] == k && a[u] < i);
            }
        }
        __syncthreads();
        if (threadIdx.x < n) {
            l.key[place] = k;
            l.at[place] = i;
        }
        __syncthreads();
        return;
    }
    uint32_t size = 512;
    while (size < n)
        size <<= 1;
    for (uint32_t j = n + threadIdx.x; j < size; j += NT) {
        l.key[j] = 0;
        l.at[j] = 0xffffffffu;
    }
    for (uint32_t len = 2; len <= size; len <<= 1)
        for (uint32_t gap = len >> 1; gap > 0; gap >>= 1) {
            __syncthreads();
            for (uint32_t p = threadIdx.x; p < size / 2; p += NT) {
                const uint32_t a = 2 * p - (p & (gap - 1)), b = a + gap;
                const K ka = l.key[a], kb = l.key[b];
                const uint32_t ia = l.at[a], ib = l.at[b];
                const bool ordered = ka > kb || (ka == kb && ia < ib);
                if (ordered != ((a & len) == 0)) {
                    l.key[a] = kb;
                    l.key[b] = ka;
                    l.at[a] = ib;
                    l.at[b] = ia;
                }
            }
        }
    __syncthreads();
}

// ------------------------------------------------------------- one entry of many

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


// Entries (key, index) that a workgroup holds, PER a thread.
template <typename K, int PER> struct Held {
    K key[PER];
    uint32_t at[PER];
};
template <typename K> struct SelectShared {
    Digit<unsigned long long> digit;
    unsigned long long bins[256];
    K varying[2][16];
    uint32_t left[16];
    K key;
    uint32_t at;
};

// In the order (key descending, index ascending), or by index alone (BY_INDEX), the entry at which
// the running sum of the measures reaches `need` (1 <= need <= their sum; entries of measure 0 do
// not count): its key and index in sh, after a barrier. 8 bits a step, from the highest bit in
// which the keys differ, until one entry is left.
template <int NT, bool BY_INDEX, typename K, int PER>
__device__ __forceinline__ void select_entry(const Held<K, PER> &e, const unsigned long long (&measure)[PER],
                                             unsigned long long need, int index_bits, SelectShared<K> &sh)
{
    bool in[PER];
#pragma unroll
    for (int b = 0; b < PER; b++)
        in[b] = measure[b] != 0;
    int shift = index_bits > 8 ? index_bits - 8 : 0;
    bool by_key = !BY_INDEX;
    if (by_key) {
        K some = 0, all = 0; // bits set in some key, bits clear in some key
#pragma unroll
        for (int b = 0; b < PER; b++)
            if (in[b]) {
                some |= e.key[b];
                all |= ~e.key[b];
            }
        some = block_reduce<NT>(some, OpOr(), sh.varying[0]);
        all = block_reduce<NT>(all, OpOr(), sh.varying[1]);
        const K varying = some & all;
        const int top = varying == 0 ? -1 : (sizeof(K) == 8 ? 63 - __builtin_clzll(varying) : 31 - __builtin_clz((uint32_t)varying));
        if (top < 0)
            by_key = false;
        else
            shift = top > 7 ? top - 7 : 0;
    }
    for (int step = 0; step < (int)sizeof(K) + 4; step++) { // at most every byte of a key and an index
        for (uint32_t b = threadIdx.x; b < 256; b += NT)
            sh.bins[b] = 0;
        __syncthreads();
        uint32_t digit[PER];
#pragma unroll
        for (int b = 0; b < PER; b++) {
            digit[b] = (by_key ? (uint32_t)(e.key[b] >> shift) : ~e.at[b] >> shift) & 255u;
            if (in[b])
                atomicAdd(&sh.bins[digit[b]], measure[b]);
        }
        const Digit<unsigned long long> d = find_digit(sh.bins, need, &sh.digit);
        need = d.left;
        uint32_t left = 0;
#pragma unroll
        for (int b = 0; b < PER; b++) {
            in[b] = in[b] && digit[b] == d.digit;
            left += in[b];
        }
        left = block_reduce<NT>(left, OpSum(), sh.left);
        if (left == 1) {
#pragma unroll
            for (int b = 0; b < PER; b++)
                if (in[b]) {
                    sh.key = e.key[b];
                    sh.at = e.at[b];
                }
            __syncthreads();
            return;
        }
        if (shift > 0) {
            shift = shift > 8 ? shift - 8 : 0;
        } else { // equal keys: by index
            by_key = false;
            shift = index_bits > 8 ? index_bits - 8 : 0;
        }
    }
}

// What a bound's search keeps in LDS.
struct BoundScratch {
    uint32_t bins[256];
    uint32_t bin, wave_min_at;
};

// A bound that at least k of the row's values reach, from the largest value of each of this
// thread's G groups: a histogram of the group maxima in 256 even steps from the row's maximum
// m down to their smallest finite one, and the smallest group maximum in the bins that
// together hold k groups. Minus infinity where fewer than k groups have a finite maximum.
template <int NT, int G, typename T>
__device__ __forceinline__ T bound_of(const T (&group)[G], T m, uint32_t k, BoundScratch &sc, T *red)
{
    T low = INFINITY;
#pragma unroll
    for (int g = 0; g < G; g++)
        if (group[g] > -INFINITY)
            low = group[g] < low ? group[g] : low;
    for (uint32_t b = threadIdx.x; b < 256; b += NT)
        sc.bins[b] = 0;
    low = -block_reduce<NT>(-low, OpMax(), red);
    if constexpr (NT == 64)
        __syncthreads();
    const T scale = (T)255.9 / (m - low);
    auto bin_of = [&](T v) -> uint32_t { // any monotone map will do: the bound is a group's own maximum
        const float x = (float)((m - v) * scale);
        return x < 255.0f ? (uint32_t)x : (x >= 255.0f ? 255u : 0u);
    };
#pragma unroll
    for (int g = 0; g < G; g++)
        if (group[g] > -INFINITY)
            atomicAdd(&sc.bins[bin_of(group[g])], 1u);
    if (threadIdx.x == 0)
        sc.bin = 256;
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t first = 4 * threadIdx.x;
        uint32_t b[4], own = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            b[i] = sc.bins[first + i];
            own += b[i];
        }
        uint32_t before = wave_inclusive_sum(own) - own;
        if (before < k && k <= before + own) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (before < k && k <= before + b[i])
                    sc.bin = first + i;
                before += b[i];
            }
        }
    }
    __syncthreads();
    const uint32_t last = sc.bin;
    if (last == 256)
        return -INFINITY;
    T least = INFINITY;
#pragma unroll
    for (int g = 0; g < G; g++)
        if (group[g] > -INFINITY && bin_of(group[g]) <= last)
            least = group[g] < least ? group[g] : least;
    return -block_reduce<NT>(-least, OpMax(), red + 16);
}

// ---------------------------------------------------------------- digit by digit

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
