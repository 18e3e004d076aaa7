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

#include <type_traits>

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
// own ones. One at a time: it serves rare rows, in kernels whose registers it must not raise.
template <typename S, int NT, typename F>
__device__ __forceinline__ void each_vec(const S *row, uint32_t n, F f)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>;
    const uint32_t vecs = (n + N - 1) / N;
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < vecs; i += NT) {
        T v[N];
        unpack<S>(load_vec(row, i, n), v);
        f(v, i * N, n - i * N < N ? n - i * N : N);
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
    // Of M values the indices of those that `wanted` says, value i at index index_of(i); their keys
    // are put in by fill_keys, all at once.
    template <int M, typename T, typename W, typename I>
    __device__ __forceinline__ void add_of(const T *v, W wanted, I index_of)
    {
        static_assert(M <= 32, "one bit a value");
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < M; i++)
            mask |= wanted(v[i], i) ? 1u << i : 0u;
        if (mask) {
            uint32_t j = atomicAdd(&count, (uint32_t)__builtin_popcount(mask));
            for (; mask; mask &= mask - 1, j++)
                if (j < CAP)
                    at[j] = index_of(__builtin_ctz(mask));
        }
    }
    // The indices of the values that reach t (t > minus infinity) in those of a thread's M vectors whose
    // largest values do; vector_of(i, f) calls f(index) for the vectors of group i, and they are read again
    // (they are in the caches): few lanes have any, and hardly one has two.
    template <int M, typename S, typename T, typename V>
    __device__ __forceinline__ void add_from(const S *row, const T (&largest)[M], T t, V vectors_of)
    {
        constexpr int N = kVec<S>;
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < M; i++)
            mask |= largest[i] >= t ? 1u << i : 0u;
        for (; mask; mask &= mask - 1)
            vectors_of(__builtin_ctz(mask), [&](uint32_t vec) {
                T v[N];
                unpack<S>(load_whole(row, vec), v);
                add_of<N>(v, [&](T x, int) { return x >= t; }, [&](int e) { return vec * N + (uint32_t)e; });
            });
    }
    // Whole workgroup, after a barrier; ends with one.
    template <int NT, typename S> __device__ __forceinline__ void fill_keys(const S *row)
    {
        const uint32_t n = count < CAP ? count : CAP;
        for (uint32_t j = threadIdx.x; j < n; j += NT)
            key[j] = key_of((typename StatOf<S>::T)row[at[j]]);
        __syncthreads();
    }
};

// The value of another lane, address = 4 * lane.
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int address) { return (uint32_t)__builtin_amdgcn_ds_bpermute(address, (int)v); }
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int address)
{
    return (uint64_t)of_lane((uint32_t)(v >> 32), address) << 32 | of_lane((uint32_t)v, address);
}

// One exchange step of a sort held in registers: lane pairs `gap` apart, `lower` the one that
// keeps what comes first where `up`.
template <typename K> __device__ __forceinline__ void exchange(K &key, uint32_t &at, K other_key, uint32_t other_at, bool first)
{
    const bool before = (other_key > key) | ((other_key == key) & (other_at < at));
    const bool take = before == first;
    key = take ? other_key : key;
    at = take ? other_at : at;
}

// Sorts the list's first n entries, E a thread (n <= E * NT), by a bitonic network on registers:
// entry e * NT + thread, so that steps of less than 64 stay in a wave (no barrier), steps of NT and
// more in a thread, and only those between go through LDS.
template <int NT, int E, typename K, int CAP> __device__ __forceinline__ void sort_in_registers(List<K, CAP> &l, uint32_t n)
{
    K key[E];
    uint32_t at[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint32_t j = e * NT + threadIdx.x;
        key[e] = j < n ? l.key[j] : 0;
        at[e] = j < n ? l.at[j] : 0xffffffffu - j; // distinct: ties among the empty places too
    }
    uint32_t size = 64; // at most CAP
    while (size < n)
        size <<= 1;
    auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t j = e * NT + threadIdx.x;
            if (j < size) {
                l.key[j] = key[e];
                l.at[j] = at[e];
            }
        }
    };
    for (uint32_t len = 2; len <= size; len <<= 1)
        for (uint32_t gap = len >> 1; gap > 0; gap >>= 1) {
            if (gap >= NT) {
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int g = 1; g < E; g <<= 1)
                        if (gap == (uint32_t)g * NT && !(e & g) && (e | g) < E) {
                            const bool up = ((e * NT + threadIdx.x) & len) == 0;
                            const K ka = key[e];
                            const uint32_t ia = at[e];
                            exchange(key[e], at[e], key[e | g], at[e | g], up);
                            exchange(key[e | g], at[e | g], ka, ia, !up);
                        }
            } else if (gap < 64) {
                const int address = (int)(((threadIdx.x & 63) ^ gap) << 2);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const uint32_t j = e * NT + threadIdx.x;
                    const K ko = of_lane(key[e], address);
                    const uint32_t io = of_lane(at[e], address);
                    exchange(key[e], at[e], ko, io, ((j & gap) == 0) == ((j & len) == 0));
                }
            } else {
                __syncthreads();
                put();
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const uint32_t j = e * NT + threadIdx.x, o = j ^ gap;
                    if (j < size)
                        exchange(key[e], at[e], l.key[o], l.at[o], ((j & gap) == 0) == ((j & len) == 0));
                }
            }
        }
    __syncthreads();
    put();
    __syncthreads();
}

// What the sort keeps in LDS beside the list.
constexpr uint32_t kSortBins = 512;
template <typename T> struct SortShared {
    uint32_t bins[kSortBins + 1], waves[16], crowded;
    T red[16];
};

// Sorts the list's first n entries by key descending, index ascending (n <= CAP); whole
// workgroup, ends with a barrier. m: the largest value. The entries are counted into even
// steps of their values, put into the steps' places, and then each finds its own among the
// few of its step; where a step is crowded (equal values, an outlier) a network sorts them.
// Measured in a row's 31 us at n = 547 with 1024 threads: a network over LDS 14.5 us, one on
// registers 9, this 2.
template <int NT, typename T, typename K, int CAP>
__device__ __forceinline__ void sort_list(List<K, CAP> &l, uint32_t n, T m, SortShared<T> &sh)
{
    constexpr int E = (CAP + NT - 1) / NT;
    constexpr uint32_t kCrowd = 32, kEach = (kSortBins + NT - 1) / NT;
    K key[E];
    uint32_t at[E], bin[E];
    T low = INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint32_t j = e * NT + threadIdx.x;
        key[e] = j < n ? l.key[j] : 0;
        at[e] = j < n ? l.at[j] : 0;
        const T v = key[e] ? value_of(key[e]) : (T)-INFINITY;
        low = v > -INFINITY && v < low ? v : low;
    }
    for (uint32_t b = threadIdx.x; b <= kSortBins; b += NT)
        sh.bins[b] = 0;
    if (threadIdx.x == 0)
        sh.crowded = 0;
    low = -block_reduce<NT>(-low, OpMax(), sh.red);
    const T scale = (T)(kSortBins - 2) / (m - low);
    // Counted one bin up: after the sums, bin b starts where bins[b] says.
#pragma unroll
    for (int e = 0; e < E; e++) {
        const T v = key[e] ? value_of(key[e]) : (T)-INFINITY;
        const float x = v == m ? 0.0f : (float)((m - v) * scale);
        bin[e] = x < (float)(kSortBins - 1) ? (uint32_t)x : kSortBins - 1; // a NaN too: infinities
        if ((uint32_t)e * NT + threadIdx.x < n && atomicAdd(&sh.bins[bin[e] + 1], 1u) >= kCrowd)
            sh.crowded = 1;
    }
    __syncthreads();
    if (sh.crowded) {
        __syncthreads();
        sort_in_registers<NT, E>(l, n);
        return;
    }
    uint32_t count[kEach], own = 0;
#pragma unroll
    for (uint32_t b = 0; b < kEach; b++) {
        const uint32_t i = threadIdx.x * kEach + b;
        count[b] = i < kSortBins ? sh.bins[i + 1] : 0;
        own += count[b];
    }
    uint32_t upto = wave_inclusive_sum(own);
    if ((threadIdx.x & 63) == 63)
        sh.waves[threadIdx.x / 64] = upto;
    __syncthreads();
    for (uint32_t w = 0; w < threadIdx.x / 64; w++)
        upto += sh.waves[w];
    uint32_t before = upto - own;
#pragma unroll
    for (uint32_t b = 0; b < kEach; b++) {
        const uint32_t i = threadIdx.x * kEach + b;
        if (i < kSortBins)
            sh.bins[i + 1] = before; // while its bin fills, then its end
        before += count[b];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if ((uint32_t)e * NT + threadIdx.x < n) {
            const uint32_t j = atomicAdd(&sh.bins[bin[e] + 1], 1u);
            l.key[j] = key[e];
            l.at[j] = at[e];
        }
    __syncthreads();
    uint32_t place[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        place[e] = 0;
        if ((uint32_t)e * NT + threadIdx.x < n) {
            const uint32_t first = sh.bins[bin[e]], last = sh.bins[bin[e] + 1];
            place[e] = first;
            for (uint32_t j = first; j < last; j++)
                place[e] += (l.key[j] > key[e]) | ((l.key[j] == key[e]) & (l.at[j] < at[e]));
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++)
        if ((uint32_t)e * NT + threadIdx.x < n) {
            l.key[place[e]] = key[e];
            l.at[place[e]] = at[e];
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


template <typename K> struct SelectShared {
    Digit<unsigned long long> digit;
    unsigned long long bins[256];
    uint32_t counts[256];
    K varying[2][16];
    K key;
    uint32_t at;
};

// Among `count` entries, entry(j) giving (key, index), in the order (key descending, index
// ascending) or by index alone (BY_INDEX): the entry at which the running sum of
// measure(key, index) reaches `need` (1 <= need <= their sum; entries of measure 0 do not count).
// Its key and index are in sh after a barrier. 8 bits a step, from the highest bit in which the
// keys differ, until one entry is left; indices are below 2^index_bits and differ.
template <int NT, bool BY_INDEX, typename K, typename E, typename M>
__device__ __forceinline__ void select_entry(uint32_t count, E entry, M measure, unsigned long long need, int index_bits,
                                             SelectShared<K> &sh)
{
    K key_bits = 0, key_mask = 0;          // of the key, found so far
    uint32_t at_bits = 0, at_mask = 0;     // of the index' complement
    int shift = index_bits > 8 ? index_bits - 8 : 0;
    bool by_key = !BY_INDEX;
    if (by_key) {
        K some = 0, none = 0; // bits set in some key, bits clear in some key
        for (uint32_t j = threadIdx.x; j < count; j += NT) {
            const K key = entry(j).key;
            some |= key;
            none |= ~key;
        }
        some = block_reduce<NT>(some, OpOr(), sh.varying[0]);
        none = block_reduce<NT>(none, OpOr(), sh.varying[1]);
        const K varying = some & none;
        key_bits = some & ~none; // the bits that all share
        key_mask = ~varying;
        const int top = varying == 0 ? -1 : (sizeof(K) == 8 ? 63 - __builtin_clzll(varying) : 31 - __builtin_clz((uint32_t)varying));
        if (top < 0)
            by_key = false;
        else
            shift = top > 7 ? top - 7 : 0;
    }
    for (int step = 0; step < (int)sizeof(K) + 5; step++) { // at most every byte of a key and an index
        for (uint32_t b = threadIdx.x; b < 256; b += NT) {
            sh.bins[b] = 0;
            sh.counts[b] = 0;
        }
        __syncthreads();
        auto digit_of = [&](const auto &e) { return (by_key ? (uint32_t)(e.key >> shift) : ~e.at >> shift) & 255u; };
        auto in = [&](const auto &e) { return (BY_INDEX || (e.key & key_mask) == key_bits) && (~e.at & at_mask) == at_bits; };
        for (uint32_t j = threadIdx.x; j < count; j += NT) {
            const auto e = entry(j);
            if (in(e)) {
                const unsigned long long w = measure(e.key, e.at);
                if (w) {
                    atomicAdd(&sh.bins[digit_of(e)], w);
                    atomicAdd(&sh.counts[digit_of(e)], 1u);
                }
            }
        }
        const Digit<unsigned long long> d = find_digit(sh.bins, need, &sh.digit);
        need = d.left;
        if (by_key) {
            key_bits |= (K)d.digit << shift;
            key_mask |= (K)255 << shift;
        } else {
            at_bits |= d.digit << shift;
            at_mask |= 255u << shift;
        }
        if (sh.counts[d.digit] == 1) {
            for (uint32_t j = threadIdx.x; j < count; j += NT) {
                const auto e = entry(j);
                if (in(e) && measure(e.key, e.at)) {
                    sh.key = e.key;
                    sh.at = e.at;
                }
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
        __syncthreads(); // the counts are read
    }
}

// What a bound's search keeps in LDS.
struct BoundScratch {
    uint32_t bins[256];
    uint32_t bin[2];
};
template <typename T> struct Bounds {
    T t[2];
};

// Bounds that at least k[0], and k[1], of the values reach, from the largest value of each of this
// thread's G groups: a histogram of the group maxima in 256 even steps from the row's maximum
// m down to their smallest finite one, and the smallest group maximum in the bins that
// together hold k groups. Minus infinity where fewer than k groups have a finite maximum.
// `red`: 3 x 16 places.
template <int NT, int G, int COUNT, typename T>
__device__ __forceinline__ Bounds<T> bounds_of(const T (&group)[G], T m, const uint32_t (&k)[COUNT], BoundScratch &sc, T *red)
{
    T low = INFINITY;
#pragma unroll
    for (int g = 0; g < G; g++)
        if (group[g] > -INFINITY)
            low = group[g] < low ? group[g] : low;
    for (uint32_t b = threadIdx.x; b < 256; b += NT)
        sc.bins[b] = 0;
    if (threadIdx.x < COUNT)
        sc.bin[threadIdx.x] = 256;
    low = -block_reduce<NT>(-low, OpMax(), red);
    if constexpr (NT == 64)
        __syncthreads();
    const T scale = (T)255.9 / (m - low);
    auto bin_of = [&](T v) -> uint32_t { // any monotone map will do: the bound is a group's own maximum
        const float x = (float)((m - v) * scale);
        return x < 255.0f ? (uint32_t)x : (x >= 255.0f ? 255u : 0u);
    };
    uint32_t bin[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        bin[g] = group[g] > -INFINITY ? bin_of(group[g]) : 256;
        if (bin[g] < 256)
            atomicAdd(&sc.bins[bin[g]], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t first = 4 * threadIdx.x;
        uint32_t b[4], own = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            b[i] = sc.bins[first + i];
            own += b[i];
        }
        const uint32_t upto = wave_inclusive_sum(own);
#pragma unroll
        for (int c = 0; c < COUNT; c++) {
            uint32_t before = upto - own;
            if (before < k[c] && k[c] <= upto) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (before < k[c] && k[c] <= before + b[i])
                        sc.bin[c] = first + i;
                    before += b[i];
                }
            }
        }
    }
    __syncthreads();
    Bounds<T> out;
#pragma unroll
    for (int c = 0; c < COUNT; c++) {
        const uint32_t last = sc.bin[c];
        T least = INFINITY;
#pragma unroll
        for (int g = 0; g < G; g++)
            if (bin[g] <= last && bin[g] < 256)
                least = group[g] < least ? group[g] : least;
        least = -block_reduce<NT>(-least, OpMax(), red + 16 * (c + 1));
        out.t[c] = last == 256 ? (T)-INFINITY : least;
    }
    return out;
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
