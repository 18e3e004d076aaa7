// Sampling of one token a row with temperature, top-k, top-p and min-p from a given uniform
// random number.
//
// With m the row's maximum and 1/T rounded to binary32:
//   z = (l - m) rounded to binary32, times 1/T, rounded;   w = floor(2^40 exp(z)), 2^40 at the maximum
//   S_k  = the first top_k of the order (value descending, index ascending)
//   S_p  = the shortest prefix of S_k that holds floor(P mass(S_k) / 2^31), P = floor(2^31 top_p)
//   kept = the tokens of S_p with w >= 2^40 min_p
//   the token is the first kept one, by index, at which the running mass passes
//   floor(U mass(kept) / 2^31), U = floor(2^31 u).
// Weights are integers, so every mass is exact whatever the order of its additions: a row's
// token does not depend on how the row is split over lanes, and a tie never does. A token below
// 2^-40 of the largest weight is never drawn. The exponential is the library's binary32 one.
//
// What bounds it: not the one read of the logits but the steps that wait for the whole row (maximum,
// bound or masses, list, place in the order, drawing), each a few barriers and trips to memory, over
// up to three launches. One row of 128000 bf16 with top-k and top-p takes 17 us of kernel in one launch,
// 64 x 50257 f32 with top-p 6 + 14 + 24 us, 512 x 152000 bf16 of mixed settings 52 + 53 + 59 us
// (156 MB: 32 us at the rate of a copy). Rows whose lists do not suffice, and every top_k above 1024, are
// searched digit by digit by one workgroup each: 64 x 50257 f32 with top-k 2000 273 us a call, with top-p
// over equal logits 713; 512 x 152000 bf16 with top-p over equal logits 8.4 ms.
#include "pcu_kernels.hpp"
#include "pcu_select.hpp"

#include <type_traits>

#pragma clang fp contract(off)

namespace pcu {

namespace {

typedef unsigned long long mass_t;
constexpr mass_t kOne = 1ull << 40;

// A sum complete here: the compiler may not put off its additions and hold the masses instead (the
// kernels on long rows took 94 registers for that, 5 workgroups a CU for 7).
__device__ __forceinline__ void added(mass_t &sum) { asm volatile("" : "+v"(sum)); }

// floor(mass * part / 2^31), mass <= 2^62 (2^22 weights of 2^40), part <= 2^31: below 2^63 throughout.
__device__ __forceinline__ mass_t share_of(mass_t mass, uint32_t part)
{
    return (mass >> 31) * part + (((mass & 0x7fffffffull) * part) >> 31);
}

template <typename T> struct Weight {
    T m;
    float inv;
    __device__ __forceinline__ mass_t operator()(T v) const
    {
        // Equal to m (also where m is infinite): 1. A NaN converts to 0 below.
        const float z = (float)(v == m ? (T)0 : v - m) * inv;
        // e <= 1, so e 2^40 has 9 bits above its lower word; both words are exact truncations.
        const float high = expf(z) * 256.0f;
        const float low = __builtin_amdgcn_fractf(high) * 4294967296.0f;
        return (mass_t)(uint32_t)high << 32 | (uint32_t)low;
    }
};

// A row's settings, as the kernels use them.
struct Settings {
    bool ok;      // all in their ranges
    uint32_t k;   // n: no limit
    float inv;    // 1 / T
    mass_t least; // 2^40 min_p
    uint32_t part, draw; // 2^31 top_p, 2^31 u
    __device__ __forceinline__ bool nucleus() const { return part < 0x80000000u; }
};
__device__ __forceinline__ Settings settings_of(const SampleArgs &g, uint64_t row)
{
    const float temperature = g.temperature ? g.temperature[row] : g.temperature_all;
    const int32_t top_k = g.top_k ? g.top_k[row] : g.top_k_all;
    const float top_p = g.top_p ? g.top_p[row] : g.top_p_all, min_p = g.min_p ? g.min_p[row] : g.min_p_all;
    const float uniform = g.uniform[row];
    Settings s;
    s.ok = temperature >= 0.0f && temperature < INFINITY && top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f &&
           min_p <= 1.0f && uniform >= 0.0f && uniform < 1.0f;
    s.k = top_k <= 0 || top_k >= (int64_t)g.vocab ? g.vocab : (uint32_t)top_k;
    s.inv = 1.0f / temperature;
    if (s.inv == INFINITY) { // the limit: the maximum of lowest index
        s.inv = 1.0f;
        s.k = 1;
    }
    s.least = (mass_t)ceil((double)min_p * (double)kOne);
    s.part = (uint32_t)((double)top_p * 2147483648.0);
    s.draw = (uint32_t)((double)uniform * 2147483648.0);
    return s;
}

__device__ __forceinline__ void put_token(const SampleArgs &g, uint64_t row, int32_t token, float log_prob)
{
    put(g.tokens + row, token);
    if (g.log_prob)
        put(g.log_prob + row, log_prob);
}

// A row from which nothing can be drawn; an invalid setting is a fault. One thread.
__device__ __forceinline__ void no_token(const SampleArgs &g, uint64_t row, bool ok)
{
    if (!ok) {
        atomicMin(g.fault, (unsigned long long)pack_fault(g.first_row + row, kInvalid));
        gate_record(g.gate);
    }
    put_token(g, row, -1, -INFINITY);
}

// The prefix of S_k = (tk, ck) that holds `need` (1 <= need <= mass of S_k).
template <typename S, int NT, typename K, typename W>
__device__ __forceinline__ Prefix<K> select_mass(const S *row, uint32_t n, Prefix<K> pk, mass_t need, const W &weight,
                                                 mass_t *bins, Digit<mass_t> *found)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>;
    const mass_t edge = pk.t == 0 ? 0 : pk.c * weight(value_of(pk.t));
    K prefix = 0;
    for (int shift = (int)sizeof(K) * 8 - 8; shift >= 0; shift -= 8) {
        for (uint32_t b = threadIdx.x; b < 256; b += NT)
            bins[b] = 0;
        __syncthreads();
        if (threadIdx.x == 0 && edge && ((pk.t ^ prefix) >> shift) < 256)
            atomicAdd(&bins[(uint32_t)(pk.t >> shift) & 255u], edge);
        each_vec<S, NT>(row, n, [&](const T *v, uint32_t, uint32_t count) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                const K key = key_of(v[i]);
                if (i < count && key > pk.t && ((key ^ prefix) >> shift) < 256)
                    atomicAdd(&bins[(uint32_t)(key >> shift) & 255u], weight(v[i]));
                one_at_a_time();
            }
        });
        const Digit<mass_t> d = find_digit(bins, need, found);
        prefix |= (K)d.digit << shift;
        need = d.left;
    }
    const mass_t w = weight(value_of(prefix));
    return {prefix, (uint32_t)((need + w - 1) / w)};
}

constexpr uint32_t kSteps = 1024; // of a row's weights in the nucleus search

// The last token of a prefix of the order: kept are the values above `value`, and those equal to it
// up to index `at`.
template <typename T> struct Last {
    T value;
    uint32_t at;
    __device__ __forceinline__ bool keeps(T v, uint32_t i) const { return v > value || (v == value && i <= at); }
};

// The index of the c-th value (from 1) of key t, for a prefix found digit by digit.
template <typename S, int NT, typename K>
__device__ __forceinline__ Last<typename StatOf<S>::T> last_of(const S *s, uint32_t n, Prefix<K> p, uint32_t *wave_ties, uint32_t *at_out)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>, W = NT / 64;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const uint32_t vecs = (n + N - 1) / N, run = (vecs + W - 1) / W;
    const uint32_t first = wave * run, last = first + run < vecs ? first + run : vecs;
    uint32_t ties = 0;
    wave_run(s, n, first, last, [&](const T *v, uint32_t, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            ties += i < count && key_of(v[i]) == p.t;
        return false;
    });
    ties = wave_reduce(ties, OpSum());
    if (lane == 0)
        wave_ties[wave] = ties;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t w = 0; w < wave; w++)
        before += wave_ties[w];
    if (before < p.c && p.c <= before + ties)
        wave_run(s, n, first, last, [&](const T *v, uint32_t at, uint32_t count) {
            uint32_t own = 0;
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                own += i < count && key_of(v[i]) == p.t;
            const uint32_t upto = wave_inclusive_sum(own);
            uint32_t rank = before + upto - own;
            if (rank < p.c && p.c <= rank + own) {
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    if (i < count && key_of(v[i]) == p.t && ++rank == p.c)
                        *at_out = at + i;
            }
            before += from_lane(upto, 63);
            return before >= p.c;
        });
    __syncthreads();
    return {value_of(p.t), *at_out};
}

// What the searches of one row by one workgroup keep in LDS.
template <typename T, int NT> struct DrawShared {
    Digit<uint32_t> count_digit;
    Digit<mass_t> mass_digit;
    mass_t red[4][16], tiles[16];
    uint32_t wave_ties[16], found_at, end;
    SelectShared<typename KeyOf<T>::K> select;
    mass_t steps[kSteps]; // masses of the steps of z, then bins of other searches
};

// The steps of z by which masses are counted: any map that falls with the value will do. Weights of z
// below -27.8 are 0.
template <typename T> struct StepOf {
    T m;
    float scale;
    // `low`: the row's smallest finite value where it is known (a flat row gets finer steps).
    __device__ __forceinline__ StepOf(T mx, float inv, T low = -INFINITY) : m(mx)
    {
        const float range = (float)(mx - low) * inv;
        scale = inv * ((float)kSteps / (range > 0.0f && range < 28.0f ? range : 28.0f));
    }
    __device__ __forceinline__ uint32_t operator()(T v) const
    {
        const float x = (float)(m - v) * scale;
        return x < (float)(kSteps - 1) ? (uint32_t)x : kSteps - 1; // a NaN (equal infinities) too
    }
};

// Among the steps' masses: the total, what a nucleus of `part` of it needs, the step in which it
// ends and the mass before that step.
struct End {
    mass_t need, above;
    uint32_t step;
};
template <typename T, int NT>
__device__ __forceinline__ End find_end(DrawShared<T, NT> &sh, uint32_t part)
{
    constexpr uint32_t each = kSteps / NT;
    mass_t own = 0;
#pragma unroll
    for (uint32_t b = 0; b < each; b++)
        own += sh.steps[threadIdx.x * each + b];
    const mass_t upto = wave_inclusive_sum(own);
    if ((threadIdx.x & 63) == 63)
        sh.red[0][threadIdx.x / 64] = upto;
    __syncthreads();
    mass_t before = upto - own, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < NT / 64; w++) {
        before += w < threadIdx.x / 64 ? sh.red[0][w] : 0;
        total += sh.red[0][w];
    }
    mass_t need = share_of(total, part);
    need = need ? need : 1; // at least one token
    if (before < need && need <= before + own) {
#pragma unroll
        for (uint32_t b = 0; b < each; b++) {
            const mass_t here = sh.steps[threadIdx.x * each + b];
            if (before < need && need <= before + here) {
                sh.end = threadIdx.x * each + b;
                sh.mass_digit.left = before;
            }
            before += here;
        }
    }
    __syncthreads();
    return {need, sh.mass_digit.left, sh.end};
}

// One entry of a list, and a list in LDS or in global memory (written by other workgroups of the
// launch, so read past the caches that they do not share).
template <typename K> struct Entry {
    K key;
    uint32_t at;
};
template <typename K> struct LocalList {
    const K *key;
    const uint32_t *at;
    __device__ __forceinline__ Entry<K> operator()(uint32_t j) const { return {key[j], at[j]}; }
};
template <typename K> struct SharedList {
    const K *key;
    const uint32_t *at;
    __device__ __forceinline__ Entry<K> operator()(uint32_t j) const
    {
        return {__hip_atomic_load(key + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
                __hip_atomic_load(at + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)};
    }
};
__device__ __forceinline__ int index_bits(uint32_t n) { return n > 1 ? 32 - __builtin_clz(n - 1) : 1; }

// The nucleus' last token, digit by digit over the whole row (of the prefix pk, its last token `last`).
template <typename S, int NT, typename T, typename W>
__device__ __forceinline__ Last<T> nucleus_exactly(const S *s, uint32_t n, Prefix<typename KeyOf<T>::K> pk, mass_t need,
                                                   const W &weight, DrawShared<T, NT> &sh)
{
    const auto pp = select_mass<S, NT>(s, n, pk, need, weight, sh.steps, &sh.mass_digit);
    return last_of<S, NT>(s, n, pp, sh.wave_ties, &sh.found_at);
}

// The mass of the list's entries.
template <int NT, typename L, typename M> __device__ __forceinline__ mass_t mass_of_list(uint32_t count, L list, M measure, mass_t *lds)
{
    mass_t sum = 0;
    for (uint32_t j = threadIdx.x; j < count; j += NT) {
        const auto e = list(j);
        sum += measure(e.key, e.at);
    }
    return block_reduce<NT>(sum, OpSum(), lds);
}

// Entries that are drawn from one a thread, which reads the whole list twice: 1 x 128000 bf16 with top-k
// 50 and top-p 27 us a call, 40 from the list digit by digit; 32 x 50257 f32 with top-k 100, lists of 96
// to 128, 43 and 37.
constexpr uint32_t kFew = 96;

// Draws from a list of at most kFew entries in LDS, one a thread, which holds the first top_k of the order
// (or all of it that is finite): each entry counts the entries before it in the order with
// their mass, and then, among the kept ones, the mass before it by index. `w`: NT + 4 places.
// need: what the nucleus has to hold, 0 for `part` of the mass of the first top_k.
template <int NT, typename K, typename W>
__device__ __forceinline__ void draw_from_few(const SampleArgs &g, uint64_t row, const Settings &set, K *key, uint32_t *at,
                                              uint32_t count, mass_t need, const W &weight, mass_t *w, mass_t *red)
{
    constexpr uint32_t kAtOnce = 4; // reads in flight
    const uint32_t tid = threadIdx.x;
    const bool in = tid < count;
    const K k = in ? key[tid] : 0;
    const uint32_t i = in ? at[tid] : 0xffffffffu;
    mass_t own = in ? weight(value_of(k)) : 0;
    w[tid] = own;
    if (tid < kAtOnce) {
        key[count + tid] = 0; // after every entry
        at[count + tid] = 0xffffffffu;
        if (count + tid >= NT)
            w[count + tid] = 0;
    }
    __syncthreads();
    uint32_t rank = 0;
    mass_t before = 0;
    for (uint32_t j = 0; j < count; j += kAtOnce) {
        K o[kAtOnce];
        uint32_t a[kAtOnce];
        mass_t x[kAtOnce];
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; u++) {
            o[u] = key[j + u];
            a[u] = at[j + u];
            x[u] = w[j + u];
        }
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; u++) {
            const bool earlier = (o[u] > k) | ((o[u] == k) & (a[u] < i));
            rank += earlier;
            before += earlier ? x[u] : 0;
        }
    }
    if (rank >= set.k)
        own = 0;
    if (set.nucleus()) {
        if (need == 0) {
            need = share_of(block_reduce<NT>(own, OpSum(), red), set.part);
            need = need ? need : 1;
        }
        if (before >= need)
            own = 0;
    }
    if (own < set.least)
        own = 0;
    const mass_t total = block_reduce<NT>(own, OpSum(), red + 16); // its barrier: the weights are read
    w[tid] = own;
    __syncthreads();
    mass_t running = 0;
    for (uint32_t j = 0; j < count; j += kAtOnce) {
        uint32_t a[kAtOnce];
        mass_t x[kAtOnce];
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; u++) {
            a[u] = at[j + u];
            x[u] = w[j + u];
        }
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; u++)
            running += a[u] < i ? x[u] : 0;
    }
    const mass_t target = share_of(total, set.draw);
    if (running <= target && target < running + own) {
        put_token(g, row, (int32_t)i, logf((float)own / (float)total));
    }
}

// Draws from a list of `count` entries, which holds the first top_k of the order (or all of it that is
// finite). need: what the nucleus has to hold, 0 for `part` of their mass.
template <typename T, int NT, typename L, typename W>
__device__ __forceinline__ void draw_from_list(const SampleArgs &g, uint64_t row, const Settings &set, L list, uint32_t count,
                                               mass_t need, const W &weight, DrawShared<T, NT> &sh)
{
    using K = typename KeyOf<T>::K;
    const int bits = index_bits(g.vocab);
    // Kept are the entries up to this one of the order.
    K last_key = 0;
    uint32_t last_at = 0xffffffffu;
    auto kept = [&](K key, uint32_t at) -> mass_t {
        return key > last_key || (key == last_key && at <= last_at) ? weight(value_of(key)) : 0;
    };
    if (count > set.k) {
        select_entry<NT, false>(count, list, [](K, uint32_t) -> mass_t { return 1; }, set.k, bits, sh.select);
        last_key = sh.select.key;
        last_at = sh.select.at;
    }
    if (set.nucleus()) {
        if (need == 0) {
            need = share_of(mass_of_list<NT>(count, list, kept, sh.red[0]), set.part);
            need = need ? need : 1;
        }
        select_entry<NT, false>(count, list, kept, need, bits, sh.select);
        last_key = sh.select.key;
        last_at = sh.select.at;
    }
    auto drawn = [&](K key, uint32_t at) -> mass_t {
        const mass_t w = kept(key, at);
        return w >= set.least ? w : 0;
    };
    // The first by index at which the running mass passes the target.
    const mass_t total = mass_of_list<NT>(count, list, drawn, sh.red[1]);
    select_entry<NT, true>(count, list, drawn, share_of(total, set.draw) + 1, bits, sh.select);
    if (threadIdx.x == 0)
        put_token(g, row, (int32_t)sh.select.at, logf((float)weight(value_of(sh.select.key)) / (float)total));
}

// Draws along vectors [from, to) of the row (`mass_of` a value and its index). total 0: the vectors
// are the whole row, and its mass is counted first; else `target` of it lies in the vectors.
// `lds`: 16 places.
template <typename S, typename F>
__device__ __forceinline__ void draw_along(const SampleArgs &g, uint64_t row, const S *s, uint32_t from, uint32_t to,
                                           uint32_t draw, mass_t total, mass_t target, F mass_of, mass_t *lds)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>, NT = 256, U = 4;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63, n = g.vocab;
    auto mass_in = [&](const u32x4 &raw, uint32_t i, mass_t *w) {
        T v[N];
        unpack<S>(raw, v);
        mass_t sum = 0;
#pragma unroll
        for (uint32_t e = 0; e < N; e++) {
            const mass_t x = i < to && i * N + e < n ? mass_of(v[e], i * N + e) : 0;
            if (w)
                w[e] = x;
            sum += x;
            if (e % 4 == 3) { // eight exponentials at once would take the registers of two waves
                added(sum);
                one_at_a_time();
            }
        }
        return sum;
    };
    auto load = [&](uint32_t i) { return i < to ? load_vec(s, i, n) : minus_infinities<S>(); };
    if (total == 0) {
        mass_t own = 0;
        for (uint32_t i = from + threadIdx.x; i < to; i += NT * U) {
            u32x4 raw[U];
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                raw[u] = load(i + u * NT);
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                own += mass_in(raw[u], i + u * NT, nullptr);
        }
        total = block_reduce<NT>(own, OpSum(), lds);
        target = share_of(total, draw);
        __syncthreads();
    }
    // Tiles of one vector a thread, four at a time: the masses of each tile's four waves, in index
    // order, then within the wave that holds the target.
    for (uint32_t at = from; at < to; at += NT * U) {
        u32x4 raw[U];
#pragma unroll
        for (uint32_t t = 0; t < U; t++)
            raw[t] = load(at + t * NT + threadIdx.x);
#pragma unroll
        for (uint32_t t = 0; t < U; t++) {
            const mass_t sum = wave_reduce(mass_in(raw[t], at + t * NT + threadIdx.x, nullptr), OpSum());
            if (lane == 0)
                lds[t * 4 + wave] = sum;
        }
        __syncthreads();
        const mass_t here = lane < 4 * U ? lds[lane] : 0, upto = wave_inclusive_sum(here), all = from_lane(upto, 63);
        if (target >= all) {
            target -= all;
            __syncthreads(); // the masses are read
            continue;
        }
        const int cell = __builtin_ctzll(__ballot(upto > target));
        target -= from_lane(upto - here, cell);
        if (wave != (uint32_t)cell % 4)
            return;
        const uint32_t i = at + (uint32_t)cell / 4 * NT + threadIdx.x;
        mass_t w[N];
        const mass_t own = mass_in(load(i), i, w), before = wave_inclusive_sum(own) - own;
        if (before <= target && target < before + own) {
            mass_t running = before;
#pragma unroll
            for (uint32_t e = 0; e < N; e++) {
                if (running <= target && target < running + w[e])
                    put_token(g, row, (int32_t)(i * N + e), logf((float)w[e] / (float)total));
                running += w[e];
            }
        }
        return;
    }
}

// ------------------------------------------------------- short rows: one workgroup a row
//
// The row in registers. Rows with a top_k that a list can hold: the list of the first top_k and
// everything else in LDS. Rows with a nucleus: the masses of even steps of z, then the list of the
// values down to the step in which the nucleus ends, or, when that is long, of that step alone.
// Then the drawing: over the list, or over the row. (A group of the bound's is a vector at least: a top_k
// of more than the row has vectors has no bound, and where all of the row do not fit the list it
// is found digit by digit.)
template <typename S, int NT, int R> __device__ __forceinline__ void sample_row(const SampleArgs &g)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    __shared__ BoundScratch bound;
    __shared__ T red_t[3][16];
    __shared__ DrawShared<T, NT> sh;
    constexpr uint32_t kCap = 2048;
    __shared__ List<K, kCap> list;
    const uint32_t tid = threadIdx.x;
    const uint64_t row = row_of_block();
    if (row >= g.rows)
        return;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t n = g.vocab;
    const Settings set = settings_of(g, row);
    const Row<S, NT, R> held(s, n);
    if (block_gate_closed(g.gate)) // after the loads: they need not wait for it
        return;

    constexpr int G = 4;
    T group[G];
#pragma unroll
    for (int i = 0; i < G; i++)
        group[i] = -INFINITY;
    group[0] = OpMax()(group[0], held.extra);
    held.walk([&](const T *v, uint32_t, int step) {
        T top = v[0];
#pragma unroll
        for (uint32_t i = 1; i < N; i++)
            top = OpMax()(top, v[i]);
        group[step % G] = OpMax()(group[step % G], top);
    });
    T m = OpMax()(OpMax()(group[0], group[1]), OpMax()(group[2], group[3]));
    m = block_reduce<NT>(m, OpMax(), red_t[0]);
    if (!set.ok || m == -INFINITY) {
        if (tid == 0)
            no_token(g, row, set.ok);
        return;
    }
    const Weight<T> weight{m, set.inv};
    const LocalList<K> entries{list.key, list.at};
    if (tid == 0)
        list.count = 0;
    __syncthreads();
    // Adds the row's wanted values to the list; its length.
    auto gather = [&](auto wanted) {
        held.walk([&](const T *v, uint32_t at, int) {
            list.template add_of<N>(v, [&](T x, int i) { return x > -INFINITY && wanted(x, at + i); },
                                    [&](int i) { return at + i; });
        });
        if (held.has_extra && held.extra > -INFINITY && wanted(held.extra, held.extra_at()))
            list.add(key_of(held.extra), held.extra_at());
        __syncthreads();
        const uint32_t count = list.count;
        list.template fill_keys<NT>(s);
        return count;
    };

    if (set.k < n && set.k <= kLogitMaxK) {
        const uint32_t top_k[1] = {set.k};
        const T t = bounds_of<NT>(group, m, top_k, bound, red_t[1]).t[0];
        const uint32_t count = gather([&](T v, uint32_t) { return v >= t; });
        if (count <= kFew) {
            draw_from_few<NT>(g, row, set, list.key, list.at, count, 0, weight, sh.steps, sh.red[0]);
            return;
        }
        if (count <= kCap) {
            draw_from_list(g, row, set, entries, count, 0, weight, sh);
            return;
        }
        if (tid == 0)
            list.count = 0;
        __syncthreads();
    }
    Last<T> last{-INFINITY, 0xffffffffu};
    Prefix<K> pk{0, 0};
    if (set.k < n) {
        pk = select_count<S, NT>(s, n, set.k, reinterpret_cast<uint32_t *>(sh.steps), &sh.count_digit);
        if (pk.t)
            last = last_of<S, NT>(s, n, pk, sh.wave_ties, &sh.found_at);
    }
    if (set.nucleus()) {
        for (uint32_t b = tid; b < kSteps; b += NT)
            sh.steps[b] = 0;
        __syncthreads();
        const StepOf<T> step_of(m, set.inv);
        auto add = [&](T v, uint32_t i) {
            if (last.keeps(v, i))
                if (const mass_t w = weight(v))
                    atomicAdd(&sh.steps[step_of(v)], w);
        };
        held.walk([&](const T *v, uint32_t at, int) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                add(v[i], at + i);
        });
        if (held.has_extra)
            add(held.extra, held.extra_at());
        __syncthreads();
        const End end = find_end(sh, set.part);
        uint32_t count = gather([&](T v, uint32_t i) { return step_of(v) <= end.step && last.keeps(v, i); });
        if (count <= kFew) {
            draw_from_few<NT>(g, row, set, list.key, list.at, count, end.need, weight, sh.steps, sh.red[0]);
            return;
        }
        if (count <= kCap) {
            draw_from_list(g, row, set, entries, count, end.need, weight, sh);
            return;
        }
        if (tid == 0)
            list.count = 0;
        __syncthreads();
        count = gather([&](T v, uint32_t i) { return step_of(v) == end.step && last.keeps(v, i); });
        if (count <= kCap) {
            select_entry<NT, false>(count, entries, [&](K key, uint32_t) { return weight(value_of(key)); },
                                    end.need - end.above, index_bits(n), sh.select);
            last = Last<T>{value_of(sh.select.key), sh.select.at};
        } else {
            last = nucleus_exactly<S, NT>(s, n, pk, end.need, weight, sh);
        }
    }
    auto mass_of = [&](T v, uint32_t i) -> mass_t {
        if (!last.keeps(v, i))
            return 0;
        const mass_t w = weight(v);
        return w >= set.least ? w : 0;
    };
    draw_along<S>(g, row, s, 0u, (n + N - 1) / N, set.draw, 0, 0, mass_of, sh.tiles);
}

// A call of its own ends its program in this kernel (close).
template <typename S, int NT, int R> __global__ __launch_bounds__(NT) void k_sample(SampleArgs g, ProgramClose close)
{
    sample_row<S, NT, R>(g);
    program_close_block(close);
}

// The drawing of a row whose lists did not suffice, or whose top_k no list holds: everything digit
// by digit over the whole row.
template <typename S, int NT, typename T>
__device__ __forceinline__ void draw_by_search(const SampleArgs &g, uint64_t row, const S *s, const Settings &set, T m, DrawShared<T, NT> &sh)
{
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    const uint32_t n = g.vocab;
    const Weight<T> weight{m, set.inv};
    Last<T> last{-INFINITY, 0xffffffffu};
    Prefix<K> pk{0, 0};
    if (set.k < n) {
        pk = select_count<S, NT>(s, n, set.k, reinterpret_cast<uint32_t *>(sh.steps), &sh.count_digit);
        if (pk.t)
            last = last_of<S, NT>(s, n, pk, sh.wave_ties, &sh.found_at);
    }
    if (set.nucleus()) {
        mass_t mass = 0;
        each_vec<S, NT>(s, n, [&](const T *v, uint32_t at, uint32_t values) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                if (i < values && last.keeps(v[i], at + i))
                    mass += weight(v[i]);
                added(mass);
            }
        });
        mass = share_of(block_reduce<NT>(mass, OpSum(), sh.red[0]), set.part);
        last = nucleus_exactly<S, NT>(s, n, pk, mass ? mass : 1, weight, sh);
    }
    draw_along<S>(g, row, s, 0u, (n + N - 1) / N, set.draw, 0, 0,
                      [&](T v, uint32_t i) -> mass_t {
                          const mass_t w = last.keeps(v, i) ? weight(v) : 0;
                          return w >= set.least ? w : 0;
                      },
                      sh.tiles);
}

// ------------------------------------------------- long rows: a row split over workgroups
//
// Each row is cut into chunks of consecutive vectors, one workgroup each, and the steps above
// become up to three launches, the last chunk of a row to finish doing what needs the whole row:
//   first: the chunk's maximum. A row whose top_k a list can hold: the chunk's values beyond a bound
//          that top_k of them reach go to the row's list, and the last chunk draws from it.
//          (Such a row's chunks take every chunks-th block of vectors, so that they hold alike values
//          wherever the row's large ones lie. Where top_k times the chunks would make the list long,
//          the bound is one that the chunk's share of top_k reaches, and the list is made in the
//          second launch from the lowest of the bounds.)
//   weigh: with the row's maximum, the chunk's mass, and the last chunk draws in the chunk that
//          holds the target; or a nucleus row's masses by steps of z, and the last chunk finds
//          the step in which the nucleus ends
//   edge:  for a nucleus, the values of that step into the row's list; the last chunk finds the
//          nucleus' last token among them and draws in the chunk that holds the target
// One workgroup would take an exponential of every logit of its row at the rate of one CU: a
// nucleus of a row of 152000 took 280 us.
enum : uint32_t {
    kRowNone,    // an invalid setting
    kRowList,    // done in the first launch
    kRowBound,   // a list made in the second
    kRowNucleus,
    kRowPlain,
    kRowSearch,  // top_k beyond any list
};

struct RowState {
    mass_t need, above; // of the nucleus
    uint32_t count;     // of the row's list; past its capacity: not whole
    uint32_t step;      // in which the nucleus ends
    uint32_t done[3];   // chunks that have finished each launch
};

template <typename T> struct ChunkPart {
    T m;
    T t; // a bound that the chunk's share of top_k reaches; for a nucleus row the smallest value above
         // minus infinity
};

constexpr uint32_t kRowCap = 8192; // of a row's list
constexpr int kChunkThreads = 256;
constexpr int kChunkListCap = 1024, kEdgeListCap = 2048; // in LDS

template <typename T> struct SplitArgs {
    SampleArgs g;
    uint32_t chunks, chunk_vecs;
    ChunkPart<T> *part;  // rows x chunks
    mass_t *chunk_mass;  // rows x chunks: kept before the nucleus' last step, or kept
    mass_t *steps;       // rows x chunks x kSteps
    RowState *state;     // rows, zero between calls
    typename KeyOf<T>::K *key; // rows x kRowCap
    uint32_t *at;              // rows x kRowCap
};

// Whether the chunks' own lists of the top `k` make the row's: then the first launch ends the row, but
// its last chunk takes a list of all of them, up to half as many again as the bounds were made for.
// (32 x 50257 f32 in 12 chunks, microseconds a call: top-k 50 28, 35 with a second launch; top-k 100 43 and
// 41; top-k 300 68 and 42.)
constexpr uint64_t kListAtOnce = 1024;
__host__ __device__ inline bool list_at_once(uint64_t k, uint32_t chunks) { return k * chunks <= kListAtOnce; }
static_assert(kListAtOnce / 2 * 3 / 2 <= kChunkListCap, "a chunk's list of k <= kListAtOnce / 2 values fits");
__device__ __forceinline__ uint32_t kind_of(const Settings &s, uint32_t n, uint32_t chunks)
{
    if (!s.ok)
        return kRowNone;
    if (s.k < n)
        return s.k > kLogitMaxK ? kRowSearch : (list_at_once(s.k, chunks) ? kRowList : kRowBound);
    return s.nucleus() ? kRowNucleus : kRowPlain;
}

// What a chunk hands to the others of its row within a launch is written through the caches that
// they do not share (put), and is complete (a wait for the wave's own stores, then the barrier)
// before the workgroup counts itself as done.
// Whether this workgroup is the last of the row's chunks; whole workgroup, at most once a launch, and
// by all of the row's chunks or by none.
__device__ __forceinline__ bool last_chunk(uint32_t *done, uint32_t chunks)
{
    __shared__ bool last;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        last = atomicAdd(done, 1u) + 1u == chunks;
        if (last)
            put(done, 0u); // as the next call expects it
    }
    __syncthreads();
    return last;
}

// How a chunk left a launch: without having counted itself for its row, or counted, as the last or not.
enum Left : int { kUncounted, kCounted, kCountedLast };

// The vectors of one chunk of the row, then (last chunk) the values after the last whole vector.
template <typename S> struct Chunk {
    using T = typename StatOf<S>::T;
    static constexpr uint32_t N = kVec<S>;
    const S *s;
    uint32_t first, step, past, rest, n;
    __device__ __forceinline__ Chunk(const S *row, uint32_t count, uint32_t chunk, uint32_t chunks, uint32_t vecs, bool apart)
        : s(row), n(count)
    {
        const uint32_t whole = count / N;
        if (apart) {
            first = chunk * kChunkThreads;
            step = chunks * kChunkThreads;
            past = whole;
        } else {
            first = chunk * vecs;
            step = kChunkThreads;
            past = first + vecs < whole ? first + vecs : whole;
        }
        rest = chunk == chunks - 1 ? whole * N + threadIdx.x : n;
    }
    // f(values, their number, index of the first) for each vector, four loads in flight; places
    // past the chunk hold minus infinity.
    template <typename F> __device__ __forceinline__ void vectors(F f) const
    {
        constexpr int U = 4;
        for (uint32_t i = first + threadIdx.x; i < past; i += step * U) {
            u32x4 in[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                in[u] = i + u * step < past ? load_whole(s, i + u * step) : minus_infinities<S>();
#pragma unroll
            for (int u = 0; u < U; u++) {
                T v[N];
                unpack<S>(in[u], v);
                f(v, std::integral_constant<int, (int)N>(), (i + u * step) * N);
                one_at_a_time();
            }
        }
        if (rest < n) {
            const T v[1] = {(T)s[rest]};
            f(v, std::integral_constant<int, 1>(), rest);
        }
    }
    // f(value, index)
    template <typename F> __device__ __forceinline__ void each(F f) const
    {
        vectors([&](const T *v, auto count, uint32_t at) {
#pragma unroll
            for (int k = 0; k < count; k++) {
                f(v[k], at + k);
                if (k % 4 == 3)
                    one_at_a_time();
            }
        });
    }
    // The largest values of this thread's vectors, every eighth of them in one group.
    static constexpr int kGroups = 8;
    __device__ __forceinline__ void largest(T (&group)[kGroups]) const
    {
#pragma unroll
        for (int g = 0; g < kGroups; g++)
            group[g] = -INFINITY;
        for (uint32_t i = first + threadIdx.x; i < past; i += step * kGroups) {
            u32x4 in[kGroups];
#pragma unroll
            for (int g = 0; g < kGroups; g++)
                in[g] = i + g * step < past ? load_whole(s, i + g * step) : minus_infinities<S>();
#pragma unroll
            for (int g = 0; g < kGroups; g++) {
                T v[N];
                unpack<S>(in[g], v);
#pragma unroll
                for (uint32_t e = 0; e < N; e++)
                    group[g] = OpMax()(group[g], v[e]);
            }
        }
    }
    // The values that reach t (above minus infinity) into the list, from the vectors of the groups
    // that do; whole workgroup, ends with a barrier.
    template <typename L> __device__ __forceinline__ void gather(L &list, const T (&group)[kGroups], T t) const
    {
        if (threadIdx.x == 0)
            list.count = 0;
        __syncthreads();
        list.add_from(s, group, t, [&](int g, auto f) {
            for (uint32_t i = first + threadIdx.x + (uint32_t)g * step; i < past; i += step * kGroups)
                f(i);
        });
        if (rest < n && (T)s[rest] >= t)
            list.add(0, rest);
        __syncthreads();
        list.template fill_keys<kChunkThreads>(s);
    }
    // The wanted values into the list; whole workgroup, ends with a barrier.
    template <typename L, typename W> __device__ __forceinline__ void gather(L &list, W wanted) const
    {
        if (threadIdx.x == 0)
            list.count = 0;
        __syncthreads();
        vectors([&](const T *v, auto count, uint32_t at) {
            list.template add_of<decltype(count)::value>(v, [&](T x, int) { return wanted(x); }, [&](int k) { return at + k; });
        });
        __syncthreads();
        list.template fill_keys<kChunkThreads>(s);
    }
};

// A workgroup's list handed to its row's: one place reserved for all of it. A list that does not
// fit sets the row's count beyond the capacity.
template <typename K, int CAP, typename T>
__device__ __forceinline__ void hand_over(const SplitArgs<T> &a, uint64_t row, const List<K, CAP> &list)
{
    __shared__ uint32_t base;
    const uint32_t count = list.count;
    if (count == 0)
        return;
    if (threadIdx.x == 0)
        base = atomicAdd(&a.state[row].count, count > CAP ? kRowCap + 1u : count);
    __syncthreads();
    const uint32_t to = base;
    if (count > CAP || to + count > kRowCap)
        return;
    for (uint32_t j = threadIdx.x; j < count; j += kChunkThreads) {
        put(&a.key[row * kRowCap + to + j], list.key[j]);
        put(&a.at[row * kRowCap + to + j], list.at[j]);
    }
}

// The row's list for its last chunk: its length (past kRowCap: not whole), and in LDS what of it may
// belong to the first `k` of the order (not whole past CAP): all of it, or, of up to 8 entries a
// thread, what reaches a bound from the threads' largest.
template <typename K, int CAP, typename T>
__device__ __forceinline__ uint32_t take_list(const SplitArgs<T> &a, uint64_t row, uint32_t k, T m, List<K, CAP> &local,
                                              BoundScratch &bound, T *red)
{
    __shared__ uint32_t count;
    if (threadIdx.x == 0) {
        count = get(&a.state[row].count);
        put(&a.state[row].count, 0u);
        local.count = 0;
    }
    __syncthreads();
    const uint32_t n = count;
    constexpr int U = 8, NT = kChunkThreads;
    if (n > U * NT)
        local.count = n;
    if (n > U * NT) {
        __syncthreads();
        return n;
    }
    const SharedList<K> list{a.key + row * kRowCap, a.at + row * kRowCap};
    Entry<K> e[U];
    K top = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t j = threadIdx.x + u * NT;
        e[u] = j < n ? list(j) : Entry<K>{0, 0};
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        top = e[u].key > top ? e[u].key : top;
    K least = 1; // no entry has key 0
    if (n > 128 && k < n) {
        const T group[1] = {top ? value_of(top) : (T)-INFINITY};
        const uint32_t wanted[1] = {k};
        const T t = bounds_of<NT>(group, m, wanted, bound, red).t[0];
        least = t > -INFINITY ? key_of(t) : least;
    }
    uint32_t own = 0;
#pragma unroll
    for (int u = 0; u < U; u++)
        own += e[u].key >= least;
    if (own) {
        uint32_t to = atomicAdd(&local.count, own);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (e[u].key >= least) {
                if (to < CAP) {
                    local.key[to] = e[u].key;
                    local.at[to] = e[u].at;
                }
                to++;
            }
    }
    __syncthreads();
    return n;
}

// Draws from the row's list.
template <typename S, typename T, typename K, int CAP>
__device__ __forceinline__ void draw_from_row(const SplitArgs<T> &a, uint64_t row, const Settings &set, T m,
                                              List<K, CAP> &local, BoundScratch &bound, T *red, DrawShared<T, kChunkThreads> &sh)
{
    const uint32_t count = take_list(a, row, set.k, m, local, bound, red), here = local.count;
    const Weight<T> weight{m, set.inv};
    if (count > kRowCap)
        draw_by_search<S, kChunkThreads>(a.g, row, static_cast<const S *>(a.g.logits) + row * a.g.stride, set, m, sh);
    else if (here <= kFew)
        draw_from_few<kChunkThreads>(a.g, row, set, local.key, local.at, here, 0, weight, sh.steps, sh.red[0]);
    else if (here <= CAP)
        draw_from_list(a.g, row, set, LocalList<K>{local.key, local.at}, here, 0, weight, sh);
    else
        draw_from_list(a.g, row, set, SharedList<K>{a.key + row * kRowCap, a.at + row * kRowCap}, count, 0, weight, sh);
}

// Draws in the chunk that holds the target; `in_chunk` the chunks' kept masses, in LDS.
template <typename S, typename T, typename F>
__device__ __forceinline__ void draw_in_chunk(const SplitArgs<T> &a, uint64_t row, const Settings &set, const mass_t *in_chunk,
                                              F mass_of, mass_t *lds)
{
    constexpr uint32_t N = kVec<S>;
    mass_t total = 0;
    for (uint32_t c = 0; c < a.chunks; c++)
        total += in_chunk[c];
    mass_t target = share_of(total, set.draw);
    uint32_t c = 0;
    while (c < a.chunks - 1 && target >= in_chunk[c])
        target -= in_chunk[c++];
    const uint32_t from = c * a.chunk_vecs, to = c == a.chunks - 1 ? (a.g.vocab + N - 1) / N : from + a.chunk_vecs;
    draw_along<S>(a.g, row, static_cast<const S *>(a.g.logits) + row * a.g.stride, from, to, set.draw, total,
                                 target, mass_of, lds);
}

// The row's maximum, and the lowest of the chunks' bounds or smallest values; one chunk a lane.
template <typename T> __device__ __forceinline__ ChunkPart<T> row_part(const SplitArgs<T> &a, uint64_t row)
{
    const uint32_t lane = threadIdx.x & 63;
    ChunkPart<T> p{-INFINITY, INFINITY};
    if (lane < a.chunks)
        p = {get(&a.part[row * a.chunks + lane].m), get(&a.part[row * a.chunks + lane].t)};
    return {wave_reduce(p.m, OpMax()), -wave_reduce(-p.t, OpMax())};
}

// The lowest finite value.
template <typename T> __device__ __forceinline__ T lowest() { return sizeof(T) == 8 ? (T)-1.7976931348623157e308 : (T)-3.402823466e38f; }

template <typename S> __device__ __forceinline__ Left sample_first(const SplitArgs<typename StatOf<S>::T> &a)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr int NT = kChunkThreads;
    if (block_gate_closed(a.g.gate))
        return kUncounted;
    __shared__ BoundScratch bound;
    __shared__ T red[4][16];
    __shared__ List<K, kChunkListCap> list;
    __shared__ DrawShared<T, NT> sh;
    const uint64_t row = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, n = a.g.vocab;
    const Settings set = settings_of(a.g, row);
    const uint32_t kind = kind_of(set, n, a.chunks);
    if (kind == kRowNone) {
        if (chunk == 0 && threadIdx.x == 0)
            no_token(a.g, row, false);
        return kUncounted;
    }
    const Chunk<S> part(static_cast<const S *>(a.g.logits) + row * a.g.stride, n, chunk, a.chunks, a.chunk_vecs,
                        kind == kRowList || kind == kRowBound);
    T largest[Chunk<S>::kGroups];
    part.largest(largest);
    const T rest = part.rest < n ? (T)part.s[part.rest] : (T)-INFINITY;
    T group[4]; // half as many for the bounds
#pragma unroll
    for (int i = 0; i < 4; i++)
        group[i] = OpMax()(largest[i], largest[i + 4]);
    group[0] = OpMax()(group[0], rest);
    T m = OpMax()(OpMax()(group[0], group[1]), OpMax()(group[2], group[3]));
    m = block_reduce<NT>(m, OpMax(), red[0]);
    T t = -INFINITY, own = -INFINITY;
    if (kind == kRowList || kind == kRowBound) {
        const uint32_t top_k[2] = {(set.k + a.chunks - 1) / a.chunks, set.k};
        const Bounds<T> b = bounds_of<NT>(group, m, top_k, bound, red[1]);
        t = b.t[0];
        own = b.t[1];
    } else if (kind == kRowNucleus) {
        t = INFINITY;
        part.each([&](T v, uint32_t) { t = v > -INFINITY && v < t ? v : t; });
        t = -block_reduce<NT>(-t, OpMax(), red[1]);
    }
    if (threadIdx.x == 0) {
        put(&a.part[blockIdx.x].m, m);
        put(&a.part[blockIdx.x].t, t);
    }
    if (kind != kRowList)
        return kUncounted;
    own = own > lowest<T>() ? own : lowest<T>(); // minus infinity is never drawn
    part.gather(list, largest, own);
    hand_over(a, row, list);
    if (!last_chunk(&a.state[row].done[0], a.chunks))
        return kCounted;
    const T top = row_part(a, row).m;
    if (top == -INFINITY) {
        if (threadIdx.x == 0)
            no_token(a.g, row, true);
        return kCountedLast;
    }
    draw_from_row<S>(a, row, set, top, list, bound, red[0], sh);
    return kCountedLast;
}

template <typename S> __device__ __forceinline__ Left sample_weigh(const SplitArgs<typename StatOf<S>::T> &a)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr int NT = kChunkThreads;
    if (block_gate_closed(a.g.gate))
        return kUncounted;
    __shared__ BoundScratch bound;
    __shared__ T red[4][16];
    __shared__ List<K, kChunkListCap> list;
    __shared__ DrawShared<T, NT> sh;
    __shared__ mass_t in_chunk[64];
    const uint64_t row = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, n = a.g.vocab;
    const Settings set = settings_of(a.g, row);
    const uint32_t kind = kind_of(set, n, a.chunks);
    if (kind == kRowNone || kind == kRowList)
        return kUncounted;
    const auto [m, low] = row_part(a, row);
    const S *s = static_cast<const S *>(a.g.logits) + row * a.g.stride;
    if (m == -INFINITY || kind == kRowSearch) {
        if (chunk != 0)
            return kUncounted;
        if (m > -INFINITY)
            draw_by_search<S, NT>(a.g, row, s, set, m, sh);
        else if (threadIdx.x == 0)
            no_token(a.g, row, true);
        return kUncounted;
    }
    const Chunk<S> part(s, n, chunk, a.chunks, a.chunk_vecs, kind == kRowBound);
    const Weight<T> weight{m, set.inv};
    if (kind == kRowBound) {
        const T t = low > lowest<T>() ? low : lowest<T>();
        part.gather(list, [&](T v) { return v >= t; });
        hand_over(a, row, list);
        if (!last_chunk(&a.state[row].done[1], a.chunks))
            return kCounted;
        draw_from_row<S>(a, row, set, m, list, bound, red[0], sh);
        return kCountedLast;
    }
    if (kind == kRowPlain) {
        auto mass_of = [&](T v, uint32_t) -> mass_t {
            const mass_t w = weight(v);
            return w >= set.least ? w : 0;
        };
        mass_t own = 0;
        part.each([&](T v, uint32_t at) {
            own += mass_of(v, at);
            added(own);
        });
        own = block_reduce<NT>(own, OpSum(), sh.red[0]);
        if (threadIdx.x == 0)
            put(&a.chunk_mass[blockIdx.x], own);
        if (!last_chunk(&a.state[row].done[1], a.chunks))
            return kCounted;
        if (threadIdx.x < a.chunks)
            in_chunk[threadIdx.x] = get(&a.chunk_mass[row * a.chunks + threadIdx.x]);
        __syncthreads();
        draw_in_chunk<S>(a, row, set, in_chunk, mass_of, sh.tiles);
        return kCountedLast;
    }
    for (uint32_t b = threadIdx.x; b < kSteps; b += NT)
        sh.steps[b] = 0;
    __syncthreads();
    const StepOf<T> step_of(m, set.inv, low);
    part.each([&](T v, uint32_t) {
        if (const mass_t w = weight(v))
            atomicAdd(&sh.steps[step_of(v)], w);
    });
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kSteps; b += NT)
        put(&a.steps[(uint64_t)blockIdx.x * kSteps + b], sh.steps[b]);
    if (!last_chunk(&a.state[row].done[1], a.chunks))
        return kCounted;
    // The step in which the nucleus ends, from the sums of the chunks' steps; 16 loads in flight.
    const mass_t *steps = a.steps + row * a.chunks * kSteps;
    constexpr uint32_t E = kSteps / NT, U = 4;
    mass_t sum[E] = {};
    for (uint32_t c = 0; c < a.chunks; c += U) {
        mass_t x[U][E];
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
#pragma unroll
            for (uint32_t e = 0; e < E; e++)
                x[u][e] = c + u < a.chunks ? get(&steps[(c + u) * kSteps + e * NT + threadIdx.x]) : 0;
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
#pragma unroll
            for (uint32_t e = 0; e < E; e++)
                sum[e] += x[u][e];
    }
#pragma unroll
    for (uint32_t e = 0; e < E; e++)
        sh.steps[e * NT + threadIdx.x] = sum[e];
    __syncthreads();
    const End end = find_end(sh, set.part);
    if (threadIdx.x == 0) {
        a.state[row].need = end.need;
        a.state[row].above = end.above;
        a.state[row].step = end.step;
    }
    return kCountedLast;
}

template <typename S> __device__ __forceinline__ Left sample_edge(const SplitArgs<typename StatOf<S>::T> &a)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr int NT = kChunkThreads;
    constexpr uint32_t N = kVec<S>;
    if (block_gate_closed(a.g.gate))
        return kUncounted;
    __shared__ BoundScratch bound;
    __shared__ T red[4][16];
    __shared__ List<K, kEdgeListCap> list;
    __shared__ DrawShared<T, NT> sh;
    __shared__ mass_t in_chunk[64];
    const uint64_t row = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, n = a.g.vocab;
    const Settings set = settings_of(a.g, row);
    if (kind_of(set, n, a.chunks) != kRowNucleus)
        return kUncounted;
    const auto [m, low] = row_part(a, row);
    if (m == -INFINITY)
        return kUncounted;
    const S *s = static_cast<const S *>(a.g.logits) + row * a.g.stride;
    const Chunk<S> part(s, n, chunk, a.chunks, a.chunk_vecs, false);
    const StepOf<T> step_of(m, set.inv, low);
    const Weight<T> weight{m, set.inv};
    const uint32_t end = a.state[row].step;
    part.gather(list, [&](T v) { return v > -INFINITY && step_of(v) == end; });
    // The chunk's mass before the step, or what min_p leaves of it.
    mass_t own = 0;
    if (set.least > 0) {
        part.each([&](T v, uint32_t) {
            if (v > -INFINITY && step_of(v) < end) {
                const mass_t w = weight(v);
                own += w >= set.least ? w : 0;
                added(own);
            }
        });
    } else {
#pragma unroll
        for (uint32_t e = 0; e < kSteps / NT; e++) {
            const mass_t here = a.steps[(uint64_t)blockIdx.x * kSteps + e * NT + threadIdx.x];
            own += e * NT + threadIdx.x < end ? here : 0;
        }
    }
    own = block_reduce<NT>(own, OpSum(), sh.red[0]);
    if (threadIdx.x == 0)
        put(&a.chunk_mass[blockIdx.x], own);
    __syncthreads();
    hand_over(a, row, list);
    if (!last_chunk(&a.state[row].done[2], a.chunks))
        return kCounted;
    const uint32_t count = take_list(a, row, kRowCap, m, list, bound, red[0]);
    if (count > kRowCap) {
        draw_by_search<S, NT>(a.g, row, s, set, m, sh);
        return kCountedLast;
    }
    if (threadIdx.x < a.chunks)
        in_chunk[threadIdx.x] = get(&a.chunk_mass[row * a.chunks + threadIdx.x]);
    Last<T> last;
    auto finish = [&](auto entries) {
        select_entry<NT, false>(count, entries, [&](K key, uint32_t) { return weight(value_of(key)); },
                                a.state[row].need - a.state[row].above, index_bits(n), sh.select);
        last = Last<T>{value_of(sh.select.key), sh.select.at};
        for (uint32_t j = threadIdx.x; j < count; j += NT) {
            const auto e = entries(j);
            const mass_t w = weight(value_of(e.key));
            // The values after the last whole vector belong to the last chunk.
            const uint32_t c = e.at / (a.chunk_vecs * N);
            if (last.keeps(value_of(e.key), e.at) && w >= set.least)
                atomicAdd(&in_chunk[c < a.chunks ? c : a.chunks - 1], w);
        }
    };
    if (list.count <= kEdgeListCap)
        finish(LocalList<K>{list.key, list.at});
    else
        finish(SharedList<K>{a.key + row * kRowCap, a.at + row * kRowCap});
    __syncthreads();
    draw_in_chunk<S>(a, row, set, in_chunk,
                     [&](T v, uint32_t i) -> mass_t {
                         const mass_t w = last.keeps(v, i) ? weight(v) : 0;
                         return w >= set.least ? w : 0;
                     },
                     sh.tiles);
    return kCountedLast;
}

// The end of the program by a call's last launch (close), number `launch` of it: every workgroup counts
// itself once for its row, here where its way through the launch did not; the last of a row takes
// the row's ticket, and the last ticket ends the program. So no workgroup is left that reads the call's
// arrays once the caller may write them again: a chunk of a row that an earlier launch finished, or
// that another chunk draws from alone, still reads the row's settings, however late it starts.
template <typename T>
__device__ __forceinline__ void close_rows(const SplitArgs<T> &a, const ProgramClose &c, int launch, Left left)
{
    if (c.words == nullptr || left == kCounted)
        return;
    if (left == kUncounted && !last_chunk(&a.state[blockIdx.x / a.chunks].done[launch], a.chunks))
        return;
    __shared__ int last;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0)
        last = atomicAdd(c.ticket, 1u) + 1u == a.g.rows;
    __syncthreads();
    if (last && threadIdx.x < 64) {
        __atomic_thread_fence(__ATOMIC_ACQUIRE);
        if (threadIdx.x == 0)
            *c.ticket = 0u; // every row has its ticket
        program_close_wave(c);
    }
}

template <typename S> __global__ __launch_bounds__(kChunkThreads) void k_sample_first(SplitArgs<typename StatOf<S>::T> a, ProgramClose close)
{
    close_rows(a, close, 0, sample_first<S>(a));
}
template <typename S> __global__ __launch_bounds__(kChunkThreads) void k_sample_weigh(SplitArgs<typename StatOf<S>::T> a, ProgramClose close)
{
    close_rows(a, close, 1, sample_weigh<S>(a));
}
template <typename S> __global__ __launch_bounds__(kChunkThreads) void k_sample_edge(SplitArgs<typename StatOf<S>::T> a, ProgramClose close)
{
    close_rows(a, close, 2, sample_edge<S>(a));
}

// ------------------------------------------------------------------------- launches

struct Split {
    uint32_t chunks, vecs;
};

// Chunks of long rows: 1536 workgroups for the chip, as far as each has four vectors a thread, at most
// about 16384 logits each (512 x 152000 bf16 of mixed settings: 181 us a call; 217 with twice as many
// to a chunk, 307 with half); at most 32 a row (the nucleus adds up 8 KB for each), and two at least, so
// that 1024 values are sought among 2048 groups.
Split split_of(uint64_t rows, uint32_t vocab, uint32_t per_vec)
{
    const uint64_t want = (1536 + rows - 1) / rows, most = vocab / (4 * kChunkThreads * per_vec), least = vocab / 16384;
    uint64_t chunks = want < most ? want : most;
    chunks = chunks < least ? least : chunks;
    chunks = chunks < 2 ? 2 : (chunks > 32 ? 32 : chunks);
    const uint32_t whole = vocab / per_vec;
    const uint32_t vecs = (uint32_t)((whole + chunks - 1) / chunks);
    return Split{(whole + vecs - 1) / vecs, vecs};
}

constexpr uint64_t kSlabRows = 1024; // rows that share one scratch

// Rows of up to 1024 whole vectors are one workgroup's: one launch, the row in registers (microseconds a
// call, and split: 1024 x 8000 bf16 of mixed settings 64 and 91, 64 x 4000 f32 with top-k 21 and 28, 1024
// rows with top-p 59 and 67, 64 rows 53 and 49).
bool short_row(const SampleArgs &g, uint32_t per_vec) { return g.vocab / per_vec <= 256 * 4; }

// Whether a row may have a nucleus.
bool has_nucleus(const SampleArgs &g) { return g.top_p || g.top_p_all < 1.0f; }

// Bytes of the scratch of up to kSlabRows rows; lays it out at `base` where `a` is given.
template <typename S> size_t scratch_t(const SampleArgs &g, SplitArgs<typename StatOf<S>::T> *a, char *base)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    const uint64_t rows = g.rows < kSlabRows ? g.rows : kSlabRows;
    const Split sp = split_of(rows, g.vocab, kVec<S>);
    const uint64_t parts = rows * sp.chunks;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return base + here;
    };
    char *part = take(parts * sizeof(ChunkPart<T>)), *mass = take(parts * sizeof(mass_t));
    char *steps = take(has_nucleus(g) ? parts * kSteps * sizeof(mass_t) : 0);
    char *key = take(rows * kRowCap * sizeof(K)), *places = take(rows * kRowCap * 4);
    if (a)
        *a = SplitArgs<T>{g, sp.chunks, sp.vecs, (ChunkPart<T> *)part, (mass_t *)mass, (mass_t *)steps, nullptr,
                          (K *)key, (uint32_t *)places};
    return at;
}

SampleArgs rows_from(const SampleArgs &all, uint64_t from, uint64_t most)
{
    SampleArgs g = all;
    const uint64_t size = all.dtype == kLogitF64 ? 8 : all.dtype == kLogitF32 ? 4 : 2;
    g.rows = all.rows - from < most ? all.rows - from : most;
    g.first_row = from;
    g.logits = static_cast<const char *>(all.logits) + from * all.stride * size;
    g.uniform += from;
    g.tokens += from;
    for (const float **p : {&g.temperature, &g.top_p, &g.min_p})
        if (*p)
            *p += from;
    if (g.top_k)
        g.top_k += from;
    if (g.log_prob)
        g.log_prob += from;
    return g;
}

template <typename S> hipError_t launch_t(hipStream_t s, const SampleArgs &all, void *scratch, void *state, const ProgramClose &close)
{
    using T = typename StatOf<S>::T;
    if (short_row(all, kVec<S>)) {
        hipLaunchKernelGGL((k_sample<S, 256, 4>), row_grid(all.rows), dim3(256), 0, s, all, close);
        return hipGetLastError();
    }
    for (uint64_t from = 0; from < all.rows; from += kSlabRows) {
        SplitArgs<T> a;
        scratch_t<S>(all, &a, static_cast<char *>(scratch));
        a.state = static_cast<RowState *>(state);
        a.g = rows_from(all, from, kSlabRows);
        const dim3 parts((unsigned)(a.g.rows * a.chunks)), block(kChunkThreads);
        // Every row's list is made and drawn from in the first launch where top_k says so for all.
        const bool lists = !all.top_k && all.top_k_all > 0 && (uint32_t)all.top_k_all < all.vocab &&
                           list_at_once((uint64_t)all.top_k_all, a.chunks);
        const bool edges = !lists && has_nucleus(all);
        const ProgramClose none;
        hipLaunchKernelGGL((k_sample_first<S>), parts, block, 0, s, a, lists ? close : none);
        if (!lists)
            hipLaunchKernelGGL((k_sample_weigh<S>), parts, block, 0, s, a, edges ? none : close);
        if (edges)
            hipLaunchKernelGGL((k_sample_edge<S>), parts, block, 0, s, a, close);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess)
            return err;
    }
    return hipSuccess;
}

} // namespace

size_t sample_scratch_bytes(const SampleArgs &g)
{
    if (g.rows == 0)
        return 0;
    switch (g.dtype) {
    case kLogitF32: return short_row(g, kVec<float>) ? 0 : scratch_t<float>(g, nullptr, nullptr);
    case kLogitF64: return short_row(g, kVec<double>) ? 0 : scratch_t<double>(g, nullptr, nullptr);
    case kLogitBf16: return short_row(g, kVec<__bf16>) ? 0 : scratch_t<__bf16>(g, nullptr, nullptr);
    default: return short_row(g, kVec<_Float16>) ? 0 : scratch_t<_Float16>(g, nullptr, nullptr);
    }
}

size_t sample_state_bytes() { return kSlabRows * sizeof(RowState); }

hipError_t launch_sample(hipStream_t s, const SampleArgs &g, void *scratch, void *state, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.rows == 0)
        return hipSuccess;
    if (g.rows > kCloseMaxBlocks)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    switch (g.dtype) {
    case kLogitF32: return launch_t<float>(s, g, scratch, state, close);
    case kLogitF64: return launch_t<double>(s, g, scratch, state, close);
    case kLogitBf16: return launch_t<__bf16>(s, g, scratch, state, close);
    default: return launch_t<_Float16>(s, g, scratch, state, close);
    }
}

} // namespace pcu
