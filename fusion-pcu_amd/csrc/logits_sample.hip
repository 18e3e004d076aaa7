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
#include "pcu_kernels.hpp"
#include "pcu_select.hpp"

#include <type_traits>

#pragma clang fp contract(off)

namespace pcu {

namespace {

typedef unsigned long long mass_t;
constexpr mass_t kOne = 1ull << 40;

// floor(mass * part / 2^31), mass < 2^62, part <= 2^31.
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

// A row from which nothing can be drawn; an invalid setting is a fault. One thread.
__device__ __forceinline__ void no_token(const SampleArgs &g, uint64_t row, bool ok)
{
    if (!ok) {
        atomicMin(g.fault, (unsigned long long)pack_fault(g.first_row + row, kInvalid));
        gate_record(g.gate);
    }
    g.tokens[row] = -1;
    if (g.log_prob)
        g.log_prob[row] = -INFINITY;
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
            }
        });
        const Digit<mass_t> d = find_digit(bins, need, found);
        prefix |= (K)d.digit << shift;
        need = d.left;
    }
    const mass_t w = weight(value_of(prefix));
    return {prefix, (uint32_t)((need + w - 1) / w)};
}

constexpr int kPerThread = 8; // entries of a list that a thread holds
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
    mass_t red[4][16];
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

// A list in registers, with the weights of its entries.
template <typename T> struct Entries {
    Held<typename KeyOf<T>::K, kPerThread> e;
    mass_t w[kPerThread];
    template <int NT, typename W>
    __device__ __forceinline__ Entries(const typename KeyOf<T>::K *key, const uint32_t *at, uint32_t count, const W &weight,
                                       std::integral_constant<int, NT>)
    {
#pragma unroll
        for (int b = 0; b < kPerThread; b++) {
            const uint32_t j = threadIdx.x + b * NT;
            e.key[b] = j < count ? key[j] : 0;
            e.at[b] = j < count ? at[j] : 0xffffffffu;
            w[b] = j < count ? weight(value_of(e.key[b])) : 0;
        }
    }
    template <int NT> __device__ __forceinline__ mass_t mass(mass_t *lds) const
    {
        mass_t sum = 0;
#pragma unroll
        for (int b = 0; b < kPerThread; b++)
            sum += w[b];
        return block_reduce<NT>(sum, OpSum(), lds);
    }
    // Leaves the entries up to `last` of the order.
    template <typename K> __device__ __forceinline__ void cut(K key, uint32_t at)
    {
#pragma unroll
        for (int b = 0; b < kPerThread; b++)
            if (!(e.key[b] > key || (e.key[b] == key && e.at[b] <= at)))
                w[b] = 0;
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

// Draws from a list of `count` entries, which holds the first top_k of the order (or all of it that is
// finite). need: what the nucleus has to hold, 0 for `part` of their mass.
template <typename T, int NT, typename W>
__device__ __forceinline__ void draw_from_list(const SampleArgs &g, uint64_t row, const Settings &set,
                                               const typename KeyOf<T>::K *key, const uint32_t *at, uint32_t count,
                                               mass_t need, const W &weight, DrawShared<T, NT> &sh)
{
    const int bits = index_bits(g.vocab);
    Entries<T> list(key, at, count, weight, std::integral_constant<int, NT>());
    if (count > set.k) {
        mass_t one[kPerThread];
#pragma unroll
        for (int b = 0; b < kPerThread; b++)
            one[b] = threadIdx.x + b * NT < count;
        select_entry<NT, false>(list.e, one, set.k, bits, sh.select);
        list.cut(sh.select.key, sh.select.at);
    }
    if (set.nucleus()) {
        if (need == 0) {
            need = share_of(list.template mass<NT>(sh.red[0]), set.part);
            need = need ? need : 1;
        }
        select_entry<NT, false>(list.e, list.w, need, bits, sh.select);
        list.cut(sh.select.key, sh.select.at);
    }
#pragma unroll
    for (int b = 0; b < kPerThread; b++)
        list.w[b] = list.w[b] >= set.least ? list.w[b] : 0;
    // The first by index at which the running mass passes the target.
    const mass_t total = list.template mass<NT>(sh.red[1]);
    select_entry<NT, true>(list.e, list.w, share_of(total, set.draw) + 1, bits, sh.select);
#pragma unroll
    for (int b = 0; b < kPerThread; b++)
        if (list.w[b] && list.e.at[b] == sh.select.at) {
            g.tokens[row] = (int32_t)list.e.at[b];
            if (g.log_prob)
                g.log_prob[row] = logf((float)list.w[b] / (float)total);
        }
}

// Draws along vectors [from, to) of the row (`mass_of` a value and its index). total 0: the vectors
// are the whole row, and its mass is counted first; else `target` of it lies in the vectors.
template <typename S, int NT, typename F>
__device__ __forceinline__ void draw_along(const SampleArgs &g, uint64_t row, const S *s, uint32_t from, uint32_t to,
                                           uint32_t draw, mass_t total, mass_t target, F mass_of, mass_t *lds)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>, W = NT / 64;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63, n = g.vocab;
    // The mass of each wave's run, in index order; then along the run that holds the target.
    const uint32_t run = (to - from + W - 1) / W;
    const uint32_t first = from + wave * run < to ? from + wave * run : to, past = first + run < to ? first + run : to;
    mass_t own = 0;
    wave_run(s, n, first, past, [&](const T *v, uint32_t at, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (i < count)
                own += mass_of(v[i], at + i);
        return false;
    });
    own = wave_reduce(own, OpSum());
    if (lane == 0)
        lds[wave] = own;
    __syncthreads();
    if (total == 0) {
        for (uint32_t w = 0; w < W; w++)
            total += lds[w];
        target = share_of(total, draw);
    }
    uint32_t holder = 0;
    while (holder < W - 1 && target >= lds[holder])
        target -= lds[holder++];
    if (wave != holder)
        return;
    wave_run(s, n, first, past, [&](const T *v, uint32_t at, uint32_t count) {
        mass_t w[N], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < N; i++) {
            w[i] = i < count ? mass_of(v[i], at + i) : 0;
            sum += w[i];
        }
        const mass_t upto = wave_inclusive_sum(sum);
        const uint64_t there = __ballot(upto > target);
        if (there) {
            if (lane == (uint32_t)__builtin_ctzll(there)) {
                mass_t running = upto - sum;
#pragma unroll
                for (uint32_t i = 0; i < N; i++) {
                    if (running <= target && target < running + w[i]) {
                        g.tokens[row] = (int32_t)(at + i);
                        if (g.log_prob)
                            g.log_prob[row] = logf((float)w[i] / (float)total);
                    }
                    running += w[i];
                }
            }
            return true;
        }
        target -= from_lane(upto, 63);
        return false;
    });
}

// ------------------------------------------------------- short rows: one workgroup a row
//
// The row in registers. Rows with a top_k that a list can hold: the list of the first top_k and
// everything else in LDS. Rows with a nucleus: the masses of even steps of z, then the list of the
// values down to the step in which the nucleus ends, or, when that is long, of that step alone.
// Then the drawing: over the list, or over the row.
template <typename S, int NT, int R> __global__ __launch_bounds__(NT) void k_sample(SampleArgs g)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    if (block_gate_closed(g.gate))
        return;
    __shared__ BoundScratch bound;
    __shared__ T red_t[3][16];
    __shared__ DrawShared<T, NT> sh;
    constexpr uint32_t kCap = kPerThread * NT;
    __shared__ List<K, kCap> list;
    const uint32_t tid = threadIdx.x;
    const uint64_t row = blockIdx.x;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t n = g.vocab;
    const Settings set = settings_of(g, row);
    const Row<S, NT, R> held(s, n);

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
    if (tid == 0)
        list.count = 0;
    __syncthreads();
    // Adds the row's wanted values to the list; its length.
    auto gather = [&](auto wanted) {
        held.walk([&](const T *v, uint32_t at, int) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                if (v[i] > -INFINITY && wanted(v[i], at + i))
                    list.add(key_of(v[i]), at + i);
        });
        if (held.has_extra && held.extra > -INFINITY && wanted(held.extra, held.extra_at()))
            list.add(key_of(held.extra), held.extra_at());
        __syncthreads();
        const uint32_t count = list.count;
        __syncthreads();
        return count;
    };

    if (set.k < n && set.k <= kLogitMaxK) {
        const T t = bound_of<NT>(group, m, set.k, bound, red_t[1]);
        const uint32_t count = gather([&](T v, uint32_t) { return v >= t; });
        if (count <= kCap) {
            draw_from_list(g, row, set, list.key, list.at, count, 0, weight, sh);
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
        if (count <= kCap) {
            draw_from_list(g, row, set, list.key, list.at, count, end.need, weight, sh);
            return;
        }
        if (tid == 0)
            list.count = 0;
        __syncthreads();
        count = gather([&](T v, uint32_t i) { return step_of(v) == end.step && last.keeps(v, i); });
        if (count <= kCap) {
            const Entries<T> in(list.key, list.at, count, weight, std::integral_constant<int, NT>());
            select_entry<NT, false>(in.e, in.w, end.need - end.above, index_bits(n), sh.select);
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
    draw_along<S, NT>(g, row, s, 0u, (n + N - 1) / N, set.draw, 0, 0, mass_of, sh.red[3]);
}

// ------------------------------------------------- long rows: a row split over workgroups
//
// Each row is cut into chunks of consecutive vectors, and the steps above become launches:
//   1. each chunk's maximum; for a row whose top_k a list can hold, a bound that the chunk's share
//      of top_k values reaches (such a row's chunks take every chunks-th block of vectors, so
//      that they hold alike values wherever the row's large ones lie)
//   2. with the row's maximum: the values beyond the lowest of the bounds into the row's list; or
//      a nucleus row's masses by steps of z; or the mass of the chunk
//   3. for a nucleus: the step in which it ends, and the chunks' masses before it
//   4. for a nucleus: the values of that step into the row's list
//   5. the drawing: from the list; or in the chunk that holds the target
// One workgroup would take an exponential of every logit of its row at the rate of one CU: a
// nucleus of a row of 152000 took 280 us.
enum : uint32_t { kRowNone, kRowList, kRowNucleus, kRowPlain, kRowSearch };

struct RowState {
    mass_t need, above; // of the nucleus
    uint32_t count;     // of the row's list; past its capacity: not whole
    uint32_t step;      // in which the nucleus ends
};

template <typename T> struct ChunkPart {
    T m;
    T t; // the bound; for a nucleus row the smallest value above minus infinity
};

template <typename T> struct SplitArgs {
    SampleArgs g;
    uint32_t chunks, chunk_vecs;
    ChunkPart<T> *part;  // rows x chunks
    mass_t *chunk_mass;  // rows x chunks: kept before the nucleus' last step, or kept
    mass_t *steps;       // rows x chunks x kSteps
    RowState *state;     // rows
    typename KeyOf<T>::K *key; // rows x kRowCap
    uint32_t *at;              // rows x kRowCap
};

__device__ __forceinline__ uint32_t kind_of(const Settings &s, uint32_t n)
{
    if (!s.ok)
        return kRowNone;
    if (s.k < n)
        return s.k <= kLogitMaxK ? kRowList : kRowSearch;
    return s.nucleus() ? kRowNucleus : kRowPlain;
}

constexpr int kChunkThreads = 256, kRowThreads = 1024;
constexpr uint32_t kRowCap = kPerThread * kRowThreads; // of a row's list

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
    // f(value, index, group of 4)
    template <typename F> __device__ __forceinline__ void each(F f) const
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
#pragma unroll
                for (uint32_t e = 0; e < N; e++)
                    f(v[e], (i + u * step) * N + e, u);
            }
        }
        if (rest < n)
            f((T)s[rest], rest, 0);
    }
};

template <typename S> __global__ __launch_bounds__(kChunkThreads) void k_sample_max(SplitArgs<typename StatOf<S>::T> a)
{
    using T = typename StatOf<S>::T;
    constexpr int NT = kChunkThreads;
    if (block_gate_closed(a.g.gate))
        return;
    __shared__ BoundScratch bound;
    __shared__ T red[3][16];
    const uint64_t row = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, n = a.g.vocab;
    const Settings set = settings_of(a.g, row);
    const uint32_t kind = kind_of(set, n);
    if (chunk == 0 && threadIdx.x == 0)
        a.state[row].count = 0;
    const Chunk<S> part(static_cast<const S *>(a.g.logits) + row * a.g.stride, n, chunk, a.chunks, a.chunk_vecs,
                        kind == kRowList);
    T group[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    part.each([&](T v, uint32_t, int u) { group[u] = OpMax()(group[u], v); });
    T m = OpMax()(OpMax()(group[0], group[1]), OpMax()(group[2], group[3]));
    m = block_reduce<NT>(m, OpMax(), red[0]);
    T t = -INFINITY;
    if (kind == kRowList) {
        t = bound_of<NT>(group, m, (set.k + a.chunks - 1) / a.chunks, bound, red[1]);
    } else if (kind == kRowNucleus) {
        t = INFINITY;
        part.each([&](T v, uint32_t, int) { t = v > -INFINITY && v < t ? v : t; });
        t = -block_reduce<NT>(-t, OpMax(), red[1]);
    }
    if (threadIdx.x == 0)
        a.part[blockIdx.x] = ChunkPart<T>{m, t};
}

// The row's maximum, and the lowest of the chunks' bounds or smallest values; one chunk a lane.
template <typename T> __device__ __forceinline__ ChunkPart<T> row_part(const SplitArgs<T> &a, uint64_t row)
{
    const uint32_t lane = threadIdx.x & 63;
    ChunkPart<T> p{-INFINITY, INFINITY};
    if (lane < a.chunks)
        p = a.part[row * a.chunks + lane];
    return {wave_reduce(p.m, OpMax()), -wave_reduce(-p.t, OpMax())};
}

// A workgroup's list handed to its row's: one place reserved for all of it. A list that does not
// fit sets the row's count beyond the capacity.
template <typename K, int CAP, typename T>
__device__ __forceinline__ void hand_over(const SplitArgs<T> &a, uint64_t row, const List<K, CAP> &list, uint32_t *base)
{
    const uint32_t count = list.count;
    if (count == 0)
        return;
    if (threadIdx.x == 0)
        *base = atomicAdd(&a.state[row].count, count > CAP ? (uint32_t)kRowCap + 1u : count);
    __syncthreads();
    const uint32_t to = *base;
    if (count > CAP || to + count > kRowCap)
        return;
    for (uint32_t j = threadIdx.x; j < count; j += kChunkThreads) {
        a.key[row * kRowCap + to + j] = list.key[j];
        a.at[row * kRowCap + to + j] = list.at[j];
    }
}

constexpr int kChunkListCap = 1024;

template <typename S> __global__ __launch_bounds__(kChunkThreads) void k_sample_weigh(SplitArgs<typename StatOf<S>::T> a)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr int NT = kChunkThreads;
    if (block_gate_closed(a.g.gate))
        return;
    __shared__ union {
        mass_t steps[kSteps];
        List<K, kChunkListCap> list;
    } sh;
    __shared__ mass_t red[16];
    __shared__ uint32_t base;
    const uint64_t row = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, n = a.g.vocab;
    const Settings set = settings_of(a.g, row);
    const uint32_t kind = kind_of(set, n);
    const auto [m, low] = row_part(a, row);
    if (kind == kRowNone || kind == kRowSearch || m == -INFINITY)
        return;
    const Chunk<S> part(static_cast<const S *>(a.g.logits) + row * a.g.stride, n, chunk, a.chunks, a.chunk_vecs,
                        kind == kRowList);
    if (kind == kRowList) {
        const T t = low;
        if (threadIdx.x == 0)
            sh.list.count = 0;
        __syncthreads();
        part.each([&](T v, uint32_t at, int) {
            if (v >= t && v > -INFINITY)
                sh.list.add(key_of(v), at);
        });
        __syncthreads();
        hand_over(a, row, sh.list, &base);
        return;
    }
    const Weight<T> weight{m, set.inv};
    if (kind == kRowPlain) {
        mass_t own = 0;
        part.each([&](T v, uint32_t, int) {
            const mass_t w = weight(v);
            own += w >= set.least ? w : 0;
        });
        own = block_reduce<NT>(own, OpSum(), red);
        if (threadIdx.x == 0)
            a.chunk_mass[blockIdx.x] = own;
        return;
    }
    for (uint32_t b = threadIdx.x; b < kSteps; b += NT)
        sh.steps[b] = 0;
    __syncthreads();
    const StepOf<T> step_of(m, set.inv, low);
    part.each([&](T v, uint32_t, int) {
        if (const mass_t w = weight(v))
            atomicAdd(&sh.steps[step_of(v)], w);
    });
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kSteps; b += NT)
        a.steps[(uint64_t)blockIdx.x * kSteps + b] = sh.steps[b];
}

// The step in which each nucleus ends, and the chunks' masses before it.
template <typename T> __global__ __launch_bounds__(kRowThreads) void k_sample_end(SplitArgs<T> a)
{
    constexpr int NT = kRowThreads;
    if (block_gate_closed(a.g.gate))
        return;
    __shared__ DrawShared<T, NT> sh;
    const uint64_t row = blockIdx.x;
    const Settings set = settings_of(a.g, row);
    if (kind_of(set, a.g.vocab) != kRowNucleus || row_part(a, row).m == -INFINITY)
        return;
    static_assert(kSteps == NT, "one step a thread");
    const mass_t *steps = a.steps + row * a.chunks * kSteps;
    mass_t sum = 0;
#pragma unroll 8
    for (uint32_t c = 0; c < a.chunks; c++)
        sum += steps[c * kSteps + threadIdx.x];
    sh.steps[threadIdx.x] = sum;
    __syncthreads();
    const End end = find_end(sh, set.part);
    if (threadIdx.x == 0) {
        a.state[row].need = end.need;
        a.state[row].above = end.above;
        a.state[row].step = end.step;
    }
    for (uint32_t c = threadIdx.x / 64; c < a.chunks; c += NT / 64) {
        mass_t before = 0;
#pragma unroll 8
        for (uint32_t b = threadIdx.x & 63; b < end.step; b += 64)
            before += steps[c * kSteps + b];
        before = wave_reduce(before, OpSum());
        if ((threadIdx.x & 63) == 0)
            a.chunk_mass[row * a.chunks + c] = before;
    }
}

// The values of the step in which the nucleus ends; where min_p cuts, the chunk's kept mass before it.
template <typename S> __global__ __launch_bounds__(kChunkThreads) void k_sample_edge(SplitArgs<typename StatOf<S>::T> a)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr int NT = kChunkThreads;
    if (block_gate_closed(a.g.gate))
        return;
    __shared__ List<K, kChunkListCap> list;
    __shared__ mass_t red[16];
    __shared__ uint32_t base;
    const uint64_t row = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, n = a.g.vocab;
    const Settings set = settings_of(a.g, row);
    const auto [m, low] = row_part(a, row);
    if (kind_of(set, n) != kRowNucleus || m == -INFINITY)
        return;
    const Chunk<S> part(static_cast<const S *>(a.g.logits) + row * a.g.stride, n, chunk, a.chunks, a.chunk_vecs, false);
    const StepOf<T> step_of(m, set.inv, low);
    const uint32_t end = a.state[row].step;
    if (threadIdx.x == 0)
        list.count = 0;
    __syncthreads();
    part.each([&](T v, uint32_t at, int) {
        if (v > -INFINITY && step_of(v) == end)
            list.add(key_of(v), at);
    });
    if (set.least > 0) {
        const Weight<T> weight{m, set.inv};
        mass_t own = 0;
        part.each([&](T v, uint32_t, int) {
            if (v > -INFINITY && step_of(v) < end) {
                const mass_t w = weight(v);
                own += w >= set.least ? w : 0;
            }
        });
        own = block_reduce<NT>(own, OpSum(), red);
        if (threadIdx.x == 0)
            a.chunk_mass[blockIdx.x] = own;
    }
    __syncthreads();
    hand_over(a, row, list, &base);
}

template <typename S> __global__ __launch_bounds__(kRowThreads) void k_sample_draw(SplitArgs<typename StatOf<S>::T> a)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr int NT = kRowThreads;
    constexpr uint32_t N = kVec<S>;
    if (block_gate_closed(a.g.gate))
        return;
    __shared__ DrawShared<T, NT> sh;
    __shared__ mass_t in_chunk[64];
    const SampleArgs &g = a.g;
    const uint64_t row = blockIdx.x;
    const uint32_t n = g.vocab, tid = threadIdx.x;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const Settings set = settings_of(g, row);
    const T m = row_part(a, row).m;
    if (!set.ok || m == -INFINITY) {
        if (tid == 0)
            no_token(g, row, set.ok);
        return;
    }
    uint32_t kind = kind_of(set, n);
    const Weight<T> weight{m, set.inv};
    const uint32_t count = kind == kRowList || kind == kRowNucleus ? a.state[row].count : 0;
    Last<T> last{-INFINITY, 0xffffffffu};
    if (count > kRowCap)
        kind = kRowSearch;
    const K *key = a.key + row * kRowCap;
    const uint32_t *at = a.at + row * kRowCap;
    if (kind == kRowList) {
        draw_from_list(g, row, set, key, at, count, 0, weight, sh);
        return;
    }
    auto mass_of = [&](T v, uint32_t i) -> mass_t {
        if (!last.keeps(v, i))
            return 0;
        const mass_t w = weight(v);
        return w >= set.least ? w : 0;
    };
    const uint32_t vecs = (n + N - 1) / N;
    if (kind == kRowSearch) {
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
                for (uint32_t i = 0; i < N; i++)
                    if (i < values && last.keeps(v[i], at + i))
                        mass += weight(v[i]);
            });
            mass = share_of(block_reduce<NT>(mass, OpSum(), sh.red[0]), set.part);
            last = nucleus_exactly<S, NT>(s, n, pk, mass ? mass : 1, weight, sh);
        }
        draw_along<S, NT>(g, row, s, 0u, vecs, set.draw, 0, 0, mass_of, sh.red[3]);
        return;
    }
    if (tid < a.chunks)
        in_chunk[tid] = a.chunk_mass[row * a.chunks + tid];
    __syncthreads();
    if (kind == kRowNucleus) {
        Entries<T> in(key, at, count, weight, std::integral_constant<int, NT>());
        select_entry<NT, false>(in.e, in.w, a.state[row].need - a.state[row].above, index_bits(n), sh.select);
        last = Last<T>{value_of(sh.select.key), sh.select.at};
        in.cut(sh.select.key, sh.select.at);
#pragma unroll
        for (int b = 0; b < kPerThread; b++) {
            // The values after the last whole vector belong to the last chunk.
            const uint32_t c = in.e.at[b] / (a.chunk_vecs * N);
            if (in.w[b] && in.w[b] >= set.least)
                atomicAdd(&in_chunk[c < a.chunks ? c : a.chunks - 1], in.w[b]);
        }
        __syncthreads();
    }
    mass_t total = 0;
    for (uint32_t c = 0; c < a.chunks; c++)
        total += in_chunk[c];
    mass_t target = share_of(total, set.draw);
    uint32_t c = 0;
    while (c < a.chunks - 1 && target >= in_chunk[c])
        target -= in_chunk[c++];
    const uint32_t from = c * a.chunk_vecs, to = c == a.chunks - 1 ? vecs : from + a.chunk_vecs;
    draw_along<S, NT>(g, row, s, from, to, set.draw, total, target, mass_of, sh.red[3]);
}

// ------------------------------------------------------------------------- launches

struct Split {
    uint32_t chunks, vecs;
};

// Chunks of long rows: of about 4096 logits where rows are few, of 16384 where they are many, at
// most 32 a row (the nucleus adds up 8 KB for each); two at least, so that 1024 values are sought
// among 2048 groups.
Split split_of(uint64_t rows, uint32_t vocab, uint32_t per_vec)
{
    uint64_t chunks = vocab / (rows < 64 ? 4096 : 16384);
    chunks = chunks < 2 ? 2 : (chunks > 32 ? 32 : chunks);
    const uint32_t whole = vocab / per_vec;
    const uint32_t vecs = (uint32_t)((whole + chunks - 1) / chunks);
    return Split{(whole + vecs - 1) / vecs, vecs};
}

constexpr uint64_t kSlabRows = 1024; // rows that share one scratch

// Rows of up to 1024 whole vectors are one workgroup's.
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
    char *part = take(parts * sizeof(ChunkPart<T>)), *mass = take(parts * sizeof(mass_t)), *state = take(rows * sizeof(RowState));
    char *steps = take(has_nucleus(g) ? parts * kSteps * sizeof(mass_t) : 0);
    char *key = take(rows * kRowCap * sizeof(K)), *places = take(rows * kRowCap * 4);
    if (a)
        *a = SplitArgs<T>{g, sp.chunks, sp.vecs, (ChunkPart<T> *)part, (mass_t *)mass, (mass_t *)steps, (RowState *)state,
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

template <typename S> hipError_t launch_t(hipStream_t s, const SampleArgs &all, void *scratch)
{
    using T = typename StatOf<S>::T;
    if (short_row(all, kVec<S>)) {
        hipLaunchKernelGGL((k_sample<S, 256, 4>), dim3((unsigned)all.rows), dim3(256), 0, s, all);
        return hipGetLastError();
    }
    for (uint64_t from = 0; from < all.rows; from += kSlabRows) {
        SplitArgs<T> a;
        scratch_t<S>(all, &a, static_cast<char *>(scratch));
        a.g = rows_from(all, from, kSlabRows);
        const dim3 parts((unsigned)(a.g.rows * a.chunks)), rows((unsigned)a.g.rows);
        hipLaunchKernelGGL((k_sample_max<S>), parts, dim3(kChunkThreads), 0, s, a);
        hipLaunchKernelGGL((k_sample_weigh<S>), parts, dim3(kChunkThreads), 0, s, a);
        if (has_nucleus(all)) {
            hipLaunchKernelGGL((k_sample_end<T>), rows, dim3(kRowThreads), 0, s, a);
            hipLaunchKernelGGL((k_sample_edge<S>), parts, dim3(kChunkThreads), 0, s, a);
        }
        hipLaunchKernelGGL((k_sample_draw<S>), rows, dim3(kRowThreads), 0, s, a);
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

hipError_t launch_sample(hipStream_t s, const SampleArgs &g, void *scratch)
{
    if (g.rows == 0)
        return hipSuccess;
    switch (g.dtype) {
    case kLogitF32: return launch_t<float>(s, g, scratch);
    case kLogitF64: return launch_t<double>(s, g, scratch);
    case kLogitBf16: return launch_t<__bf16>(s, g, scratch);
    default: return launch_t<_Float16>(s, g, scratch);
    }
}

} // namespace pcu
