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
        if (v == m)
            return kOne;
        const float z = (float)(v - m) * inv;
        const uint32_t e = __float_as_uint(expf(z)); // at most 1, or NaN
        const int shift = (int)(e >> 23) - (127 + 23 - 40);
        const uint32_t frac = (e & 0x7fffffu) | 0x800000u;
        const mass_t w = shift >= 0 ? (mass_t)frac << shift : (mass_t)(frac >> (shift < -31 ? 31 : -shift));
        return v < m ? w : 0; // a NaN has no weight
    }
};

struct Settings {
    float temperature, top_p, min_p, uniform;
    int top_k;
};

__device__ __forceinline__ bool settings_ok(const Settings &s)
{
    return s.temperature >= 0.0f && s.temperature < INFINITY && s.top_p >= 0.0f && s.top_p <= 1.0f &&
           s.min_p >= 0.0f && s.min_p <= 1.0f && s.uniform >= 0.0f && s.uniform < 1.0f;
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

// Inclusive sums over the workgroup's threads, and the total.
template <int NT> struct BlockSums {
    mass_t upto, total;
};
template <int NT> __device__ __forceinline__ BlockSums<NT> block_sums(mass_t v, mass_t *lds)
{
    const mass_t in = wave_inclusive_sum(v);
    if ((threadIdx.x & 63) == 63)
        lds[threadIdx.x / 64] = in;
    __syncthreads();
    mass_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < NT / 64; w++) {
        before += w < threadIdx.x / 64 ? lds[w] : 0;
        total += lds[w];
    }
    return {before + in, total};
}

constexpr int kListCap = 2048;
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
            before += __shfl(upto, 63, 64);
            return before >= p.c;
        });
    __syncthreads();
    return {value_of(p.t), *at_out};
}

// One workgroup a row, the row in registers where it fits. Rows with a top_k that a list can hold:
// the list of the first top_k and everything else in LDS. Rows with a nucleus: the masses of
// even steps of z, then the list of the values down to the step in which the nucleus ends, or,
// when that is long, of that step alone. Then the drawing: over the list, or over the row.
template <typename S, int NT, int R> __global__ __launch_bounds__(NT) void k_sample(SampleArgs g)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    if (block_gate_closed(g.gate))
        return;
    __shared__ BoundScratch bound;
    __shared__ Digit<uint32_t> count_digit;
    __shared__ Digit<mass_t> mass_digit;
    __shared__ T red_t[3][16];
    __shared__ mass_t red_m[4][16];
    __shared__ uint32_t wave_ties[16], found_at;
    __shared__ List<K, kListCap> list;
    __shared__ mass_t steps[kSteps]; // masses of the steps of z, then weights of the list
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint64_t row = blockIdx.x;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t n = g.vocab;
    Settings set;
    set.temperature = g.temperature ? g.temperature[row] : g.temperature_all;
    set.top_k = g.top_k ? g.top_k[row] : g.top_k_all;
    set.top_p = g.top_p ? g.top_p[row] : g.top_p_all;
    set.min_p = g.min_p ? g.min_p[row] : g.min_p_all;
    set.uniform = g.uniform[row];
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

    const bool ok = settings_ok(set);
    if (!ok || m == -INFINITY) {
        if (tid == 0) {
            if (!ok) {
                atomicMin(g.fault, (unsigned long long)pack_fault(row, kInvalid));
                gate_record(g.gate);
            }
            g.tokens[row] = -1;
            if (g.log_prob)
                g.log_prob[row] = -INFINITY;
        }
        return;
    }
    float inv = 1.0f / set.temperature;
    uint32_t k = set.top_k <= 0 || set.top_k >= (int64_t)n ? n : (uint32_t)set.top_k;
    if (inv == INFINITY) {
        inv = 1.0f;
        k = 1;
    }
    const Weight<T> weight{m, inv};
    const mass_t least = (mass_t)ceil((double)set.min_p * (double)kOne);
    const uint32_t part = (uint32_t)((double)set.top_p * 2147483648.0);
    const uint32_t draw = (uint32_t)((double)set.uniform * 2147483648.0);
    const bool nucleus = part < 0x80000000u;

    // The prefix from which tokens are drawn: as a list (`listed` entries, sorted), or by its
    // last token.
    uint32_t listed = 0;
    Last<T> last{-INFINITY, 0xffffffffu};
    mass_t need = ~0ull; // what the nucleus has to hold
    if (k < n && k <= kLogitMaxK) {
        if (tid == 0)
            list.count = 0;
        const T t = bound_of<NT>(group, m, k, bound, red_t[1]);
        held.walk([&](const T *v, uint32_t at, int) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                if (v[i] >= t && v[i] > -INFINITY)
                    list.add(key_of(v[i]), at + i);
        });
        if (held.has_extra && held.extra >= t && held.extra > -INFINITY)
            list.add(key_of(held.extra), held.extra_at());
        __syncthreads();
        listed = list.count;
        __syncthreads();
        if (listed <= kListCap) {
            sort_list<NT>(list, listed);
            listed = listed < k ? listed : k; // fewer: the row has no more finite values
        } else {
            listed = 0;
        }
    }
    if (listed == 0) {
        Prefix<K> pk{0, 0};
        if (k < n) {
            pk = select_count<S, NT>(s, n, k, reinterpret_cast<uint32_t *>(steps), &count_digit);
            if (pk.t)
                last = last_of<S, NT>(s, n, pk, wave_ties, &found_at);
        }
        if (nucleus) {
            // Masses by steps of z; the weights of z below -27.8 are 0.
            for (uint32_t b = tid; b < kSteps; b += NT)
                steps[b] = 0;
            if (tid == 0)
                list.count = 0;
            __syncthreads();
            const float scale = inv * (float)(kSteps / 28.0);
            auto step_of = [&](T v) { return (float)(m - v) * scale; };
            auto add = [&](T v, uint32_t i) {
                if (last.keeps(v, i)) {
                    const mass_t w = weight(v);
                    if (w) {
                        const float x = step_of(v);
                        atomicAdd(&steps[x < (float)(kSteps - 1) ? (uint32_t)x : kSteps - 1], w);
                    }
                }
            };
            held.walk([&](const T *v, uint32_t at, int) {
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    add(v[i], at + i);
            });
            if (held.has_extra)
                add(held.extra, held.extra_at());
            __syncthreads();
            // The step in which the nucleus ends, and the mass before it.
            constexpr uint32_t each = kSteps / NT;
            mass_t own = 0;
#pragma unroll
            for (uint32_t b = 0; b < each; b++)
                own += steps[tid * each + b];
            const BlockSums<NT> sums = block_sums<NT>(own, red_m[0]);
            need = share_of(sums.total, part);
            need = need ? need : 1; // at least one token
            mass_t before = sums.upto - own;
            if (before < need && need <= sums.upto) {
#pragma unroll
                for (uint32_t b = 0; b < each; b++) {
                    const mass_t here = steps[tid * each + b];
                    if (before < need && need <= before + here) {
                        bound.bin = tid * each + b;
                        mass_digit.left = before;
                    }
                    before += here;
                }
            }
            __syncthreads();
            const uint32_t end = bound.bin;
            const mass_t above = mass_digit.left;
            // Everything down to that step, if it fits the list, else that step alone.
            auto in_step = [&](T v, uint32_t i) {
                const float x = step_of(v);
                const uint32_t b = x < (float)(kSteps - 1) ? (uint32_t)x : kSteps - 1;
                return b == end && last.keeps(v, i);
            };
            auto to_step = [&](T v, uint32_t i) {
                const float x = step_of(v);
                const uint32_t b = x < (float)(kSteps - 1) ? (uint32_t)x : kSteps - 1;
                return b <= end && last.keeps(v, i);
            };
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
            listed = gather(to_step);
            if (listed <= kListCap) {
                sort_list<NT>(list, listed);
            } else {
                if (tid == 0)
                    list.count = 0;
                __syncthreads();
                const uint32_t count = gather(in_step);
                listed = 0;
                if (count <= kListCap) {
                    sort_list<NT>(list, count);
                    // The first entry at which the mass reaches `need` is the last one kept.
                    constexpr uint32_t per = kListCap / NT;
                    mass_t w[per], sum = 0;
#pragma unroll
                    for (uint32_t b = 0; b < per; b++) {
                        const uint32_t j = tid * per + b;
                        w[b] = j < count ? weight(value_of(list.key[j])) : 0;
                        sum += w[b];
                    }
                    const BlockSums<NT> in = block_sums<NT>(sum, red_m[1]);
                    mass_t upto = above + in.upto - sum;
#pragma unroll
                    for (uint32_t b = 0; b < per; b++) {
                        if (upto < need && need <= upto + w[b])
                            found_at = tid * per + b;
                        upto += w[b];
                    }
                    __syncthreads();
                    last = Last<T>{value_of(list.key[found_at]), list.at[found_at]};
                } else {
                    const Prefix<K> pp = select_mass<S, NT>(s, n, pk, need, weight, steps, &mass_digit);
                    last = last_of<S, NT>(s, n, pp, wave_ties, &found_at);
                }
            }
        }
    }

    if (listed) {
        // Weights of the sorted list, and how many of them are kept.
        constexpr uint32_t per = kListCap / NT;
        mass_t w[per], sum = 0;
#pragma unroll
        for (uint32_t b = 0; b < per; b++) {
            const uint32_t j = tid * per + b;
            w[b] = j < listed ? weight(value_of(list.key[j])) : 0;
            sum += w[b];
        }
        BlockSums<NT> in = block_sums<NT>(sum, red_m[0]);
        if (nucleus && need == ~0ull) {
            need = share_of(in.total, part);
            need = need ? need : 1;
        }
        mass_t before = in.upto - sum, own = 0;
#pragma unroll
        for (uint32_t b = 0; b < per; b++) {
            const mass_t here = w[b];
            if (!(before < need) || here < least)
                w[b] = 0;
            before += here;
            own += w[b];
        }
        const mass_t total = block_reduce<NT>(own, OpSum(), red_m[1]);
        // The first by index at which the running mass passes the target: digit by digit of the
        // index, 8 bits each.
        mass_t target = share_of(total, draw) + 1;
        uint32_t prefix = 0;
        mass_t *const bins = steps;
        for (int shift = 16; shift >= 0; shift -= 8) {
            for (uint32_t b = tid; b < 256; b += NT)
                bins[b] = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t b = 0; b < per; b++) {
                const uint32_t j = tid * per + b;
                if (w[b]) {
                    const uint32_t at = ~list.at[j] & 0xffffffu; // larger for smaller indices
                    if (((at ^ prefix) >> shift) < 256)
                        atomicAdd(&bins[(at >> shift) & 255u], w[b]);
                }
            }
            const Digit<mass_t> d = find_digit(bins, target, &mass_digit);
            prefix |= d.digit << shift;
            target = d.left;
        }
        const uint32_t token = ~prefix & 0xffffffu;
#pragma unroll
        for (uint32_t b = 0; b < per; b++) {
            const uint32_t j = tid * per + b;
            if (w[b] && list.at[j] == token) {
                g.tokens[row] = (int32_t)token;
                if (g.log_prob)
                    g.log_prob[row] = logf((float)w[b] / (float)total);
            }
        }
        return;
    }

    // Over the row: the mass of each wave's run of it in index order, then along the run that
    // holds the target.
    constexpr uint32_t W = NT / 64;
    const uint32_t wave = tid / 64;
    auto mass_of = [&](T v, uint32_t i) -> mass_t {
        if (!last.keeps(v, i))
            return 0;
        const mass_t w = weight(v);
        return w >= least ? w : 0;
    };
    const uint32_t vecs = (n + N - 1) / N, run = (vecs + W - 1) / W;
    const uint32_t first = wave * run, past = first + run < vecs ? first + run : vecs;
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
        red_m[3][wave] = own;
    __syncthreads();
    mass_t total = 0;
    for (uint32_t w = 0; w < W; w++)
        total += red_m[3][w];
    mass_t target = share_of(total, draw);
    uint32_t holder = 0;
    while (holder < W - 1 && target >= red_m[3][holder])
        target -= red_m[3][holder++];
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
        target -= __shfl(upto, 63, 64);
        return false;
    });
}

template <typename S> hipError_t launch_t(hipStream_t s, const SampleArgs &g)
{
    const uint32_t vecs = g.vocab / kVec<S>;
    const dim3 grid((unsigned)g.rows);
    if (vecs <= 256 * 4)
        hipLaunchKernelGGL((k_sample<S, 256, 4>), grid, dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((k_sample<S, 1024, 0>), grid, dim3(1024), 0, s, g);
    return hipGetLastError();
}

} // namespace

hipError_t launch_sample(hipStream_t s, const SampleArgs &g)
{
    if (g.rows == 0)
        return hipSuccess;
    switch (g.dtype) {
    case kLogitF32: return launch_t<float>(s, g);
    case kLogitF64: return launch_t<double>(s, g);
    case kLogitBf16: return launch_t<__bf16>(s, g);
    default: return launch_t<_Float16>(s, g);
    }
}

} // namespace pcu
