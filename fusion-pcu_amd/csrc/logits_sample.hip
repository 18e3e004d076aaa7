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

template <typename S, int NT> __global__ __launch_bounds__(NT) void k_sample(SampleArgs g)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    constexpr uint32_t W = NT / 64;
    if (block_gate_closed(g.gate))
        return;
    __shared__ mass_t bins[256];
    __shared__ Digit<uint32_t> count_digit;
    __shared__ Digit<mass_t> mass_digit;
    __shared__ T red_t[16];
    __shared__ mass_t red_m[16], wave_mass[16];
    __shared__ uint32_t wave_ties[16];
    const uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid & 63;
    const uint64_t row = blockIdx.x;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t n = g.vocab;
    Settings set;
    set.temperature = g.temperature ? g.temperature[row] : g.temperature_all;
    set.top_k = g.top_k ? g.top_k[row] : g.top_k_all;
    set.top_p = g.top_p ? g.top_p[row] : g.top_p_all;
    set.min_p = g.min_p ? g.min_p[row] : g.min_p_all;
    set.uniform = g.uniform[row];

    T m = -INFINITY;
    each_vec<S, NT>(s, n, [&](const T *v, uint32_t, uint32_t) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            m = OpMax()(m, v[i]);
    });
    m = block_reduce<NT>(m, OpMax(), red_t);

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

    // (t, c) of the prefix from which tokens are drawn; t = 0: all of the row.
    Prefix<K> kept{0, 0};
    if (k < n)
        kept = select_count<S, NT>(s, n, k, reinterpret_cast<uint32_t *>(bins), &count_digit);
    if (part < 0x80000000u) {
        mass_t mass = 0;
        each_vec<S, NT>(s, n, [&](const T *v, uint32_t, uint32_t count) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                if (i < count && key_of(v[i]) > kept.t)
                    mass += weight(v[i]);
        });
        mass = block_reduce<NT>(mass, OpSum(), red_m);
        if (kept.t)
            mass += kept.c * weight(value_of(kept.t));
        const mass_t need = share_of(mass, part);
        if (need == 0)
            kept = Prefix<K>{key_of(m), 1};
        else
            kept = select_mass<S, NT>(s, n, kept, need, weight, bins, &mass_digit);
    }

    // Each wave's part of the row in index order: its mass and its values equal to t.
    const mass_t tie_w = kept.t == 0 ? 0 : weight(value_of(kept.t));
    const mass_t tie = tie_w >= least ? tie_w : 0;
    auto above = [&](T v) -> mass_t {
        if (!(key_of(v) > kept.t))
            return 0;
        const mass_t w = weight(v);
        return w >= least ? w : 0;
    };
    const uint32_t vecs = (n + N - 1) / N, run = (vecs + W - 1) / W;
    const uint32_t first = wave * run, last = first + run < vecs ? first + run : vecs;
    mass_t mass = 0;
    uint32_t ties = 0;
    wave_run(s, n, first, last, [&](const T *v, uint32_t, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (i < count) {
                mass += above(v[i]);
                ties += kept.t != 0 && key_of(v[i]) == kept.t;
            }
        return false;
    });
    mass = wave_reduce(mass, OpSum());
    ties = wave_reduce(ties, OpSum());
    if (lane == 0) {
        wave_mass[wave] = mass;
        wave_ties[wave] = ties;
    }
    __syncthreads();
    mass_t total = 0;
    uint32_t left = kept.c;
    for (uint32_t w = 0; w < W; w++) {
        const uint32_t here = wave_ties[w] < left ? wave_ties[w] : left;
        total += wave_mass[w] + here * tie;
        left -= here;
    }
    mass_t target = share_of(total, (uint32_t)((double)set.uniform * 2147483648.0));
    // The wave whose part holds the target, and what is left of the target and the ties there.
    left = kept.c;
    uint32_t holder = 0;
    for (uint32_t w = 0; w < W; w++) {
        const uint32_t here = wave_ties[w] < left ? wave_ties[w] : left;
        const mass_t in = wave_mass[w] + here * tie;
        if (target < in) {
            holder = w;
            break;
        }
        target -= in;
        left -= here;
    }
    if (wave != holder)
        return;
    wave_run(s, n, first, last, [&](const T *v, uint32_t at, uint32_t count) {
        uint32_t own_ties = 0;
        mass_t own = 0;
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (i < count) {
                own += above(v[i]);
                own_ties += kept.t != 0 && key_of(v[i]) == kept.t;
            }
        const uint32_t ties_upto = wave_inclusive_sum(own_ties);
        const uint32_t ties_before = ties_upto - own_ties;
        uint32_t mine = ties_before >= left ? 0 : (own_ties < left - ties_before ? own_ties : left - ties_before);
        own += mine * tie;
        const mass_t upto = wave_inclusive_sum(own);
        const uint64_t there = __ballot(upto > target);
        if (there) {
            if (lane == (uint32_t)__builtin_ctzll(there)) {
                mass_t run_mass = upto - own;
                uint32_t token = 0;
                mass_t drawn = 0;
                bool done = false;
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    if (i < count && !done) {
                        mass_t w = above(v[i]);
                        if (kept.t != 0 && key_of(v[i]) == kept.t && mine) {
                            w = tie;
                            mine--;
                        }
                        run_mass += w;
                        if (run_mass > target) {
                            token = at + i;
                            drawn = w;
                            done = true;
                        }
                    }
                g.tokens[row] = (int32_t)token;
                if (g.log_prob)
                    g.log_prob[row] = logf((float)drawn / (float)total);
            }
            return true;
        }
        target -= __shfl(upto, 63, 64);
        const uint32_t all = __shfl(ties_upto, 63, 64);
        left -= all < left ? all : left;
        return false;
    });
}

template <typename S> hipError_t launch_t(hipStream_t s, const SampleArgs &g)
{
    if (g.vocab <= 8192)
        hipLaunchKernelGGL((k_sample<S, 256>), dim3((unsigned)g.rows), dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((k_sample<S, 1024>), dim3((unsigned)g.rows), dim3(1024), 0, s, g);
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
