// The k largest logits of each row, in order, with the row's log-sum-exp.
//
//   order: value descending, then index ascending (-0 equal to +0, NaN after minus infinity)
//   log_sum = log sum_v exp(l_v / T)
// The prefix (t, c) of k values is found digit by digit of the key; its values are then
// gathered into LDS, the c values equal to t by index, and sorted there.
#include "pcu_kernels.hpp"
#include "pcu_select.hpp"

#pragma clang fp contract(off)

namespace pcu {

namespace {

// Sorts `size` (a power of two) entries, by key descending and index ascending; whole workgroup.
template <int NT, typename K> __device__ __forceinline__ void sort_entries(K *key, uint32_t *at, uint32_t size)
{
    for (uint32_t len = 2; len <= size; len <<= 1)
        for (uint32_t gap = len >> 1; gap > 0; gap >>= 1) {
            __syncthreads();
            for (uint32_t p = threadIdx.x; p < size / 2; p += NT) {
                const uint32_t a = 2 * p - (p & (gap - 1)), b = a + gap;
                const K ka = key[a], kb = key[b];
                const uint32_t ia = at[a], ib = at[b];
                const bool ordered = ka > kb || (ka == kb && ia < ib);
                if (ordered != ((a & len) == 0)) {
                    key[a] = kb;
                    key[b] = ka;
                    at[a] = ib;
                    at[b] = ia;
                }
            }
        }
    __syncthreads();
}

template <typename S, int NT> __global__ __launch_bounds__(NT) void k_top(TopArgs g)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    constexpr uint32_t W = NT / 64;
    if (block_gate_closed(g.gate))
        return;
    __shared__ uint32_t bins[256];
    __shared__ Digit<uint32_t> digit;
    __shared__ T red_m[16], red_s[16];
    __shared__ uint32_t wave_ties[16], entries;
    __shared__ K key[kLogitMaxK];
    __shared__ uint32_t place[kLogitMaxK];
    const uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid & 63;
    const uint64_t row = blockIdx.x;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t n = g.vocab, k = g.k < n ? g.k : n;

    if (g.log_sum) {
        T m = -INFINITY;
        each_vec<S, NT>(s, n, [&](const T *v, uint32_t, uint32_t) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                m = OpMax()(m, v[i]);
        });
        m = block_reduce<NT>(m, OpMax(), red_m);
        const Expo<T> ex(m, (T)1 / (T)g.temperature);
        T sum = 0;
        each_vec<S, NT>(s, n, [&](const T *v, uint32_t, uint32_t) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                sum += ex(v[i]);
        });
        sum = block_reduce<NT>(sum, OpSum(), red_s);
        if (tid == 0)
            static_cast<T *>(g.log_sum)[row] = ex.log_sum(sum);
    }
    uint32_t size = 1;
    while (size < k)
        size <<= 1;
    if (k > 0) {
        const Prefix<K> top = select_count<S, NT>(s, n, k, bins, &digit);
        for (uint32_t j = tid; j < size; j += NT) {
            key[j] = 0;
            place[j] = 0xffffffffu; // after every entry of the same key
        }
        if (tid == 0)
            entries = 0;
        // Each wave's run of the row, in order: its values equal to t, then all entries.
        const uint32_t vecs = (n + N - 1) / N, run = (vecs + W - 1) / W;
        const uint32_t first = wave * run, last = first + run < vecs ? first + run : vecs;
        uint32_t ties = 0;
        wave_run(s, n, first, last, [&](const T *v, uint32_t, uint32_t count) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                ties += i < count && key_of(v[i]) == top.t;
            return false;
        });
        ties = wave_reduce(ties, OpSum());
        if (lane == 0)
            wave_ties[wave] = ties;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t w = 0; w < wave; w++)
            before += wave_ties[w];
        wave_run(s, n, first, last, [&](const T *v, uint32_t at, uint32_t count) {
            uint32_t own = 0;
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                own += i < count && key_of(v[i]) == top.t;
            const uint32_t upto = wave_inclusive_sum(own);
            uint32_t rank = before + upto - own;
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                const K x = key_of(v[i]);
                if (i < count && (x > top.t || (x == top.t && rank < top.c))) {
                    const uint32_t j = atomicAdd(&entries, 1u);
                    key[j] = x;
                    place[j] = at + i;
                }
                rank += i < count && x == top.t;
            }
            before += __shfl(upto, 63, 64);
            return false;
        });
        sort_entries<NT>(key, place, size);
    }
    S *values = static_cast<S *>(g.values) + row * g.k;
    int32_t *indices = g.indices + row * g.k;
    for (uint32_t j = tid; j < g.k; j += NT) {
        values[j] = j < k ? s[place[j]] : (S)-INFINITY;
        indices[j] = j < k ? (int32_t)place[j] : -1;
    }
}

template <typename S> hipError_t launch_t(hipStream_t s, const TopArgs &g)
{
    if (g.vocab <= 8192)
        hipLaunchKernelGGL((k_top<S, 256>), dim3((unsigned)g.rows), dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((k_top<S, 1024>), dim3((unsigned)g.rows), dim3(1024), 0, s, g);
    return hipGetLastError();
}

} // namespace

hipError_t launch_top(hipStream_t s, const TopArgs &g)
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
