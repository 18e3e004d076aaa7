// The k largest logits of each row, in order, with the row's log-sum-exp.
//
//   order: value descending, then index ascending (-0 equal to +0, NaN after minus infinity)
//   log_sum = log sum_v exp(l_v / T)
// One workgroup a row, the row in registers where it fits: one read, the maximum and the sum of
// exponentials, a bound from the maxima of groups of the row, the values that reach it gathered
// and sorted in LDS (see pcu_select.hpp).
//
// Many rows are bound by their one read: 2048 x 32000 bf16 with k = 64 takes 33.8 us of kernel, 3.9
// TB/s, where a copy reaches 4.9; 511 x 50257 f32 with k = 500 takes 41 us, 2.5 TB/s: a row
// takes a CU's registers whole, and its list and sort lie open behind its read. A few short rows are a
// chain of barriers: 64 x 1000 f32 with k = 8 takes 8.4 us, the end of the program among them. A row is one
// workgroup's however few there are (1 x 128000 bf16, k 50: 28 us a call; 64 x 131072 f32 46), and rows whose
// largest values lie side by side or are equal fill the list (2048 x 32000 bf16, k 64, sorted rows 307
// us a call, equal logits 990).
#include "pcu_kernels.hpp"
#include "pcu_select.hpp"

#pragma clang fp contract(off)

namespace pcu {

namespace {

// The list's place for a row whose values beyond the bound do not fit it: the prefix of k values
// found digit by digit, its entries gathered, those equal to t by index.
template <typename S, int NT, typename K, int CAP>
__device__ __forceinline__ void gather_exactly(const S *s, uint32_t n, uint32_t k, List<K, CAP> &list, uint32_t *bins,
                                               Digit<uint32_t> *digit, uint32_t *wave_ties)
{
    using T = typename StatOf<S>::T;
    constexpr uint32_t N = kVec<S>, W = NT / 64;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const Prefix<K> top = select_count<S, NT>(s, n, k, bins, digit);
    if (threadIdx.x == 0)
        list.count = 0;
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
            if (i < count && (x > top.t || (x == top.t && rank < top.c)))
                list.add(x, at + i);
            rank += i < count && x == top.t;
        }
        before += from_lane(upto, 63);
        return false;
    });
    __syncthreads();
}

// G groups a thread, each of one vector at least, so that a row has NT * G groups or as many as it has
// vectors. At least twice as many as k keep the list short. Short rows of 16-bit logits have fewer: the
// bound is low, or there is none where k is above the vectors, and a list that overflows is made
// digit by digit (2048 x 4000 bf16: k 200 61 us a call, k 300 52, k 600 100; 2048 x 8000: k 600 88, k 1000 198).
template <typename S, int NT, int R, int G, int CAP> __device__ __forceinline__ void top_row(const TopArgs &g)
{
    using T = typename StatOf<S>::T;
    using K = typename KeyOf<T>::K;
    constexpr uint32_t N = kVec<S>;
    __shared__ BoundScratch bound;
    __shared__ Digit<uint32_t> digit;
    __shared__ T red[4][16];
    __shared__ uint32_t wave_ties[16];
    __shared__ List<K, CAP> list;
    __shared__ SortShared<T> sort;
    const uint32_t tid = threadIdx.x;
    const uint64_t row = row_of_block();
    if (row >= g.rows)
        return;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t n = g.vocab, k = g.k < n ? g.k : n;
    const Row<S, NT, R> held(s, n);
    if (block_gate_closed(g.gate)) // after the loads: they need not wait for it
        return;

    T group[G], largest[R ? R : 1]; // of the groups, and of each held vector
#pragma unroll
    for (int i = 0; i < G; i++)
        group[i] = -INFINITY;
    group[0] = held.extra > -INFINITY ? held.extra : (T)-INFINITY;
    held.walk([&](const T *v, uint32_t, int step) {
        T top = v[0];
#pragma unroll
        for (uint32_t i = 1; i < N; i++)
            top = OpMax()(top, v[i]);
        if constexpr (R > 0)
            largest[step] = top;
        group[step % G] = OpMax()(group[step % G], top);
    });
    T m = group[0];
#pragma unroll
    for (int i = 1; i < G; i++)
        m = OpMax()(m, group[i]);
    m = block_reduce<NT>(m, OpMax(), red[0]);
    if (g.log_sum) {
        const Expo<T> ex(m, (T)1 / (T)g.temperature);
        T sum = ex(held.extra);
        held.walk([&](const T *v, uint32_t, int) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                sum += ex(v[i]);
        });
        sum = block_reduce<NT>(sum, OpSum(), red[1]);
        if (tid == 0)
            put(static_cast<T *>(g.log_sum) + row, ex.log_sum(sum));
    }
    if (k > 0) {
        if (tid == 0)
            list.count = 0;
        const uint32_t wanted[1] = {k};
        const T t = bounds_of<NT>(group, m, wanted, bound, red[2]).t[0]; // its barriers order the count
        if (R > 0 && t > -INFINITY)
            list.add_from(s, largest, t, [&](int r, auto f) { f(tid + (uint32_t)r * NT); });
        else
            held.walk([&](const T *v, uint32_t at, int) {
                if (at < held.whole * N) // a held vector past the row is all minus infinity
                    list.template add_of<N>(v, [&](T x, int) { return x >= t; }, [&](int i) { return at + i; });
            });
        if (held.has_extra && held.extra >= t)
            list.add(key_of(held.extra), held.extra_at());
        __syncthreads();
        list.template fill_keys<NT>(s);
        // Fewer than k: the rest of the row are NaNs.
        uint32_t found = list.count;
        __syncthreads();
        if (found > CAP || found < k) {
            gather_exactly<S, NT>(s, n, k, list, bound.bins, &digit, wave_ties);
            found = k;
        }
        sort_list<NT>(list, found, m, sort);
    }
    S *values = static_cast<S *>(g.values) + row * g.k;
    int32_t *indices = g.indices + row * g.k;
    for (uint32_t j = tid; j < g.k; j += NT) {
        put(values + j, j < k ? s[list.at[j]] : (S)-INFINITY);
        put(indices + j, j < k ? (int32_t)list.at[j] : -1);
    }
}

// A call of its own of at most kCloseMaxBlocks rows ends its program in this kernel (close) instead of
// a launch of 4 us; with every row's ticket on the one counter 2048 x 32000 bf16 took 106 us a call for
// 48.
template <typename S, int NT, int R, int G, int CAP>
__global__ __launch_bounds__(NT) void k_top(TopArgs g, ProgramClose close)
{
    top_row<S, NT, R, G, CAP>(g);
    program_close_block(close);
}

template <typename S, int NT, int R> hipError_t launch_row(hipStream_t s, const TopArgs &g, const ProgramClose &close)
{
    const dim3 grid = row_grid(g.rows), block(NT);
    if (g.k * 4 <= NT)
        hipLaunchKernelGGL((k_top<S, NT, R, 1, 512>), grid, block, 0, s, g, close);
    else
        hipLaunchKernelGGL((k_top<S, NT, R, 4, 2048>), grid, block, 0, s, g, close);
    return hipGetLastError();
}

// As few threads as hold the row, with at most 16 vectors each, since the reductions' and the list's
// barriers cost by the wave. Microseconds a call, against the next form:
//   256 x 4 to 256 x 16: 2048 x 4096 f32, k 16, 24.9 and 34
//   256 x 16 to 1024 x 4: 2048 x 32000 bf16, k 64, 57 and 62; k above 256 overflows the list too
//     often (512 x 16000 f32: k 300 30 with 1024 x 4 and 41, k 1000 47 and 149)
//   512 x 16 to 1024 x 16: 512 x 32000 f32, k 64, 29 and 50
//   1024 x 16 to a row read again for each walk: 511 x 50257 f32, k 500, 51 and 63. (Binary64 with
//     that many would spill.)
template <typename S> hipError_t launch_t(hipStream_t s, const TopArgs &g, const ProgramClose &close)
{
    const uint32_t vecs = g.vocab / kVec<S>;
    if (vecs <= 256 * 4)
        return launch_row<S, 256, 4>(s, g, close);
    if (vecs <= 256 * 16 && g.k <= 256)
        return launch_row<S, 256, 16>(s, g, close);
    if (vecs <= 1024 * 4)
        return launch_row<S, 1024, 4>(s, g, close);
    if (vecs <= 512 * 16)
        return launch_row<S, 512, 16>(s, g, close);
    if constexpr (sizeof(S) < 8)
        if (vecs <= 1024 * 16)
            return launch_row<S, 1024, 16>(s, g, close);
    return launch_row<S, 1024, 0>(s, g, close);
}

} // namespace

hipError_t launch_top(hipStream_t s, const TopArgs &g, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.rows == 0)
        return hipSuccess;
    if (g.rows > kCloseMaxBlocks)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    switch (g.dtype) {
    case kLogitF32: return launch_t<float>(s, g, close);
    case kLogitF64: return launch_t<double>(s, g, close);
    case kLogitBf16: return launch_t<__bf16>(s, g, close);
    default: return launch_t<_Float16>(s, g, close);
    }
}

} // namespace pcu
