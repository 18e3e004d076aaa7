// Distillation from a teacher's top logits, forward and backward.
//
// Row of V student logits s, k teacher entries (v_j, i_j), temperature T, weights a and b:
//   q_j  = exp(v_j / T - L), L the teacher's log-sum-exp of the whole row if it is given, else
//          that of the row's own entries;   Q = sum q_j
//   p    = softmax(s / T), p1 = softmax(s)
//   loss = a T^2 sum_j q_j (log q_j - log p[i_j])  +  b (-log p1[y])
//   ds_v = scale (a T (Q p_v - sum over i_j = v of q_j)  +  b (p1_v - [v = y]))
// The b terms are there only for rows with a label y >= 0; entries with a negative index are
// absent. A row without entries and label has loss 0 and gradient 0 whatever it holds.
//
// The gradient is dense (Q p_v everywhere) with at most k + 1 places that differ: each
// workgroup writes its dense part, and after a barrier overwrites those places with the full
// value, computed anew by the lane that owns the place's first entry, so that no atomics and no
// order are involved and duplicate indices add up.
//
// What bounds it: one read of the logits and one write of the gradient. 4096 x 128000 bf16, loss and
// gradient, takes 499 us of kernel (4.2 TB/s; a copy reaches 4.9), 1025 x 50257 f16, the gradient
// alone, 47 us (4.4 TB/s), the loss alone of 512 x 32000 f32 19 us (3.4 TB/s); a few short rows
// are a chain of loads, reductions and the program's end (64 x 1000 f64: 13 us). Medians of 32 calls.
#include "pcu_kernels.hpp"
#include "pcu_logits.hpp"

#include <type_traits>

#pragma clang fp contract(off)

namespace pcu {

namespace {

// exp(s / T - L) from a given log-sum-exp.
__device__ __forceinline__ float share(float s, float inv_t, float l) { return exp2_fast(__fmaf_rn(s, inv_t, -l) * kLog2e); }
__device__ __forceinline__ double share(double s, double inv_t, double l) { return exp(s * inv_t - l); }

template <typename T> __device__ __forceinline__ T widen_teacher(const void *values, int dtype, uint64_t i)
{
    switch (dtype) {
    case kLogitF32: return (T) static_cast<const float *>(values)[i];
    case kLogitF64: return (T) static_cast<const double *>(values)[i];
    case kLogitBf16: return (T)(float)static_cast<const __bf16 *>(values)[i];
    default: return (T)(float)static_cast<const _Float16 *>(values)[i];
    }
}

// A row's teacher entries in LDS (k places, then one for the label): the index (-1 when
// absent), q, log q and the student's logit there (kept, since the gradient may overwrite it).
template <typename T> struct Entries {
    T *q, *log_q, *s;
    int *at;
    T sum;     // Q
    int label; // -1: none
    static size_t bytes(uint32_t k) { return (k + 1) * (3 * sizeof(T) + 4); }
    __device__ __forceinline__ Entries(void *lds, uint32_t k)
        : q(static_cast<T *>(lds)), log_q(q + (k + 1)), s(log_q + (k + 1)),
          at(reinterpret_cast<int *>(s + (k + 1))), sum(0), label(-1)
    {
    }
};

// What load_entries takes from global memory first: this thread's first entry and the label. Loaded
// ahead of the row's vectors, since loads come back in order.
template <typename T> struct FirstEntry {
    int at = -1, label = -1;
    T v = 0, log_sum = 0;
    __device__ __forceinline__ FirstEntry(const DistillArgs &g, uint64_t row)
    {
        if (threadIdx.x < g.k) {
            at = g.teacher_indices[row * g.k + threadIdx.x];
            v = widen_teacher<T>(g.teacher_values, g.teacher_dtype, row * g.k + threadIdx.x);
        }
        if (g.labels)
            label = g.labels[row];
        if (g.teacher_log_sum)
            log_sum = g.teacher_log_sum_f64 ? (T) static_cast<const double *>(g.teacher_log_sum)[row]
                                            : (T) static_cast<const float *>(g.teacher_log_sum)[row];
    }
};

// Normalises the row's entries. `red`: 2 x 16 places.
template <int NT, typename T>
__device__ __forceinline__ void load_entries(const DistillArgs &g, uint64_t row, const FirstEntry<T> &ahead, Entries<T> &e, T *red)
{
    const uint32_t tid = threadIdx.x;
    uint64_t bad = kNoFault;
    const T t = (T)g.temperature;
    T top = -INFINITY;
    for (uint32_t j = tid; j < g.k; j += NT) {
        int at = j == tid ? ahead.at : g.teacher_indices[row * g.k + j];
        T z = (j == tid ? ahead.v : widen_teacher<T>(g.teacher_values, g.teacher_dtype, row * g.k + j)) / t;
        if (at >= (int64_t)g.vocab) {
            bad = pack_fault(row * (g.k + 1) + j, kInvalid) < bad ? pack_fault(row * (g.k + 1) + j, kInvalid) : bad;
            at = -1;
        }
        if (at < 0) {
            at = -1;
            z = -INFINITY;
        }
        e.at[j] = at;
        e.log_q[j] = z;
        top = OpMax()(top, z);
    }
    int y = ahead.label;
    if (y >= (int64_t)g.vocab) {
        if (tid == 0) {
            const uint64_t f = pack_fault(row * (g.k + 1) + g.k, kInvalid);
            bad = f < bad ? f : bad;
        }
        y = -1;
    }
    e.label = y < 0 ? -1 : y;
    wave_record_fault(bad, g.fault, g.gate);
    T log_sum;
    if (g.teacher_log_sum) {
        log_sum = ahead.log_sum;
    } else {
        top = block_reduce<NT>(top, OpMax(), red);
        T sum = 0;
        for (uint32_t j = tid; j < g.k; j += NT) {
            const T z = e.log_q[j];
            sum += z == -INFINITY ? (T)0 : exp(z - top);
        }
        sum = block_reduce<NT>(sum, OpSum(), red + 16);
        log_sum = top + log(sum);
        if constexpr (NT > 64)
            __syncthreads(); // red is used again below
    }
    T sum = 0;
    for (uint32_t j = tid; j < g.k; j += NT) {
        const T z = e.log_q[j];
        const T lq = z - log_sum;
        const T q = z == -INFINITY ? (T)0 : exp(lq);
        e.q[j] = q;
        e.log_q[j] = lq;
        sum += q;
    }
    if (tid == 0) {
        e.q[g.k] = 0;
        e.at[g.k] = e.label;
    }
    e.sum = block_reduce<NT>(sum, OpSum(), red);
    if constexpr (NT == 64)
        __syncthreads();
}

// Reads the student's logits at the entries' places of [c0, c1), for the two functions below;
// each lane reads and later uses its own places only.
template <int NT, typename S, typename T>
__device__ __forceinline__ void gather_entries(const DistillArgs &g, const S *s, Entries<T> &e, uint32_t c0, uint32_t c1)
{
    for (uint32_t j = threadIdx.x; j <= g.k; j += NT) {
        const int at = e.at[j];
        if (at >= (int)c0 && at < (int)c1)
            e.s[j] = (T)s[at];
    }
}

// The row's loss from the two log-sum-exps, on every thread. `red`: 2 x 16 places.
template <int NT, typename T>
__device__ __forceinline__ T row_loss(const DistillArgs &g, const Entries<T> &e, T lse, T lse1, T *red)
{
    T part = 0, hard = 0;
    const T t = (T)g.temperature;
    for (uint32_t j = threadIdx.x; j <= g.k; j += NT) {
        if (e.at[j] < 0)
            continue;
        const T v = e.s[j];
        // log p of a masked logit is minus infinity also where all are masked (not the difference of
        // two infinities), but NaN in a row that has no log-sum-exp.
        if (j == g.k) {
            hard = v == -INFINITY && lse1 == lse1 ? (T)INFINITY : lse1 - v;
        } else if (!(e.q[j] == 0)) {
            const T log_p = v == -INFINITY && lse == lse ? v : v / t - lse;
            part += e.q[j] * (e.log_q[j] - log_p);
        }
    }
    part = block_reduce<NT>(part, OpSum(), red);
    hard = block_reduce<NT>(hard, OpSum(), red + 16);
    T loss = 0;
    // In binary64: the square of a temperature leaves binary32's range before the loss does.
    if (g.distill_weight != 0 && !(e.sum == 0))
        loss += (T)(g.distill_weight * ((double)t * t) * part);
    if (g.label_weight != 0 && e.label >= 0)
        loss += (T)g.label_weight * hard;
    return loss;
}

// The places of [c0, c1) whose gradient differs from the dense part: `dense(v)` gives the dense
// gradient of a logit.
template <int NT, typename S, typename T, typename Dense>
__device__ __forceinline__ void fix_entries(const DistillArgs &g, S *grad, const Entries<T> &e, uint32_t c0,
                                            uint32_t c1, T scale, Dense dense)
{
    const T per_q = scale * (T)g.distill_weight * (T)g.temperature;
    const T per_label = scale * (T)g.label_weight;
    for (uint32_t j = threadIdx.x; j <= g.k; j += NT) {
        const int at = e.at[j];
        if (at < (int)c0 || at >= (int)c1)
            continue;
        bool first = true;
        T less = 0;
        for (uint32_t i = 0; i < g.k; i++)
            if (e.at[i] == at) {
                first = first && i >= j;
                less += e.q[i];
            }
        if (!first)
            continue;
        T value = dense(e.s[j]);
        if (per_q != 0)
            value -= less * per_q;
        if (at == e.label)
            value -= per_label;
        put(grad + at, (S)value);
    }
}

// ---------------------------------------------------- one workgroup a row, the row in registers
//
// Forward, or forward and backward, for rows of at most NT * R whole vectors (the values after
// the last whole one lie one a lane in the first wave): each thread keeps R vectors of the row,
// so that the row is read once and its gradient written once. The sums are made as the vectors
// arrive, since nothing else fills that time where one row takes a CU's registers.
// Rows of up to so many vectors end the program of a call of their own in its kernel, their gradient
// stored through the caches (64 x 1000 f64: 20.5 us a call, 21.2 with a launch for it).
constexpr uint32_t kCloseVecs = 1024;

template <typename S, int NT, int R, bool GRAD> __device__ __forceinline__ void distill_row(const DistillArgs &g)
{
    using T = typename StatOf<S>::T;
    constexpr int N = kVec<S>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ T red[7][16];
    const uint32_t tid = threadIdx.x;
    const uint64_t row = row_of_block();
    if (row >= g.rows)
        return;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t whole = g.vocab / N, rest = whole * N + tid;
    const bool has_rest = rest < g.vocab; // at most N - 1 lanes

    const FirstEntry<T> ahead(g, row);
    u32x4 raw[R];
#pragma unroll
    for (int r = 0; r < R; r++)
        raw[r] = tid + r * NT < whole ? load_held(s, r * NT, tid) : minus_infinities<S>();
    const T extra = has_rest ? (T)s[rest] : (T)-INFINITY;

    if (block_gate_closed(g.gate)) // after the loads: they need not wait for it
        return;

    Entries<T> e(lds, g.k);
    load_entries<NT>(g, row, ahead, e, red[0]);

    // Each thread's maximum and sums over the vectors as they arrive, two at a time, the sums
    // rescaled when the maximum rises.
    const T inv_t = (T)1 / (T)g.temperature;
    const bool two = g.temperature != 1.0 && (g.log_sums_out != nullptr || e.label >= 0);
    T m = extra, sum = Expo<T>(m, inv_t)(extra), sum1 = two ? Expo<T>(m, (T)1)(extra) : (T)0;
    auto add_up = [&](auto both) {
        const Pass pass = Pass::fresh();
#pragma unroll
        for (int r = 0; r < R; r += 2) {
            T v[2 * N];
            unpack<S>(raw[r], v, pass);
            unpack<S>(raw[r + 1], v + N, pass);
            T top = m;
#pragma unroll
            for (int i = 0; i < 2 * N; i++)
                top = OpMax()(top, v[i]);
            const Expo<T> ex(top, inv_t), ex1(top, (T)1);
            sum *= m == -INFINITY ? (T)1 : ex(m); // 0, or NaN, while there is no maximum
            if (both)
                sum1 *= m == -INFINITY ? (T)1 : ex1(m);
#pragma unroll
            for (int i = 0; i < 2 * N; i++) {
                sum += ex(v[i]);
                if (both)
                    sum1 += ex1(v[i]);
            }
            m = top;
            one_at_a_time();
        }
    };
    if (two)
        add_up(std::true_type());
    else
        add_up(std::false_type());
    const T own = m;
    m = block_reduce<NT>(m, OpMax(), red[2]);
    const Expo<T> ex(m, inv_t), ex1(m, (T)1);
    sum *= own == -INFINITY ? (T)1 : ex(own); // without a maximum the sum is 0, or NaN
    sum = block_reduce<NT>(sum, OpSum(), red[3]);
    if (two) {
        sum1 *= own == -INFINITY ? (T)1 : ex1(own);
        sum1 = block_reduce<NT>(sum1, OpSum(), red[4]);
    } else {
        sum1 = sum;
    }
    const T lse = ex.log_sum(sum), lse1 = two ? ex1.log_sum(sum1) : lse;
    if (tid == 0 && g.log_sums_out) {
        put(static_cast<T *>(g.log_sums_out) + 2 * row, lse);
        put(static_cast<T *>(g.log_sums_out) + 2 * row + 1, lse1);
    }
    gather_entries<NT>(g, s, e, 0u, g.vocab);
    if (g.loss) {
        const T loss = row_loss<NT>(g, e, lse, lse1, red[5]);
        if (tid == 0)
            put(static_cast<T *>(g.loss) + row, loss);
    }
    if constexpr (GRAD) {
        const T scale = g.row_scale ? static_cast<const T *>(g.row_scale)[row] : (T)1;
        T cq = scale * (T)g.distill_weight * (T)g.temperature * e.sum;
        T cl = e.label >= 0 ? scale * (T)g.label_weight : (T)0;
        if (!two) {
            cq += cl;
            cl = 0;
        }
        // Rows whose logits are all minus infinity have no probabilities.
        const T pq = cq == 0 || sum == 0 ? (T)0 : cq / sum, pl = cl == 0 || sum1 == 0 ? (T)0 : cl / sum1;
        S *grad = static_cast<S *>(g.grad) + row * g.grad_stride;
        __syncthreads(); // the entries' logits are read: the gradient may lie in the row's place
        const Pass pass = Pass::fresh();
        // The dense part; `value` gives it for one logit.
        auto write = [&](auto value) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                T v[N];
                unpack<S>(raw[r], v, pass);
#pragma unroll
                for (int i = 0; i < N; i++)
                    v[i] = value(v[i]);
                if (tid + r * NT < whole)
                    store_held<NT * R <= kCloseVecs>(grad, r * NT, tid, pack<S>(v), g.store);
                one_at_a_time();
            }
            if (has_rest)
                put(grad + rest, (S)value(extra));
            __syncthreads();
            fix_entries<NT>(g, grad, e, 0u, g.vocab, scale, value);
        };
        for (uint32_t i = g.vocab + tid; i < g.grad_cols; i += NT)
            put(grad + i, (S)0);
        const Expo<T> fq = ex.fresh(), fl = ex1.fresh(), one = pq != 0 ? fq : fl;
        const T p1 = pq != 0 ? pq : pl;
        if (p1 == 0) // nothing asks for the row (or it has no probabilities)
            write([](T) { return (T)0; });
        else if (pq == 0 || pl == 0)
            write([&](T v) { return one(v) * p1; });
        else
            write([&](T v) { return fq(v) * pq + fl(v) * pl; });
    }
}

// A call of its own ends its program in this kernel (close).
template <typename S, int NT, int R, bool GRAD>
__global__ __launch_bounds__(NT) void k_distill_row(DistillArgs g, ProgramClose close)
{
    distill_row<S, NT, R, GRAD>(g);
    program_close_block(close);
}

// ----------------------------------------------------------- a row split over workgroups
//
// Rows that no workgroup holds, and few rows of a long vocabulary: the statistics of chunks of
// a row, with the logits at the entries; then per chunk the row's two log-sum-exps from all its
// chunks and the gradient, the loss with the first (or, for the loss alone, one workgroup a row).
// 16 x 200001 f32: 6 + 13 us of kernels, the second's reads out of the caches, 29.3 us a call; with a
// launch of its own between them for the loss and the log-sum-exps 32.6.
template <typename T> struct Partial {
    T m, sum, sum1;
};

template <typename S, int NT>
__global__ __launch_bounds__(NT) void k_distill_stats(DistillArgs g, uint32_t chunks, uint32_t chunk_vecs,
                                                      Partial<typename StatOf<S>::T> *parts, typename StatOf<S>::T *picked)
{
    using T = typename StatOf<S>::T;
    constexpr int N = kVec<S>;
    constexpr int U = 4; // vectors in flight a thread
    if (block_gate_closed(g.gate))
        return;
    __shared__ T red[3][16];
    const uint64_t row = blockIdx.x / chunks;
    const uint32_t chunk = blockIdx.x % chunks;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    const uint32_t first = chunk * chunk_vecs, last = first + chunk_vecs;
    const T inv_t = (T)1 / (T)g.temperature;
    const bool two = g.temperature != 1.0;

    if (picked) { // what the loss needs, before a gradient in place overwrites it
        const uint32_t c0 = first * N, c1 = last * N < g.vocab ? last * N : g.vocab;
        for (uint32_t j = threadIdx.x; j <= g.k; j += NT) {
            const int at = j < g.k ? g.teacher_indices[row * g.k + j] : (g.labels ? g.labels[row] : -1);
            if (at >= (int)c0 && at < (int)c1)
                picked[row * (g.k + 1) + j] = (T)s[at];
        }
    }
    // Each thread's running maximum and sums, rescaled when a piece raises the maximum.
    T m = -INFINITY, sum = 0, sum1 = 0;
    for (uint32_t i = first + threadIdx.x; i < last; i += NT * U) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            raw[u] = i + u * NT < last ? load_vec(s, i + u * NT, g.vocab) : minus_infinities<S>();
        T v[U * N], top = m;
#pragma unroll
        for (int u = 0; u < U; u++)
            unpack<S>(raw[u], v + u * N);
#pragma unroll
        for (int k = 0; k < U * N; k++)
            top = OpMax()(top, v[k]);
        const Expo<T> ex(top, inv_t), ex1(top, (T)1);
        if (top != m) {
            sum = m == -INFINITY ? sum : sum * ex(m);
            sum1 = m == -INFINITY ? sum1 : sum1 * ex1(m);
            m = top;
        }
#pragma unroll
        for (int k = 0; k < U * N; k++)
            sum += ex(v[k]);
        if (two) {
#pragma unroll
            for (int k = 0; k < U * N; k++)
                sum1 += ex1(v[k]);
        }
    }
    const T top = block_reduce<NT>(m, OpMax(), red[0]);
    if (m != top && m != -INFINITY) {
        sum *= Expo<T>(top, inv_t)(m);
        sum1 *= Expo<T>(top, (T)1)(m);
    }
    sum = block_reduce<NT>(sum, OpSum(), red[1]);
    sum1 = block_reduce<NT>(sum1, OpSum(), red[2]);
    if (threadIdx.x == 0)
        parts[blockIdx.x] = Partial<T>{top, sum, two ? sum1 : sum};
}

// The row's two log-sum-exps from its chunks'. `red`: 3 x 16 places.
template <typename T> struct LogSums {
    T lse, lse1;
};
template <int NT, typename T>
__device__ __forceinline__ LogSums<T> log_sums_of(const DistillArgs &g, uint64_t row, uint32_t chunks, const Partial<T> *parts, T *red)
{
    T m = -INFINITY;
    for (uint32_t c = threadIdx.x; c < chunks; c += NT)
        m = OpMax()(m, parts[row * chunks + c].m);
    m = block_reduce<NT>(m, OpMax(), red);
    const Expo<T> ex(m, (T)1 / (T)g.temperature), ex1(m, (T)1);
    T sum = 0, sum1 = 0;
    for (uint32_t c = threadIdx.x; c < chunks; c += NT) {
        const Partial<T> p = parts[row * chunks + c];
        // A chunk of minus infinities adds nothing; one with a NaN among them hands it on.
        sum += p.m == -INFINITY ? p.sum : p.sum * ex(p.m);
        sum1 += p.m == -INFINITY ? p.sum1 : p.sum1 * ex1(p.m);
    }
    sum = block_reduce<NT>(sum, OpSum(), red + 16);
    sum1 = block_reduce<NT>(sum1, OpSum(), red + 32);
    const T lse = ex.log_sum(sum);
    return {lse, g.temperature != 1.0 ? ex1.log_sum(sum1) : lse};
}

constexpr int kFinishThreads = 256;

template <typename S>
__global__ __launch_bounds__(kFinishThreads) void k_distill_finish(DistillArgs g, uint32_t chunks,
                                                                   const Partial<typename StatOf<S>::T> *parts)
{
    using T = typename StatOf<S>::T;
    constexpr int NT = kFinishThreads;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ T red[7][16];
    const uint64_t row = blockIdx.x;
    const FirstEntry<T> ahead(g, row);
    if (block_gate_closed(g.gate))
        return;
    const LogSums<T> sums = log_sums_of<NT>(g, row, chunks, parts, red[0]);
    if (threadIdx.x == 0 && g.log_sums_out) {
        static_cast<T *>(g.log_sums_out)[2 * row] = sums.lse;
        static_cast<T *>(g.log_sums_out)[2 * row + 1] = sums.lse1;
    }
    Entries<T> e(lds, g.k);
    load_entries<NT>(g, row, ahead, e, red[3]);
    gather_entries<NT>(g, static_cast<const S *>(g.logits) + row * g.stride, e, 0u, g.vocab);
    const T loss = row_loss<NT>(g, e, sums.lse, sums.lse1, red[5]);
    if (threadIdx.x == 0)
        static_cast<T *>(g.loss)[row] = loss;
}

// The gradient of one chunk of a row, from the row's given log-sum-exps or (parts) from its chunks',
// and then the loss with the first chunk.
template <typename S, int NT>
__global__ __launch_bounds__(NT) void k_distill_grad(DistillArgs g, uint32_t chunks, uint32_t chunk_vecs,
                                                     const Partial<typename StatOf<S>::T> *parts,
                                                     const typename StatOf<S>::T *picked)
{
    using T = typename StatOf<S>::T;
    constexpr int N = kVec<S>;
    constexpr int U = 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ T red[7][16];
    const uint32_t block = row_of_block(); // rows x chunks of them, below 2^31
    const uint64_t row = block / chunks;
    const uint32_t chunk = block % chunks;
    if (row >= g.rows)
        return;
    const S *s = static_cast<const S *>(g.logits) + row * g.stride;
    S *grad = static_cast<S *>(g.grad) + row * g.grad_stride;
    const uint32_t first = chunk * chunk_vecs, last = first + chunk_vecs;
    const uint32_t c0 = first * N, c1 = last * N < g.vocab ? last * N : g.vocab;

    const FirstEntry<T> ahead(g, row);
    u32x4 raw[U]; // the first vectors come while the entries are made ready
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t i = first + threadIdx.x + u * NT;
        raw[u] = i < last ? load_vec(s, i, g.vocab) : minus_infinities<S>();
    }
    if (block_gate_closed(g.gate))
        return;
    Entries<T> e(lds, g.k);
    load_entries<NT>(g, row, ahead, e, red[0]);
    T lse, lse1;
    if (parts) {
        const LogSums<T> sums = log_sums_of<NT>(g, row, chunks, parts, red[2]);
        lse = sums.lse;
        lse1 = sums.lse1;
        if (chunk == 0) {
            for (uint32_t j = threadIdx.x; j <= g.k; j += NT)
                e.s[j] = e.at[j] >= 0 ? picked[row * (g.k + 1) + j] : (T)0;
            const T loss = row_loss<NT>(g, e, lse, lse1, red[5]);
            if (threadIdx.x == 0)
                static_cast<T *>(g.loss)[row] = loss;
        }
    } else {
        lse = static_cast<const T *>(g.log_sums_in)[2 * row];
        lse1 = static_cast<const T *>(g.log_sums_in)[2 * row + 1];
    }
    gather_entries<NT>(g, s, e, c0, c1);
    const T scale = g.row_scale ? static_cast<const T *>(g.row_scale)[row] : (T)1;
    T pq = scale * (T)g.distill_weight * (T)g.temperature * e.sum;
    T pl = e.label >= 0 ? scale * (T)g.label_weight : (T)0;
    if (g.temperature == 1.0) {
        pq += pl;
        pl = 0;
    }
    if (lse == -INFINITY) // a row of minus infinities has no probabilities
        pq = 0;
    if (lse1 == -INFINITY)
        pl = 0;
    const T inv_t = (T)1 / (T)g.temperature;
    auto dense = [&](T v) {
        T out = pq == 0 ? (T)0 : share(v, inv_t, lse) * pq;
        if (pl != 0)
            out += share(v, (T)1, lse1) * pl;
        return out;
    };
    __syncthreads(); // the entries' logits are read: the gradient may lie in the row's place
    for (uint32_t i = first + threadIdx.x; i < last; i += NT * U) {
        u32x4 now[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            now[u] = raw[u];
            const uint32_t next = i + (U + u) * NT;
            raw[u] = next < last ? load_vec(s, next, g.vocab) : minus_infinities<S>();
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            T v[N];
            unpack<S>(now[u], v);
#pragma unroll
            for (int k = 0; k < N; k++)
                v[k] = dense(v[k]);
            if (i + u * NT < last)
                store_vec(grad, i + u * NT, g.vocab, v, g.store == kStorePast);
        }
    }
    if (chunk == chunks - 1)
        for (uint32_t i = g.vocab + threadIdx.x; i < g.grad_cols; i += NT)
            grad[i] = (S)0;
    __syncthreads();
    fix_entries<NT>(g, grad, e, c0, c1, scale, dense);
}

// ------------------------------------------------------------------------- launches

// A large gradient is stored past the caches: with the logits, and the output layer that both come from
// and go to, it would not stay in the chip's 256 MiB, and the logits' own reads come faster
// (4096 x 128000 bf16 533 -> 492 us a call, 1025 x 50257 f16, 103 MB, 69 -> 59 us). A smaller one
// is left where its reader finds it.
constexpr uint64_t kPastCaches = 64ull << 20;

struct Split {
    uint32_t chunks, vecs;
};
constexpr int kSplitThreads = 256;

Split split_of(uint64_t rows, uint32_t vecs)
{
    // Enough workgroups for the chip, each with at least 4 vectors a thread.
    const uint64_t want = (2048 + rows - 1) / rows;
    vecs = vecs ? vecs : 1; // a row without logits is one chunk
    const uint64_t most = (vecs + 4 * kSplitThreads - 1) / (4 * kSplitThreads);
    const uint64_t chunks = want < most ? want : most;
    const uint32_t each = (uint32_t)((vecs + chunks - 1) / chunks);
    return Split{(vecs + each - 1) / each, each};
}

template <typename S, int NT, int R> hipError_t launch_row(hipStream_t s, const DistillArgs &g, const ProgramClose &close)
{
    const size_t lds = Entries<typename StatOf<S>::T>::bytes(g.k);
    if (g.grad)
        hipLaunchKernelGGL((k_distill_row<S, NT, R, true>), row_grid(g.rows), dim3(NT), lds, s, g, close);
    else
        hipLaunchKernelGGL((k_distill_row<S, NT, R, false>), row_grid(g.rows), dim3(NT), lds, s, g, close);
    return hipGetLastError();
}

template <typename S>
hipError_t launch_grad(hipStream_t s, const DistillArgs &g, Split sp, const Partial<typename StatOf<S>::T> *parts,
                       const typename StatOf<S>::T *picked)
{
    const size_t lds = Entries<typename StatOf<S>::T>::bytes(g.k);
    hipLaunchKernelGGL((k_distill_grad<S, kSplitThreads>), row_grid(g.rows * sp.chunks), dim3(kSplitThreads),
                       lds, s, g, sp.chunks, sp.vecs, parts, picked);
    return hipGetLastError();
}

// Vectors of a row that one workgroup holds. Binary64 with 1024 threads would spill. Fewer than 64
// long rows leave CUs idle and are split (4 x 60000 f32 27 us a call and 30 held, 16 rows 28 and 31,
// 32 x 50257 28.5 and 30; 64 rows alike).
template <typename S> constexpr uint32_t kHeldVecs = (sizeof(S) == 8 ? 512 : 1024) * 16;

template <typename S> bool held(uint64_t rows, uint32_t vecs)
{
    return vecs <= kHeldVecs<S> && (rows >= 64 || vecs <= 1024);
}

// As few threads as hold the row: a row's reductions cost by the wave, and small workgroups share a
// CU, one's loads beside another's sums. Loss and gradient in microseconds a call, against the next form:
// 4096 x 1000 f32 28 with 64 x 4 and 44 with 256 x 4; 2048 x 32000 bf16 73 with 256 x 16, 96 with
// 512 x 16; 1024 x 32000 f32 63 with 512 x 16, 78 with 1024 x 16.
template <typename S> hipError_t launch_t(hipStream_t s, const DistillArgs &g, void *scratch, const ProgramClose &close)
{
    using T = typename StatOf<S>::T;
    const uint32_t vecs = (g.vocab + kVec<S> - 1) / kVec<S>;
    if (g.log_sums_in)
        return launch_grad<S>(s, g, split_of(g.rows, vecs), nullptr, nullptr);
    if (held<S>(g.rows, vecs)) {
        if (vecs <= 64 * 4)
            return launch_row<S, 64, 4>(s, g, close);
        if (vecs <= 256 * 4)
            return launch_row<S, 256, 4>(s, g, close);
        if (vecs <= 256 * 16)
            return launch_row<S, 256, 16>(s, g, close);
        if (vecs <= 512 * 16)
            return launch_row<S, 512, 16>(s, g, close);
        if constexpr (sizeof(S) < 8)
            return launch_row<S, 1024, 16>(s, g, close);
    }
    const Split sp = split_of(g.rows, vecs);
    Partial<T> *parts = static_cast<Partial<T> *>(scratch);
    T *picked = reinterpret_cast<T *>(parts + g.rows * sp.chunks);
    hipLaunchKernelGGL((k_distill_stats<S, kSplitThreads>), dim3((unsigned)(g.rows * sp.chunks)), dim3(kSplitThreads), 0,
                       s, g, sp.chunks, sp.vecs, parts, g.grad ? picked : nullptr);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return err;
    if (g.grad)
        return launch_grad<S>(s, g, sp, parts, picked);
    hipLaunchKernelGGL((k_distill_finish<S>), dim3((unsigned)g.rows), dim3(kFinishThreads), Entries<T>::bytes(g.k), s, g,
                       sp.chunks, parts);
    return hipGetLastError();
}

template <typename S> size_t scratch_t(const DistillArgs &g)
{
    using T = typename StatOf<S>::T;
    const uint32_t vecs = (g.vocab + kVec<S> - 1) / kVec<S>;
    if (g.rows == 0 || g.log_sums_in || held<S>(g.rows, vecs))
        return 0;
    return g.rows * (split_of(g.rows, vecs).chunks * sizeof(Partial<T>) + (g.grad ? g.k + 1 : 0) * sizeof(T));
}

} // namespace

size_t distill_scratch_bytes(const DistillArgs &g)
{
    switch (g.dtype) {
    case kLogitF32: return scratch_t<float>(g);
    case kLogitF64: return scratch_t<double>(g);
    case kLogitBf16: return scratch_t<__bf16>(g);
    default: return scratch_t<_Float16>(g);
    }
}

hipError_t launch_distill(hipStream_t s, DistillArgs g, void *scratch, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.rows == 0)
        return hipSuccess;
    const uint64_t size = g.dtype == kLogitF64 ? 8 : g.dtype == kLogitF32 ? 4 : 2;
    if (g.log_sums_in || g.rows > kCloseMaxBlocks || g.vocab > kCloseVecs * 16 / size)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    if (*closed)
        g.store = kStoreThrough;
    else if (g.grad && g.rows * g.grad_cols * size > kPastCaches)
        g.store = kStorePast;
    switch (g.dtype) {
    case kLogitF32: return launch_t<float>(s, g, scratch, close);
    case kLogitF64: return launch_t<double>(s, g, scratch, close);
    case kLogitBf16: return launch_t<__bf16>(s, g, scratch, close);
    default: return launch_t<_Float16>(s, g, scratch, close);
    }
}

} // namespace pcu
