// Layer norm's forward and backward pass.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), n = (x - m) r, y = n w + b
//   g = dy w, dx = r (g - mean g - n mean(g n)), dw = sum over rows of dy n, db = sum of dy
//
// Both directions are bound by HBM: a row is read once and held in registers while its sums are
// taken. The weight's gradients are sums down the columns: every workgroup adds up its rows in
// registers, and a second launch adds up the workgroups in their order.
#include "pcu_rows.hpp"

#pragma clang fp contract(off)

namespace pcu {
namespace {

// Sum over the 16 lanes of a DPP row, the same bits in each (the rotations pair the same values
// up whatever the lane).
template <typename T> __device__ __forceinline__ T sum16(T v)
{
    v = v + dpp<0x128, 0xf>((T)0, v); // row_ror:8
    v = v + dpp<0x124, 0xf>((T)0, v);
    v = v + dpp<0x122, 0xf>((T)0, v);
    return v + dpp<0x121, 0xf>((T)0, v);
}

// Sum over 32 lanes, the same bits in each.
template <typename T> __device__ __forceinline__ T sum32(T v)
{
    v = sum16(v);
    return v + __shfl_xor(v, 16);
}

// Sums of N values over a row's LANES lanes: 16, 32, 64 or whole waves of a workgroup of NT threads, a
// row's waves side by side. lds: N * NT / 64 entries that no other sum between two barriers uses.
template <int NT, int LANES, int N, typename T> __device__ __forceinline__ void row_sums(T (&v)[N], T *lds)
{
    if constexpr (LANES == 16) {
#pragma unroll
        for (int k = 0; k < N; k++)
            v[k] = sum16(v[k]);
    } else if constexpr (LANES == 32) {
#pragma unroll
        for (int k = 0; k < N; k++)
            v[k] = sum32(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            v[k] = wave_reduce(v[k], OpSum{});
        if constexpr (LANES > 64) {
            constexpr int W = LANES / 64;
            const int wave = threadIdx.x / 64, first = wave / W * W;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int k = 0; k < N; k++)
                    lds[k * (NT / 64) + wave] = v[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; k++) {
                v[k] = lds[k * (NT / 64) + first];
#pragma unroll
                for (int w = 1; w < W; w++)
                    v[k] += lds[k * (NT / 64) + first + w];
            }
        }
    }
}

// kVec<S> weights from vector i on, in the statistics' type.
template <typename S, typename W>
__device__ __forceinline__ void load_weights(const W *w, uint32_t i, uint32_t n, typename StatOf<S>::T (&out)[kVec<S>])
{
    if constexpr (sizeof(W) == sizeof(S)) {
        unpack<W>(load_piece(w, i, n), out);
    } else {
        unpack<W>(load_piece(w, 2 * i, n), out);
        unpack<W>(load_piece(w, 2 * i + 1, n), out + 4);
    }
}

template <typename T> __device__ __forceinline__ T rsqrt_of(T v);
template <> __device__ __forceinline__ float rsqrt_of(float v) { return 1.0f / sqrtf(v); }
template <> __device__ __forceinline__ double rsqrt_of(double v) { return 1.0 / sqrt(v); }

template <typename S>
__device__ __forceinline__ void store_norm(S *row, uint32_t i, uint32_t n, const typename StatOf<S>::T *v, bool through)
{
    if (!through || (i + 1) * kVec<S> > n) {
        if (!through) {
            store_vec(row, i, n, v, false);
        } else {
#pragma unroll
            for (int e = 0; e < kVec<S>; e++)
                if (i * kVec<S> + e < n)
                    put(row + i * kVec<S> + e, (S)v[e]);
        }
    } else {
        put_vec(row + i * kVec<S>, pack<S>(v));
    }
}

// Rows of up to LANES * R vectors, held; R = 0: rows of any length, read three times by LANES = NT.
template <typename S, typename W, int NT, int LANES, int R>
__global__ __launch_bounds__(NT) void k_norm(NormArgs g, ProgramClose close)
{
    using T = typename StatOf<S>::T;
    __shared__ T lds[2][NT / 64];
    if (block_gate_closed(g.gate))
        return;
    const uint64_t r = (uint64_t)row_of_block() * (NT / LANES) + threadIdx.x / LANES;
    const bool on = r < g.rows, through = close.words != nullptr;
    const uint32_t lane = threadIdx.x % LANES, n = g.width, vecs = (n + kVec<S> - 1) / kVec<S>;
    const S *x = static_cast<const S *>(g.x) + r * g.stride;
    S *y = static_cast<S *>(g.out) + r * g.out_stride;
    const W *w = static_cast<const W *>(g.weight), *b = static_cast<const W *>(g.bias);
    // One pass of f(vector, values, how many of them are the row's).
    u32x4 held[R ? R : 1];
    auto walk = [&](auto f) {
        if constexpr (R > 0) {
#pragma unroll
            for (int q = 0; q < R; q++) {
                const uint32_t i = q * LANES + lane;
                if (on && i < vecs) {
                    T v[kVec<S>];
                    unpack<S>(held[q], v, Pass::fresh());
                    f(i, v, min(n - i * kVec<S>, (uint32_t)kVec<S>));
                }
            }
        } else {
            for (uint32_t i = lane; on && i < vecs; i += LANES) {
                T v[kVec<S>];
                unpack<S>(load_piece(x, i, n), v);
                f(i, v, min(n - i * kVec<S>, (uint32_t)kVec<S>));
            }
        }
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int q = 0; q < R; q++)
            if (on && q * LANES + lane < vecs)
                held[q] = load_piece(x, q * LANES + lane, n);
    }
    T sum[1] = {0};
    walk([&](uint32_t, const T *v, uint32_t m) {
        T t = 0;
#pragma unroll
        for (int e = 0; e < kVec<S>; e++)
            t += (uint32_t)e < m ? v[e] : (T)0;
        sum[0] += t;
    });
    row_sums<NT, LANES, 1>(sum, lds[0]);
    const T mean = sum[0] / (T)n;
    T square[1] = {0};
    walk([&](uint32_t, const T *v, uint32_t m) {
        T t = 0;
#pragma unroll
        for (int e = 0; e < kVec<S>; e++) {
            const T d = (uint32_t)e < m ? v[e] - mean : (T)0;
            t += d * d;
        }
        square[0] += t;
    });
    row_sums<NT, LANES, 1>(square, lds[1]);
    const T rstd = rsqrt_of(square[0] / (T)n + (T)g.eps);
    walk([&](uint32_t i, T *v, uint32_t) {
        T ws[kVec<S>], bs[kVec<S>];
        if (w)
            load_weights<S, W>(w, i, n, ws);
        if (b)
            load_weights<S, W>(b, i, n, bs);
#pragma unroll
        for (int e = 0; e < kVec<S>; e++) {
            v[e] = (v[e] - mean) * rstd;
            if (w)
                v[e] *= ws[e];
            if (b)
                v[e] += bs[e];
        }
        store_norm(y, i, n, v, through);
    });
    if (on && lane == 0 && g.stats) {
        T *s = static_cast<T *>(g.stats) + 2 * r;
        if (through) {
            put(s, mean);
            put(s + 1, rstd);
        } else {
            s[0] = mean;
            s[1] = rstd;
        }
    }
    program_close_block(close);
}

template <typename S, typename W, int NT, int LANES, int R>
hipError_t launch_norm_rows(hipStream_t s, const NormArgs &g, ProgramClose close, bool *closed)
{
    const uint64_t blocks = (g.rows + NT / LANES - 1) / (NT / LANES);
    if (blocks > kCloseMaxBlocks)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    hipLaunchKernelGGL((k_norm<S, W, NT, LANES, R>), row_grid(blocks), dim3(NT), 0, s, g, close);
    return hipGetLastError();
}

template <typename S, typename W> hipError_t launch_norm_t(hipStream_t s, const NormArgs &g, ProgramClose close, bool *closed)
{
    const uint32_t vecs = (g.width + kVec<S> - 1) / kVec<S>;
    if (vecs <= 16)
        return launch_norm_rows<S, W, 256, 16, 1>(s, g, close, closed);
    if (vecs <= 32)
        return launch_norm_rows<S, W, 256, 32, 1>(s, g, close, closed);
    if (vecs <= 64)
        return launch_norm_rows<S, W, 256, 64, 1>(s, g, close, closed);
    if (vecs <= 256)
        return launch_norm_rows<S, W, 256, 64, 4>(s, g, close, closed);
    if (vecs <= 1024)
        return launch_norm_rows<S, W, 256, 256, 4>(s, g, close, closed);
    if (vecs <= 4096)
        return launch_norm_rows<S, W, 1024, 1024, 4>(s, g, close, closed);
    return launch_norm_rows<S, W, 1024, 1024, 0>(s, g, close, closed);
}

// ------------------------------------------------------------------- backward
// Workgroups of NT threads, LANES a row, R vectors a lane: each takes the rows from its own on by
// the grid's step, the next one's loads under way while this one is worked on, and leaves its sums
// down the columns at part[workgroup][2][vecs * kVec].
template <typename S, typename W, int NT, int LANES, int R, bool SUMS>
__global__ __launch_bounds__(NT) void k_norm_back(NormBackArgs g, void *parts)
{
    using T = typename StatOf<S>::T;
    constexpr int G = NT / LANES, V = kVec<S>;
    extern __shared__ __align__(16) char dyn[]; // the groups' sums at the end
    __shared__ T lds[2 * NT / 64];
    if (block_gate_closed(g.gate))
        return;
    const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES, n = g.width, vecs = (n + V - 1) / V;
    const W *w = static_cast<const W *>(g.weight);
    const T inv_n = (T)1 / (T)n;
    u32x4 x[R], dy[R];
    T st[2];
    auto fetch = [&](uint64_t r) {
        const S *xr = static_cast<const S *>(g.x) + r * g.stride;
        const S *dr = static_cast<const S *>(g.gradient) + r * g.gradient_stride;
#pragma unroll
        for (int q = 0; q < R; q++)
            if (q * LANES + lane < vecs) {
                x[q] = load_piece(xr, q * LANES + lane, n);
                dy[q] = load_piece(dr, q * LANES + lane, n);
            }
        const T *s = static_cast<const T *>(g.stats) + 2 * r;
        st[0] = s[0];
        st[1] = s[1];
    };
    T dw[SUMS ? R : 1][V] = {}, db[SUMS ? R : 1][V] = {};
    const uint64_t step = (uint64_t)gridDim.x * G;
    uint64_t r = (uint64_t)blockIdx.x * G + group;
    if (r < g.rows)
        fetch(r);
    for (uint64_t r0 = (uint64_t)blockIdx.x * G; r0 < g.rows; r0 += step, r += step) {
        const bool on = r < g.rows;
        T xs[R][V], gs[R][V];
        T sum[2] = {0, 0};
        const T mean = st[0], rstd = st[1];
        if (on) {
#pragma unroll
            for (int q = 0; q < R; q++) {
                const uint32_t i = q * LANES + lane;
                if (i >= vecs)
                    continue;
                T ws[V];
                unpack<S>(x[q], xs[q]);
                unpack<S>(dy[q], gs[q]);
                if (w)
                    load_weights<S, W>(w, i, n, ws);
                T s0 = 0, s1 = 0;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const bool in = i * V + e < n;
                    xs[q][e] = in ? (xs[q][e] - mean) * rstd : (T)0;
                    gs[q][e] = in ? gs[q][e] : (T)0;
                    if constexpr (SUMS) {
                        dw[q][e] += gs[q][e] * xs[q][e];
                        db[q][e] += gs[q][e];
                    }
                    if (w)
                        gs[q][e] = in ? gs[q][e] * ws[e] : (T)0;
                    s0 += gs[q][e];
                    s1 += gs[q][e] * xs[q][e];
                }
                sum[0] += s0;
                sum[1] += s1;
            }
        }
        if (r + step < g.rows)
            fetch(r + step);
        if (g.x_gradient) {
            row_sums<NT, LANES, 2>(sum, lds);
            const T c0 = sum[0] * inv_n, c1 = sum[1] * inv_n;
            if (on) {
                S *out = static_cast<S *>(g.x_gradient) + r * g.x_gradient_stride;
#pragma unroll
                for (int q = 0; q < R; q++) {
                    const uint32_t i = q * LANES + lane;
                    if (i >= vecs)
                        continue;
#pragma unroll
                    for (int e = 0; e < V; e++)
                        xs[q][e] = rstd * (gs[q][e] - c0 - xs[q][e] * c1);
                    store_vec(out, i, n, xs[q], false);
                }
            }
            if constexpr (LANES > 64)
                __syncthreads(); // the sums' words are free again
        }
    }
    if constexpr (SUMS) {
        T *part = static_cast<T *>(parts) + (uint64_t)blockIdx.x * 2 * vecs * V;
        T *all = reinterpret_cast<T *>(dyn);
        if constexpr (LANES <= 64 && R == 1) {
            // The sums of a wave's groups by exchange, then those of the waves, all in LDS at once (33322 rows of
            // 113 binary32 values: one group after another 27.8 us, so 16.6).
#pragma unroll
            for (int o = 0; o < 2; o++) {
                T(&d)[V] = o ? db[0] : dw[0];
#pragma unroll
                for (int far = LANES; far < 64; far *= 2)
#pragma unroll
                    for (int e = 0; e < V; e++)
                        d[e] += __shfl_xor(d[e], far);
                if (o)
                    __syncthreads();
                if ((threadIdx.x & 63) < LANES && lane < vecs)
#pragma unroll
                    for (int e = 0; e < V; e++)
                        all[(threadIdx.x / 64 * vecs + lane) * V + e] = d[e];
                __syncthreads();
                for (uint32_t i = threadIdx.x; i < vecs * V; i += NT) {
                    T sum = all[i];
#pragma unroll
                    for (int k = 1; k < NT / 64; k++)
                        sum += all[k * vecs * V + i];
                    part[o * vecs * V + i] = sum;
                }
            }
        } else {
            // The groups' sums, one group after another.
            for (int k = 0; k < G; k++) {
                if ((int)group == k)
#pragma unroll
                    for (int q = 0; q < R; q++) {
                        const uint32_t i = q * LANES + lane;
                        if (i >= vecs)
                            continue;
#pragma unroll
                        for (int e = 0; e < V; e++) {
                            T *a = all + i * V + e, *c = a + vecs * V;
                            if (G == 1) {
                                part[i * V + e] = dw[q][e];
                                part[vecs * V + i * V + e] = db[q][e];
                            } else {
                                *a = k ? *a + dw[q][e] : dw[q][e];
                                *c = k ? *c + db[q][e] : db[q][e];
                            }
                        }
                    }
                if (G > 1)
                    __syncthreads();
            }
            if (G > 1)
                for (uint32_t i = threadIdx.x; i < 2 * vecs * V; i += NT)
                    part[i] = all[i];
        }
    }
}

// Rows too long to hold: for dx the two sums of each row first (one workgroup a row), then dx and (SUMS) the
// columns' sums by pieces of 1024 vectors and runs of rows.
template <typename S, typename W> __global__ __launch_bounds__(1024) void k_norm_back_sums(NormBackArgs g, void *sums)
{
    using T = typename StatOf<S>::T;
    constexpr int V = kVec<S>;
    __shared__ T lds[2 * 16];
    if (block_gate_closed(g.gate))
        return;
    const uint64_t r = row_of_block();
    if (r >= g.rows)
        return;
    const uint32_t n = g.width, vecs = (n + V - 1) / V;
    const S *xr = static_cast<const S *>(g.x) + r * g.stride, *dr = static_cast<const S *>(g.gradient) + r * g.gradient_stride;
    const W *w = static_cast<const W *>(g.weight);
    const T mean = static_cast<const T *>(g.stats)[2 * r], rstd = static_cast<const T *>(g.stats)[2 * r + 1];
    T sum[2] = {0, 0};
    for (uint32_t i = threadIdx.x; i < vecs; i += 1024) {
        T x[V], d[V], ws[V], s0 = 0, s1 = 0;
        unpack<S>(load_piece(xr, i, n), x);
        unpack<S>(load_piece(dr, i, n), d);
        if (w)
            load_weights<S, W>(w, i, n, ws);
#pragma unroll
        for (int e = 0; e < V; e++)
            if (i * V + e < n) {
                const T gv = w ? d[e] * ws[e] : d[e];
                s0 += gv;
                s1 += gv * ((x[e] - mean) * rstd);
            }
        sum[0] += s0;
        sum[1] += s1;
    }
    row_sums<1024, 1024, 2>(sum, lds);
    if (threadIdx.x == 0) {
        static_cast<T *>(sums)[2 * r] = sum[0] / (T)n;
        static_cast<T *>(sums)[2 * r + 1] = sum[1] / (T)n;
    }
}

template <typename S, typename W, bool SUMS>
__global__ __launch_bounds__(1024) void k_norm_back_wide(NormBackArgs g, const void *sums, void *parts)
{
    using T = typename StatOf<S>::T;
    constexpr int V = kVec<S>;
    if (block_gate_closed(g.gate))
        return;
    const uint32_t n = g.width, vecs = (n + V - 1) / V, i = blockIdx.y * 1024 + threadIdx.x;
    if (i >= vecs)
        return;
    const W *w = static_cast<const W *>(g.weight);
    T ws[V], dw[V] = {}, db[V] = {};
    if (w)
        load_weights<S, W>(w, i, n, ws);
    for (uint64_t r = blockIdx.x; r < g.rows; r += gridDim.x) {
        const T mean = static_cast<const T *>(g.stats)[2 * r], rstd = static_cast<const T *>(g.stats)[2 * r + 1];
        T x[V], d[V];
        unpack<S>(load_piece(static_cast<const S *>(g.x) + r * g.stride, i, n), x);
        unpack<S>(load_piece(static_cast<const S *>(g.gradient) + r * g.gradient_stride, i, n), d);
        const T c0 = g.x_gradient ? static_cast<const T *>(sums)[2 * r] : (T)0, c1 = g.x_gradient ? static_cast<const T *>(sums)[2 * r + 1] : (T)0;
#pragma unroll
        for (int e = 0; e < V; e++) {
            const T near = (x[e] - mean) * rstd;
            if constexpr (SUMS) {
                dw[e] += d[e] * near;
                db[e] += d[e];
            }
            x[e] = rstd * ((w ? d[e] * ws[e] : d[e]) - c0 - near * c1);
        }
        if (g.x_gradient)
            store_vec(static_cast<S *>(g.x_gradient) + r * g.x_gradient_stride, i, n, x, false);
    }
    if constexpr (SUMS) {
        T *part = static_cast<T *>(parts) + (uint64_t)blockIdx.x * 2 * vecs * V + i * V;
#pragma unroll
        for (int e = 0; e < V; e++) {
            part[e] = dw[e];
            part[vecs * V + e] = db[e];
        }
    }
}

// The workgroups' sums of both gradients, in their order: 64 columns a workgroup, 16 waves that each take
// every 16th workgroup's, then the waves' sums.
template <typename S, typename W>
__global__ __launch_bounds__(1024) void k_norm_back_join(NormBackArgs g, const void *parts, uint32_t count, ProgramClose close)
{
    using T = typename StatOf<S>::T;
    constexpr int V = kVec<S>;
    __shared__ T lds[2][16][64];
    if (block_gate_closed(g.gate))
        return;
    const uint32_t cols = (g.width + V - 1) / V * V, c = threadIdx.x & 63, k = threadIdx.x / 64;
    const uint32_t at = blockIdx.x * 64 + c;
    const T *from = static_cast<const T *>(parts) + at;
    T sum[2] = {0, 0};
    if (at < cols) {
        constexpr uint32_t U = 4;
        for (uint32_t p = k; p < count; p += 16 * U) {
            T x[U][2];
#pragma unroll
            for (uint32_t q = 0; q < U; q++)
#pragma unroll
                for (int o = 0; o < 2; o++)
                    x[q][o] = p + 16 * q < count ? from[((uint64_t)(p + 16 * q) * 2 + o) * cols] : (T)0;
#pragma unroll
            for (uint32_t q = 0; q < U; q++) {
                sum[0] += x[q][0];
                sum[1] += x[q][1];
            }
        }
    }
    lds[0][k][c] = sum[0];
    lds[1][k][c] = sum[1];
    __syncthreads();
    W *out = static_cast<W *>(k ? g.bias_gradient : g.weight_gradient);
    if (k < 2 && out && at < g.width) {
        T all = lds[k][0][c];
        for (int q = 1; q < 16; q++)
            all += lds[k][q][c];
        if (close.words)
            put(out + at, (W)all);
        else
            out[at] = (W)all;
    }
    program_close_block(close);
}

// How the backward pass is launched. Few rows take workgroups of 256 threads where those of 1024
// would leave CUs without one.
struct NormBackPlan {
    uint32_t threads = 1024, lanes = 0, r = 0, grid = 0; // lanes == 0: rows too long to hold
    uint64_t sums = 0, parts = 0, bytes = 0;
    NormBackPlan(const NormBackArgs &g)
    {
        const int size = logit_size_of(g.dtype);
        const uint32_t v = 16 / size, vecs = (g.width + v - 1) / v, stat = size == 8 ? 8 : 4;
        const bool want = g.weight_gradient || g.bias_gradient;
        if (vecs <= 16) lanes = 16, r = 1;
        else if (vecs <= 32) lanes = 32, r = 1;
        else if (vecs <= 64) lanes = 64, r = 1;
        else if (vecs <= 128) lanes = 64, r = 2;
        else if (vecs <= 512) lanes = 256, r = 2;
        else if (vecs <= 1024) lanes = 1024, r = 1;
        else if (vecs <= 2048) lanes = 1024, r = 2;
        if (lanes && lanes <= 256 && g.rows * lanes < 2ull * 1024 * kGfx950Cus)
            threads = 256;
        const uint64_t groups = lanes ? threads / lanes : 1, most = threads == 256 ? 512 : kGfx950Cus;
        const uint64_t need = (g.rows + groups - 1) / groups;
        grid = (uint32_t)(need < most ? need : most);
        parts = lanes || !g.x_gradient ? 0 : (g.rows * 2 * stat + 255) / 256 * 256;
        bytes = parts + (want ? (uint64_t)grid * 2 * vecs * v * stat : 0);
    }
};

template <typename S, typename W, int NT, int LANES, int R>
void launch_norm_held(hipStream_t s, const NormBackArgs &g, const NormBackPlan &p, char *sc, bool want)
{
    using T = typename StatOf<S>::T;
    const uint32_t vecs = (g.width + kVec<S> - 1) / kVec<S>;
    const uint32_t held = LANES <= 64 && R == 1 ? NT / 64 : LANES < NT ? 2 : 0;
    const uint32_t lds = want ? held * vecs * kVec<S> * (uint32_t)sizeof(T) : 0;
    if (want)
        hipLaunchKernelGGL((k_norm_back<S, W, NT, LANES, R, true>), dim3(p.grid), dim3(NT), lds, s, g, sc + p.parts);
    else
        hipLaunchKernelGGL((k_norm_back<S, W, NT, LANES, R, false>), dim3(p.grid), dim3(NT), 0, s, g, nullptr);
}

template <typename S, typename W, int NT> void launch_norm_narrow(hipStream_t s, const NormBackArgs &g, const NormBackPlan &p, char *sc, bool want)
{
    if (p.lanes == 16)
        launch_norm_held<S, W, NT, 16, 1>(s, g, p, sc, want);
    else if (p.lanes == 32)
        launch_norm_held<S, W, NT, 32, 1>(s, g, p, sc, want);
    else if (p.lanes == 64 && p.r == 1)
        launch_norm_held<S, W, NT, 64, 1>(s, g, p, sc, want);
    else if (p.lanes == 64)
        launch_norm_held<S, W, NT, 64, 2>(s, g, p, sc, want);
    else
        launch_norm_held<S, W, NT, 256, 2>(s, g, p, sc, want);
}

template <typename S, typename W>
hipError_t launch_norm_back_t(hipStream_t s, const NormBackArgs &g, void *scratch, ProgramClose close, bool *closed)
{
    const NormBackPlan p(g);
    char *sc = static_cast<char *>(scratch);
    const bool want = g.weight_gradient || g.bias_gradient;
    const uint32_t vecs = (g.width + kVec<S> - 1) / kVec<S>;
    if (!want && !g.x_gradient)
        return hipSuccess;
    if (p.grid) {
        if (p.lanes == 0) {
            const dim3 grid(p.grid, (vecs + 1023) / 1024);
            if (g.x_gradient)
                hipLaunchKernelGGL((k_norm_back_sums<S, W>), row_grid(g.rows), dim3(1024), 0, s, g, sc + p.sums);
            if (want)
                hipLaunchKernelGGL((k_norm_back_wide<S, W, true>), grid, dim3(1024), 0, s, g, sc + p.sums, sc + p.parts);
            else
                hipLaunchKernelGGL((k_norm_back_wide<S, W, false>), grid, dim3(1024), 0, s, g, sc + p.sums, nullptr);
        } else if (p.threads == 256) {
            launch_norm_narrow<S, W, 256>(s, g, p, sc, want);
        } else if (p.lanes <= 256) {
            launch_norm_narrow<S, W, 1024>(s, g, p, sc, want);
        } else if (p.r == 1) {
            launch_norm_held<S, W, 1024, 1024, 1>(s, g, p, sc, want);
        } else {
            launch_norm_held<S, W, 1024, 1024, 2>(s, g, p, sc, want);
        }
        const hipError_t e = hipGetLastError();
        if (e)
            return e;
    }
    if (!want)
        return hipSuccess;
    const uint32_t blocks = (g.width + 63) / 64;
    if (blocks > kCloseMaxBlocks)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    hipLaunchKernelGGL((k_norm_back_join<S, W>), dim3(blocks), dim3(1024), 0, s, g, sc + p.parts, p.grid, close);
    return hipGetLastError();
}

} // namespace

hipError_t launch_norm(hipStream_t s, const NormArgs &g, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.rows == 0 || (g.width == 0 && !g.stats)) // (the mean of no columns is NaN)
        return hipSuccess;
    switch (g.dtype) {
    case kLogitF32: return launch_norm_t<float, float>(s, g, close, closed);
    case kLogitF64: return launch_norm_t<double, double>(s, g, close, closed);
    case kLogitBf16:
        return g.weight_dtype == kLogitF32 ? launch_norm_t<__bf16, float>(s, g, close, closed)
                                           : launch_norm_t<__bf16, __bf16>(s, g, close, closed);
    default:
        return g.weight_dtype == kLogitF32 ? launch_norm_t<_Float16, float>(s, g, close, closed)
                                           : launch_norm_t<_Float16, _Float16>(s, g, close, closed);
    }
}

size_t norm_back_scratch_bytes(const NormBackArgs &g) { return g.width ? NormBackPlan(g).bytes : 0; }

hipError_t launch_norm_back(hipStream_t s, const NormBackArgs &g, void *scratch, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.width == 0)
        return hipSuccess;
    switch (g.dtype) {
    case kLogitF32: return launch_norm_back_t<float, float>(s, g, scratch, close, closed);
    case kLogitF64: return launch_norm_back_t<double, double>(s, g, scratch, close, closed);
    case kLogitBf16:
        return g.weight_dtype == kLogitF32 ? launch_norm_back_t<__bf16, float>(s, g, scratch, close, closed)
                                           : launch_norm_back_t<__bf16, __bf16>(s, g, scratch, close, closed);
    default:
        return g.weight_dtype == kLogitF32 ? launch_norm_back_t<_Float16, float>(s, g, scratch, close, closed)
                                           : launch_norm_back_t<_Float16, _Float16>(s, g, scratch, close, closed);
    }
}

} // namespace pcu
