// The cross entropy of an output layer, l = x W^T, loss = log(sum exp l) - l[label], and its gradients
// G = s (softmax(l) - [v = label]), dx = G W, dW = G^T x, with the logits never in memory.
//
// The loss is one product whose tiles leave a (maximum, sum of exponentials) for each row and the
// label's logit; a reduction joins them. The gradients go over the vocabulary in pieces: a piece's
// logits are made again and turned into G where they lie in registers, G goes to a buffer that the
// caches hold, and two products read it. That is one product of rows x vocab x width for a loss and four for
// a step, against three if the logits were kept (4096 x 128000: 1 GB in 16 bits, written and read twice).
//
// 16-bit features and weights go to the matrix cores as they are. Binary32 ones are split into three
// bfloat16 parts of 8 bits (exact), of whose products six are summed, smallest first: binary32's precision
// at a sixth of the 16-bit rate, against the binary32 matrix instructions' sixteenth. G is rounded
// to the operands' precision (8, 11 or 3 x 8 bits) before its products, as every training in 16 bits rounds
// the logits' gradient. It is kept relative to the largest row scale, so that rows with that
// scale, usually all, have the exact factor 1, and in binary16 2^14 times as large: the smallest
// probability it holds is then 2^-38.
#include "pcu_entropy_tile.hpp"
#include "pcu_rows.hpp"

#include <cmath>

#pragma clang fp contract(off)

namespace pcu {
namespace {

template <typename S> struct ElemOf { using T = S; };
template <> struct ElemOf<float> { using T = __bf16; };
template <typename S> constexpr int kParts = sizeof(S) == 4 ? 3 : 1;
template <typename S> constexpr float kBoost = __is_same(S, _Float16) ? 16384.0f : 1.0f;

// Rows as the tiles take them: parts, zeros past `cols` up to out_ld and past `rows` up to
// out_rows, and zeros in rows whose label is absent (labels given), whatever those hold.
struct PackArgs {
    const void *in = nullptr;
    uint64_t ld = 0;
    uint32_t rows = 0, cols = 0;
    const int32_t *labels = nullptr;
    uint32_t vocab = 0;
    uint16_t *out = nullptr;
    uint64_t plane = 0;
    uint32_t out_rows = 0, out_ld = 0;
    NodeGate gate{nullptr, 0};
};

template <typename S> __device__ __forceinline__ void pack_rows(const PackArgs &g, uint64_t block, uint64_t blocks)
{
    const uint32_t pieces = g.out_ld / 8; // of 8 values
    const uint64_t all = (uint64_t)g.out_rows * pieces;
    for (uint64_t i = block * 256 + threadIdx.x; i < all; i += blocks * 256) {
        const uint32_t r = (uint32_t)(i / pieces), c = (uint32_t)(i % pieces) * 8;
        bool on = r < g.rows && c < g.cols;
        if (on && g.labels) {
            const int32_t y = g.labels[r];
            on = y >= 0 && (uint32_t)y < g.vocab;
        }
        uint16_t *out = g.out + (uint64_t)r * g.out_ld + c;
        if constexpr (sizeof(S) == 2) {
            u32x4 raw = {0, 0, 0, 0};
            if (on)
                raw = load_piece(static_cast<const S *>(g.in) + r * g.ld, c / 8, g.cols);
            *reinterpret_cast<u32x4 *>(out) = raw;
        } else {
            float v[8] = {};
            if (on) {
                const float *row = static_cast<const float *>(g.in) + r * g.ld;
                unpack<float>(load_piece(row, c / 4, g.cols), v);
                unpack<float>(load_piece(row, c / 4 + 1, g.cols), v + 4);
            }
            u32x4 raw[3];
            split8(v, raw);
#pragma unroll
            for (int k = 0; k < 3; k++)
                *reinterpret_cast<u32x4 *>(out + k * g.plane) = raw[k];
        }
    }
}

template <typename S> __global__ __launch_bounds__(256) void k_pack(PackArgs g)
{
    if (block_gate_closed(g.gate))
        return;
    pack_rows<S>(g, blockIdx.x, gridDim.x);
}

// What the tiles and reductions know of a row.
struct RowData {
    int32_t *label;   // -1: none (or out of range: a fault)
    float *scale;     // relative to *factor; 0 where there is no label
    float *log_sum;
    float *own;       // the label's logit
    float *factor;    // what a gradient's sums are multiplied by
};

struct PrepArgs {
    const int32_t *labels = nullptr;
    const float *row_scale = nullptr;
    uint32_t rows = 0, vocab = 0;
    float boost = 1.0f;
    RowData row{};
    unsigned long long *fault = nullptr;
};

// One workgroup: labels, their faults, the largest finite |scale| and the scales relative to it.
__device__ __forceinline__ void prepare_rows(const PrepArgs &p, const NodeGate &gate)
{
    __shared__ float lds[4];
    uint64_t key = kNoFault;
    float most = 0.0f;
    for (uint32_t r = threadIdx.x; r < p.rows; r += 256) {
        int32_t y = p.labels[r];
        if (y >= 0 && (uint32_t)y >= p.vocab) {
            if (key == kNoFault)
                key = pack_fault(r, kInvalid);
            y = -1;
        }
        p.row.label[r] = y < 0 ? -1 : y;
        if (y >= 0) {
            const float s = p.row_scale ? fabsf(p.row_scale[r]) : 1.0f;
            if (s < INFINITY)
                most = fmaxf(most, s);
        }
    }
    wave_record_fault(key, p.fault, gate);
    most = block_reduce<256>(most, OpMax{}, lds);
    if (most == 0.0f)
        most = 1.0f;
    for (uint32_t r = threadIdx.x; r < p.rows; r += 256) {
        const float s = p.row_scale ? p.row_scale[r] : 1.0f;
        p.row.scale[r] = p.row.label[r] >= 0 ? s / most : 0.0f;
    }
    if (threadIdx.x == 0)
        *p.row.factor = most / p.boost;
}

// The features packed (by `blocks` workgroups), the weights packed if they are to be kept, and the
// rows prepared, by one launch.
template <typename S> __global__ __launch_bounds__(256) void k_entropy_open(PackArgs g, uint32_t blocks, PackArgs w, PrepArgs p)
{
    if (block_gate_closed(g.gate))
        return;
    if (blockIdx.x == 0)
        prepare_rows(p, g.gate);
    else if (blockIdx.x <= blocks)
        pack_rows<S>(g, blockIdx.x - 1, blocks);
    else
        pack_rows<S>(w, blockIdx.x - 1 - blocks, gridDim.x - 1 - blocks);
}

// ----------------------------------------------------------------------- tiles
struct LogitArgs {
    EntropyOperand w, x;       // rows: vocabulary, features
    uint32_t slabs = 0;        // of kSlabK
    uint32_t tiles_m = 0, tiles_n = 0;
    uint32_t first = 0;        // vocabulary of w's first row
    uint32_t vocab = 0, rows = 0;
    RowData row{};
    float2 *partial = nullptr; // [tile of the vocabulary][partial_ld], the loss
    uint32_t partial_ld = 0, partial_first = 0;
    uint32_t join = 0;         // the gradient: so many tiles' sums of a row to join first (0: they are joined)
    float *loss = nullptr;
    uint16_t *grad = nullptr;  // [row][grad_ld], the gradient, and its parts
    uint64_t grad_plane = 0;
    uint32_t grad_ld = 0;
    float boost = 1.0f;
    NodeGate gate{nullptr, 0};
};

// What exponentials are taken against, by the largest logit: that, or 0 where it is infinite (inf - inf is no number;
// against 0 the sum is the definition's, 0 or infinity).
__device__ __forceinline__ float exp_base(float most) { return fabsf(most) == INFINITY ? 0.0f : most; }

// (maximum, sum of exponentials against it) of two sets of logits together.
__device__ __forceinline__ float2 join_sums(float2 a, float2 b)
{
    const float m = fmaxf(a.x, b.x), from = exp_base(m);
    return make_float2(m, a.y * exp2_fast((a.x - from) * kLog2e) + b.y * exp2_fast((b.x - from) * kLog2e));
}

// A row's share k of SHARES of its tiles' sums, in order; share 0 joined with the others, in order, is the
// row's. Both ways that a row's sums are joined go by this, with 16 shares for few tiles.
template <uint32_t U, uint32_t SHARES = 16> __device__ __forceinline__ float2 join_share(const float2 *partial, uint32_t ld, uint32_t tiles, uint32_t n, uint32_t k)
{
    float2 a = make_float2(-INFINITY, 0.0f);
    for (uint32_t t = k; t < tiles; t += SHARES * U) {
        float2 b[U];
#pragma unroll
        for (uint32_t q = 0; q < U; q++)
            b[q] = t + SHARES * q < tiles ? partial[(uint64_t)(t + SHARES * q) * ld + n] : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (uint32_t q = 0; q < U; q++)
            a = join_sums(a, b[q]);
    }
    return a;
}
__device__ __forceinline__ float log_of(float2 a)
{
    // A NaN among the logits is not in the maximum, but in the sum.
    return (float)((double)exp_base(a.x) + (double)__builtin_amdgcn_logf(a.y) * kLn2);
}

// Vocabulary down, rows across: a lane holds 4 SM logits of each of its SN rows.
template <typename S, class Cfg, bool GRAD, bool CARRY> __global__ __launch_bounds__(Cfg::kThreads) void k_logits(LogitArgs g)
{
    using E = typename ElemOf<S>::T;
    constexpr int SM = Cfg::SM, SN = Cfg::SN, BM = Cfg::BM, BN = Cfg::BN;
    extern __shared__ __align__(16) char lds[];
    if (block_gate_closed(g.gate))
        return;
    const EntropyTile t = entropy_tile(blockIdx.x, g.tiles_m, g.tiles_n, 1);
    const uint32_t m0 = t.tm * BM, n0 = t.tn * BN;
    float *own_sum = reinterpret_cast<float *>(lds + Cfg::kTile);
    if (GRAD && g.join) {
        float2 *share = reinterpret_cast<float2 *>(lds);
        for (uint32_t i = threadIdx.x; i < 16u * BN; i += Cfg::kThreads)
            share[i] = join_share<2>(g.partial, g.partial_ld, g.join, n0 + i % BN, i / BN);
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < (uint32_t)BN; c += Cfg::kThreads) {
            float2 a = share[c];
            for (int q = 1; q < 16; q++)
                a = join_sums(a, share[q * BN + c]);
            const float l = own_sum[c] = log_of(a);
            if (t.tm == 0 && g.first == 0 && g.loss && n0 + c < g.rows)
                g.loss[n0 + c] = g.row.label[n0 + c] >= 0 ? l - g.row.own[n0 + c] : 0.0f;
        }
        __syncthreads();
    }
    // What the end needs of the rows is under way before the product.
    const uint32_t wave = threadIdx.x / 64, wm = wave / Cfg::WN * SM * 16, wn = wave % Cfg::WN * SN * 16;
    int32_t labels[SN];
    float scales[SN];
#pragma unroll
    for (int j = 0; j < SN; j++) {
        const uint32_t n = n0 + wn + acc_col(j);
        labels[j] = n < g.rows ? g.row.label[n] : -1;
        scales[j] = GRAD && n < g.rows ? g.row.scale[n] * g.boost : 0.0f;
    }
    f32x4 acc[SM][SN];
    // (The gradient's tiles go on to a whole slab of rows: those past the last one are zeros.)
    const uint32_t slabs = GRAD && n0 >= g.rows ? 0 : g.slabs * (kSlabK / Cfg::K);
    entropy_product<E, Cfg, false, false, CARRY>(g.w, g.x, m0, n0, 0, slabs, lds, acc);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t v0 = g.first + m0 + wm; // of acc[i][j][r]: v0 + acc_row(i, r)
    const bool ragged = g.first + m0 + BM > g.vocab;
    if constexpr (!GRAD) {
        float2 *red = reinterpret_cast<float2 *>(lds + Cfg::kTile);
#pragma unroll
        for (int j = 0; j < SN; j++) {
            const uint32_t n = n0 + wn + acc_col(j);
            const int32_t label = labels[j];
            if (label >= 0 && (uint32_t)label - v0 < SM * 16u) {
#pragma unroll
                for (int i = 0; i < SM; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (v0 + acc_row(i, r) == (uint32_t)label)
                            g.row.own[n] = acc[i][j][r];
            }
            if (ragged) {
#pragma unroll
                for (int i = 0; i < SM; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (v0 + acc_row(i, r) >= g.vocab)
                            acc[i][j][r] = -INFINITY;
            }
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < SM; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    m = fmaxf(m, acc[i][j][r]);
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            const float from = exp_base(m);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < SM; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    sum += exp2_fast((acc[i][j][r] - from) * kLog2e);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane < 16)
                red[wave / Cfg::WN * BN + wn + acc_col(j)] = make_float2(m, sum);
        }
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < (uint32_t)BN; c += Cfg::kThreads) {
            float2 a = red[c];
#pragma unroll
            for (int k = 1; k < Cfg::WM; k++)
                a = join_sums(a, red[k * BN + c]);
            g.partial[(uint64_t)(g.partial_first + t.tm) * g.partial_ld + n0 + c] = a;
        }
    } else {
#pragma unroll
        for (int j = 0; j < SN; j++) {
            const uint32_t n = n0 + wn + acc_col(j);
            const bool in = n < g.rows;
            const int32_t label = labels[j];
            const float scale = scales[j];
            const float log_sum = g.join ? own_sum[n - n0] : in ? g.row.log_sum[n] : 0.0f;
            const bool mine = label >= 0 && (uint32_t)label - v0 < SM * 16u;
#pragma unroll
            for (int i = 0; i < SM; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float p = exp2_fast((acc[i][j][r] - log_sum) * kLog2e);
                    if (mine && v0 + acc_row(i, r) == (uint32_t)label)
                        p -= 1.0f;
                    acc[i][j][r] = label >= 0 && !(ragged && v0 + acc_row(i, r) >= g.vocab) ? p * scale : 0.0f;
                }
        }
        // Values that need care in parts: any of the wave's.
        bool special = false;
        if constexpr (kParts<S> == 3) {
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < SN; j++)
#pragma unroll
                for (int i = 0; i < SM; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        most = max(most, __float_as_uint(acc[i][j][r]) & 0x7fffffffu);
            special = __any(most >= kLeastCut);
        }
        // Through LDS, so that a row's values are stored side by side.
        uint16_t *tile = reinterpret_cast<uint16_t *>(lds);
#pragma unroll
        for (int part = 0; part < kParts<S>; part++) {
            if (part)
                __syncthreads();
#pragma unroll
            for (int j = 0; j < SN; j++)
#pragma unroll
                for (int i = 0; i < SM; i++) {
                    uint32_t two[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if constexpr (kParts<S> == 1) {
                            typedef float f32x2 __attribute__((ext_vector_type(2)));
                            typedef S s16x2 __attribute__((ext_vector_type(2)));
                            const f32x2 x = {acc[i][j][2 * h], acc[i][j][2 * h + 1]};
                            two[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, s16x2));
                        } else {
                            // A part, and what is left for the next ones.
                            float lo = acc[i][j][2 * h], hi = acc[i][j][2 * h + 1];
                            two[h] = special ? next_part(lo, part) | next_part(hi, part) << 16 : next_parts(lo, hi, part);
                            acc[i][j][2 * h] = lo;
                            acc[i][j][2 * h + 1] = hi;
                        }
                    }
                    *reinterpret_cast<uint2 *>(tile + (wn + acc_col(j)) * Cfg::kOutPitch + wm + acc_row(i, 0)) = make_uint2(two[0], two[1]);
                }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < BN * BM / 8; i += Cfg::kThreads) {
                const uint32_t n = i / (BM / 8), c = i % (BM / 8) * 8;
                *reinterpret_cast<u32x4 *>(g.grad + part * g.grad_plane + (uint64_t)(n0 + n) * g.grad_ld + m0 + c) =
                    *reinterpret_cast<const u32x4 *>(tile + n * Cfg::kOutPitch + c);
            }
        }
    }
}

// Each row's log-sum-exp from its tiles', and its loss: 16 rows a workgroup, SHARES threads each. Of many tiles' sums
// 64 threads have one trip to memory each (8 rows of 1000 tiles: 11.4 us with 16, 9.5 so).
constexpr uint32_t kManyTiles = 256;
template <uint32_t SHARES>
__global__ __launch_bounds__(16 * SHARES) void k_entropy_loss(const float2 *partial, uint32_t ld, uint32_t tiles, uint32_t rows, RowData row,
                                                              float *loss, float *log_sum, NodeGate gate, ProgramClose close)
{
    __shared__ float2 red[SHARES][16];
    if (block_gate_closed(gate))
        return;
    const uint32_t c = threadIdx.x & 15, k = threadIdx.x / 16, n = blockIdx.x * 16 + c;
    red[k][c] = n < rows ? join_share<16, SHARES>(partial, ld, tiles, n, k) : make_float2(0.0f, 0.0f);
    __syncthreads();
    if constexpr (SHARES > 16) {
        // 16 runs of the shares first.
        if (k < 16) {
            float2 a = red[k * (SHARES / 16)][c];
            for (uint32_t q = 1; q < SHARES / 16; q++)
                a = join_sums(a, red[k * (SHARES / 16) + q][c]);
            red[k * (SHARES / 16)][c] = a;
        }
        __syncthreads();
    }
    if (k == 0 && n < rows) {
        float2 a = red[0][c];
        for (uint32_t q = 1; q < 16; q++)
            a = join_sums(a, red[q * (SHARES / 16)][c]);
        const float l = log_of(a);
        row.log_sum[n] = l;
        // Stored past the caches, in case the launch ends its program.
        if (log_sum)
            put(log_sum + n, l);
        if (loss)
            put(loss + n, row.label[n] >= 0 ? l - row.own[n] : 0.0f);
    }
    program_close_block(close);
}

struct ProductArgs {
    EntropyOperand a, b;
    uint32_t slabs = 0, splits = 1; // of kSlabK
    uint32_t tiles_m = 0, tiles_n = 0;
    float *sums = nullptr; // [split][row][sums_ld], the features' gradient
    uint64_t sums_split = 0;
    uint32_t sums_ld = 0;
    int add = 0;           // to what `sums` holds
    const float *factor = nullptr;
    void *out = nullptr;   // [vocabulary][out_ld], the weights' gradient
    uint64_t out_ld = 0;
    uint32_t out_rows = 0, out_cols = 0;
    NodeGate gate{nullptr, 0};
};

// dx: width down (from the weights, k-major), rows across (G); sums in binary32, k split.
template <typename S, class Cfg, bool CARRY> __device__ __forceinline__ void feature_tile(const ProductArgs &g, uint32_t block, char *lds)
{
    using E = typename ElemOf<S>::T;
    constexpr int SM = Cfg::SM, SN = Cfg::SN;
    const EntropyTile t = entropy_tile(block, g.tiles_m, g.tiles_n, g.splits);
    const uint32_t m0 = t.tm * Cfg::BM, n0 = t.tn * Cfg::BN;
    const uint32_t k_lo = (uint32_t)((uint64_t)g.slabs * t.split / g.splits), k_hi = (uint32_t)((uint64_t)g.slabs * (t.split + 1) / g.splits);
    f32x4 acc[SM][SN];
    entropy_product<E, Cfg, true, false, CARRY>(g.a, g.b, m0, n0, k_lo * (kSlabK / Cfg::K), k_hi * (kSlabK / Cfg::K), lds, acc);
    const uint32_t wave = threadIdx.x / 64, m = m0 + wave / Cfg::WN * SM * 16, n = n0 + wave % Cfg::WN * SN * 16;
#pragma unroll
    for (int j = 0; j < SN; j++)
#pragma unroll
        for (int i = 0; i < SM; i++) {
            f32x4 *to = reinterpret_cast<f32x4 *>(g.sums + t.split * g.sums_split + (uint64_t)(n + acc_col(j)) * g.sums_ld + m + acc_row(i, 0));
            *to = g.add ? *to + acc[i][j] : acc[i][j];
        }
}
template <typename S, class Cfg, bool CARRY> __global__ __launch_bounds__(Cfg::kThreads) void k_feature_gradient(ProductArgs g)
{
    extern __shared__ __align__(16) char lds[];
    if (!block_gate_closed(g.gate))
        feature_tile<S, Cfg, CARRY>(g, blockIdx.x, lds);
}

// dx from the splits' sums, in their order.
template <typename S>
__global__ __launch_bounds__(256) void k_feature_join(const float *sums, uint64_t split, uint32_t splits, uint32_t ld, uint32_t rows,
                                                      uint32_t cols, const float *factor, S *out, uint64_t out_ld, NodeGate gate,
                                                      ProgramClose close)
{
    if (block_gate_closed(gate))
        return;
    constexpr int V = kVec<S>;
    const uint32_t pieces = (cols + V - 1) / V;
    const float f = *factor;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)rows * pieces; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / pieces), c = (uint32_t)(i % pieces);
        float v[V] = {};
        constexpr uint32_t U = 8; // splits under way together
        for (uint32_t s = 0; s < splits; s += U) {
            f32x4 x[U][V / 4];
            const float *from = sums + s * split + (uint64_t)r * ld + c * V;
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                if (s + u < splits)
#pragma unroll
                    for (int q = 0; q < V / 4; q++)
                        x[u][q] = *reinterpret_cast<const f32x4 *>(from + u * split + 4 * q);
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                if (s + u < splits)
#pragma unroll
                    for (int e = 0; e < V; e++)
                        v[e] += x[u][e / 4][e % 4];
        }
#pragma unroll
        for (int e = 0; e < V; e++)
            v[e] *= f;
        S *row = out + r * out_ld;
        if (close.words && (c + 1) * V <= cols) {
            put_vec(row + c * V, pack<S>(v));
        } else if (close.words) {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (c * V + e < cols)
                    put(row + c * V + e, (S)v[e]);
        } else {
            store_vec(row, c, cols, v, false);
        }
    }
    program_close_block(close);
}

// dW: width down (from the features, k-major), vocabulary across (G, k-major).
template <typename S, class Cfg> __device__ __forceinline__ void weight_tile(const ProductArgs &g, uint32_t block, char *lds)
{
    using E = typename ElemOf<S>::T;
    constexpr int SM = Cfg::SM, SN = Cfg::SN, BM = Cfg::BM, BN = Cfg::BN;
    const EntropyTile t = entropy_tile(block, g.tiles_m, g.tiles_n, 1);
    const uint32_t m0 = t.tm * BM, n0 = t.tn * BN;
    f32x4 acc[SM][SN];
    entropy_product<E, Cfg, true, true, false>(g.a, g.b, m0, n0, 0, g.slabs * (kSlabK / Cfg::K), lds, acc);
    const uint32_t wave = threadIdx.x / 64, wm = wave / Cfg::WN * SM * 16, wn = wave % Cfg::WN * SN * 16;
    const float f = *g.factor;
    S *out = static_cast<S *>(g.out);
    if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int j = 0; j < SN; j++) {
            const uint32_t n = n0 + wn + acc_col(j);
            if (n >= g.out_rows)
                continue;
#pragma unroll
            for (int i = 0; i < SM; i++) {
                const uint32_t m = m0 + wm + acc_row(i, 0);
                const f32x4 v = acc[i][j] * f;
                float *to = out + (uint64_t)n * g.out_ld + m;
                typedef f32x4 f32x4_any __attribute__((aligned(4)));
                if (m + 4 <= g.out_cols)
                    *reinterpret_cast<f32x4_any *>(to) = v;
                else
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (m + e < g.out_cols)
                            to[e] = v[e];
            }
        }
    } else {
        S *tile = reinterpret_cast<S *>(lds);
        typedef S s16x4_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int j = 0; j < SN; j++)
#pragma unroll
            for (int i = 0; i < SM; i++)
                *reinterpret_cast<s16x4_t *>(tile + (wn + acc_col(j)) * Cfg::kOutPitch + wm + acc_row(i, 0)) =
                    __builtin_convertvector(acc[i][j] * f, s16x4_t);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < BN * BM / 8; i += Cfg::kThreads) {
            const uint32_t n = i / (BM / 8), c = i % (BM / 8) * 8;
            if (n0 + n >= g.out_rows || m0 + c >= g.out_cols)
                continue;
            const S *from = tile + n * Cfg::kOutPitch + c;
            S *to = out + (uint64_t)(n0 + n) * g.out_ld + m0 + c;
            if (m0 + c + 8 <= g.out_cols)
                *reinterpret_cast<u32x4_any *>(to) = *reinterpret_cast<const u32x4 *>(from);
            else
                for (uint32_t e = 0; e < 8 && m0 + c + e < g.out_cols; e++)
                    to[e] = from[e];
        }
    }
}

template <typename S, class Cfg> __global__ __launch_bounds__(Cfg::kThreads) void k_weight_gradient(ProductArgs g)
{
    extern __shared__ __align__(16) char lds[];
    if (!block_gate_closed(g.gate))
        weight_tile<S, Cfg>(g, blockIdx.x, lds);
}
// Both in one launch, `features` workgroups for the first: neither fills the CUs alone.
template <typename S, class CfgF, class CfgW, bool CARRY> __global__ __launch_bounds__(CfgF::kThreads) void k_both_gradients(ProductArgs f, uint32_t features, ProductArgs w)
{
    static_assert(CfgF::kThreads == CfgW::kThreads, "one kind of workgroup");
    extern __shared__ __align__(16) char lds[];
    if (block_gate_closed(f.gate))
        return;
    if (blockIdx.x < features)
        feature_tile<S, CfgF, CARRY>(f, blockIdx.x, lds);
    else
        weight_tile<S, CfgW>(w, blockIdx.x - features, lds);
}

// Rows of zeros: of the weights' gradient past the vocabulary, or where there are no rows.
template <typename S> __global__ __launch_bounds__(256) void k_zero_rows(S *out, uint64_t ld, uint64_t rows, uint32_t cols, NodeGate gate)
{
    if (block_gate_closed(gate))
        return;
    const uint32_t pieces = (cols + kVec<S> - 1) / kVec<S>;
    const typename StatOf<S>::T zero[kVec<S>] = {};
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (uint64_t)gridDim.x * 256)
        store_vec(out + i / pieces * ld, (uint32_t)(i % pieces), cols, zero, false);
}

// ---------------------------------------------------------------------- launches
template <typename S> struct Tiles {
    using Large = EntropyCfg<4, 2, 4, 8, 64, 2, 1>;  // 256 x 256
    using Middle = EntropyCfg<2, 2, 4, 4, 64, 2, 1>; // 128 x 128
    using Half = EntropyCfg<2, 2, 4, 2, 64, 3, 1>;   // 128 x 64
    using Thin = EntropyCfg<4, 1, 2, 2, 64, 3, 1>;   // 128 x 32
};
// Three parts leave LDS for one workgroup a CU: 8 waves of it, so that one reads while another multiplies
// (256 x 4247 x 1728 by 128 x 64 tiles: 50 us with 4 waves, 36 with 8).
template <> struct Tiles<float> {
    using Large = EntropyCfg<4, 2, 4, 4, 32, 2, 3>;  // 256 x 128
    using Middle = EntropyCfg<4, 2, 2, 4, 32, 3, 3>; // 128 x 128
    using Half = EntropyCfg<4, 2, 2, 2, 64, 2, 3>;   // 128 x 64
    using Thin = EntropyCfg<4, 1, 2, 2, 64, 2, 3>;   // 128 x 32
};

constexpr uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

enum class Side { Large, Middle, Half, Thin };
inline uint32_t side_m(Side s) { return s == Side::Large ? 256 : 128; }
inline uint32_t side_n(Side s, uint32_t parts) { return s == Side::Large ? (parts == 1 ? 256 : 128) : s == Side::Middle ? 128 : s == Side::Half ? 64 : 32; }

// What choices go by, measured: workgroups a CU, and what a slab of kSlabK takes them, in us (the
// 256 x 256 tiles of 16-bit values run at 1450 TFLOP/s, the 128 x 128 ones at 1050), the first where each CU
// has as many, the second alone on it.
struct SideTime {
    uint32_t per_cu;
    double full, alone;
};
inline SideTime side_time(Side s, uint32_t parts)
{
    if (parts == 1)
        return s == Side::Large ? SideTime{1, 1.5, 1.5} : s == Side::Middle ? SideTime{2, 1.0, 0.65} : s == Side::Half ? SideTime{2, 0.6, 0.45} : SideTime{2, 0.45, 0.4};
    return s == Side::Large ? SideTime{1, 4.2, 4.2} : s == Side::Middle ? SideTime{1, 2.4, 2.4} : s == Side::Half ? SideTime{1, 1.05, 1.05} : SideTime{1, 1.1, 1.1};
}
inline uint64_t tiles_of(Side s, uint32_t parts, uint64_t m, uint64_t n)
{
    return (m + side_m(s) - 1) / side_m(s) * ((n + side_n(s, parts) - 1) / side_n(s, parts));
}

// An m x n product's tiles, each over so many slabs: the rounds that they take on the CUs, each with its
// start and end (777 x 32003 x 1000: 83 us by 504 tiles of 256 x 256, 104 by 128 x 128).
inline double product_us(Side s, uint32_t parts, uint64_t m, uint64_t n, uint64_t slabs)
{
    const SideTime t = side_time(s, parts);
    const double tiles = (double)tiles_of(s, parts, m, n);
    if (tiles <= kGfx950Cus)
        return 8 + slabs * t.alone;
    const double n_rounds = tiles / (t.per_cu * kGfx950Cus);
    // A last round that few take runs faster.
    return (n_rounds <= 1 ? 1.0 : (n_rounds + std::ceil(n_rounds)) / 2) * ((s == Side::Large ? 14 : 8) + slabs * t.full);
}
inline Side choose(uint32_t parts, uint64_t m, uint64_t n, uint64_t slabs, bool narrow)
{
    Side best = Side::Middle;
    for (Side s : {Side::Large, Side::Half, Side::Thin})
        if ((narrow || s == Side::Large) && product_us(s, parts, m, n, slabs) < product_us(best, parts, m, n, slabs))
            best = s;
    return best;
}
// Where k can be split: by the whole work, unless a CU would have next to none of it. Few rows take
// narrower tiles, which read the weights at HBM's rate.
inline Side choose_split(uint32_t parts, uint64_t m, uint64_t rows, uint64_t slabs, bool carry)
{
    if (rows <= 64)
        return rows <= 32 && !(carry && parts == 3) ? Side::Thin : Side::Half;
    const SideTime l = side_time(Side::Large, parts), k = side_time(Side::Middle, parts);
    const double large = (double)tiles_of(Side::Large, parts, m, rows) / (l.per_cu * kGfx950Cus);
    const double middle = (double)tiles_of(Side::Middle, parts, m, rows) / (k.per_cu * kGfx950Cus);
    return large * l.full <= middle * k.full && large * slabs >= 4 ? Side::Large : Side::Middle;
}

// Binary32 weights that few rows read are split by the tiles' own workgroups, on their way to LDS, where a
// copy in parts would cost more than it saves: 6 bytes a value written, and read instead of 4 (20 rows, vocabulary 51939,
// width 896: a step of 388 us of kernels with the copy, 268 so; 128, 121922 x 2083: 2430 and 2140 a call). Tiles of one column each
// (128 rows) read them once. Small weights are in the caches, and their copy's launch is needed anyway (64, 1000 x 64: 30.7 with, 32.7 so).
constexpr uint64_t kSplitRows = 128, kSplitBytes = 8ull << 20;

// How a call goes over its vocabulary and what its scratch holds.
struct EntropyPlan {
    bool grads, pack_weights, keep_weights, carry;
    uint32_t parts, ld;    // of packed rows
    uint64_t rows_up;      // rows with padding
    uint64_t piece;        // vocabulary of a piece, a multiple of 256
    Side logits, features, weights;
    uint32_t splits, sums_ld;
    uint64_t sums_rows;
    uint64_t x, w, partial, grad, sums, label, scale, log_sum, own, factor, bytes;

    explicit EntropyPlan(const EntropyArgs &g)
    {
        grads = g.feature_gradient || g.weight_gradient;
        parts = g.dtype == kLogitF32 ? 3 : 1;
        ld = (uint32_t)round_up(g.width, kSlabK);
        rows_up = round_up(g.rows, 256);
        // 16-bit weights are read in place where direct loads can: whole slabs, 16-byte pieces, a
        // tile's rows within 32-bit offsets. Others go through registers for a loss, which reads them
        // once, and are copied for the gradients (24 rows, vocabulary 97088, width 3098: 151 us against
        // 390; a step of 29 rows, 34688 x 3211: three passes 324 us, the copy and three passes 248).
        const bool direct = g.width % kSlabK == 0 && g.weight_stride % 8 == 0 && ((uintptr_t)g.weights & 15) == 0 &&
                            g.weight_stride * 2 * 256 <= UINT32_MAX;
        const bool few = g.rows <= kSplitRows && (uint64_t)g.vocab * g.width * 4 > kSplitBytes;
        pack_weights = parts == 3 ? !few : !direct && grads;
        carry = parts == 3 ? few : !pack_weights && !direct;
        const uint64_t vocab_up = round_up(g.vocab, 256);
        const uint64_t row_bytes = 2ull * parts * ld;
        // G's piece is what the 256 MiB cache behind the L2s can hold; packed weights are kept
        // for the second pass where they are no more than 2 GiB (of 288 GB; splitting 1 GB of weights
        // takes 450 us).
        constexpr uint64_t kGradBytes = 192ull << 20, kWeightBytes = 2ull << 30;
        piece = kGradBytes / (rows_up ? rows_up * 2 * parts : 1) / 256 * 256;
        piece = piece < 256 ? 256 : piece > vocab_up ? vocab_up : piece;
        keep_weights = pack_weights && vocab_up * row_bytes <= kWeightBytes;
        if (!grads)
            piece = vocab_up;
        if (pack_weights && !keep_weights) {
            const uint64_t fit = kWeightBytes / row_bytes / 256 * 256;
            piece = piece < fit ? piece : fit < 256 ? 256 : fit;
        }
        const uint64_t within = piece < g.vocab ? piece : g.vocab, most = (within + kSlabK - 1) / kSlabK;
        logits = g.rows <= 64 ? choose_split(parts, g.vocab, g.rows, 1, carry) : choose(parts, g.vocab, g.rows, ld / kSlabK, !(carry && parts == 3));
        features = choose_split(parts, g.width, g.rows, most, carry);
        weights = choose(parts, g.width, within, (g.rows + kSlabK - 1) / kSlabK, false);
        const uint64_t tiles = tiles_of(features, parts, g.width, g.rows);
        const uint64_t per = side_time(features, parts).per_cu, want = tiles ? per * kGfx950Cus / tiles : 1;
        sums_ld = (uint32_t)round_up(g.width, 256);
        sums_rows = round_up(g.rows, side_n(features, parts));
        // Splits that fill the CUs, but no more than pay: a split's sums are written and read at 4 TB/s, 8 of
        // them in a trip to memory.
        const double best = std::sqrt(most * side_time(features, parts).full / (sums_rows * sums_ld * 8 / 4e6 + 0.15));
        const uint64_t pay = best < 1 ? 1 : (uint64_t)best, cut = want < pay ? want : pay;
        splits = (uint32_t)(cut < 1 ? 1 : cut > most ? (most ? most : 1) : cut);
        bytes = 0;
        auto take = [&](uint64_t n) {
            const uint64_t at = bytes;
            bytes += round_up(n, 256);
            return at;
        };
        x = take(rows_up * row_bytes);
        w = take(pack_weights ? (keep_weights ? vocab_up : piece) * row_bytes : 0);
        partial = take(g.log_sum_in ? 0 : (vocab_up / 128) * rows_up * 8);
        grad = take(grads ? piece * rows_up * 2 * parts : 0);
        sums = take(g.feature_gradient ? splits * sums_rows * sums_ld * 4ull : 0);
        label = take(g.rows * 4);
        scale = take(g.rows * 4);
        log_sum = take(g.rows * 4);
        own = take(g.rows * 4);
        factor = take(4);
    }
};

template <typename K> hipError_t with_lds(K *kernel, uint32_t bytes)
{
    return bytes > 65536 ? hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)
                         : hipSuccess;
}

template <typename S, class Cfg, bool GRAD, bool CARRY> hipError_t run_logits(hipStream_t s, LogitArgs a, uint64_t vocab_rows, uint64_t rows)
{
    a.tiles_m = (uint32_t)((vocab_rows + Cfg::BM - 1) / Cfg::BM);
    a.tiles_n = (uint32_t)((rows + Cfg::BN - 1) / Cfg::BN);
    hipError_t e = with_lds(k_logits<S, Cfg, GRAD, CARRY>, Cfg::kLds);
    if (e)
        return e;
    hipLaunchKernelGGL((k_logits<S, Cfg, GRAD, CARRY>), dim3(a.tiles_m * a.tiles_n), dim3(Cfg::kThreads), Cfg::kLds, s, a);
    return hipGetLastError();
}
template <typename S, class Cfg, bool GRAD> hipError_t logits_of(bool carry, hipStream_t s, const LogitArgs &a, uint64_t vocab_rows, uint64_t rows)
{
    if constexpr (sizeof(S) == 4 ? Cfg::BN > 32 : !GRAD) // (no others are chosen)
        if (carry)
            return run_logits<S, Cfg, GRAD, true>(s, a, vocab_rows, rows);
    return run_logits<S, Cfg, GRAD, false>(s, a, vocab_rows, rows);
}
template <typename S, bool GRAD> hipError_t logits_by(Side side, bool carry, hipStream_t s, const LogitArgs &a, uint64_t vocab_rows, uint64_t rows)
{
    switch (side) {
    case Side::Large: return logits_of<S, typename Tiles<S>::Large, GRAD>(carry, s, a, vocab_rows, rows);
    case Side::Middle: return logits_of<S, typename Tiles<S>::Middle, GRAD>(carry, s, a, vocab_rows, rows);
    case Side::Half: return logits_of<S, typename Tiles<S>::Half, GRAD>(carry, s, a, vocab_rows, rows);
    default: return logits_of<S, typename Tiles<S>::Thin, GRAD>(carry, s, a, vocab_rows, rows);
    }
}

template <typename S, class Cfg, bool CARRY> hipError_t launch_features(hipStream_t s, const ProductArgs &a)
{
    hipError_t e = with_lds(k_feature_gradient<S, Cfg, CARRY>, Cfg::kLds);
    if (e)
        return e;
    hipLaunchKernelGGL((k_feature_gradient<S, Cfg, CARRY>), dim3(a.tiles_m * a.tiles_n * a.splits), dim3(Cfg::kThreads), Cfg::kLds, s, a);
    return hipGetLastError();
}
template <typename S, class Cfg> hipError_t run_features(bool carry, hipStream_t s, ProductArgs a, uint64_t width, uint64_t rows)
{
    a.tiles_m = (uint32_t)((width + Cfg::BM - 1) / Cfg::BM);
    a.tiles_n = (uint32_t)((rows + Cfg::BN - 1) / Cfg::BN);
    if constexpr (sizeof(S) == 4 && Cfg::BN > 32)
        if (carry)
            return launch_features<S, Cfg, true>(s, a);
    return launch_features<S, Cfg, false>(s, a);
}
template <typename S, class Cfg> hipError_t run_weights(hipStream_t s, ProductArgs a, uint64_t width, uint64_t vocab_rows)
{
    a.tiles_m = (uint32_t)((width + Cfg::BM - 1) / Cfg::BM);
    a.tiles_n = (uint32_t)((vocab_rows + Cfg::BN - 1) / Cfg::BN);
    hipError_t e = with_lds(k_weight_gradient<S, Cfg>, Cfg::kLds);
    if (e)
        return e;
    hipLaunchKernelGGL((k_weight_gradient<S, Cfg>), dim3(a.tiles_m * a.tiles_n), dim3(Cfg::kThreads), Cfg::kLds, s, a);
    return hipGetLastError();
}

// Tiles of a row whose sums the gradient's workgroups join themselves, instead of a launch before.
constexpr uint32_t kJoinTiles = 32;

inline unsigned pack_blocks(uint64_t rows, uint64_t ld)
{
    const uint64_t n = (rows * (ld / 8) + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n > 8192 ? 8192 : n);
}

// Features' and weights' gradients of a piece in one launch, the weights' by 128 x 128 tiles.
template <typename S, class Cfg, bool CARRY> hipError_t launch_both(hipStream_t s, const ProductArgs &f, const ProductArgs &w)
{
    using Middle = typename Tiles<S>::Middle;
    constexpr uint32_t lds = Cfg::kLds > Middle::kLds ? Cfg::kLds : Middle::kLds;
    hipError_t e = with_lds(k_both_gradients<S, Cfg, Middle, CARRY>, lds);
    if (e)
        return e;
    const uint32_t features = f.tiles_m * f.tiles_n * f.splits;
    hipLaunchKernelGGL((k_both_gradients<S, Cfg, Middle, CARRY>), dim3(features + w.tiles_m * w.tiles_n), dim3(Cfg::kThreads), lds, s, f,
                       features, w);
    return hipGetLastError();
}
template <typename S, class Cfg>
hipError_t run_both(bool carry, hipStream_t s, ProductArgs f, ProductArgs w, uint64_t width, uint64_t rows, uint64_t vocab_rows)
{
    using Middle = typename Tiles<S>::Middle;
    f.tiles_m = (uint32_t)((width + Cfg::BM - 1) / Cfg::BM);
    f.tiles_n = (uint32_t)((rows + Cfg::BN - 1) / Cfg::BN);
    w.tiles_m = (uint32_t)((width + Middle::BM - 1) / Middle::BM);
    w.tiles_n = (uint32_t)((vocab_rows + Middle::BN - 1) / Middle::BN);
    if constexpr (sizeof(S) == 4)
        if (carry)
            return launch_both<S, Cfg, true>(s, f, w);
    return launch_both<S, Cfg, false>(s, f, w);
}

template <typename S> hipError_t launch_entropy_t(hipStream_t s, const EntropyArgs &g, void *scratch, ProgramClose close, bool *closed)
{
    const EntropyPlan p(g);
    char *sc = static_cast<char *>(scratch);
    const RowData row{reinterpret_cast<int32_t *>(sc + p.label), reinterpret_cast<float *>(sc + p.scale),
                      g.log_sum_in ? const_cast<float *>(g.log_sum_in) : reinterpret_cast<float *>(sc + p.log_sum),
                      reinterpret_cast<float *>(sc + p.own), reinterpret_cast<float *>(sc + p.factor)};
    hipError_t e;
    const bool whole_pass = !g.log_sum_in;
    const uint32_t slabs = p.ld / kSlabK;

    PackArgs px;
    px.in = g.features;
    px.ld = g.feature_stride;
    px.rows = (uint32_t)g.rows;
    px.cols = g.width;
    px.labels = p.grads ? g.labels : nullptr; // rows without a label reach no gradient
    px.vocab = g.vocab;
    px.out = reinterpret_cast<uint16_t *>(sc + p.x);
    px.plane = p.rows_up * p.ld;
    px.out_rows = (uint32_t)p.rows_up;
    px.out_ld = p.ld;
    px.gate = g.gate;
    PrepArgs pp;
    pp.labels = g.labels;
    pp.row_scale = g.row_scale;
    pp.rows = (uint32_t)g.rows;
    pp.vocab = g.vocab;
    pp.boost = kBoost<S>;
    pp.row = row;
    pp.fault = g.fault;
    // Parts of kept weights: one plane after another over the whole vocabulary; of others, of a piece.
    const uint64_t weight_plane = (p.keep_weights ? round_up(g.vocab, 256) : p.piece) * p.ld;
    auto pack_weights = [&](uint64_t v, uint64_t n, uint16_t *to) {
        PackArgs pw;
        pw.in = static_cast<const S *>(g.weights) + v * g.weight_stride;
        pw.ld = g.weight_stride;
        pw.rows = pw.out_rows = (uint32_t)n;
        pw.cols = g.width;
        pw.out = to;
        pw.plane = weight_plane;
        pw.out_ld = p.ld;
        pw.gate = g.gate;
        return pw;
    };
    uint16_t *const packed = reinterpret_cast<uint16_t *>(sc + p.w);
    if (g.rows) {
        const unsigned bx = pack_blocks(p.rows_up, p.ld), bw = p.keep_weights && g.vocab ? pack_blocks(g.vocab, p.ld) : 0;
        hipLaunchKernelGGL((k_entropy_open<S>), dim3(1 + bx + bw), dim3(256), 0, s, px, bx, pack_weights(0, g.vocab, packed), pp);
        if ((e = hipGetLastError()))
            return e;
    }

    const EntropyOperand x{px.out, px.plane, p.ld, (uint32_t)p.rows_up, p.ld};
    // The weights of vocabulary [v, v + n), packed here where they are not kept.
    auto weights = [&](uint64_t v, uint64_t n, EntropyOperand *o) {
        if (!p.pack_weights) {
            *o = EntropyOperand{reinterpret_cast<const uint16_t *>(static_cast<const S *>(g.weights) + v * g.weight_stride), 0, (uint32_t)g.weight_stride,
                                (uint32_t)n, g.width};
            return hipSuccess;
        }
        *o = EntropyOperand{p.keep_weights ? packed + v * p.ld : packed, weight_plane, p.ld, (uint32_t)n, p.ld};
        if (p.keep_weights)
            return hipSuccess;
        hipLaunchKernelGGL((k_pack<S>), dim3(pack_blocks(n, p.ld)), dim3(256), 0, s, pack_weights(v, n, packed));
        return hipGetLastError();
    };

    LogitArgs l;
    l.x = x;
    l.slabs = slabs;
    l.vocab = g.vocab;
    l.rows = (uint32_t)g.rows;
    l.row = row;
    l.partial = reinterpret_cast<float2 *>(sc + p.partial);
    l.partial_ld = (uint32_t)p.rows_up;
    l.grad = reinterpret_cast<uint16_t *>(sc + p.grad);
    l.grad_plane = p.rows_up * p.piece;
    l.grad_ld = (uint32_t)p.piece;
    l.boost = kBoost<S>;
    l.gate = g.gate;
    if (whole_pass && g.rows) {
        // Weights that need not be packed, or all fit when they are, take one launch.
        const uint64_t step = !p.pack_weights || p.keep_weights ? round_up(g.vocab, 256) : p.piece;
        uint32_t tiles = 0;
        for (uint64_t v = 0; v < g.vocab; v += step) {
            const uint64_t n = g.vocab - v < step ? g.vocab - v : step;
            if ((e = weights(v, n, &l.w)))
                return e;
            l.first = (uint32_t)v;
            l.partial_first = tiles;
            if ((e = logits_by<S, false>(p.logits, p.carry, s, l, n, g.rows)))
                return e;
            tiles += (uint32_t)((n + side_m(p.logits) - 1) / side_m(p.logits));
        }
        // A few tiles' sums are joined by the gradient's workgroups, each for its rows.
        if (p.grads && tiles > 0 && tiles <= kJoinTiles) {
            l.join = tiles;
            l.loss = g.loss;
        } else {
            const unsigned blocks = (unsigned)((g.rows + 15) / 16);
            const ProgramClose c = !p.grads && blocks <= kCloseMaxBlocks ? close : ProgramClose{};
            *closed = c.words != nullptr;
            if (tiles > kManyTiles)
                hipLaunchKernelGGL(k_entropy_loss<64>, dim3(blocks), dim3(1024), 0, s, l.partial, l.partial_ld, tiles, (uint32_t)g.rows, row,
                               g.loss, g.log_sum_out, g.gate, c);
            else
                hipLaunchKernelGGL(k_entropy_loss<16>, dim3(blocks), dim3(256), 0, s, l.partial, l.partial_ld, tiles, (uint32_t)g.rows, row,
                               g.loss, g.log_sum_out, g.gate, c);
            if ((e = hipGetLastError()))
                return e;
        }
    }
    if (!p.grads)
        return hipSuccess;

    ProductArgs f;
    f.sums = reinterpret_cast<float *>(sc + p.sums);
    f.sums_split = p.sums_rows * p.sums_ld;
    f.sums_ld = p.sums_ld;
    f.splits = p.splits;
    f.gate = g.gate;
    ProductArgs d;
    d.a = EntropyOperand{x.p, x.plane, x.ld, (uint32_t)round_up(g.rows, kSlabK), x.ld};
    d.slabs = (uint32_t)((g.rows + kSlabK - 1) / kSlabK);
    d.factor = row.factor;
    d.out_ld = g.weight_gradient_stride;
    d.out_cols = g.width;
    d.gate = g.gate;
    const uint64_t vocab = g.rows ? g.vocab : 0;
    for (uint64_t v = 0; v < vocab; v += p.piece) {
        const uint64_t n = vocab - v < p.piece ? vocab - v : p.piece;
        if ((e = weights(v, n, &l.w)))
            return e;
        l.first = (uint32_t)v;
        // Rows up to a whole slab: the weights' gradient reads those.
        if ((e = logits_by<S, true>(p.logits, p.carry, s, l, n, round_up(g.rows, kSlabK))))
            return e;
        f.a = l.w;
        f.b = EntropyOperand{l.grad, l.grad_plane, l.grad_ld, (uint32_t)p.rows_up, l.grad_ld};
        f.slabs = (uint32_t)((n + kSlabK - 1) / kSlabK);
        f.add = v > 0;
        d.b = EntropyOperand{l.grad, l.grad_plane, l.grad_ld, d.a.rows, l.grad_ld};
        d.out = static_cast<S *>(g.weight_gradient) + v * g.weight_gradient_stride;
        d.out_rows = (uint32_t)n;
        // (The narrowest tiles of binary32 have fewer waves.)
        constexpr bool kThinToo = Tiles<S>::Thin::kThreads == Tiles<S>::Middle::kThreads;
        if (g.feature_gradient && g.weight_gradient && p.weights == Side::Middle &&
            (p.features == Side::Middle || p.features == Side::Half || (kThinToo && p.features == Side::Thin))) {
            if (p.features == Side::Middle)
                e = run_both<S, typename Tiles<S>::Middle>(p.carry, s, f, d, g.width, g.rows, n);
            else if (p.features == Side::Half)
                e = run_both<S, typename Tiles<S>::Half>(p.carry, s, f, d, g.width, g.rows, n);
            else if constexpr (kThinToo)
                e = run_both<S, typename Tiles<S>::Thin>(p.carry, s, f, d, g.width, g.rows, n);
            if (e)
                return e;
            continue;
        }
        if (g.feature_gradient) {
            e = p.features == Side::Large    ? run_features<S, typename Tiles<S>::Large>(p.carry, s, f, g.width, g.rows)
                : p.features == Side::Middle ? run_features<S, typename Tiles<S>::Middle>(p.carry, s, f, g.width, g.rows)
                : p.features == Side::Half   ? run_features<S, typename Tiles<S>::Half>(p.carry, s, f, g.width, g.rows)
                                             : run_features<S, typename Tiles<S>::Thin>(p.carry, s, f, g.width, g.rows);
            if (e)
                return e;
        }
        if (g.weight_gradient) {
            e = p.weights == Side::Large ? run_weights<S, typename Tiles<S>::Large>(s, d, g.width, n) : run_weights<S, typename Tiles<S>::Middle>(s, d, g.width, n);
            if (e)
                return e;
        }
    }
    // Rows past the vocabulary first: the features' gradient may end the program.
    if (g.weight_gradient && g.weight_gradient_rows > vocab) {
        const uint64_t rows = g.weight_gradient_rows - vocab, n = (rows * ((g.width + kVec<S> - 1) / kVec<S>) + 255) / 256;
        hipLaunchKernelGGL((k_zero_rows<S>), dim3((unsigned)(n > 8192 ? 8192 : n)), dim3(256), 0, s,
                           static_cast<S *>(g.weight_gradient) + vocab * g.weight_gradient_stride, g.weight_gradient_stride, rows,
                           g.width, g.gate);
        if ((e = hipGetLastError()))
            return e;
    }
    if (g.feature_gradient && g.rows) {
        const uint64_t n = (g.rows * ((g.width + kVec<S> - 1) / kVec<S>) + 255) / 256;
        if (n > kCloseMaxBlocks)
            close = ProgramClose{};
        *closed = close.words != nullptr;
        hipLaunchKernelGGL((k_feature_join<S>), dim3((unsigned)(n > 8192 ? 8192 : n)), dim3(256), 0, s, f.sums, f.sums_split,
                           vocab ? p.splits : 0, f.sums_ld, (uint32_t)g.rows, g.width, row.factor, static_cast<S *>(g.feature_gradient),
                           g.feature_gradient_stride, g.gate, close);
        return hipGetLastError();
    }
    return hipSuccess;
}

} // namespace

size_t entropy_scratch_bytes(const EntropyArgs &g) { return EntropyPlan(g).bytes; }

hipError_t launch_entropy(hipStream_t s, const EntropyArgs &g, void *scratch, ProgramClose close, bool *closed)
{
    *closed = false;
    switch (g.dtype) {
    case kLogitF32: return launch_entropy_t<float>(s, g, scratch, close, closed);
    case kLogitBf16: return launch_entropy_t<__bf16>(s, g, scratch, close, closed);
    default: return launch_entropy_t<_Float16>(s, g, scratch, close, closed);
    }
}

} // namespace pcu
