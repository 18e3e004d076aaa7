// Embedding lookup with scaling, and the table's gradient.
//
//   out[i] = scale * table[t_i]                 (a negative token: zeros)
//   grad[v] = base[v] + scale * (sum of g[i] over the i with t_i = v, i ascending, long sums in parts)
//
// The gradient sorts the tokens (stable, so a row's terms are added in one order whatever the
// launch did); then every row of the table is written once, by the lanes that own it: no atomics on
// values, no second pass over the table to clear it. Both directions are bound by HBM.
#include "pcu_rows.hpp"

#include <type_traits>

#pragma clang fp contract(off)

namespace pcu {
namespace {

// Lanes a row takes: a row's 16-byte vectors, as a power of two of at most 64.
inline int row_lanes(uint32_t vecs)
{
    int t = 1;
    while (t < 64 && (uint32_t)t < vecs)
        t *= 2;
    return t;
}

// A vector of a row, stored past the caches by a launch that ends its program.
template <typename S> __device__ __forceinline__ void store_row(S *row, uint32_t i, uint32_t n, const typename StatOf<S>::T *v, bool through)
{
    if (!through) {
        store_vec(row, i, n, v, false);
        return;
    }
    const uint32_t at = i * kVec<S>;
    if (at + kVec<S> <= n) {
        put_vec(row + at, pack<S>(v));
    } else {
#pragma unroll
        for (int e = 0; e < kVec<S>; e++)
            if (at + e < n)
                put(row + at + e, (S)v[e]);
    }
}

// `lanes` lanes a row (a power of two of at most 64), 256 threads a workgroup.
template <typename S> __global__ __launch_bounds__(256) void k_embed(EmbedArgs g, int lanes, ProgramClose close)
{
    using T = typename StatOf<S>::T;
    if (block_gate_closed(g.gate))
        return;
    const uint32_t lane = threadIdx.x & (lanes - 1), per_block = 256 / lanes;
    const uint64_t i = (uint64_t)row_of_block() * per_block + threadIdx.x / lanes;
    const uint32_t vecs = (g.width + kVec<S> - 1) / kVec<S>;
    const T scale = (T)g.scale;
    uint64_t key = kNoFault;
    if (i < g.rows) {
        const int32_t t = g.tokens[i];
        S *out = static_cast<S *>(g.out) + i * g.out_stride;
        if (t >= 0 && (uint64_t)t < g.vocab) {
            const S *row = static_cast<const S *>(g.table) + (uint64_t)t * g.table_stride;
            for (uint32_t v0 = lane; v0 < vecs; v0 += 4 * lanes) {
                u32x4 raw[4];
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (v0 + q * lanes < vecs)
                        raw[q] = load_piece(row, v0 + q * lanes, g.width);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (v0 + q * lanes < vecs) {
                        T x[kVec<S>];
                        unpack<S>(raw[q], x);
#pragma unroll
                        for (int e = 0; e < kVec<S>; e++)
                            x[e] *= scale;
                        store_row(out, v0 + q * lanes, g.width, x, close.words != nullptr);
                    }
            }
        } else {
            if (t >= 0)
                key = pack_fault(i, kInvalid);
            const T zero[kVec<S>] = {};
            for (uint32_t v = lane; v < vecs; v += lanes)
                store_row(out, v, g.width, zero, close.words != nullptr);
        }
    }
    wave_record_fault(key, g.fault, g.gate);
    program_close_block(close);
}

template <typename S> hipError_t launch_embed_t(hipStream_t s, const EmbedArgs &g, ProgramClose close, bool *closed)
{
    const int lanes = row_lanes((g.width + kVec<S> - 1) / kVec<S>);
    const uint64_t blocks = (g.rows + 256 / lanes - 1) / (256 / lanes);
    if (blocks > kCloseMaxBlocks)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    hipLaunchKernelGGL((k_embed<S>), row_grid(blocks), dim3(256), 0, s, g, lanes, close);
    return hipGetLastError();
}

// ------------------------------------------------------------------ sorting tokens
// Keys are the tokens, absent and invalid ones as `vocab` (they come last and are not summed).
// Two stable counting passes over half of the key's bits each (at most 12). A tile of keys is
// ranked by one workgroup: its waves take consecutive runs of it, 64 keys at a time, and lanes with
// equal digits find each other by one ballot for each bit.
constexpr int kSortTile = 2048, kSortThreads = 512, kSortRounds = kSortTile / kSortThreads;
constexpr int kSortWaves = kSortThreads / 64;
// The most that one workgroup sorts alone, of 1024 threads (4096 tokens, 1000 x 64 in binary32: a call that sorts by
// tiles in 4 launches 37 us, 33 so; all tokens the same 57 and 43).
constexpr int kSortAlone = 8192;

__device__ __forceinline__ uint32_t token_key(const int32_t *tokens, uint64_t i, uint32_t vocab)
{
    const int32_t t = tokens[i];
    return t >= 0 && (uint32_t)t < vocab ? (uint32_t)t : vocab;
}

// Of the lanes with the same digit (and `on`): those before this one, and all of them.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool on)
{
    uint64_t same = __ballot(on);
    for (int b = 0; b < bits; b++) {
        const uint64_t set = __ballot((digit >> b) & 1);
        same &= (digit >> b) & 1 ? set : ~set;
    }
    return same;
}

// How often each digit occurs in a tile: counts[tile][digit].
__global__ __launch_bounds__(kSortThreads) void k_sort_count(EmbedBackArgs g, const uint32_t *keys, int shift, int bits,
                                                             uint32_t *counts)
{
    extern __shared__ uint32_t hist[];
    if (block_gate_closed(g.gate))
        return;
    const uint32_t bins = 1u << bits;
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads)
        hist[b] = 0;
    __syncthreads();
    uint64_t key = kNoFault;
    for (int r = 0; r < kSortRounds; r++) {
        const uint64_t i = (uint64_t)blockIdx.x * kSortTile + r * kSortThreads + threadIdx.x;
        if (i < g.rows) {
            uint32_t k;
            if (keys) {
                k = keys[i];
            } else {
                const int32_t t = g.tokens[i];
                if (t >= 0 && (uint32_t)t >= g.vocab && key == kNoFault)
                    key = pack_fault(i, kInvalid);
                k = token_key(g.tokens, i, g.vocab);
            }
            atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
        }
    }
    wave_record_fault(key, g.fault, g.gate);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads)
        counts[(uint64_t)blockIdx.x * bins + b] = hist[b];
}

// Ranks of a tile's keys among the tile's equal digits, wave by wave: rank[r] within the wave, and
// wave_count[wave][digit], the wave's number of each digit.
template <int THREADS, int ROUNDS, typename Key>
__device__ __forceinline__ void rank_tile(Key key_at, uint64_t n, uint64_t tile0, int shift, int bits,
                                          uint32_t (&k)[ROUNDS], uint32_t (&rank)[ROUNDS], uint32_t *wave_count)
{
    const uint32_t bins = 1u << bits, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    uint32_t *mine = wave_count + wave * bins;
    for (uint32_t b = threadIdx.x; b < bins * THREADS / 64; b += THREADS)
        wave_count[b] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const uint64_t i = tile0 + wave * (ROUNDS * 64) + r * 64 + lane;
        const bool on = i < n;
        k[r] = on ? key_at(i) : ~0u;
        const uint32_t d = (k[r] >> shift) & (bins - 1);
        const uint64_t same = same_digit(d, bits, on);
        const uint64_t before = same & ((1ull << lane) - 1);
        const uint32_t base = on ? mine[d] : 0;
        rank[r] = base + (uint32_t)__popcll(before);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (on && before == 0)
            mine[d] = base + (uint32_t)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
}

// Exclusive prefix over a tile's or launch's bins, in place: v[b] becomes the sum before bin b.
template <int THREADS> __device__ __forceinline__ void scan_bins(uint32_t *v, uint32_t bins, uint32_t *part)
{
    const uint32_t each = (bins + THREADS - 1) / THREADS, b0 = threadIdx.x * each;
    uint32_t sum = 0;
    for (uint32_t b = b0; b < b0 + each && b < bins; b++)
        sum += v[b];
    const uint32_t upto = wave_upto(sum, OpSum{}, 0u);
    if ((threadIdx.x & 63) == 63)
        part[threadIdx.x / 64] = upto;
    __syncthreads();
    uint32_t at = upto - sum;
    for (uint32_t w = 0; w < threadIdx.x / 64; w++)
        at += part[w];
    for (uint32_t b = b0; b < b0 + each && b < bins; b++) {
        const uint32_t n = v[b];
        v[b] = at;
        at += n;
    }
    __syncthreads();
}

// One workgroup a digit: its count in each tile becomes its count in the tiles before, and its
// count in all of them goes to totals.
__global__ __launch_bounds__(kSortThreads) void k_sort_scan(EmbedBackArgs g, int bits, uint32_t tiles, uint32_t *counts,
                                                            uint32_t *totals)
{
    __shared__ uint32_t part[kSortWaves];
    if (block_gate_closed(g.gate))
        return;
    uint32_t before = 0;
    for (uint32_t t0 = 0; t0 < tiles; t0 += kSortThreads) {
        const uint32_t t = t0 + threadIdx.x;
        uint32_t *c = counts + ((uint64_t)t << bits) + blockIdx.x;
        const uint32_t n = t < tiles ? *c : 0, upto = wave_upto(n, OpSum{}, 0u);
        if ((threadIdx.x & 63) == 63)
            part[threadIdx.x / 64] = upto;
        __syncthreads();
        uint32_t at = before + upto - n;
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; w++) {
            at += w < threadIdx.x / 64 ? part[w] : 0;
            before += part[w];
        }
        if (t < tiles)
            *c = at;
        __syncthreads();
    }
    if (threadIdx.x == 0)
        totals[blockIdx.x] = before;
}

// Moves a tile's keys and places to where the digit's order puts them: after all smaller digits,
// and after the digit in the tiles before.
__global__ __launch_bounds__(kSortThreads) void k_sort_move(EmbedBackArgs g, const uint32_t *keys, const uint32_t *places,
                                                            int shift, int bits, const uint32_t *counts, const uint32_t *totals, uint32_t tiles,
                                                            uint32_t *keys_out, uint32_t *places_out)
{
    extern __shared__ uint32_t lds[];
    if (block_gate_closed(g.gate))
        return;
    const uint32_t bins = 1u << bits, wave = threadIdx.x / 64;
    uint32_t *first = lds, *wave_count = lds + bins, *part = wave_count + bins * kSortWaves;
    uint32_t k[kSortRounds], rank[kSortRounds];
    rank_tile<kSortThreads, kSortRounds>([&](uint64_t i) { return keys ? keys[i] : token_key(g.tokens, i, g.vocab); }, g.rows,
              (uint64_t)blockIdx.x * kSortTile, shift, bits, k, rank, wave_count);
    // A digit's count in all tiles; without totals (few tiles) the tiles' counts are added up here.
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t all = totals ? totals[b] : 0;
        for (uint32_t t = 0; !totals && t < tiles; t++)
            all += counts[(uint64_t)t * bins + b];
        first[b] = all;
    }
    __syncthreads();
    scan_bins<kSortThreads>(first, bins, part);
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads) {
        uint32_t at = first[b] + (totals ? counts[(uint64_t)blockIdx.x * bins + b] : 0);
        for (uint32_t t = 0; !totals && t < blockIdx.x; t++)
            at += counts[(uint64_t)t * bins + b];
        for (int w = 0; w < kSortWaves; w++) {
            const uint32_t n = wave_count[w * bins + b];
            wave_count[w * bins + b] = at;
            at += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; r++) {
        const uint64_t i = (uint64_t)blockIdx.x * kSortTile + wave * (kSortTile / kSortWaves) + r * 64 + (threadIdx.x & 63);
        if (i < g.rows) {
            const uint32_t to = wave_count[wave * bins + ((k[r] >> shift) & (bins - 1))] + rank[r];
            keys_out[to] = k[r];
            places_out[to] = places ? places[i] : (uint32_t)i;
        }
    }
}

// Both passes in one workgroup, through LDS.
template <int THREADS, int ROUNDS> __global__ __launch_bounds__(THREADS) void k_sort_one(EmbedBackArgs g, int bits, uint32_t *keys_out, uint32_t *places_out)
{
    extern __shared__ uint32_t lds[];
    if (block_gate_closed(g.gate))
        return;
    const uint32_t bins = 1u << bits, wave = threadIdx.x / 64, lane = threadIdx.x & 63, n = (uint32_t)g.rows;
    uint32_t *first = lds, *wave_count = lds + bins, *part = wave_count + bins * (THREADS / 64);
    uint32_t *mid_key = part + THREADS / 64, *mid_place = mid_key + THREADS * ROUNDS;
    uint64_t key = kNoFault;
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        const int32_t t = g.tokens[i];
        if (t >= 0 && (uint32_t)t >= g.vocab && key == kNoFault)
            key = pack_fault(i, kInvalid);
    }
    wave_record_fault(key, g.fault, g.gate);
    for (int pass = 0; pass < 2; pass++) {
        uint32_t k[ROUNDS], rank[ROUNDS];
        rank_tile<THREADS, ROUNDS>([&](uint64_t i) { return pass ? mid_key[i] : token_key(g.tokens, i, g.vocab); }, n, 0, pass * bits, bits,
                  k, rank, wave_count);
        for (uint32_t b = threadIdx.x; b < bins; b += THREADS) {
            uint32_t all = 0;
            for (int w = 0; w < THREADS / 64; w++)
                all += wave_count[w * bins + b];
            first[b] = all;
        }
        __syncthreads();
        scan_bins<THREADS>(first, bins, part);
        for (uint32_t b = threadIdx.x; b < bins; b += THREADS) {
            uint32_t at = first[b];
            for (int w = 0; w < THREADS / 64; w++) {
                const uint32_t c = wave_count[w * bins + b];
                wave_count[w * bins + b] = at;
                at += c;
            }
        }
        uint32_t place[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t i = wave * (ROUNDS * 64) + r * 64 + lane;
            place[r] = pass && i < n ? mid_place[i] : i;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t i = wave * (ROUNDS * 64) + r * 64 + lane;
            if (i < n) {
                const uint32_t to = wave_count[wave * bins + ((k[r] >> (pass * bits)) & (bins - 1))] + rank[r];
                (pass ? keys_out : mid_key)[to] = k[r];
                (pass ? places_out : mid_place)[to] = place[r];
            }
        }
        __syncthreads();
    }
}

// --------------------------------------------------------------------- summing
// First of the sorted keys [lo, lo + len) that is at least v; a wave looks at 64 of them at a time.
__device__ __forceinline__ uint32_t lower_bound(const uint32_t *keys, uint32_t lo, uint32_t len, uint32_t v)
{
    while (len > 0) {
        const uint32_t step = (len + 63) / 64, at = (threadIdx.x & 63) * step;
        const uint32_t below = (uint32_t)__popcll(__ballot(at < len && keys[lo + min(at, len - 1)] < v));
        if (below == 0)
            break;
        const uint32_t skip = (below - 1) * step + 1;
        lo += skip;
        len = min(step - 1, len - skip);
    }
    return lo;
}

// A wave takes the rows whose first term is one of kStarts sorted ones. Rows of more than kLong terms
// are added up by several waves, kLong terms each from the row's first on (a part; which other tokens there are makes
// no difference to a row's sum), whose sums are added in order afterwards. The other rows that begin in a wave's share end within its 64 lanes.
constexpr uint32_t kStarts = 16, kLong = 48;
static_assert(kStarts - 1 + kLong < 64, "a short row's end is in sight");

// sum += terms [lo, hi) of the sorted order, vector v of each, one after another.
template <typename S, typename P, typename T>
__device__ __forceinline__ void add_terms(const EmbedBackArgs &g, const P *places, uint32_t lo, uint32_t hi, uint32_t v,
                                          T (&sum)[kVec<S>])
{
    constexpr int U = 8;
    for (uint32_t j = lo; j < hi; j += U) {
        u32x4 raw[U];
#pragma unroll
        for (int q = 0; q < U; q++)
            if (j + q < hi)
                raw[q] = load_piece(static_cast<const S *>(g.gradient) + (uint64_t)places[j + q] * g.gradient_stride, v, g.width);
#pragma unroll
        for (int q = 0; q < U; q++)
            if (j + q < hi) {
                T x[kVec<S>];
                unpack<S>(raw[q], x);
#pragma unroll
                for (int e = 0; e < kVec<S>; e++)
                    sum[e] += x[e];
            }
    }
}

// Row `row`, vector v: base (raw; zeros without one) plus scale times `sum`.
template <typename S, typename T>
__device__ __forceinline__ void write_sum(const EmbedBackArgs &g, uint32_t row, uint32_t v, const u32x4 &base, const T (&sum)[kVec<S>],
                                          bool through = false)
{
    const T scale = (T)g.scale;
    T y[kVec<S>];
    if (g.base) {
        unpack<S>(base, y);
#pragma unroll
        for (int e = 0; e < kVec<S>; e++)
            y[e] += scale * sum[e];
    } else {
#pragma unroll
        for (int e = 0; e < kVec<S>; e++)
            y[e] = scale * sum[e];
    }
    S *out = static_cast<S *>(g.out) + (uint64_t)row * g.out_stride;
    if (through)
        store_row(out, v, g.width, y, true);
    else
        store_vec(out, v, g.width, y, g.past);
}
template <typename S> __device__ __forceinline__ u32x4 load_base(const EmbedBackArgs &g, uint32_t row, uint32_t v)
{
    return g.base ? load_piece(static_cast<const S *>(g.base) + (uint64_t)row * g.base_stride, v, g.width) : u32x4{0, 0, 0, 0};
}

// Row sums of the runs of equal keys that begin at sorted terms [16 chunk, 16 chunk + 16), but long
// ones. Rows of 64 vectors or more (lanes 64): all control is scalar, and the terms are walked across the
// rows' ends, so that their loads, and the bases' with them, are under way together. Narrower rows: each
// group of `lanes` lanes takes every so-manieth run. vec: the lane's vector.
template <typename S, bool BASE>
__device__ __forceinline__ void sum_runs(const EmbedBackArgs &g, const uint32_t *keys, const uint32_t *places, uint32_t chunk, int lanes,
                                         uint32_t vec, bool on)
{
    using T = typename StatOf<S>::T;
    constexpr int U = BASE ? 4 : 8, V = kVec<S>;
    const uint32_t n = (uint32_t)g.rows, lane = threadIdx.x & 63, at = chunk * kStarts + lane;
    const uint32_t key = at < n ? keys[at] : ~0u, place = at < n ? places[at] : 0;
    uint32_t prev = __shfl_up(key, 1);
    if (lane == 0)
        prev = at > 0 ? keys[at - 1] : ~0u;
    const uint64_t change = __ballot(key != prev), after = change >> 1 >> lane;
    const uint32_t len = after ? (uint32_t)__builtin_ctzll(after) + 1 : 64 - lane; // beyond sight: long
    const uint64_t starts = __ballot(lane < kStarts && key != prev && key < g.vocab && len <= kLong);
    if (lanes == 64) {
        const uint64_t upto = change & (~0ull >> (63 - lane));
        uint64_t terms = __ballot(upto && (starts >> (63 - __builtin_clzll(upto | 1)) & 1));
        const uint64_t lasts = terms & change >> 1;
        T sum[V] = {};
        while (terms) {
            u32x4 raw[U], base[U];
            uint64_t t = terms;
#pragma unroll
            for (int q = 0; q < U; q++, t &= t - 1)
                if (t) {
                    const int l = __builtin_ctzll(t);
                    if (on) {
                        raw[q] = load_piece(static_cast<const S *>(g.gradient) + (uint64_t)from_lane(place, l) * g.gradient_stride, vec, g.width);
                        if (BASE && lasts >> l & 1)
                            base[q] = load_base<S>(g, from_lane(key, l), vec);
                    }
                }
#pragma unroll
            for (int q = 0; q < U; q++, terms &= terms - 1)
                if (terms) {
                    const int l = __builtin_ctzll(terms);
                    T x[V];
                    unpack<S>(raw[q], x);
#pragma unroll
                    for (int e = 0; e < V; e++)
                        sum[e] += x[e];
                    if (lasts >> l & 1) {
                        if (on)
                            write_sum<S>(g, from_lane(key, l), vec, base[q], sum);
#pragma unroll
                        for (int e = 0; e < V; e++)
                            sum[e] = 0;
                    }
                }
        }
        return;
    }
    const uint32_t runs = (uint32_t)__popcll(starts), subs = 64 / lanes;
    uint64_t left = starts;
    for (uint32_t r = 0; r < runs; r += subs) {
        // This group's run: the (lane / lanes)-th of those left.
        uint64_t mine = left;
        for (uint32_t k = 0; k < lane / lanes; k++)
            mine &= mine - 1;
        for (uint32_t k = 0; k < subs; k++)
            left &= left - 1;
        const int l = mine ? __builtin_ctzll(mine) : 0;
        const uint32_t row = __shfl(key, l), terms = __shfl(len, l);
        if (mine && on) {
            const u32x4 base = load_base<S>(g, row, vec);
            T sum[V] = {};
            add_terms<S>(g, places + chunk * kStarts, l, l + terms, vec, sum);
            write_sum<S>(g, row, vec, base, sum);
        }
    }
}

// A few tokens: no sort, one launch. Its first workgroups (`sums` of them) add up the rows of every
// token that occurs for the first time: a wave takes a token and 64 vectors of the row, and finds the
// token's other places by looking all of them over. The others fill the rest of the table's gradient with
// zeros or its base, `each` vectors side by side; they leave out the rows that occur. 511 tokens,
// 50257 x 768 F32: as two launches, all rows filled and then some written again, 22 and 10 us (a plain
// fill of the 154 MB takes 22.6, past the caches 27); waves that looked for the tokens of 16 rows each
// took 41 to 46, and sorting first 55 in three launches.
constexpr uint32_t kDirect = 1024, kFillBlocks = 8 * kGfx950Cus;
constexpr uint32_t kFillRows = (1u << 22) / kFillBlocks + 2; // rows that a workgroup's vectors can lie in

template <typename S>
__device__ __forceinline__ void fill_rows(const EmbedBackArgs &g, const uint32_t *keys, uint32_t block, uint64_t each, bool through)
{
    __shared__ uint32_t occurs[(kFillRows + 31) / 32];
    const uint32_t n = (uint32_t)g.rows, vecs = (g.width + kVec<S> - 1) / kVec<S>;
    const uint64_t lo = block * each, hi = min(lo + each, (uint64_t)g.vocab * vecs);
    if (lo >= hi)
        return;
    const uint32_t row0 = (uint32_t)(lo / vecs);
    for (uint32_t w = threadIdx.x; w < (kFillRows + 31) / 32; w += 256)
        occurs[w] = 0;
    __syncthreads();
    // The rows that occur, from the sorted keys or (few tokens) from all of them.
    const uint32_t first = keys ? lower_bound(keys, 0, n, row0) : 0;
    const uint32_t last = keys ? lower_bound(keys, 0, n, min((uint32_t)((hi - 1) / vecs) + 1, g.vocab)) : n;
    for (uint32_t i = first + threadIdx.x; i < last; i += 256) {
        const uint32_t t = keys ? keys[i] : (uint32_t)g.tokens[i]; // an absent one is no row's
        if (t - row0 < kFillRows)
            atomicOr(&occurs[(t - row0) / 32], 1u << ((t - row0) & 31));
    }
    __syncthreads();
    // Row and vector of each step by addition: a division a vector is dearer than its store.
    const uint32_t down = 256 / vecs, along = 256 % vecs;
    uint32_t row = (uint32_t)((lo + threadIdx.x) / vecs), v = (uint32_t)((lo + threadIdx.x) % vecs);
    constexpr int U = 4;
    for (uint64_t i = lo + threadIdx.x; i < hi; i += 256 * U) {
        u32x4 raw[U];
        uint32_t rows[U], at[U];
#pragma unroll
        for (int q = 0; q < U; q++) {
            rows[q] = row;
            at[q] = v;
            if (i + 256 * q >= hi || occurs[(row - row0) / 32] >> ((row - row0) & 31) & 1)
                rows[q] = ~0u;
            else
                raw[q] = load_base<S>(g, row, v);
            row += down;
            v += along;
            if (v >= vecs) {
                v -= vecs;
                row++;
            }
        }
#pragma unroll
        for (int q = 0; q < U; q++)
            if (rows[q] != ~0u) {
                typename StatOf<S>::T y[kVec<S>];
                unpack<S>(raw[q], y);
                S *out = static_cast<S *>(g.out) + (uint64_t)rows[q] * g.out_stride;
                if (through)
                    store_row(out, at[q], g.width, y, true);
                else
                    store_vec(out, at[q], g.width, y, g.past);
            }
    }
}

template <typename S>
__global__ __launch_bounds__(256) void k_embed_first(EmbedBackArgs g, uint32_t across, uint32_t sums, uint64_t each, ProgramClose close)
{
    using T = typename StatOf<S>::T;
    constexpr int V = kVec<S>, N = kDirect / 64;
    if (block_gate_closed(g.gate))
        return;
    if (blockIdx.x >= sums) {
        fill_rows<S>(g, nullptr, blockIdx.x - sums, each, close.words != nullptr);
        program_close_block(close);
        return;
    }
    const uint32_t n = (uint32_t)g.rows, lane = threadIdx.x & 63, vecs = (g.width + V - 1) / V;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = unit / across;
    const uint32_t v = unit % across * 64 + lane;
    const int32_t t = i < n ? g.tokens[i] : -1;
    const bool valid = t >= 0 && (uint32_t)t < g.vocab;
    wave_record_fault(t >= 0 && !valid && lane == 0 ? pack_fault(i, kInvalid) : kNoFault, g.fault, g.gate);
    uint64_t same[N]; // bit l of same[q]: place 64 q + l
    bool first = valid;
    if (valid) {
        int32_t other[N];
#pragma unroll
        for (int q = 0; q < N; q++)
            other[q] = (uint32_t)q * 64 + lane < n ? g.tokens[q * 64 + lane] : -1;
#pragma unroll
        for (int q = 0; q < N; q++) {
            same[q] = __ballot(other[q] == t);
            if ((uint32_t)q < i / 64 ? same[q] != 0 : (uint32_t)q == i / 64 && (same[q] & ((1ull << (i & 63)) - 1)))
                first = false;
        }
    }
    if (first) {
        const u32x4 base = v < vecs ? load_base<S>(g, t, v) : u32x4{};
        T sum[V] = {};
        // U terms' loads under way together, no branch between them: past the last term it is read again (1024 terms
        // of one token, 64 wide: 102 us with a branch a load, 65 so; 16 at a time 63).
        auto add_terms = [&](auto count, auto load, uint64_t &left, int q) {
            constexpr int U = decltype(count)::value;
            u32x4 raw[U];
            uint64_t l = left;
            uint32_t place = 0;
#pragma unroll
            for (int k = 0; k < U; k++) {
                place = l ? __builtin_ctzll(l) : place;
                raw[k] = load(static_cast<const S *>(g.gradient) + (uint64_t)(q * 64 + place) * g.gradient_stride);
                l &= l - 1;
            }
#pragma unroll
            for (int k = 0; k < U; k++) {
                T x[V];
                unpack<S>(raw[k], x);
#pragma unroll
                for (int e = 0; e < V; e++)
                    sum[e] += left ? x[e] : (T)0; // (no sum is -0)
                left &= left - 1;
            }
        };
        auto add_all = [&](auto load) {
            for (int q = 0; q < N; q++)
                for (uint64_t left = same[q]; left;)
                    if (left & (left - 1))
                        add_terms(std::integral_constant<int, 8>{}, load, left, q);
                    else
                        add_terms(std::integral_constant<int, 1>{}, load, left, q);
        };
        const uint32_t mine = min(v, vecs - 1);
        if (__all((mine + 1) * V <= g.width))
            add_all([&](const S *row) { return load_whole(row, mine); });
        else
            add_all([&](const S *row) { return load_piece(row, mine, g.width); });
        if (v < vecs)
            write_sum<S>(g, t, v, base, sum, close.words != nullptr);
    }
    program_close_block(close);
}

// The rows at the ends of a window of kLong sorted terms: how many of these are its first key's and its last key's, and how
// many terms more those keys have right before and behind the window (64 for 64 or more). At most two long rows have a part
// that begins in a window: its first key's, unless the row ends before, and its last key's.
struct Window {
    uint32_t lo, hi, first, last, head, tail, before, behind;
    __device__ __forceinline__ Window(const uint32_t *keys, uint32_t n, uint32_t c)
    {
        const uint32_t lane = threadIdx.x & 63;
        lo = c * kLong;
        hi = min(lo + kLong, n);
        const uint32_t m = hi - lo, key = lane < m ? keys[lo + lane] : ~0u;
        first = from_lane(key, 0);
        last = from_lane(key, (int)m - 1);
        const uint64_t in = (1ull << m) - 1; // m <= 48
        head = (uint32_t)__builtin_ctzll(~(__ballot(key == first) & in));
        tail = (uint32_t)__builtin_clzll(~((__ballot(key == last) & in) << (64 - m)));
        before = run_length(lane < lo ? keys[lo - 1 - lane] : ~0u, first);
        behind = run_length(hi + lane < n ? keys[hi + lane] : ~0u, last);
    }
    static __device__ __forceinline__ uint32_t run_length(uint32_t key, uint32_t of)
    {
        const uint64_t other = ~__ballot(key == of);
        return other ? (uint32_t)__builtin_ctzll(other) : 64;
    }
    __device__ __forceinline__ bool head_long() const { return before + head + (head == hi - lo ? behind : 0) > kLong; }
    __device__ __forceinline__ bool tail_long() const { return tail + behind + (tail == hi - lo ? before : 0) > kLong; }
};

// The sum of terms [lo, hi), vector vec, of a wave whose groups of `lanes` lanes take a share each.
template <typename S>
__device__ __forceinline__ void leave_part(const EmbedBackArgs &g, const uint32_t *places, uint32_t lo, uint32_t hi, int lanes, uint32_t vec,
                                           bool on, typename StatOf<S>::T *out)
{
    using T = typename StatOf<S>::T;
    constexpr int V = kVec<S>;
    const uint32_t lane = threadIdx.x & 63, subs = 64 / lanes, each = (hi - lo + subs - 1) / subs, sub = lane / lanes;
    const uint32_t a = min(lo + sub * each, hi), b = min(a + each, hi);
    T sum[V] = {};
    if (on)
        add_terms<S>(g, places, a, b, vec, sum);
    T all[V];
#pragma unroll
    for (int e = 0; e < V; e++) {
        all[e] = __shfl(sum[e], lane & (lanes - 1));
        for (uint32_t k = 1; k < subs; k++)
            all[e] += __shfl(sum[e], (lane & (lanes - 1)) + k * lanes);
        if (on && sub == 0)
            out[e] = all[e];
    }
}

// Workgroups [0, runs): waves with the rows that begin in their terms; [runs, parts): waves that leave the
// sums of the long rows' parts that begin in window c, its first row's in slot 2 c and its last row's in 2 c + 1, a
// wave each (2560 tokens, 111 x 384: a call of 53 us with one wave for both, 44 so); the others fill the rows that do not
// occur. A wave takes 64 vectors of the rows, of `across`.
template <typename S, bool BASE>
__global__ __launch_bounds__(256) void k_embed_sum(EmbedBackArgs g, const uint32_t *keys, const uint32_t *places, int lanes,
                                                   uint32_t across, uint32_t runs, uint32_t parts, uint64_t each, void *sums)
{
    using T = typename StatOf<S>::T;
    if (block_gate_closed(g.gate))
        return;
    if (blockIdx.x >= parts) {
        fill_rows<S>(g, keys, blockIdx.x - parts, each, false);
        return;
    }
    const uint32_t n = (uint32_t)g.rows, vecs = (g.width + kVec<S> - 1) / kVec<S>, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const bool of_runs = blockIdx.x < runs;
    const uint32_t unit = (blockIdx.x - (of_runs ? 0 : runs)) * 4 + wave, slot = unit / across;
    const uint32_t vec = unit % across * 64 + (threadIdx.x & (lanes - 1));
    if (of_runs) {
        if (slot * kStarts < n)
            sum_runs<S, BASE>(g, keys, places, slot, lanes, vec, vec < vecs);
        return;
    }
    const uint32_t c = slot / 2;
    if (c * kLong >= n)
        return;
    const Window p(keys, n, c);
    uint32_t at = n, end = n;
    if (slot & 1) {
        if (p.last != p.first && p.last < g.vocab && p.tail_long()) {
            at = p.hi - p.tail;
            end = at + kLong;
        }
    } else if (p.first < g.vocab && p.head_long()) {
        const uint32_t start = p.before < 64 ? p.lo - p.before : lower_bound(keys, 0, p.lo, p.first); // of the row
        at = start + (p.lo - start + kLong - 1) / kLong * kLong;
        end = min(at + kLong, p.lo + p.head + (p.lo + p.head == p.hi ? p.behind : 0));
    }
    if (at < end)
        leave_part<S>(g, places, at, end, lanes, vec, vec < vecs, static_cast<T *>(sums) + ((uint64_t)slot * vecs + vec) * kVec<S>);
}

// The long rows, each by the window in which it begins.
template <typename S>
__global__ __launch_bounds__(256) void k_embed_join(EmbedBackArgs g, const uint32_t *keys, int lanes, uint32_t across, const void *sums)
{
    using T = typename StatOf<S>::T;
    constexpr int V = kVec<S>;
    if (block_gate_closed(g.gate))
        return;
    const uint32_t n = (uint32_t)g.rows, vecs = (g.width + V - 1) / V, unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t c = unit / across, vec = unit % across * 64 + (threadIdx.x & 63);
    if (c * kLong >= n)
        return;
    const Window p(keys, n, c);
    if (p.last >= g.vocab || !p.tail_long() || (p.tail == p.hi - p.lo && p.before > 0))
        return;
    const uint32_t end = p.behind < 64 ? p.hi + p.behind : lower_bound(keys, p.hi, n - p.hi, p.last + 1);
    if (vec >= vecs || (threadIdx.x & 63) >= (uint32_t)lanes)
        return;
    const T *from = static_cast<const T *>(sums) + (uint64_t)vec * V;
    const uint64_t part = (uint64_t)vecs * V;
    const uint32_t more = (end - (p.hi - p.tail) - 1) / kLong; // parts after the first, one a window
    T sum[V];
#pragma unroll
    for (int e = 0; e < V; e++)
        sum[e] = from[(2 * (uint64_t)c + (p.first == p.last ? 0 : 1)) * part + e];
    constexpr uint32_t U = 8;
    for (uint32_t j = 1; j <= more; j += U) {
        T x[U][V];
#pragma unroll
        for (uint32_t q = 0; q < U; q++)
            if (j + q <= more)
#pragma unroll
                for (int e = 0; e < V; e++)
                    x[q][e] = from[2 * (uint64_t)(c + j + q) * part + e];
#pragma unroll
        for (uint32_t q = 0; q < U; q++)
            if (j + q <= more)
#pragma unroll
                for (int e = 0; e < V; e++)
                    sum[e] += x[q][e];
    }
    write_sum<S>(g, p.last, vec, load_base<S>(g, p.last, vec), sum);
}

// What the gradient's scratch holds: sorted keys and places, those of the first pass, the tiles'
// digit counts and the launch's, and the long rows' parts.
struct EmbedPlan {
    int bits;             // of each of the two digits
    uint32_t tiles, lds;  // of the sort
    bool one;             // a single workgroup sorts
    uint64_t keys, counts, totals, parts, bytes;
    explicit EmbedPlan(const EmbedBackArgs &g)
    {
        bytes = 0;
        if (g.rows <= kDirect) // no sort
            return;
        bits = 1;
        while ((1ull << (2 * bits)) <= g.vocab) // the largest key is vocab
            bits++;
        const uint64_t bins = 1ull << bits;
        tiles = (uint32_t)((g.rows + kSortTile - 1) / kSortTile);
        lds = (uint32_t)((bins * (1 + kSortWaves) + kSortWaves) * 4);
        one = g.rows <= kSortTile ? bits <= 11 : g.rows <= kSortAlone && bits <= 10; // keys and places fit beside the counts in 160 KiB
        const int size = logit_size_of(g.dtype);
        const uint64_t vecs = ((uint64_t)g.width * size + 15) / 16, stat = size == 8 ? 8 : 4;
        auto take = [&](uint64_t n) {
            const uint64_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        keys = take(4 * 4 * g.rows);
        counts = take(one ? 0 : bins * tiles * 4);
        totals = take(one ? 0 : bins * 4);
        parts = take((g.rows + kLong - 1) / kLong * 2 * vecs * (16 / size) * stat);
    }
};

// Tiles whose counts the moving workgroups add up themselves.
constexpr uint32_t kFewTiles = 32;

// A kernel whose LDS is beyond what a launch may have unasked.
template <typename K> hipError_t allow_lds(K *kernel, uint32_t bytes)
{
    return bytes > 65536 ? hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)
                         : hipSuccess;
}

template <int THREADS, int ROUNDS> hipError_t sort_alone(hipStream_t s, const EmbedBackArgs &g, int bits, uint32_t *keys, uint32_t *places)
{
    constexpr uint32_t W = THREADS / 64;
    const uint32_t bins = 1u << bits, lds = (bins * (1 + W) + W + 2 * THREADS * ROUNDS) * 4;
    const hipError_t e = allow_lds(k_sort_one<THREADS, ROUNDS>, lds);
    if (e)
        return e;
    hipLaunchKernelGGL((k_sort_one<THREADS, ROUNDS>), dim3(1), dim3(THREADS), lds, s, g, bits, keys, places);
    return hipGetLastError();
}

template <typename S> hipError_t launch_embed_back_t(hipStream_t s, EmbedBackArgs g, void *scratch, ProgramClose close, bool *closed)
{
    const EmbedPlan p(g);
    const uint32_t vecs = (g.width + kVec<S> - 1) / kVec<S>;
    const int lanes = row_lanes(vecs);
    const uint32_t across = (vecs + lanes - 1) / lanes;
    // Vectors of the table that are filled, if no row keeps its place, by how many workgroups.
    const uint64_t all = g.base && g.base == g.out ? 0 : (uint64_t)g.vocab * vecs, wanted = (all + 1023) / 1024;
    const uint64_t fill = wanted < kFillBlocks ? wanted : kFillBlocks, each = fill ? ((all + fill - 1) / fill + 255) / 256 * 256 : 0;
    if (g.rows <= kDirect) {
        const uint32_t sums = (uint32_t)((g.rows * across + 3) / 4), blocks = sums + (uint32_t)fill;
        if (blocks == 0)
            return hipSuccess;
        if (blocks > kCloseMaxBlocks)
            close = ProgramClose{};
        *closed = close.words != nullptr;
        hipLaunchKernelGGL((k_embed_first<S>), dim3(blocks), dim3(256), 0, s, g, across, sums, each, close);
        return hipGetLastError();
    }
    // Where every row is read and written, storing past the caches is the faster way (32768 tokens,
    // 32000 x 2048 bf16 with a base: 129 and 162 us).
    g.past = g.base && (uint64_t)g.vocab * g.width * sizeof(S) > 64u << 20;
    char *sc = static_cast<char *>(scratch);
    uint32_t *keys = reinterpret_cast<uint32_t *>(sc + p.keys), *places = keys + g.rows;
    uint32_t *mid_keys = places + g.rows, *mid_places = mid_keys + g.rows;
    uint32_t *counts = reinterpret_cast<uint32_t *>(sc + p.counts), *totals = reinterpret_cast<uint32_t *>(sc + p.totals);
    hipError_t e;
    if (p.one) {
        if ((e = g.rows <= kSortTile ? sort_alone<kSortThreads, kSortRounds>(s, g, p.bits, keys, places)
                                     : sort_alone<1024, kSortAlone / 1024>(s, g, p.bits, keys, places)))
            return e;
    } else {
        if ((e = allow_lds(k_sort_move, p.lds)))
            return e;
        const uint32_t bins = 1u << p.bits;
        for (int pass = 0; pass < 2; pass++) {
            const uint32_t *in = pass ? mid_keys : nullptr;
            hipLaunchKernelGGL(k_sort_count, dim3(p.tiles), dim3(kSortThreads), bins * 4, s, g, in, pass * p.bits, p.bits, counts);
            if (p.tiles > kFewTiles)
                hipLaunchKernelGGL(k_sort_scan, dim3(bins), dim3(kSortThreads), 0, s, g, p.bits, p.tiles, counts, totals);
            hipLaunchKernelGGL(k_sort_move, dim3(p.tiles), dim3(kSortThreads), p.lds, s, g, in, pass ? mid_places : nullptr,
                               pass * p.bits, p.bits, counts, p.tiles > kFewTiles ? totals : nullptr, p.tiles, pass ? keys : mid_keys, pass ? places : mid_places);
        }
    }
    const uint32_t runs = (uint32_t)(((g.rows + kStarts - 1) / kStarts * across + 3) / 4);
    const uint64_t windows = (g.rows + kLong - 1) / kLong;
    const uint32_t parts = (uint32_t)((windows * 2 * across + 3) / 4), joins = (uint32_t)((windows * across + 3) / 4);
    const dim3 grid(runs + parts + (uint32_t)fill);
    if (g.base)
        hipLaunchKernelGGL((k_embed_sum<S, true>), grid, dim3(256), 0, s, g, keys, places, lanes, across, runs, runs + parts, each, sc + p.parts);
    else
        hipLaunchKernelGGL((k_embed_sum<S, false>), grid, dim3(256), 0, s, g, keys, places, lanes, across, runs, runs + parts, each, sc + p.parts);
    hipLaunchKernelGGL((k_embed_join<S>), dim3(joins), dim3(256), 0, s, g, keys, lanes, across, sc + p.parts);
    return hipGetLastError();
}

// A gradient of no values: its tokens are looked at all the same.
__global__ __launch_bounds__(256) void k_token_check(EmbedBackArgs g, ProgramClose close)
{
    if (block_gate_closed(g.gate))
        return;
    uint64_t key = kNoFault;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < g.rows; i += (uint64_t)gridDim.x * 256) {
        const int32_t t = g.tokens[i];
        if (t >= 0 && (uint32_t)t >= g.vocab && key == kNoFault)
            key = pack_fault(i, kInvalid);
    }
    wave_record_fault(key, g.fault, g.gate);
    program_close_block(close);
}

hipError_t launch_token_check(hipStream_t s, const EmbedBackArgs &g, ProgramClose close, bool *closed)
{
    if (g.rows == 0)
        return hipSuccess;
    const uint64_t need = (g.rows + 255) / 256;
    const unsigned blocks = (unsigned)(need < 2048 ? need : 2048);
    if (blocks > kCloseMaxBlocks)
        close = ProgramClose{};
    *closed = close.words != nullptr;
    hipLaunchKernelGGL(k_token_check, dim3(blocks), dim3(256), 0, s, g, close);
    return hipGetLastError();
}

} // namespace

hipError_t launch_embed(hipStream_t s, const EmbedArgs &g, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.rows == 0)
        return hipSuccess;
    switch (g.dtype) { // (rows without columns have tokens to check)
    case kLogitF32: return launch_embed_t<float>(s, g, close, closed);
    case kLogitF64: return launch_embed_t<double>(s, g, close, closed);
    case kLogitBf16: return launch_embed_t<__bf16>(s, g, close, closed);
    default: return launch_embed_t<_Float16>(s, g, close, closed);
    }
}

size_t embed_back_scratch_bytes(const EmbedBackArgs &g) { return g.width && g.vocab ? EmbedPlan(g).bytes : 0; }

hipError_t launch_embed_back(hipStream_t s, const EmbedBackArgs &g, void *scratch, ProgramClose close, bool *closed)
{
    *closed = false;
    if (g.width == 0 || g.vocab == 0)
        return launch_token_check(s, g, close, closed);
    switch (g.dtype) {
    case kLogitF32: return launch_embed_back_t<float>(s, g, scratch, close, closed);
    case kLogitF64: return launch_embed_back_t<double>(s, g, scratch, close, closed);
    case kLogitBf16: return launch_embed_back_t<__bf16>(s, g, scratch, close, closed);
    default: return launch_embed_back_t<_Float16>(s, g, scratch, close, closed);
    }
}

} // namespace pcu
