// Matrix-core tiles of the output layer's cross entropy (gfx950): 16-bit operands, F32 sums.
//
// A workgroup makes a BM x BN tile of C = A B, k in slabs of K. An operand's slab lies in LDS as
// it lies in memory, either k-contiguous (K values of a row of A or column of B side by side) or k-major
// (`T`: K rows of BM or BN values), and comes there by direct loads, one or more slabs ahead, or (A
// alone, where its rows do not start at multiples of 16 bytes or end inside a slab) through registers. A lane of the
// 16 x 16 x 32 instruction takes 8 consecutive k of one row or column: one 16-byte read of a
// k-contiguous slab, two transposing 8-byte reads of a k-major one. The 16-byte pieces of a slab's
// row are permuted by the row (in the loads' addresses, so that LDS stays dense): by half of it (a
// quarter in slabs of 32) where k is contiguous, and by twice its bits 0, 1 and 3 where it is k-major, so that the 16 lanes (32 of
// a transposing read) that are served at once touch all 256 bytes of LDS's banks.
//
// What bounds the tiles is power: the clock falls to 1.7 GHz under them. On random values the
// 16 x 16 x 32 instruction alone reaches 2290 TFLOP/s, the 32 x 32 x 16 one 1940 (both 2400 on zeros).
#pragma once

#include "pcu_gemm_stage.hpp"
#include "pcu_logits.hpp"

#pragma clang fp contract(off)

namespace pcu {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename E> __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c)
{
    if constexpr (__is_same(E, __bf16))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr int kSlabK = 64; // operands are padded to whole slabs of the longer kind

// Binary32 operands come as three parts of 8 bits, exact together: the value rounded to 8 bits, then its rest. A rest
// is at most half a step, so the second part is at most 2^-8 of the value and the third 2^-17. Of the nine
// products of two operands' parts the three smallest are left out: at most 2 * 2^-25 + 2^-34 of the whole together, of
// either sign (normal values: 0.9 * 2^-24 at most, 0 on average; parts cut off instead of rounded left out up to
// 8 * 2^-24, always towards zero, 0.7 * 2^-24 on average, and took a loss of 2 rows, 83776 x 3648, 351 us instead of 359). Small ones are added first. All
// parts of a slab lie in LDS at once: 6 products for 3 + 3 parts read. (Parts pair by pair through the
// 16-bit tiles: 1024 x 50257 x 768 1.93 ms a step, 64 x 1000 x 64 55 us; so 1.73 ms and 40.)
constexpr int kPartPairs = 6;
__device__ constexpr int kPartA[kPartPairs] = {2, 0, 1, 1, 0, 0}, kPartB[kPartPairs] = {0, 2, 1, 0, 1, 0};

// From here on 8 bits round to infinity; such a value's first part is cut off instead.
constexpr uint32_t kLeastCut = 0x7f7f8000u;

// A value rounded to its first 8 bits (of its rest: part 1 and 2), as a bfloat16; v becomes what is left. An infinity is
// (1, 0, infinity), each with its sign: of the products that are kept, its last part meets the other operand's first
// part alone, which is zero only if the value is, and its first part gives two infinities their product. (As a first
// part it would meet the zeros that follow every value of few bits, and their product is NaN.) A NaN is its first part.
__device__ __forceinline__ uint32_t next_part(float &v, int part)
{
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7f800000u) == 0x7f800000u) {
        const bool nan = b & 0x7fffffu;
        return part == 0 ? (b >> 16 & 0x8000u) | (nan ? 0x7fc0u : 0x3f80u) : part == 2 && !nan ? b >> 16 : 0u;
    }
    const uint32_t to = part < 2 && (b & 0x7fffffffu) < kLeastCut ? b + 0x8000u : b; // (the last rest has 8 bits)
    v -= __uint_as_float(to & 0xffff0000u); // exact
    return to >> 16;
}

// Part `part` of two values below kLeastCut, side by side; they become what is left.
__device__ __forceinline__ uint32_t next_parts(float &a, float &b, int part)
{
    const uint32_t half = part < 2 ? 0x8000u : 0u, lo = __float_as_uint(a) + half, hi = __float_as_uint(b) + half;
    if (part < 2) { // exact
        a -= __uint_as_float(lo & 0xffff0000u);
        b -= __uint_as_float(hi & 0xffff0000u);
    }
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

// The parts of 8 values.
__device__ __forceinline__ void split8(const float (&v)[8], u32x4 (&raw)[3])
{
    uint32_t most = 0;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
        x[e] = v[e];
    }
    if (most < kLeastCut) {
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                raw[k][e / 2] = next_parts(x[e], x[e + 1], k);
    } else {
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                raw[k][e / 2] = next_part(x[e], k) | next_part(x[e + 1], k) << 16;
    }
}

// WM x WN waves, each with SM x SN subtiles of 16 x 16; slabs of K, STAGES of them in LDS, of PARTS parts.
template <int WM_, int WN_, int SM_, int SN_, int K_, int STAGES, int PARTS> struct EntropyCfg {
    static constexpr int WM = WM_, WN = WN_, SM = SM_, SN = SN_, K = K_, kStages = STAGES, kParts = PARTS;
    static_assert((K == 32 || K == 64) && (PARTS == 1 || PARTS == 3), "slabs");
    static constexpr int BM = WM * SM * 16, BN = WN * SN * 16, kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int kSlabA = BM * K * 2, kSlabB = BN * K * 2, kStage = PARTS * (kSlabA + kSlabB); // bytes
    static constexpr int kOutPitch = BM + 8; // of a 16-bit output tile in LDS, in values
    static constexpr int kTile = kStages * kStage > BN * kOutPitch * 2 ? kStages * kStage : BN * kOutPitch * 2;
    static constexpr int kReduce = WM * BN * 8; // bytes for a reduction over the tile's rows
    static constexpr int kLds = kTile + kReduce;
    static_assert(kLds + 64 <= 160 * 1024, "LDS");
};
// Where acc[i][j][r] of a lane lies in its wave's tile.
__device__ __forceinline__ uint32_t acc_row(int i, int r) { return 16 * i + 4 * ((threadIdx.x & 63) / 16) + r; }
__device__ __forceinline__ uint32_t acc_col(int j) { return 16 * j + (threadIdx.x & 15); }

// One operand: `ld` values from row to row (k-contiguous: rows of C; k-major: k), `plane` from one
// 16-bit part of a binary32 operand to the next. Past `rows` rows and (k-major) `cols` columns the last
// ones are read again: what they give is not stored, or meets zeros in the other operand.
// Through registers, what lies past `cols` (of k, too) is zero and never read.
struct EntropyOperand {
    const uint16_t *p = nullptr;
    uint64_t plane = 0;
    uint32_t ld = 0, rows = 0, cols = 0;
};

// How the pieces of a k-major slab's row are permuted.
__device__ __forceinline__ uint32_t k_major_swap(uint32_t k) { return 2 * ((k & 3) | (k >> 1 & 4)); }

__device__ __forceinline__ uint32_t k_contiguous_swap(uint32_t row, int k) { return k == 64 ? row / 2 & 7 : row / 4 & 3; }

// What operands that go through registers are made of.
template <int PARTS> struct SourceOf { typedef uint16_t T; };
template <> struct SourceOf<3> { typedef uint32_t T; };

template <class Cfg, int ROWS, bool T> struct SlabLoader {
    static constexpr int K = Cfg::K, IPW = ROWS * K / 512 / Cfg::kWaves; // 1 KiB loads a wave and part
    static_assert(IPW * 512 * Cfg::kWaves == ROWS * K, "every wave loads as much");
    static constexpr int kPieces = (T ? ROWS : K) / 8; // 16-byte pieces of a row
    static_assert(!T || kPieces >= 16, "the permutation stays within a row");
    uint32_t off[IPW];
    __device__ __forceinline__ int row_of(int wave, int q) const { return ((wave * IPW + q) * 64 + (threadIdx.x & 63)) / kPieces; }
    // at: the tile's first row (k-contiguous) or column (k-major).
    __device__ __forceinline__ void init(const EntropyOperand &o, uint32_t at, int wave)
    {
        const uint32_t piece = (threadIdx.x & 63) % kPieces;
#pragma unroll
        for (int q = 0; q < IPW; q++) {
            const uint32_t r = row_of(wave, q);
            if constexpr (!T)
                off[q] = min(r, o.rows - 1 - at) * o.ld * 2 + (piece ^ k_contiguous_swap(r, K)) * 16;
            else
                off[q] = r * o.ld * 2 + min((piece ^ k_major_swap(r)) * 8, o.cols - 8 - at) * 2;
        }
    }
    // The slab of k0, all its parts, into `lds`.
    __device__ __forceinline__ void load(const EntropyOperand &o, uint32_t at, uint32_t k0, uint32_t lds, int wave) const
    {
        // Past the last row (padding to whole slabs) the last one is read again.
        const bool over = T && k0 + K > o.rows;
        const uint32_t k1 = T ? min(k0, o.rows - 1) : k0;
#pragma unroll
        for (int part = 0; part < Cfg::kParts; part++) {
            const uint16_t *base = o.p + part * o.plane + (T ? (uint64_t)k1 * o.ld + at : (uint64_t)at * o.ld + k0);
#pragma unroll
            for (int q = 0; q < IPW; q++) {
                uint32_t from = off[q];
                if (T && over) {
                    const uint32_t k = row_of(wave, q), to = min(k0 + k, o.rows - 1) - k1;
                    from -= (k - to) * o.ld * 2;
                }
                load_lds<4>(base, from, __builtin_amdgcn_readfirstlane(lds + part * ROWS * K * 2 + (wave * IPW + q) * 1024));
            }
        }
    }
};

// The same through registers, for rows at any alignment of their type and of any length. Where tiles take
// three parts, the rows are binary32 values (`p` points to those) and are split here.
template <class Cfg, int ROWS, bool T> struct SlabCarrier {
    static constexpr int K = Cfg::K, IPW = ROWS * K / 512 / Cfg::kWaves, kPieces = (T ? ROWS : K) / 8;
    static constexpr int kHeld = Cfg::kParts == 3 ? 2 : 1; // 16-byte vectors of 8 values
    typedef typename SourceOf<Cfg::kParts>::T Source;
    static constexpr int kLoads = IPW * kHeld;
    u32x4 held[IPW][kHeld];
    // Takes kLoads loads, or more where this is true.
    static __device__ __forceinline__ bool is_ragged(const EntropyOperand &o, uint32_t at, uint32_t k0) { return (T ? at + ROWS : k0 + K) > o.cols; }
    __device__ __forceinline__ void fetch(const EntropyOperand &o, uint32_t at, uint32_t k0, int wave)
    {
        const uint32_t lane = threadIdx.x & 63;
        const bool ragged = is_ragged(o, at, k0);
#pragma unroll
        for (int q = 0; q < IPW; q++) {
            const uint32_t r = ((wave * IPW + q) * 64 + lane) / kPieces, piece = lane % kPieces;
            const uint32_t row = min((T ? k0 : at) + r, o.rows - 1);
            const uint32_t c = (T ? at : k0) + (T ? piece ^ k_major_swap(r) : piece ^ k_contiguous_swap(r, K)) * 8;
            const Source *from = reinterpret_cast<const Source *>(o.p) + (uint64_t)row * o.ld + c;
            if (!ragged || c + 8 <= o.cols) {
#pragma unroll
                for (int h = 0; h < kHeld; h++)
                    held[q][h] = *reinterpret_cast<const u32x4_any *>(from + h * (8 / kHeld));
            } else {
                u32x4 raw[kHeld] = {};
#pragma unroll
                for (uint32_t e = 0; e < 8; e++)
                    if (c + e < o.cols) {
                        if constexpr (kHeld == 2)
                            raw[e / 4][e % 4] = from[e];
                        else
                            raw[0][e / 2] |= (uint32_t)from[e] << (16 * (e & 1));
                    }
#pragma unroll
                for (int h = 0; h < kHeld; h++)
                    held[q][h] = raw[h];
            }
        }
    }
    __device__ __forceinline__ void stash(char *slab, int wave) const
    {
#pragma unroll
        for (int q = 0; q < IPW; q++) {
            char *to = slab + (wave * IPW + q) * 1024 + (threadIdx.x & 63) * 16;
            if constexpr (kHeld == 2) {
                float v[8];
                u32x4 raw[3];
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] = __uint_as_float(held[q][e / 4][e % 4]);
                split8(v, raw);
#pragma unroll
                for (int part = 0; part < 3; part++)
                    *reinterpret_cast<u32x4 *>(to + part * ROWS * K * 2) = raw[part];
            } else {
                *reinterpret_cast<u32x4 *>(to) = held[q][0];
            }
        }
    }
};

// Fragments of an operand's slab (one part): subtile i of S, 32 values of k from 32 kk on.
template <int K, int ROWS, int S, bool T> struct SlabReader {
    uint32_t at[T ? S : K / 32];
    // first: the wave's first row or column of the slab.
    __device__ __forceinline__ void init(uint32_t first)
    {
        const uint32_t lane = threadIdx.x & 63;
        if constexpr (!T) {
            // Row first + lane % 16, piece 4 kk + lane / 16.
#pragma unroll
            for (int kk = 0; kk < K / 32; kk++)
                at[kk] = (first + (lane & 15)) * K * 2 + (((4 * kk + lane / 16) ^ k_contiguous_swap(lane & 15, K)) * 16);
        } else {
            // Lanes 16 g ..: k 8 g .. of 16 columns; a lane reads 4 columns of row j / 4.
            const uint32_t j = lane & 15, g = lane / 16, row = 8 * g + j / 4;
#pragma unroll
            for (int i = 0; i < S; i++) {
                const uint32_t c = (first + 16 * i) / 8 + (j & 3) / 2;
                at[i] = row * ROWS * 2 + ((c ^ k_major_swap(row)) * 16) + (j & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ s16x8 read(const char *slab, int i, int kk) const
    {
        if constexpr (!T) {
            return *reinterpret_cast<const s16x8 *>(slab + at[kk] + i * 16 * K * 2);
        } else {
            const char *p = slab + at[i] + kk * 32 * ROWS * 2;
            typedef __attribute__((address_space(3))) s16x4 *P;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * ROWS * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// Tile (tm, tn) and split of workgroup `bid`: workgroups go round-robin to the 8 XCDs, so each of
// those gets a contiguous run of the order, in which 8 tile-rows share each of B's panels.
struct EntropyTile {
    uint32_t tm, tn, split;
};
__device__ __forceinline__ EntropyTile entropy_tile(uint32_t bid, uint32_t tiles_m, uint32_t tiles_n, uint32_t splits)
{
    const uint32_t all = tiles_m * tiles_n * splits, xcd = bid % 8;
    uint32_t l = xcd * (all / 8) + min(xcd, all % 8) + bid / 8;
    EntropyTile t;
    t.split = l / (tiles_m * tiles_n);
    l %= tiles_m * tiles_n;
    const uint32_t per = 8 * tiles_n, first = l / per * 8, rows = min(tiles_m - first, 8u);
    t.tm = first + l % per % rows;
    t.tn = l % per / rows;
    return t;
}

// acc = the tile of A B over slabs [k_lo, k_hi). a, b: the operands; m0, n0: the tile's first row and
// column; lds: Cfg::kTile bytes. CARRY: A goes through registers. No LDS is read after
// the last barrier.
template <typename E, class Cfg, bool TA, bool TB, bool CARRY>
__device__ __forceinline__ void entropy_product(const EntropyOperand &a, const EntropyOperand &b, uint32_t m0, uint32_t n0, uint32_t k_lo,
                                                uint32_t k_hi, char *lds, f32x4 (&acc)[Cfg::SM][Cfg::SN])
{
    constexpr int SM = Cfg::SM, SN = Cfg::SN, K = Cfg::K;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    SlabLoader<Cfg, Cfg::BM, TA> la;
    SlabCarrier<Cfg, Cfg::BM, TA> ca;
    SlabLoader<Cfg, Cfg::BN, TB> lb;
    SlabReader<K, Cfg::BM, SM, TA> ra;
    SlabReader<K, Cfg::BN, SN, TB> rb;
    if constexpr (!CARRY)
        la.init(a, m0, wave);
    lb.init(b, n0, wave);
    ra.init(wave / Cfg::WN * SM * 16);
    rb.init(wave % Cfg::WN * SN * 16);
#pragma unroll
    for (int i = 0; i < SM; i++)
#pragma unroll
        for (int j = 0; j < SN; j++)
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (k_lo >= k_hi)
        return;
    const uint32_t lds0 = lds_address(lds);
    uint32_t slab = k_lo; // the next one to load
    const uint32_t steps = k_hi - k_lo;
    auto issue = [&](int stage) __attribute__((always_inline)) {
        if constexpr (CARRY)
            ca.fetch(a, m0, slab * K, wave);
        else
            la.load(a, m0, slab * K, lds0 + stage * Cfg::kStage, wave);
        lb.load(b, n0, slab * K, lds0 + stage * Cfg::kStage + Cfg::kParts * Cfg::kSlabA, wave);
        slab++;
    };
    auto compute = [&](int stage) __attribute__((always_inline)) {
        const char *sa = lds + stage * Cfg::kStage, *sb = sa + Cfg::kParts * Cfg::kSlabA;
#pragma unroll
        for (int kk = 0; kk < K / 32; kk++) {
            s16x8 fa[Cfg::kParts][SM], fb[Cfg::kParts][SN];
#pragma unroll
            for (int part = 0; part < Cfg::kParts; part++) {
#pragma unroll
                for (int j = 0; j < SN; j++)
                    fb[part][j] = rb.read(sb + part * Cfg::kSlabB, j, kk);
#pragma unroll
                for (int i = 0; i < SM; i++)
                    fa[part][i] = ra.read(sa + part * Cfg::kSlabA, i, kk);
            }
#pragma unroll
            for (int pair = Cfg::kParts == 1 ? kPartPairs - 1 : 0; pair < kPartPairs; pair++)
#pragma unroll
                for (int i = 0; i < SM; i++)
#pragma unroll
                    for (int j = 0; j < SN; j++)
                        acc[i][j] = mfma16<E>(fa[kPartA[pair]][i], fb[kPartB[pair]][j], acc[i][j]);
        }
    };
    if constexpr (CARRY && Cfg::kParts == 3) {
        // A's slabs two ahead: one in registers while the next one's loads are under way, too (2 rows, vocabulary
        // 83776, width 3648 in binary32: one ahead 396 us, 344 so; 16-bit rows, of which more workgroups share a
        // CU, took 172 us so for 24, 97088 x 3098, 153 below).
        SlabCarrier<Cfg, Cfg::BM, TA> cb;
        auto fetch = [&](SlabCarrier<Cfg, Cfg::BM, TA> &c, uint32_t s) __attribute__((always_inline)) {
            asm volatile("" ::: "memory"); // after B's loads
            if (k_lo + s < k_hi)
                c.fetch(a, m0, (k_lo + s) * K, wave);
            asm volatile("" ::: "memory");
        };
        // Slab s + 1, fetched after B's loads of slab s, may stay under way.
        auto arrive = [&](const SlabCarrier<Cfg, Cfg::BM, TA> &c, int stage, uint32_t s) __attribute__((always_inline)) {
            c.stash(lds + stage * Cfg::kStage, wave);
            if (s + 1 < steps && !c.is_ragged(a, m0, (k_lo + s + 1) * K))
                wait_loads_but<SlabCarrier<Cfg, Cfg::BM, TA>::kLoads>();
            else
                wait_lds_loads();
            __syncthreads();
        };
        auto load_b = [&](int stage, uint32_t s) __attribute__((always_inline)) {
            lb.load(b, n0, (k_lo + s) * K, lds0 + stage * Cfg::kStage + Cfg::kParts * Cfg::kSlabA, wave);
        };
        fetch(ca, 0);
        load_b(0, 0);
        fetch(cb, 1);
        arrive(ca, 0, 0);
        for (uint32_t s = 0; s < steps; s += 2) {
            if (s + 1 < steps)
                load_b(1, s + 1);
            fetch(ca, s + 2);
            compute(0);
            if (s + 1 < steps) {
                arrive(cb, 1, s + 1);
                if (s + 2 < steps)
                    load_b(0, s + 2);
                fetch(cb, s + 3);
                compute(1);
                if (s + 2 < steps)
                    arrive(ca, 0, s + 2);
            }
        }
        __syncthreads();
    } else if constexpr (Cfg::kStages == 2 || CARRY) {
        auto arrive = [&](int stage) __attribute__((always_inline)) {
            if constexpr (CARRY)
                ca.stash(lds + stage * Cfg::kStage, wave); // (again what was fetched last, past the last slab)
            wait_lds_loads();
            __syncthreads();
        };
        issue(0);
        arrive(0);
        // Two slabs a trip, so that each stage's addresses are constants. (The conditions stand where
        // the compiler keeps the sums in registers: leaving the loop amid a trip spilled them.)
        for (uint32_t s = 0; s < steps; s += 2) {
            if (s + 1 < steps)
                issue(1);
            compute(0);
            arrive(1);
            if (s + 1 < steps) {
                if (s + 2 < steps)
                    issue(0);
                compute(1);
                arrive(0);
            }
        }
    } else {
        // kStages - 1 slabs ahead. A slab is there when no more than the later ones' loads are
        // outstanding and every wave has come to the barrier; then every wave is done with the slab
        // before, too, whose stage the next load takes.
        constexpr int N = Cfg::kStages, kLoads = Cfg::kParts * (SlabLoader<Cfg, Cfg::BM, TA>::IPW + SlabLoader<Cfg, Cfg::BN, TB>::IPW);
#pragma unroll
        for (int st = 0; st < N - 1; st++)
            if ((uint32_t)st < steps)
                issue(st);
        for (uint32_t s = 0; s < steps; s += N) {
#pragma unroll
            for (int st = 0; st < N; st++) {
                if (s + st >= steps)
                    break;
                if (s + st + N - 2 < steps)
                    wait_loads_but<(N - 2) * kLoads>();
                else
                    wait_lds_loads();
                __syncthreads();
                if (s + st + N - 1 < steps)
                    issue((st + N - 1) % N);
                compute(st);
            }
        }
        __syncthreads();
    }
}

} // namespace pcu
