// Pieces of rows whose length is no multiple of 16 bytes.
#pragma once

#include "pcu_logits.hpp"

namespace pcu {

// Vector i of a row of n values; places past the row's end read as zero, vectors past it too. The
// last, partial one is the row's last 16 bytes, moved down: one load, where value by value takes as many
// trips to memory (6572 tokens of 62 bfloat16 values: 42 us for the sums, 23 now).
template <typename S> __device__ __forceinline__ u32x4 load_piece(const S *row, uint32_t i, uint32_t n)
{
    constexpr uint32_t V = kVec<S>;
    const uint32_t at = i * V;
    if (at + V <= n)
        return load_whole(row, i);
    u32x4 raw = {0, 0, 0, 0};
    if (at >= n)
        return raw;
    if (n >= V) {
        const u32x4 last = *reinterpret_cast<const u32x4_any *>(row + (n - V));
        const uint64_t lo = (uint64_t)last[1] << 32 | last[0], hi = (uint64_t)last[3] << 32 | last[2];
        const uint32_t bits = (at + V - n) * 8 * (uint32_t)sizeof(S); // 16 .. 112
        const uint64_t a = bits < 64 ? lo >> bits | hi << (64 - bits) : hi >> (bits - 64), b = bits < 64 ? hi >> bits : 0;
        return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)};
    }
    // A row shorter than a vector.
#pragma unroll
    for (uint32_t e = 0; e < V; e++)
        if (at + e < n) {
            if constexpr (sizeof(S) == 2)
                raw[e / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[at + e]) << (16 * (e & 1));
            else
#pragma unroll
                for (uint32_t w = 0; w < sizeof(S) / 4; w++)
                    raw[e * (sizeof(S) / 4) + w] = reinterpret_cast<const uint32_t *>(row + at + e)[w];
        }
    return raw;
}

} // namespace pcu
