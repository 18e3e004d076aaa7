// Argument checks that the native operators' entry points share.
#pragma once

#include "pcu_runtime.hpp"

#include <cmath>

namespace pcu {

inline uint64_t logit_size(uint32_t dtype) { return dtype == PCU_F64 ? 8 : dtype == PCU_F32 ? 4 : 2; }
inline uint64_t stat_size(uint32_t dtype) { return dtype == PCU_F64 ? 8 : 4; }

// A pointer to values of `size` bytes: the kernels load and store them whole (null passes).
inline bool aligned(const void *p, uint64_t size) { return ((uintptr_t)p & (size - 1)) == 0; }

// Bytes from the first element of `rows` strided rows of `cols` to past the last one.
inline uint64_t strided_bytes(uint64_t rows, uint64_t cols, uint64_t stride, uint64_t size)
{
    return rows && cols ? ((rows - 1) * stride + cols) * size : 0;
}

// A weight that is a number in the statistics' type.
inline bool valid_weight(uint32_t dtype, double weight)
{
    return dtype == PCU_F64 ? std::isfinite(weight) : std::isfinite((float)weight);
}

// An output against one input.
struct Range {
    const void *p;
    uint64_t bytes;
};
template <size_t N> bool overlaps_any(Range out, const Range (&in)[N])
{
    for (const Range &r : in)
        if (ranges_overlap(out.p, out.bytes, r.p, r.bytes))
            return true;
    return false;
}

// Opens a call on `ctx` as the other op entry points do.
inline Ctx *enter(pcu_ctx *ctx, pcu_status *st)
{
    Ctx *c = reinterpret_cast<Ctx *>(ctx);
    if (!c) {
        g_thread_error = "null context";
        *st = PCU_ERR_ARGUMENT;
        return nullptr;
    }
    *st = c->start_op();
    return *st ? nullptr : c;
}

} // namespace pcu
