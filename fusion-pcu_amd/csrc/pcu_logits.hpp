// Device helpers of the operators on logits (top logits, distillation, sampling): 16-byte
// vectors of a row in any of the four types, reductions over a workgroup and the order of a
// row's values.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pcu_device.hpp"

#pragma clang fp contract(off)

namespace pcu {

// The type that a row's statistics are held in: 32 bits, 64 for binary64 rows.
template <typename S> struct StatOf { using T = float; };
template <> struct StatOf<double> { using T = double; };

// One 16-byte piece of a row. Rows start at any multiple of their type's size (odd
// vocabularies, padded strides), and the hardware loads and stores 16 bytes at any address:
// a misaligned piece costs at most one more cache line for each wave's kilobyte.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename S> constexpr int kVec = 16 / (int)sizeof(S);

// One pass over a row that a thread holds in registers. The compiler would keep what one pass
// unpacks for the next (twice the registers for 16-bit rows, and spills), so each pass unpacks with
// constants that it does not know to be those of the pass before.
struct Pass {
    uint32_t shift = 16, upper = 0xffff0000u, zero = 0;
    static __device__ __forceinline__ Pass fresh()
    {
        Pass p;
        asm volatile("" : "+s"(p.shift), "+s"(p.upper), "+s"(p.zero));
        return p;
    }
};

template <typename S>
__device__ __forceinline__ void unpack(const u32x4 &raw, typename StatOf<S>::T *out, const Pass &p = Pass{})
{
    if constexpr (sizeof(S) == 8) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            out[i] = __longlong_as_double((long long)(((uint64_t)raw[2 * i + 1] << 32) | raw[2 * i]));
    } else if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            out[i] = __uint_as_float(raw[i]);
    } else if constexpr (__is_same(S, __bf16)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            out[2 * i] = __uint_as_float(raw[i] << p.shift);
            out[2 * i + 1] = __uint_as_float(raw[i] & p.upper);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = raw[i] | p.zero;
            out[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w);
            out[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
        }
    }
}

// Between the vectors of a held row: the scheduler otherwise unpacks many of them at once.
__device__ __forceinline__ void one_at_a_time() { __builtin_amdgcn_sched_barrier(0); }

// Values rounded once (to nearest even) to the row's type.
template <typename S> __device__ __forceinline__ u32x4 pack(const typename StatOf<S>::T *v)
{
    u32x4 raw;
    if constexpr (sizeof(S) == 8) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint64_t b = (uint64_t)__double_as_longlong(v[i]);
            raw[2 * i] = (uint32_t)b;
            raw[2 * i + 1] = (uint32_t)(b >> 32);
        }
    } else if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            raw[i] = __float_as_uint(v[i]);
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef S s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x2 two = {v[2 * i], v[2 * i + 1]};
            raw[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, s16x2));
        }
    }
    return raw;
}

template <typename S> __device__ __forceinline__ u32x4 minus_infinities()
{
    if constexpr (sizeof(S) == 8)
        return u32x4{0u, 0xfff00000u, 0u, 0xfff00000u};
    else if constexpr (sizeof(S) == 4)
        return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
    else if constexpr (__is_same(S, __bf16))
        return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
    else
        return u32x4{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};
}

// Whole vector i of a row. The 32-bit byte offset (a row has at most 2^22 values) lets the
// row's address stay in scalar registers.
template <typename S> __device__ __forceinline__ u32x4 load_whole(const S *row, uint32_t i)
{
    return *reinterpret_cast<const u32x4_any *>(reinterpret_cast<const char *>(row) + i * 16u);
}

// The same where a thread holds many vectors of the row: vector `step` + i, `step` the same for
// the workgroup. The address of the step is kept scalar and unknown to the compiler, which
// otherwise adds every step to a 64-bit address in vector registers and keeps those.
template <typename S> __device__ __forceinline__ u32x4 load_held(const S *row, uint32_t step, uint32_t i)
{
    typedef const __attribute__((address_space(1))) char *P;
    P base = (P) reinterpret_cast<const char *>(row) + step * 16u;
    asm volatile("" : "+s"(base));
    return *(const __attribute__((address_space(1))) u32x4_any *)(base + i * 16u);
}
// Stores and loads past the caches that the chip's parts do not share: what a workgroup hands to
// others of its launch, and results of a launch that ends its program itself (the caller may read
// them from another stream before the kernel's own end has written the caches back).
template <typename V> __device__ __forceinline__ void put(V *p, V v)
{
    if constexpr (sizeof(V) == 2)
        __hip_atomic_store(reinterpret_cast<uint16_t *>(p), __builtin_bit_cast(uint16_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else
        __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V> __device__ __forceinline__ V get(const V *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// A vector, as words, or as values where 2-byte values are not aligned to words.
template <typename S> __device__ __forceinline__ void put_vec(S *p, const u32x4 &raw)
{
    if (sizeof(S) == 2 && (reinterpret_cast<uintptr_t>(p) & 2)) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            put(reinterpret_cast<uint16_t *>(p) + e, (uint16_t)(raw[e / 2] >> (e & 1 ? 16 : 0)));
    } else {
#pragma unroll
        for (int w = 0; w < 4; w++)
            put(reinterpret_cast<uint32_t *>(p) + w, raw[w]);
    }
}

__device__ __forceinline__ void apart() { asm volatile(""); }
// THROUGH: the kernel may be one that ends its program.
template <bool THROUGH, typename S>
__device__ __forceinline__ void store_held(S *row, uint32_t step, uint32_t i, const u32x4 &raw, int how)
{
    typedef __attribute__((address_space(1))) char *P;
    typedef __attribute__((address_space(1))) u32x4_any *V;
    P base = (P) reinterpret_cast<char *>(row) + step * 16u;
    asm volatile("" : "+s"(base));
    if (how == kStorePast) {
        apart(); // or the two stores would become one, and an ordinary one
        __builtin_nontemporal_store(raw, (V)(base + i * 16u));
        apart();
    } else if (THROUGH && how == kStoreThrough) {
        put_vec(row + (step + i) * kVec<S>, raw);
    } else {
        *(V)(base + i * 16u) = raw;
    }
}

// Vector i of a row of n values; places past the row's end read as minus infinity, whole
// vectors past it too.
template <typename S> __device__ __forceinline__ u32x4 load_vec(const S *row, uint32_t i, uint32_t n)
{
    const uint32_t at = i * kVec<S>;
    if (at + kVec<S> <= n)
        return load_whole(row, i);
    u32x4 raw = minus_infinities<S>();
    if (at < n) {
        if constexpr (sizeof(S) == 2) {
            for (uint32_t e = 0; at + e < n; e++) {
                const uint32_t b = __builtin_bit_cast(uint16_t, row[at + e]);
                const uint32_t keep = e & 1 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
                for (uint32_t w = 0; w < 4; w++)
                    if (w == e / 2)
                        raw[w] = (raw[w] & keep) | (e & 1 ? b << 16 : b);
            }
        } else {
            constexpr uint32_t W = sizeof(S) / 4;
            const uint32_t *words = reinterpret_cast<const uint32_t *>(row + at);
#pragma unroll
            for (uint32_t w = 0; w < 4; w++)
                if (at + w / W < n)
                    raw[w] = words[w];
        }
    }
    return raw;
}

template <typename S>
__device__ __forceinline__ void store_vec(S *row, uint32_t i, uint32_t n, const typename StatOf<S>::T *v, bool past)
{
    const uint32_t at = i * kVec<S>;
    if (at + kVec<S> <= n) {
        if (past) {
            apart();
            __builtin_nontemporal_store(pack<S>(v), reinterpret_cast<u32x4_any *>(reinterpret_cast<char *>(row) + i * 16u));
            apart();
        } else
            *reinterpret_cast<u32x4_any *>(reinterpret_cast<char *>(row) + i * 16u) = pack<S>(v);
    } else {
#pragma unroll
        for (int e = 0; e < kVec<S>; e++)
            if (at + e < n)
                row[at + e] = (S)v[e];
    }
}

// One workgroup a row: a launch's threads have to stay below 2^32 along each axis of its grid, so many
// rows take its second axis too. Rows past the last one (~0 below) have workgroups without work.
constexpr uint32_t kRowsAlong = 1u << 20;
inline dim3 row_grid(uint64_t rows)
{
    return rows <= kRowsAlong ? dim3((unsigned)rows) : dim3(kRowsAlong, (unsigned)((rows + kRowsAlong - 1) / kRowsAlong));
}
__device__ __forceinline__ uint32_t row_of_block() { return blockIdx.y * kRowsAlong + blockIdx.x; }

// --------------------------------------------------------- reductions of a workgroup
struct OpMax {
    template <typename T> __device__ __forceinline__ T none() const { return (T)-INFINITY; }
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
};
struct OpSum {
    template <typename T> __device__ __forceinline__ T none() const { return (T)0; }
    template <typename T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct OpOr {
    template <typename T> __device__ __forceinline__ T none() const { return (T)0; }
    template <typename T> __device__ __forceinline__ T operator()(T a, T b) const { return a | b; }
};

// v of the lane that DPP control C names, `none` where there is none or row mask M leaves the
// lane's row of 16 out.
template <int C, int M, typename T> __device__ __forceinline__ T dpp(T none, T v)
{
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), C, M, 0xf, false));
    } else {
        const uint64_t n = __builtin_bit_cast(uint64_t, none), x = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)n, (int)(uint32_t)x, C, M, 0xf, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(n >> 32), (int)(x >> 32), C, M, 0xf, false);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    }
}
// v folded over lanes 0 .. own, in one fixed order (`none` is op's neutral value). Shifts within
// rows of 16 lanes, then the rows' totals handed on: no LDS.
template <typename T, typename Op> __device__ __forceinline__ T wave_upto(T v, Op op, T none)
{
    v = op(dpp<0x111, 0xf>(none, v), v); // row_shr:1
    v = op(dpp<0x112, 0xf>(none, v), v);
    v = op(dpp<0x114, 0xf>(none, v), v);
    v = op(dpp<0x118, 0xf>(none, v), v);
    v = op(dpp<0x142, 0xa>(none, v), v); // row_bcast:15 to rows 1 and 3
    v = op(dpp<0x143, 0xc>(none, v), v); // row_bcast:31 to rows 2 and 3
    return v;
}
template <typename T> __device__ __forceinline__ T from_lane(T v, int lane)
{
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const uint64_t x = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    }
}
template <typename T, typename Op> __device__ __forceinline__ T wave_reduce(T v, Op op)
{
    return from_lane(wave_upto(v, op, op.template none<T>()), 63);
}

// Every thread gets the result, folded in one fixed order. `lds`: NT / 64 entries that no
// other reduction between the same two barriers uses.
template <int NT, typename T, typename Op> __device__ __forceinline__ T block_reduce(T v, Op op, T *lds)
{
    v = wave_reduce(v, op);
    if constexpr (NT == 64)
        return v;
    if ((threadIdx.x & 63) == 0)
        lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++)
        v = op(v, lds[w]);
    return v;
}

// ------------------------------------------------------------------ exponentials
// Binary32: the hardware's 2^x (1 ulp) on a product that already holds log2(e).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLn2 = 0.69314718055994530942;

// exp((s - m) / T) of the row's values against a fixed m. Binary32: the difference first (it
// is exact near m, and m / T itself may overflow where T is small), then 2^x of the product.
template <typename T> struct Expo;
template <> struct Expo<float> {
    float m, inv_t, c;
    __device__ __forceinline__ Expo(float mx, float it) : m(mx == -INFINITY ? 0.0f : mx), inv_t(it), c(it * kLog2e) {}
    __device__ __forceinline__ float operator()(float s) const { return exp2_fast((s - m) * c); }
    // The same function for another pass (see Pass): its differences are not kept either.
    __device__ __forceinline__ Expo fresh() const
    {
        Expo e = *this;
        asm volatile("" : "+v"(e.m));
        return e;
    }
    // log(sum of exp(s / T)) from the sum of the above.
    __device__ __forceinline__ float log_sum(float sum) const
    {
        return (float)((double)m * inv_t + (double)__builtin_amdgcn_logf(sum) * kLn2);
    }
};
template <> struct Expo<double> {
    double inv_t, m;
    __device__ __forceinline__ Expo(double mx, double it) : inv_t(it), m(mx == -INFINITY ? 0.0 : mx) {}
    __device__ __forceinline__ double operator()(double s) const { return exp((s - m) * inv_t); }
    __device__ __forceinline__ Expo fresh() const
    {
        Expo e = *this;
        asm volatile("" : "+v"(e.m));
        return e;
    }
    __device__ __forceinline__ double log_sum(double sum) const { return m * inv_t + log(sum); }
};

} // namespace pcu
