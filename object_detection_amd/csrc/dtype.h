// Element types of the class-head operators (norm.hip, linear.hip, logprob.hip): fp32, bfloat16 and fp16 in memory,
// fp32 in registers.  Not part of the C ABI.
#pragma once
#include <type_traits>
#include "detbox_internal.h"

namespace detbox {

// Calls fn with a value of the element type that `dtype` (DETBOX_F32 / _BF16 / _F16) stands for; false if it is none.
template <typename F>
inline bool with_dtype(int dtype, F &&fn) {
    switch (dtype) {
        case DETBOX_F32: fn(float{}); return true;
        case DETBOX_BF16: fn(__bf16{}); return true;
        case DETBOX_F16: fn(_Float16{}); return true;
    }
    return false;
}

inline size_t dtype_size(int dtype) { return dtype == DETBOX_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == DETBOX_F32 || dtype == DETBOX_BF16 || dtype == DETBOX_F16; }

// Element i of a buffer whose type is known at run time only (per-column parameters: the branch is uniform).
__device__ inline float load_as_float(const void *p, int dtype, int64_t i) {
    if (dtype == DETBOX_F32) return static_cast<const float *>(p)[i];
    if (dtype == DETBOX_BF16) return (float)static_cast<const __bf16 *>(p)[i];
    return (float)static_cast<const _Float16 *>(p)[i];
}
__device__ inline void store_from_float(void *p, int dtype, int64_t i, float v) {
    if (dtype == DETBOX_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == DETBOX_BF16) static_cast<__bf16 *>(p)[i] = (__bf16)v;
    else static_cast<_Float16 *>(p)[i] = (_Float16)v;
}

// Sixteen bytes of elements from any address that is a multiple of the element's size: rows of odd length start anywhere, and
// the memory pipeline takes a wide access at any such address.
typedef uint32_t detbox_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t detbox_u4_at2 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef uint32_t detbox_u4_at4 __attribute__((ext_vector_type(4), aligned(4), may_alias));
template <typename T> using raw_pack = std::conditional_t<sizeof(T) == 2, detbox_u4_at2, detbox_u4_at4>;
template <typename T> constexpr int VEC_OF = 16 / (int)sizeof(T);
template <typename T>
__device__ inline detbox_u4 load_raw(const T *p) { return *reinterpret_cast<const raw_pack<T> *>(p); }
// The same for data that is not read again soon: it does not displace what is.
template <typename T>
__device__ inline detbox_u4 load_raw_nt(const T *p) { return __builtin_nontemporal_load(reinterpret_cast<const raw_pack<T> *>(p)); }
template <typename T>
__device__ inline void unpack(float (&v)[VEC_OF<T>], const detbox_u4 u) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        const t8 t = __builtin_bit_cast(t8, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
    }
}
template <typename T>
__device__ inline void store_pack(T *p, const float (&v)[VEC_OF<T>]) {
    detbox_u4 u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(v[i]);
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        t8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
        u = __builtin_bit_cast(detbox_u4, t);
    }
    *reinterpret_cast<raw_pack<T> *>(p) = u;
}
template <typename T>
__device__ inline void load_pack(float (&v)[VEC_OF<T>], const T *p) { unpack<T>(v, load_raw<T>(p)); }
// Packs u = 0 .. U-1 of a row of C >= VEC elements at c + u * step, any of them partly or wholly behind its end (those read as
// `fill`).  All U loads are issued before the first is looked at; the address of one that would pass the end is moved back.
template <typename T, int U>
__device__ inline void load_packs_to_end(float (&v)[U][VEC_OF<T>], const T *row, int64_t c, int64_t step, int64_t C, float fill) {
    constexpr int VEC = VEC_OF<T>;
    detbox_u4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw<T>(row + (c + u * step + VEC <= C ? c + u * step : C - VEC));
#pragma unroll
    for (int u = 0; u < U; ++u) unpack<T>(v[u], raw[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (c + u * step + VEC > C) {
            // what was loaded are the row's last VEC elements: the wanted ones move down, the fill moves in
            const int64_t by = c + u * step + VEC - C;
#pragma unroll
            for (int b = VEC / 2; b > 0; b >>= 1)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[u][i] = (by & b) ? (i + b < VEC ? v[u][i + b < VEC ? i + b : 0] : fill) : v[u][i];
            if (by >= VEC) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[u][i] = fill;
            }
        }
}
// A pack whose first `by` elements are not wanted (0 < by): the rest moved down, zeros behind them.
template <typename T>
__device__ inline detbox_u4 moved_down(detbox_u4 u, int64_t by) {
    if (by >= VEC_OF<T>) return detbox_u4{0, 0, 0, 0};
    const int bits = (int)by * 8 * (int)sizeof(T);
    const unsigned long long lo = ((unsigned long long)u[1] << 32) | u[0], hi = ((unsigned long long)u[3] << 32) | u[2];
    const unsigned long long l = bits >= 64 ? hi >> (bits - 64) : (lo >> bits) | (hi << (64 - bits)), h = bits >= 64 ? 0 : hi >> bits;
    return detbox_u4{(uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32)};
}
// The first n of a pack; the rest reads as `fill` and is not touched in memory.
template <typename T>
__device__ inline void load_pack(float (&v)[VEC_OF<T>], const T *p, int64_t n, float fill) {
    if (n >= VEC_OF<T>) {
        load_pack<T>(v, p);
    } else {
#pragma unroll
        for (int i = 0; i < VEC_OF<T>; ++i) v[i] = i < n ? (float)p[i] : fill;
    }
}
template <typename T>
__device__ inline void store_pack(T *p, int64_t n, const float (&v)[VEC_OF<T>]) {
    if (n >= VEC_OF<T>) {
        store_pack<T>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC_OF<T>; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// Sum and maximum over groups of G consecutive lanes, in every lane of the group.
template <int G>
__device__ inline float group_sum(float v) {
    if constexpr (G > 1) v += lane_xor_f32<1>(v);
    if constexpr (G > 2) v += lane_xor_f32<2>(v);
    if constexpr (G > 4) v += lane_xor_f32<4>(v);
    if constexpr (G > 8) v += lane_xor_f32<8>(v);
    if constexpr (G > 16) v += lane_xor_f32<16>(v);
    if constexpr (G > 32) v += lane_xor_f32<32>(v);
    return v;
}
template <int G>
__device__ inline float group_max(float v) {
    if constexpr (G > 1) v = fmaxf(v, lane_xor_f32<1>(v));
    if constexpr (G > 2) v = fmaxf(v, lane_xor_f32<2>(v));
    if constexpr (G > 4) v = fmaxf(v, lane_xor_f32<4>(v));
    if constexpr (G > 8) v = fmaxf(v, lane_xor_f32<8>(v));
    if constexpr (G > 16) v = fmaxf(v, lane_xor_f32<16>(v));
    if constexpr (G > 32) v = fmaxf(v, lane_xor_f32<32>(v));
    return v;
}
template <int G>
__device__ inline uint64_t group_max_u64(uint64_t v) {
#define DETBOX_STEP(J) if constexpr (G > J) { const uint64_t o = lane_xor_u64<J>(v); v = o > v ? o : v; }
    DETBOX_STEP(1) DETBOX_STEP(2) DETBOX_STEP(4) DETBOX_STEP(8) DETBOX_STEP(16) DETBOX_STEP(32)
#undef DETBOX_STEP
    return v;
}

// exp through the hardware's power of two; off by a few steps of fp32 and 2^-24 |d| relative
__device__ inline float fast_exp(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }

}  // namespace detbox
