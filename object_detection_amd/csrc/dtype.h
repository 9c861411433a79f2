// Element types of the class-head operators (norm.hip, linear.hip, logprob.hip): fp32, bfloat16 and fp16 in memory,
// fp32 in registers.  Not part of the C ABI.
#pragma once
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

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ inline float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

}  // namespace detbox
