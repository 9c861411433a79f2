// Second step of the column sums (gradients of per-column parameters): adds the rows of partial sums that the workgroups of a
// first pass left.  Not part of the C ABI.
#pragma once
#include "dtype.h"

namespace detbox {

// part [rows][cols]; column c goes to out0[c] (c < cut) or out1[c - cut], either may be null.  32 columns and 32 slices of the
// rows per workgroup, the slices added in order: latency bound, 1024 rows take a few microseconds.  Workgroups take several groups of
// columns where there are more than COLUMN_GROUPS of them: a launch has less than 2^32 threads.
constexpr int64_t COLUMN_GROUPS = 1 << 20;
template <int UNUSED = 0>
__global__ __launch_bounds__(1024) void column_join_kernel(const float *__restrict__ part, int rows, int64_t cols, int64_t cut,
                                                           int dtype, void *out0, void *out1) {
    __shared__ float s[32][33];
    const int slice = threadIdx.x >> 5;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < cols; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + (threadIdx.x & 31);
        float a = 0.f;
        if (c < cols) {
#pragma unroll 8
            for (int r = slice; r < rows; r += 32) a += part[(int64_t)r * cols + c];
        }
        s[slice][threadIdx.x & 31] = a;
        __syncthreads();
        if (slice == 0 && c < cols) {
            a = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) a += s[i][threadIdx.x];
            void *out = c < cut ? out0 : out1;
            if (out) store_from_float(out, dtype, c < cut ? c : c - cut, a);
        }
        __syncthreads();
    }
}

inline void column_join(const float *part, int rows, int64_t cols, int64_t cut, int dtype, void *out0, void *out1, hipStream_t s) {
    const int64_t groups = (cols + 31) / 32;
    column_join_kernel<><<<dim3((unsigned)(groups < COLUMN_GROUPS ? groups : COLUMN_GROUPS)), dim3(1024), 0, s>>>(part, rows, cols, cut, dtype, out0, out1);
}

}  // namespace detbox
