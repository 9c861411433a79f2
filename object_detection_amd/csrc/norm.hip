// Layer normalisation over the last axis, forward and backward.
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), h = (x - mu) * r, y = h * w + b
//   gw = g * w:  grad_x = r * (gw - mean(gw) - h * mean(gw * h)),  grad_w = sum over rows of g * h,  grad_b = sum of g
// All statistics and sums are fp32; every output is rounded once.
#include "dtype.h"

using namespace detbox;

namespace {

constexpr int NORM_BLOCK = 256;
constexpr int NORM_SLICES = 256;      // row slices whose partial column sums the second step adds up

__device__ inline float block_sum(float v, float *s) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < NORM_BLOCK / 64; ++w) t += s[w];
    return t;
}

template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void norm_forward_kernel(const T *__restrict__ x, int64_t ldx, int pdt, const void *weight,
                                                                  const void *bias, int64_t rows, int64_t D, float eps,
                                                                  T *__restrict__ y, float *__restrict__ stats) {
    __shared__ float s[NORM_BLOCK / 64];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx;
        float a = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += NORM_BLOCK) a += (float)xr[i];
        const float mean = block_sum(a, s) / (float)D;
        a = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += NORM_BLOCK) { const float d = (float)xr[i] - mean; a = fmaf(d, d, a); }
        const float rstd = 1.0f / sqrtf(block_sum(a, s) / (float)D + eps);
        for (int64_t i = threadIdx.x; i < D; i += NORM_BLOCK) {
            float h = ((float)xr[i] - mean) * rstd;
            if (weight) h *= load_as_float(weight, pdt, i);
            if (bias) h += load_as_float(bias, pdt, i);
            y[row * D + i] = (T)h;
        }
        if (stats && threadIdx.x == 0) { stats[2 * row] = mean; stats[2 * row + 1] = rstd; }
    }
}

template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void norm_grad_x_kernel(const T *__restrict__ g, int64_t ldg, const T *__restrict__ x,
                                                                 int64_t ldx, int pdt, const void *weight,
                                                                 const float *__restrict__ stats, int64_t rows, int64_t D,
                                                                 T *__restrict__ gx) {
    __shared__ float s[NORM_BLOCK / 64];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx, *gr = g + row * ldg;
        const float mean = stats[2 * row], rstd = stats[2 * row + 1];
        float a = 0.f, b = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += NORM_BLOCK) {
            const float gw = (float)gr[i] * (weight ? load_as_float(weight, pdt, i) : 1.0f);
            a += gw;
            b = fmaf(gw, ((float)xr[i] - mean) * rstd, b);
        }
        a = block_sum(a, s) / (float)D;
        b = block_sum(b, s) / (float)D;
        for (int64_t i = threadIdx.x; i < D; i += NORM_BLOCK) {
            const float gw = (float)gr[i] * (weight ? load_as_float(weight, pdt, i) : 1.0f);
            const float h = ((float)xr[i] - mean) * rstd;
            gx[row * D + i] = (T)((gw - a - h * b) * rstd);
        }
    }
}

// partial column sums: part[0][slice][D] of g * h, part[1][slice][D] of g
template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void norm_columns_kernel(const T *__restrict__ g, int64_t ldg, const T *__restrict__ x,
                                                                  int64_t ldx, const float *__restrict__ stats, int64_t rows,
                                                                  int64_t D, int slices, float *__restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * NORM_BLOCK + threadIdx.x;
    if (c >= D) return;
    const int sl = blockIdx.y;
    float a = 0.f, b = 0.f;
    for (int64_t row = sl; row < rows; row += slices) {
        const float gv = (float)g[row * ldg + c];
        a = fmaf(gv, ((float)x[row * ldx + c] - stats[2 * row]) * stats[2 * row + 1], a);
        b += gv;
    }
    part[(int64_t)sl * D + c] = a;
    part[((int64_t)slices + sl) * D + c] = b;
}

__global__ __launch_bounds__(NORM_BLOCK) void norm_columns_join_kernel(const float *__restrict__ part, int64_t D, int slices,
                                                                       int pdt, void *gw, void *gb) {
    const int64_t c = (int64_t)blockIdx.x * NORM_BLOCK + threadIdx.x;
    if (c >= D) return;
    float a = 0.f, b = 0.f;
    for (int sl = 0; sl < slices; ++sl) {
        a += part[(int64_t)sl * D + c];
        b += part[((int64_t)slices + sl) * D + c];
    }
    if (gw) store_from_float(gw, pdt, c, a);
    if (gb) store_from_float(gb, pdt, c, b);
}

int slices_of(int64_t rows) { return (int)(rows < NORM_SLICES ? (rows < 1 ? 1 : rows) : NORM_SLICES); }
unsigned row_grid(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

int check_norm(int dtype, const void *x, int64_t ldx, int pdt, int64_t rows, int64_t D) {
    DETBOX_CHECK_ARG(dtype_ok(dtype) && dtype_ok(pdt), "unknown element type");
    DETBOX_CHECK_ARG(rows >= 0 && D >= 1 && rows < (1ll << 40) && D < (1ll << 31), "bad size");
    DETBOX_CHECK_ARG(ldx >= D, "row stride below the row length");
    DETBOX_CHECK_ARG(rows == 0 || x, "null pointer");
    return DETBOX_OK;
}

}  // namespace

extern "C" int detbox_layer_norm_forward(int dtype, const void *x, int64_t ldx, int param_dtype, const void *weight,
                                         const void *bias, int64_t rows, int64_t D, float eps, void *y, float *stats,
                                         void *stream) {
    if (int rc = check_norm(dtype, x, ldx, param_dtype, rows, D)) return rc;
    if (rows == 0) return DETBOX_OK;
    DETBOX_CHECK_ARG(y, "null pointer");
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("layer_norm_forward", s);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        norm_forward_kernel<T><<<dim3(row_grid(rows)), dim3(NORM_BLOCK), 0, s>>>(
            static_cast<const T *>(x), ldx, param_dtype, weight, bias, rows, D, eps, static_cast<T *>(y), stats);
    });
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}

extern "C" size_t detbox_layer_norm_backward_workspace_bytes(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1) return 0;
    return (size_t)2 * slices_of(rows) * (size_t)D * sizeof(float);
}

extern "C" int detbox_layer_norm_backward(int dtype, const void *grad_y, int64_t ldg, const void *x, int64_t ldx,
                                          int param_dtype, const void *weight, const float *stats, int64_t rows, int64_t D,
                                          void *grad_x, void *grad_weight, void *grad_bias, void *workspace,
                                          size_t workspace_bytes, void *stream) {
    if (int rc = check_norm(dtype, x, ldx, param_dtype, rows, D)) return rc;
    DETBOX_CHECK_ARG(ldg >= D, "row stride below the row length");
    DETBOX_CHECK_ARG(rows == 0 || (grad_y && stats), "null pointer");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool columns = grad_weight || grad_bias;
    const int slices = slices_of(rows);
    float *part = static_cast<float *>(workspace);
    if (columns && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < detbox_layer_norm_backward_workspace_bytes(rows, D))) {
        set_error("%s: workspace missing, misaligned or too small", __func__);
        return DETBOX_ERR_WORKSPACE;
    }
    ProfScope ps("layer_norm_backward", s);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const T *g = static_cast<const T *>(grad_y), *xx = static_cast<const T *>(x);
        if (grad_x && rows)
            norm_grad_x_kernel<T><<<dim3(row_grid(rows)), dim3(NORM_BLOCK), 0, s>>>(g, ldg, xx, ldx, param_dtype, weight, stats, rows,
                                                                                   D, static_cast<T *>(grad_x));
        if (columns)
            norm_columns_kernel<T><<<dim3((unsigned)((D + NORM_BLOCK - 1) / NORM_BLOCK), slices), dim3(NORM_BLOCK), 0, s>>>(
                g, ldg, xx, ldx, stats, rows, D, slices, part);
    });
    DETBOX_LAUNCH_CHECK();
    if (columns) {
        norm_columns_join_kernel<<<dim3((unsigned)((D + NORM_BLOCK - 1) / NORM_BLOCK)), dim3(NORM_BLOCK), 0, s>>>(
            part, D, slices, param_dtype, grad_weight, grad_bias);
        DETBOX_LAUNCH_CHECK();
    }
    return DETBOX_OK;
}
