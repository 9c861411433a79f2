// Layer normalisation over the last axis, forward and backward.
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), h = (x - mu) * r, y = h * w + b
//   gw = g * w:  grad_x = r * (gw - mean(gw) - h * mean(gw * h)),  grad_w = sum over rows of g * h,  grad_b = sum of g
// All statistics and sums are fp32; every output is rounded once.
//
// HBM bound (240174 x 1024 bf16: forward 225 us = 4.4 TB/s, backward 271 us = 5.4 TB/s); a single row is bound by latency, its
// parameters and its elements one after the other (1 x 1024: 6 us).  A row lives in the registers of a group of 4, 16, 64, 256, 512
// or 1024 lanes, 8 or 16 elements each, so that it is read once and the deviations are squared about the mean itself.
// A lane keeps the parameters of its columns, and in the backward pass their gradients, in registers over all the rows its group
// takes; the groups' sums meet in LDS, the workgroups' in the workspace.  Rows of more than 16384 elements are walked three times.
#include "columns.h"

using namespace detbox;

namespace {

constexpr int NORM_BLOCK = 256;
constexpr int64_t LONG_ROW = 16384;
constexpr int LONG_SLICES = 256;

__device__ inline float block_sum(float v, float *s) {
    v = group_sum<64>(v);
    const int waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < waves; ++w) t += s[w];
    return t;
}
// Two sums at once over the G lanes of a group, in every lane.
template <int G>
__device__ inline void group_sum2(float &a, float &b, float *s) {
    a = group_sum<(G < 64 ? G : 64)>(a);
    b = group_sum<(G < 64 ? G : 64)>(b);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { s[threadIdx.x >> 6] = a; s[W + (threadIdx.x >> 6)] = b; }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { a += s[w]; b += s[W + w]; }
    }
}

// Parameters of a lane's columns as fp32; `fill` where there is none.
template <int VEC, int NV, int G>
__device__ inline void load_columns(float (&v)[NV][VEC], const void *p, int dtype, int lane, int D, float fill) {
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int c = (q * G + lane) * VEC + i;
            v[q][i] = p && c < D ? load_as_float(p, dtype, c) : fill;
        }
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(G < NORM_BLOCK ? NORM_BLOCK : G) void norm_forward_kernel(
    const T *__restrict__ x, int64_t ldx, int pdt, const void *weight, const void *bias, int64_t rows, int D, float eps,
    T *__restrict__ y, float *__restrict__ stats) {
    constexpr int VEC = VEC_OF<T>, BLOCK = G < NORM_BLOCK ? NORM_BLOCK : G, PER = BLOCK / G;
    __shared__ float s[G > 64 ? 2 * G / 64 : 1];
    const int lane = threadIdx.x % G;
    const float inv_d = 1.0f / (float)D;
    float w[NV][VEC], b[NV][VEC];
    load_columns<VEC, NV, G>(w, weight, pdt, lane, D, 1.f);
    load_columns<VEC, NV, G>(b, bias, pdt, lane, D, 0.f);
    for (int64_t row0 = (int64_t)blockIdx.x * PER; row0 < rows; row0 += (int64_t)gridDim.x * PER) {
        const int64_t row = row0 + threadIdx.x / G;
        const bool live = row < rows;
        const T *xr = x + (live ? row : row0) * ldx;
        float v[NV][VEC];
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int c = (q * G + lane) * VEC;
            load_pack<T>(v[q], xr + c, D - c, 0.f);
        }
        float a = 0.f, z = 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) a += v[q][i];
        group_sum2<G>(a, z, s);
        const float mean = a * inv_d;
        a = 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[q][i] = (q * G + lane) * VEC + i < D ? v[q][i] - mean : 0.f;
                a = fmaf(v[q][i], v[q][i], a);
            }
        group_sum2<G>(a, z, s);
        const float rstd = 1.0f / sqrtf(fmaf(a, inv_d, eps));
        if (!live) continue;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int c = (q * G + lane) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[q][i] = fmaf(v[q][i] * rstd, w[q][i], b[q][i]);
            store_pack<T>(y + row * D + c, D - c, v[q]);
        }
        if (stats && lane == 0) { stats[2 * row] = mean; stats[2 * row + 1] = rstd; }
    }
}

// part [workgroups][2 D]: sums of g * h, then of g, over the workgroup's rows; null: no column sums wanted.
template <typename T, int G, int NV>
__global__ __launch_bounds__(G < NORM_BLOCK ? NORM_BLOCK : G) void norm_backward_kernel(
    const T *__restrict__ g, int64_t ldg, const T *__restrict__ x, int64_t ldx, int pdt, const void *weight,
    const float *__restrict__ stats, int64_t rows, int D, T *__restrict__ gx, float *__restrict__ part) {
    constexpr int VEC = VEC_OF<T>, BLOCK = G < NORM_BLOCK ? NORM_BLOCK : G, PER = BLOCK / G, WIDTH = G * NV * VEC;
    __shared__ float s[G > 64 ? 2 * G / 64 : PER * WIDTH];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_d = 1.0f / (float)D;
    float w[NV][VEC], sh[NV][VEC], sg[NV][VEC];
    load_columns<VEC, NV, G>(w, weight, pdt, lane, D, 1.f);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sh[q][i] = sg[q][i] = 0.f;
    for (int64_t row0 = (int64_t)blockIdx.x * PER; row0 < rows; row0 += (int64_t)gridDim.x * PER) {
        const int64_t row = row0 + group;
        const bool live = row < rows;
        const T *xr = x + (live ? row : row0) * ldx, *gr = g + (live ? row : row0) * ldg;
        const float mean = stats[2 * (live ? row : row0)], rstd = stats[2 * (live ? row : row0) + 1];
        float h[NV][VEC], v[NV][VEC];
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int c = (q * G + lane) * VEC;
            load_pack<T>(h[q], xr + c, D - c, 0.f);
            load_pack<T>(v[q], gr + c, live ? D - c : 0, 0.f);          // 0 behind the row: nothing is added there
        }
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[q][i] = (q * G + lane) * VEC + i < D ? (h[q][i] - mean) * rstd : 0.f;
                if (live) {
                    sh[q][i] = fmaf(v[q][i], h[q][i], sh[q][i]);
                    sg[q][i] += v[q][i];
                }
                v[q][i] *= w[q][i];
                a += v[q][i];
                b = fmaf(v[q][i], h[q][i], b);
            }
        if (gx) {
            group_sum2<G>(a, b, s);
            a *= inv_d;
            b *= inv_d;
            if (live) {
#pragma unroll
                for (int q = 0; q < NV; ++q) {
                    const int c = (q * G + lane) * VEC;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[q][i] = (v[q][i] - fmaf(h[q][i], b, a)) * rstd;
                    store_pack<T>(gx + row * D + c, D - c, v[q]);
                }
            }
        }
    }
    if (!part) return;
    float *mine = part + (int64_t)blockIdx.x * 2 * D;
    if constexpr (G > 64) {
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int c = (q * G + lane) * VEC + i;
                if (c < D) { mine[c] = sh[q][i]; mine[D + c] = sg[q][i]; }
            }
    } else {
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < NV; ++q)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[group * WIDTH + (q * G + lane) * VEC + i] = turn ? sg[q][i] : sh[q][i];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += BLOCK) {
                float t = 0.f;
                for (int k = 0; k < PER; ++k) t += s[k * WIDTH + c];
                mine[turn * D + c] = t;
            }
        }
    }
}

// ---- rows too long for registers -----------------------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(1024) void norm_long_forward_kernel(const T *__restrict__ x, int64_t ldx, int pdt, const void *weight,
                                                                 const void *bias, int64_t rows, int64_t D, float eps,
                                                                 T *__restrict__ y, float *__restrict__ stats) {
    __shared__ float s[16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx;
        float a = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += 1024) a += (float)xr[i];
        const float mean = block_sum(a, s) / (float)D;
        a = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += 1024) { const float d = (float)xr[i] - mean; a = fmaf(d, d, a); }
        const float rstd = 1.0f / sqrtf(block_sum(a, s) / (float)D + eps);
        for (int64_t i = threadIdx.x; i < D; i += 1024) {
            float h = ((float)xr[i] - mean) * rstd;
            if (weight) h *= load_as_float(weight, pdt, i);
            if (bias) h += load_as_float(bias, pdt, i);
            y[row * D + i] = (T)h;
        }
        if (stats && threadIdx.x == 0) { stats[2 * row] = mean; stats[2 * row + 1] = rstd; }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_long_grad_x_kernel(const T *__restrict__ g, int64_t ldg, const T *__restrict__ x,
                                                                int64_t ldx, int pdt, const void *weight,
                                                                const float *__restrict__ stats, int64_t rows, int64_t D,
                                                                T *__restrict__ gx) {
    __shared__ float s[16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx, *gr = g + row * ldg;
        const float mean = stats[2 * row], rstd = stats[2 * row + 1];
        float a = 0.f, b = 0.f;
        for (int64_t i = threadIdx.x; i < D; i += 1024) {
            const float gw = (float)gr[i] * (weight ? load_as_float(weight, pdt, i) : 1.0f);
            a += gw;
            b = fmaf(gw, ((float)xr[i] - mean) * rstd, b);
        }
        a = block_sum(a, s) / (float)D;
        b = block_sum(b, s) / (float)D;
        for (int64_t i = threadIdx.x; i < D; i += 1024) {
            const float gw = (float)gr[i] * (weight ? load_as_float(weight, pdt, i) : 1.0f);
            const float h = ((float)xr[i] - mean) * rstd;
            gx[row * D + i] = (T)((gw - a - h * b) * rstd);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void norm_long_columns_kernel(const T *__restrict__ g, int64_t ldg, const T *__restrict__ x,
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
    part[(int64_t)sl * 2 * D + c] = a;
    part[(int64_t)sl * 2 * D + D + c] = b;
}

// ---- host ----------------------------------------------------------------------------------------------------------------

int64_t at_most(int64_t v, int64_t most) { return v < most ? v : most; }

// Lanes per row for rows of D <= LONG_ROW elements: the group of 16 elements per lane that holds them.
int lanes_of(int64_t D) { return D <= 64 ? 4 : D <= 256 ? 16 : D <= 1024 ? 64 : D <= 4096 ? 256 : D <= 8192 ? 512 : 1024; }

// Workgroups of the backward pass, each of which leaves one row of partial sums: four per CU, one of 1024 threads.
int workgroups_of(int64_t rows, int64_t D) {
    if (D > LONG_ROW) return (int)at_most(rows < 1 ? 1 : rows, LONG_SLICES);
    const int G = lanes_of(D), per = G < NORM_BLOCK ? NORM_BLOCK / G : 1;
    const int64_t need = (rows + per - 1) / per;
    return (int)at_most(need < 1 ? 1 : need, G == 1024 ? 256 : 1024);
}

// Calls fn(integral_constant<G>, integral_constant<NV>) for the smallest group that holds a row.
template <typename T, typename F>
void with_group(int64_t D, F &&fn) {
    constexpr int W = 8 / VEC_OF<T>;                                   // packs per eight elements
    auto call = [&](auto g, auto nv) { fn(g, nv); };
    using std::integral_constant;
    switch (lanes_of(D)) {
        case 4: call(integral_constant<int, 4>{}, integral_constant<int, 2 * W>{}); break;
        case 16:
            if (D <= 128) call(integral_constant<int, 16>{}, integral_constant<int, W>{});
            else call(integral_constant<int, 16>{}, integral_constant<int, 2 * W>{});
            break;
        case 64:
            if (D <= 512) call(integral_constant<int, 64>{}, integral_constant<int, W>{});
            else call(integral_constant<int, 64>{}, integral_constant<int, 2 * W>{});
            break;
        case 256:
            if (D <= 2048) call(integral_constant<int, 256>{}, integral_constant<int, W>{});
            else call(integral_constant<int, 256>{}, integral_constant<int, 2 * W>{});
            break;
        case 512: call(integral_constant<int, 512>{}, integral_constant<int, 2 * W>{}); break;
        default: call(integral_constant<int, 1024>{}, integral_constant<int, 2 * W>{});
    }
}

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
        const T *xx = static_cast<const T *>(x);
        T *yy = static_cast<T *>(y);
        if (D > LONG_ROW) {
            norm_long_forward_kernel<T><<<dim3((unsigned)at_most(rows, 65536)), dim3(1024), 0, s>>>(xx, ldx, param_dtype, weight, bias,
                                                                                                  rows, D, eps, yy, stats);
            return;
        }
        with_group<T>(D, [&](auto g, auto nv) {
            constexpr int G = decltype(g)::value, BLOCK = G < NORM_BLOCK ? NORM_BLOCK : G, PER = BLOCK / G;
            // eight workgroups per CU: each loads the parameters once
            const int64_t grid = at_most((rows + PER - 1) / PER, G == 1024 ? 512 : 2048);
            norm_forward_kernel<T, G, decltype(nv)::value><<<dim3((unsigned)grid), dim3(BLOCK), 0, s>>>(
                xx, ldx, param_dtype, weight, bias, rows, (int)D, eps, yy, stats);
        });
    });
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}

extern "C" size_t detbox_layer_norm_backward_workspace_bytes(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1) return 0;
    return (size_t)2 * workgroups_of(rows, D) * (size_t)D * sizeof(float);
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
    const int wgs = workgroups_of(rows, D);
    float *part = columns ? static_cast<float *>(workspace) : nullptr;
    if (columns && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < detbox_layer_norm_backward_workspace_bytes(rows, D))) {
        set_error("%s: workspace missing, misaligned or too small", __func__);
        return DETBOX_ERR_WORKSPACE;
    }
    if (!columns && (!grad_x || rows == 0)) return DETBOX_OK;
    ProfScope ps("layer_norm_backward", s);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const T *g = static_cast<const T *>(grad_y), *xx = static_cast<const T *>(x);
        T *gx = rows ? static_cast<T *>(grad_x) : nullptr;
        if (D > LONG_ROW) {
            if (gx)
                norm_long_grad_x_kernel<T><<<dim3((unsigned)at_most(rows, 65536)), dim3(1024), 0, s>>>(g, ldg, xx, ldx, param_dtype,
                                                                                                     weight, stats, rows, D, gx);
            if (columns)
                norm_long_columns_kernel<T><<<dim3((unsigned)((D + NORM_BLOCK - 1) / NORM_BLOCK), wgs), dim3(NORM_BLOCK), 0, s>>>(
                    g, ldg, xx, ldx, stats, rows, D, wgs, part);
            return;
        }
        with_group<T>(D, [&](auto lanes, auto nv) {
            constexpr int G = decltype(lanes)::value, BLOCK = G < NORM_BLOCK ? NORM_BLOCK : G;
            norm_backward_kernel<T, G, decltype(nv)::value><<<dim3((unsigned)wgs), dim3(BLOCK), 0, s>>>(
                g, ldg, xx, ldx, param_dtype, weight, stats, rows, (int)D, gx, part);
        });
    });
    DETBOX_LAUNCH_CHECK();
    if (columns) {
        column_join(part, wgs, 2 * D, D, param_dtype, grad_weight, grad_bias, s);
        DETBOX_LAUNCH_CHECK();
    }
    return DETBOX_OK;
}
