// Matrix product with bias, activation and residual in its epilogue, forward and backward.
//   z = x W^T + b,  y = act(z) + residual          x [M,K], W [N,K], y [M,N]
//   dz = g * act'(z),  grad_x = dz W,  grad_W = dz^T x,  grad_b = sum over rows of dz,  grad_residual = g
// Products are summed in fp32.  What is rounded to the type of x before it is multiplied: dz (when g is wider than x or
// there is an activation) and the z that the derivative is taken at; both are operands of the same matrix instructions as
// x and W, which have that type.
#include "dtype.h"

using namespace detbox;

namespace {

__device__ inline float sigmoid_f(float z) { return 1.0f / (1.0f + expf(-z)); }

__device__ inline float act_value(float z, int act) {
    switch (act) {
        case DETBOX_ACTIVATION_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case DETBOX_ACTIVATION_GELU: return z < -1e4f ? 0.f : 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case DETBOX_ACTIVATION_SILU: return z < -1e4f ? 0.f : z * sigmoid_f(z);
        case DETBOX_ACTIVATION_SIGMOID: return sigmoid_f(z);
    }
    return z;
}

// The derivative; z is kept off the infinities, where the products below would be 0 * inf.
__device__ inline float act_slope(float z, int act) {
    if (act == DETBOX_ACTIVATION_RELU) return z > 0.f ? 1.f : (z != z ? z : 0.f);
    z = z > 1e4f ? 1e4f : (z < -1e4f ? -1e4f : z);
    if (act == DETBOX_ACTIVATION_GELU)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    if (act == DETBOX_ACTIVATION_SILU) { const float p = sigmoid_f(z); return p * (1.0f + z * (1.0f - p)); }
    if (act == DETBOX_ACTIVATION_SIGMOID) { const float p = sigmoid_f(z); return p * (1.0f - p); }
    return 1.f;
}

struct Epilogue {
    const void *bias; int bias_dtype;
    const void *residual; int64_t ldr;      // element type of the output
    int act;
    void *pre;                              // z in the type of x, or null
    int out_dtype;
};

constexpr int TILE = 64, TILE_K = 16;

// C[m,n] = sum_k A[m * am + k * ak] * B[n * bn + k * bk]: every layout through element loads and fp32 arithmetic
template <typename T>
__global__ __launch_bounds__(256) void gemm_any_kernel(const T *__restrict__ A, int64_t am, int64_t ak, const T *__restrict__ B,
                                                       int64_t bn, int64_t bk, int64_t M, int64_t N, int64_t K, Epilogue ep,
                                                       void *C, int64_t tiles_n, int64_t tiles) {
    __shared__ float sa[TILE_K][TILE + 4], sb[TILE_K][TILE + 4];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t m0 = tile / tiles_n * TILE, n0 = tile % tiles_n * TILE;
        float acc[4][4] = {};
        for (int64_t k0 = 0; k0 < K; k0 += TILE_K) {
            __syncthreads();
            for (int e = threadIdx.x; e < TILE * TILE_K; e += 256) {
                const int k = ak == 1 ? e % TILE_K : e / TILE, m = ak == 1 ? e / TILE_K : e % TILE;
                sa[k][m] = m0 + m < M && k0 + k < K ? (float)A[(m0 + m) * am + (k0 + k) * ak] : 0.f;
            }
            for (int e = threadIdx.x; e < TILE * TILE_K; e += 256) {
                const int k = bk == 1 ? e % TILE_K : e / TILE, n = bk == 1 ? e / TILE_K : e % TILE;
                sb[k][n] = n0 + n < N && k0 + k < K ? (float)B[(n0 + n) * bn + (k0 + k) * bk] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < TILE_K; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
        }
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
                if (m >= M || n >= N) continue;
                float z = acc[i][j];
                if (ep.bias) z += load_as_float(ep.bias, ep.bias_dtype, n);
                if (ep.pre) static_cast<T *>(ep.pre)[m * N + n] = (T)z;
                z = act_value(z, ep.act);
                if (ep.residual) z += load_as_float(ep.residual, ep.out_dtype, m * ep.ldr + n);
                store_from_float(C, ep.out_dtype, m * N + n, z);
            }
    }
}

// dz = g * act'(pre) in the type of x, and partial column sums of the unrounded dz per row slice
template <typename T>
__global__ __launch_bounds__(256) void linear_slope_kernel(const void *g, int gdt, int64_t ldg, const T *__restrict__ pre, int act,
                                                           int64_t M, int64_t N, int slices, T *__restrict__ dz,
                                                           float *__restrict__ part) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float a = 0.f;
    for (int64_t row = blockIdx.y; row < M; row += slices) {
        float v = load_as_float(g, gdt, row * ldg + c);
        if (pre) v *= act_slope((float)pre[row * N + c], act);
        if (dz) dz[row * N + c] = (T)v;
        a += v;
    }
    if (part) part[(int64_t)blockIdx.y * N + c] = a;
}

__global__ __launch_bounds__(256) void linear_bias_join_kernel(const float *__restrict__ part, int64_t N, int slices, int bdt,
                                                               void *gb) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float a = 0.f;
    for (int sl = 0; sl < slices; ++sl) a += part[(int64_t)sl * N + c];
    store_from_float(gb, bdt, c, a);
}

int slices_of(int64_t rows) { return (int)(rows < 256 ? (rows < 1 ? 1 : rows) : 256); }

bool act_ok(int act) { return act >= DETBOX_ACTIVATION_NONE && act <= DETBOX_ACTIVATION_SIGMOID; }

template <typename T>
void gemm(const T *A, int64_t am, int64_t ak, const T *B, int64_t bn, int64_t bk, int64_t M, int64_t N, int64_t K,
          const Epilogue &ep, void *C, hipStream_t s) {
    const int64_t tn = (N + TILE - 1) / TILE, tiles = (M + TILE - 1) / TILE * tn;
    gemm_any_kernel<T><<<dim3((unsigned)(tiles < (1 << 20) ? tiles : (1 << 20))), dim3(256), 0, s>>>(A, am, ak, B, bn, bk, M, N, K, ep,
                                                                                                     C, tn, tiles);
}

int check_linear(int dtype, int act, int64_t ldx, int64_t ldw, int64_t M, int64_t N, int64_t K) {
    DETBOX_CHECK_ARG(dtype_ok(dtype), "unknown element type");
    DETBOX_CHECK_ARG(act_ok(act), "unknown activation");
    DETBOX_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31), "bad size");
    DETBOX_CHECK_ARG(ldx >= K && ldw >= K, "row stride below the row length");
    return DETBOX_OK;
}

}  // namespace

extern "C" size_t detbox_linear_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
    (void)dtype; (void)M; (void)N; (void)K;
    return 0;
}

extern "C" int detbox_linear_forward(int dtype, int activation, const void *x, int64_t ldx, const void *weight, int64_t ldw,
                                     int bias_dtype, const void *bias, const void *residual, int64_t ldr, int64_t M, int64_t N,
                                     int64_t K, int out_dtype, void *y, void *pre_activation, void *workspace,
                                     size_t workspace_bytes, void *stream) {
    if (int rc = check_linear(dtype, activation, ldx, ldw, M, N, K)) return rc;
    DETBOX_CHECK_ARG(out_dtype == dtype || out_dtype == DETBOX_F32, "the output has the type of x or fp32");
    DETBOX_CHECK_ARG(dtype_ok(bias_dtype), "unknown element type");
    DETBOX_CHECK_ARG(!residual || ldr >= N, "row stride below the row length");
    if (M == 0) return DETBOX_OK;
    DETBOX_CHECK_ARG(x && weight && y, "null pointer");
    (void)workspace; (void)workspace_bytes;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("linear_forward", s);
    const Epilogue ep{bias, bias_dtype, residual, ldr, activation, pre_activation, out_dtype};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        gemm<T>(static_cast<const T *>(x), ldx, 1, static_cast<const T *>(weight), ldw, 1, M, N, K, ep, y, s);
    });
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}

extern "C" size_t detbox_linear_backward_workspace_bytes(int dtype, int activation, int grad_dtype, int64_t M, int64_t N, int64_t K) {
    if (!dtype_ok(dtype) || M < 0 || N < 1 || K < 1) return 0;
    size_t b = align_up((size_t)slices_of(M) * (size_t)N * sizeof(float), 256);
    if (activation != DETBOX_ACTIVATION_NONE || grad_dtype != dtype) b += align_up((size_t)M * (size_t)N * dtype_size(dtype), 256);
    return b;
}

extern "C" int detbox_linear_backward(int dtype, int activation, int grad_dtype, const void *grad_y, int64_t ldg,
                                      const void *pre_activation, const void *x, int64_t ldx, const void *weight, int64_t ldw,
                                      int64_t M, int64_t N, int64_t K, void *grad_x, void *grad_weight, int bias_dtype,
                                      void *grad_bias, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_linear(dtype, activation, ldx, ldw, M, N, K)) return rc;
    DETBOX_CHECK_ARG(grad_dtype == dtype || grad_dtype == DETBOX_F32, "the gradient has the type of x or fp32");
    DETBOX_CHECK_ARG(dtype_ok(bias_dtype), "unknown element type");
    DETBOX_CHECK_ARG(ldg >= N, "row stride below the row length");
    DETBOX_CHECK_ARG(M == 0 || (grad_y && (activation == DETBOX_ACTIVATION_NONE || pre_activation)), "null pointer");
    DETBOX_CHECK_ARG(M == 0 || ((!grad_x || weight) && (!grad_weight || x)), "null pointer");
    if (!workspace || (uintptr_t)workspace % 256 ||
        workspace_bytes < detbox_linear_backward_workspace_bytes(dtype, activation, grad_dtype, M, N, K)) {
        set_error("%s: workspace missing, misaligned or too small", __func__);
        return DETBOX_ERR_WORKSPACE;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("linear_backward", s);
    const int slices = slices_of(M);
    Carver ws(workspace);
    float *part = ws.take<float>((size_t)slices * N);
    const bool slope = activation != DETBOX_ACTIVATION_NONE, convert = slope || grad_dtype != dtype;
    const Epilogue plain{nullptr, 0, nullptr, 0, DETBOX_ACTIVATION_NONE, nullptr, dtype};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        T *dz = convert ? ws.take<T>((size_t)M * N) : nullptr;
        if (convert || grad_bias)
            linear_slope_kernel<T><<<dim3((unsigned)((N + 255) / 256), slices), dim3(256), 0, s>>>(
                grad_y, grad_dtype, ldg, slope ? static_cast<const T *>(pre_activation) : nullptr, activation, M, N, slices, dz,
                grad_bias ? part : nullptr);
        const T *z = convert ? dz : static_cast<const T *>(grad_y);
        const int64_t ldz = convert ? N : ldg;
        if (grad_x && M) gemm<T>(z, ldz, 1, static_cast<const T *>(weight), 1, ldw, M, K, N, plain, grad_x, s);
        if (grad_weight) gemm<T>(z, 1, ldz, static_cast<const T *>(x), 1, ldx, N, K, M, plain, grad_weight, s);
    });
    DETBOX_LAUNCH_CHECK();
    if (grad_bias) {
        linear_bias_join_kernel<<<dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s>>>(part, N, slices, bias_dtype, grad_bias);
        DETBOX_LAUNCH_CHECK();
    }
    return DETBOX_OK;
}
