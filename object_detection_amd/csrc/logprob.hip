// Log probability of a given label, entropy and best alternatives of every row of logits, forward and backward.
//   m = max(x), s = sum exp(x - m), log p_j = (x_j - m) - log s
//   entropy = log s - sum exp(x - m) (x - m) / s;  alternatives: the top_k largest x (lower index first among equals)
//   grad_j = g (1[j = label] - p_j) - h p_j (log p_j + entropy), g and h the incoming gradients of the two
// A row whose label lies outside [0, C) does not take part: log probability 0, g taken as 0.  A row of -inf only has no
// distribution: log probability -inf, entropy 0, alternatives 0 .. top_k-1 with -inf, gradient 0.
#include "dtype.h"

using namespace detbox;

namespace {

constexpr int LP_BLOCK = 256;

// NaN ranks above everything, -0 equals +0; the lower index is the larger word among equal values
__device__ inline uint64_t rank_word(float v, int64_t i) {
    const uint32_t k = v != v ? 0xffffffffu : okey_from_bits(__float_as_uint(v));
    return ((uint64_t)k << 32) | (uint32_t)~(uint32_t)i;
}

template <typename T>
__global__ __launch_bounds__(LP_BLOCK) void logprob_forward_kernel(const T *__restrict__ x, int64_t ld,
                                                                   const int64_t *__restrict__ labels, int64_t rows, int64_t C,
                                                                   int top_k, float *__restrict__ log_probs,
                                                                   float *__restrict__ entropy, float *__restrict__ top_lp,
                                                                   int64_t *__restrict__ top_ids, float *__restrict__ stats) {
    __shared__ float s1[LP_BLOCK / 64], s2[LP_BLOCK / 64];
    __shared__ uint64_t sw[LP_BLOCK / 64];
    const int w = threadIdx.x >> 6;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ld;
        float m = -INFINITY;
        for (int64_t i = threadIdx.x; i < C; i += LP_BLOCK) m = fmaxf(m, (float)xr[i]);
        m = wave_max(m);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s1[w] = m;
        __syncthreads();
        for (int k = 0; k < LP_BLOCK / 64; ++k) m = fmaxf(m, s1[k]);
        const bool empty = m == -INFINITY;
        const float ref = empty ? 0.f : m;
        float a = 0.f, b = 0.f;
        for (int64_t i = threadIdx.x; i < C; i += LP_BLOCK) {
            const float d = (float)xr[i] - ref, e = expf(d);
            a += e;
            b = fmaf(e, fmaxf(d, -1e30f), b);
        }
        a = wave_sum(a);
        b = wave_sum(b);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { s1[w] = a; s2[w] = b; }
        __syncthreads();
        a = b = 0.f;
        for (int k = 0; k < LP_BLOCK / 64; ++k) { a += s1[k]; b += s2[k]; }
        const float ls = logf(a);
        // a row of -inf and NaN only: the maximum is -inf, the sum is NaN, and the row's values are NaN
        const bool none = empty && a == 0.f;
        if (threadIdx.x == 0) {
            const int64_t t = labels[row];
            log_probs[row] = t < 0 || t >= C ? 0.f : none ? -INFINITY : ((float)xr[t] - ref) - ls;
            if (entropy) entropy[row] = none ? 0.f : ls - b / a;
            if (stats) { stats[2 * row] = ref; stats[2 * row + 1] = a; }
        }
        uint64_t last = ~0ull;
        for (int k = 0; k < top_k; ++k) {
            uint64_t best = 0;
            for (int64_t i = threadIdx.x; i < C; i += LP_BLOCK) {
                const uint64_t r = rank_word((float)xr[i], i);
                if (r < last || k == 0) best = r > best ? r : best;
            }
            for (int o = 32; o > 0; o >>= 1) { const uint64_t r = __shfl_xor(best, o); best = r > best ? r : best; }
            __syncthreads();
            if ((threadIdx.x & 63) == 0) sw[w] = best;
            __syncthreads();
            for (int q = 0; q < LP_BLOCK / 64; ++q) best = sw[q] > best ? sw[q] : best;
            last = best;
            if (threadIdx.x == 0) {
                const int64_t i = (uint32_t)~(uint32_t)best;
                top_ids[row * top_k + k] = i;
                top_lp[row * top_k + k] = none ? -INFINITY : ((float)xr[i] - ref) - ls;
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(LP_BLOCK) void logprob_backward_kernel(const T *__restrict__ x, int64_t ld,
                                                                    const int64_t *__restrict__ labels, int64_t rows, int64_t C,
                                                                    const float *__restrict__ stats,
                                                                    const float *__restrict__ entropy,
                                                                    const float *__restrict__ grad_lp,
                                                                    const float *__restrict__ grad_ent, T *__restrict__ gx) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ld;
        const float ref = stats[2 * row], sum = stats[2 * row + 1], ls = logf(sum);
        const int64_t t = labels[row];
        const bool part = t >= 0 && t < C;
        const float g = grad_lp && part ? grad_lp[row] : 0.f, h = grad_ent ? grad_ent[row] : 0.f, H = grad_ent ? entropy[row] : 0.f;
        for (int64_t i = threadIdx.x; i < C; i += LP_BLOCK) {
            float r = 0.f;
            if (sum != 0.f && (part || grad_ent)) {      // a row that does not take part has gradient 0 whatever it holds
                const float d = (float)xr[i] - ref, p = expf(d) / sum;
                r = ((part && i == t) ? g : 0.f) - g * p;
                if (grad_ent) r -= h * (p * (fmaxf(d, -1e30f) - ls + H));
            }
            gx[row * C + i] = (T)r;
        }
    }
}

int check_logprob(int dtype, const void *logits, int64_t ld, const int64_t *labels, int64_t rows, int64_t C) {
    DETBOX_CHECK_ARG(dtype_ok(dtype), "unknown element type");
    DETBOX_CHECK_ARG(rows >= 0 && C >= 1 && rows < (1ll << 40) && C < (1ll << 31), "bad size");
    DETBOX_CHECK_ARG(ld >= C, "row stride below the row length");
    DETBOX_CHECK_ARG(rows == 0 || (logits && labels), "null pointer");
    return DETBOX_OK;
}
unsigned row_grid(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

}  // namespace

extern "C" size_t detbox_label_log_probs_workspace_bytes(int64_t rows, int64_t C, int top_k) {
    (void)rows; (void)C; (void)top_k;
    return 0;
}

extern "C" int detbox_label_log_probs_forward(int dtype, const void *logits, int64_t ld, const int64_t *labels, int64_t rows,
                                              int64_t C, int top_k, float *log_probs, float *entropy, float *top_log_probs,
                                              int64_t *top_ids, float *stats, void *workspace, size_t workspace_bytes,
                                              void *stream) {
    if (int rc = check_logprob(dtype, logits, ld, labels, rows, C)) return rc;
    DETBOX_CHECK_ARG(top_k >= 0 && top_k <= C, "top_k outside 0 .. C");
    if (top_k > DETBOX_MAX_ALTERNATIVES) {
        set_error("%s: top_k beyond DETBOX_MAX_ALTERNATIVES", __func__);
        return DETBOX_ERR_UNSUPPORTED;
    }
    if (rows == 0) return DETBOX_OK;
    DETBOX_CHECK_ARG(log_probs && (top_k == 0 || (top_log_probs && top_ids)), "null pointer");
    (void)workspace; (void)workspace_bytes;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("label_log_probs_forward", s);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        logprob_forward_kernel<T><<<dim3(row_grid(rows)), dim3(LP_BLOCK), 0, s>>>(
            static_cast<const T *>(logits), ld, labels, rows, C, top_k, log_probs, entropy, top_log_probs, top_ids, stats);
    });
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}

extern "C" int detbox_label_log_probs_backward(int dtype, const void *logits, int64_t ld, const int64_t *labels, int64_t rows,
                                               int64_t C, const float *stats, const float *entropy, const float *grad_log_probs,
                                               const float *grad_entropy, void *grad_logits, void *stream) {
    if (int rc = check_logprob(dtype, logits, ld, labels, rows, C)) return rc;
    if (rows == 0) return DETBOX_OK;
    DETBOX_CHECK_ARG(stats && grad_logits && (!grad_entropy || entropy), "null pointer");
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("label_log_probs_backward", s);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        logprob_backward_kernel<T><<<dim3(row_grid(rows)), dim3(LP_BLOCK), 0, s>>>(
            static_cast<const T *>(logits), ld, labels, rows, C, stats, entropy, grad_log_probs, grad_entropy,
            static_cast<T *>(grad_logits));
    });
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}
