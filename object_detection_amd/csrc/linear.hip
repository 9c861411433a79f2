// Matrix product with bias, activation and residual in its epilogue, forward and backward.
//   z = x W^T + b,  y = act(z) + residual          x [M,K], W [N,K], y [M,N]
//   dz = g * act'(z),  grad_x = dz W,  grad_W = dz^T x,  grad_b = sum over rows of dz,  grad_residual = g
// Products are summed in fp32.  What is rounded to the type of x before it is multiplied: dz (when g is wider than x or
// there is an activation) and the z that the derivative is taken at; both are operands of the same matrix instructions as
// x and W, which have that type.  For fp16 a dz that is rounded is first brought into that type's range by a power of two,
// which the products take out again: a mean over many rows has gradients below fp16's smallest step, a scaled loss some beyond
// its largest value.
//
// Bounds: a long contraction is bound by the matrix instructions (8192^3 bf16, 20 training steps in a row: 1.15-1.19
// PFLOP/s on average in all three products, 1.24-1.28 at best), a short one by memory (RetinaNet's class logits, 480348 x 256
// bf16 by 81, fp32 out: 97 us = 4.2 TB/s), few rows by the read of the weight and its latency (4 x 4096 by 4096: 9.8 us = 3.4 TB/s).
//
// One tile kernel serves all three products.  Each operand lies in memory either along the contraction (x, W forward) or
// across it (W in grad_x; dz and x in grad_W); both come into LDS as they lie, 16 bytes at a time, and only the read of a
// fragment differs: a plain 16-byte read, or the transposing LDS read of 16-bit elements.
#include "columns.h"

using namespace detbox;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const void __attribute__((address_space(1))) *gptr_t;
typedef void __attribute__((address_space(3))) *lptr_t;

__device__ inline float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z)); }

// Normal distribution function by Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26 (error below 1.5e-7 / 2, 2.8e-7
// at most as measured in fp32 arithmetic, on [-8, 8]);
// e is exp(-z^2 / 2), which the slope needs as well.
__device__ inline float normal_cdf(float z, float e) {
    const float u = fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, u, 1.0f));
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    const float tail = 0.5f * q * t * e;
    return z < 0.f ? tail : 1.0f - tail;
}

__device__ inline float relu_f(float z) { return z > 0.f ? z : (z != z ? z : 0.f); }
__device__ inline float gelu_f(float z) { return z < -1e4f ? 0.f : z * normal_cdf(z, fast_exp(-0.5f * z * z)); }
__device__ inline float silu_f(float z) { return z < -1e4f ? 0.f : z * sigmoid_f(z); }
// The derivatives; z is kept off the infinities, where the products would be 0 * inf.
__device__ inline float bounded(float z) { return z > 1e4f ? 1e4f : (z < -1e4f ? -1e4f : z); }
__device__ inline float relu_slope(float z) { return z > 0.f ? 1.f : (z != z ? z : 0.f); }
__device__ inline float gelu_slope(float z) {
    z = bounded(z);
    const float e = fast_exp(-0.5f * z * z);
    return fmaf(z * 0.39894228040143268f, e, normal_cdf(z, e));
}
__device__ inline float silu_slope(float z) {
    z = bounded(z);
    const float p = sigmoid_f(z);
    return p * (1.0f + z * (1.0f - p));
}
__device__ inline float sigmoid_slope(float z) { const float p = sigmoid_f(z); return p * (1.0f - p); }

struct Epilogue {
    const void *bias; int bias_dtype;
    const void *residual; int64_t ldr;      // element type of the output
    int act;
    void *pre; int pre_dtype;               // z, or null
    void *out; int out_dtype;
    const float *unscale = nullptr;         // factor on the sums (in device memory), or null
};

// Four values with one (uniform) choice of the activation.
#define DETBOX_FOUR(f) f32x4{f(z[0]), f(z[1]), f(z[2]), f(z[3])}
__device__ inline f32x4 act4(f32x4 z, int act) {
    switch (act) {
        case DETBOX_ACTIVATION_RELU: return DETBOX_FOUR(relu_f);
        case DETBOX_ACTIVATION_GELU: return DETBOX_FOUR(gelu_f);
        case DETBOX_ACTIVATION_SILU: return DETBOX_FOUR(silu_f);
        case DETBOX_ACTIVATION_SIGMOID: return DETBOX_FOUR(sigmoid_f);
    }
    return z;
}
__device__ inline f32x4 slope4(f32x4 z, int act) {
    switch (act) {
        case DETBOX_ACTIVATION_RELU: return DETBOX_FOUR(relu_slope);
        case DETBOX_ACTIVATION_GELU: return DETBOX_FOUR(gelu_slope);
        case DETBOX_ACTIVATION_SILU: return DETBOX_FOUR(silu_slope);
        case DETBOX_ACTIVATION_SIGMOID: return DETBOX_FOUR(sigmoid_slope);
    }
    return f32x4{1.f, 1.f, 1.f, 1.f};
}
#undef DETBOX_FOUR

// Four elements as they were loaded: a pack of fp32, or the first eight bytes of 16-bit ones.
__device__ inline f32x4 widen4(detbox_u4 u, int dtype) {
    if (dtype == DETBOX_F32) return __builtin_bit_cast(f32x4, u);
    f32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint16_t h = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
        v[j] = dtype == DETBOX_BF16 ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
    }
    return v;
}

// n <= 4 consecutive elements of a buffer whose type is known at run time, from any address of an element
typedef uint32_t detbox_u2_at2 __attribute__((ext_vector_type(2), aligned(2), may_alias));
__device__ inline f32x4 load4(const void *p, int dtype, int64_t i, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        if (dtype == DETBOX_F32) return __builtin_bit_cast(f32x4, load_raw<float>(static_cast<const float *>(p) + i));
        const detbox_u2_at2 u = *reinterpret_cast<const detbox_u2_at2 *>(static_cast<const uint16_t *>(p) + i);
        return widen4(detbox_u4{u[0], u[1], 0, 0}, dtype);
    }
    for (int j = 0; j < n; ++j) v[j] = load_as_float(p, dtype, i + j);
    return v;
}
__device__ inline void store4(void *p, int dtype, int64_t i, int n, f32x4 v) {
    if (n >= 4) {
        if (dtype == DETBOX_F32) {
            *reinterpret_cast<detbox_u4_at4 *>(static_cast<float *>(p) + i) = __builtin_bit_cast(detbox_u4, v);
            return;
        }
        detbox_u2_at2 u;
        if (dtype == DETBOX_BF16) {
            typedef __bf16 b4 __attribute__((ext_vector_type(4)));
            u = __builtin_bit_cast(detbox_u2_at2, __builtin_convertvector(v, b4));
        } else {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            u = __builtin_bit_cast(detbox_u2_at2, __builtin_convertvector(v, h4));
        }
        *reinterpret_cast<detbox_u2_at2 *>(static_cast<uint16_t *>(p) + i) = u;
        return;
    }
    for (int j = 0; j < n; ++j) store_from_float(p, dtype, i + j, v[j]);
}

// z as it is kept for the slope.  fp16 holds nothing between 0 and 2^-24: what lies there is kept as the latter, since relu's
// slope is 1 at any z above 0 and 0 at 0 itself (the other slopes are the same at both to 2^-24).
__device__ inline f32x4 kept(f32x4 z, bool half) {
    if (half) {
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = z[j] > 0.f ? fmaxf(z[j], 0x1p-24f) : z[j];
    }
    return z;
}

// Four neighbouring sums of a row, columns n .. n + 3 (those below N), through the epilogue.  `row` is the row's offset in the
// outputs, `res_row` that in the residual: kept by the caller, since a 64-bit product per four elements costs more than
// everything else here.
__device__ inline void finish4(const Epilogue &ep, int64_t row, int64_t res_row, int n, int N, f32x4 z) {
    const int left = N - n < 4 ? N - n : 4;
    if (left <= 0) return;
    if (ep.unscale) z *= *ep.unscale;
    if (ep.bias) z += load4(ep.bias, ep.bias_dtype, n, left);
    if (ep.pre) store4(ep.pre, ep.pre_dtype, row + n, left, kept(z, ep.pre_dtype == DETBOX_F16));
    if (ep.act != DETBOX_ACTIVATION_NONE) z = act4(z, ep.act);
    if (ep.residual) z += load4(ep.residual, ep.out_dtype, res_row + n, left);
    store4(ep.out, ep.out_dtype, row + n, left, z);
}

// ---- tile kernel ---------------------------------------------------------------------------------------------------------

// An operand: `rows` rows of the output's axis, contraction length in GemmArgs.  ACROSS == false: element (r, k) at
// p[r * ld + k]; ACROSS == true: at p[k * ld + r].  extent: how far the axis that lies in order may be read (to the end of a
// padded row where what is behind the operand's own end is zero).
template <typename T>
struct Operand { const T *p; int64_t ld; int64_t rows, extent; };

template <typename T>
struct GemmArgs {
    Operand<T> a, b;            // output rows m from a, columns n from b
    int64_t K;
    int tiles_m, tiles_n, splits;
    int64_t steps_per_split;    // contraction steps of one piece
    Epilogue ep;
    float *part;                // [splits][M][N] where splits > 1
};

// A step of the contraction is 128 bytes per row: 64 elements of 16 bits or 32 of fp32, eight chunks of 16 bytes.
template <typename T> constexpr int STEP_K = 128 / (int)sizeof(T);

// Where the chunks of a step lie in LDS.  Along: chunk c of row r at slot c ^ (r & 7) of the row's 128 bytes, so that the 16
// rows a fragment read touches spread over all banks.  Across: rows of the contraction, each ROWS elements in units of 16
// (one fragment's width); unit u of row k at u ^ swizzle(k), which spreads the rows that one read touches.
template <typename T, int ROWS>
__device__ inline int across_swizzle(int k) {
    static_assert((ROWS & (ROWS - 1)) == 0, "units are swapped in powers of two");
    return (sizeof(T) == 2 ? (k & 3) | ((k >> 3) & 1) << 2 : (k >> 2) & 3) & (ROWS / 16 - 1);
}

__device__ const uint4 zero_chunk = {0, 0, 0, 0};

// The chunks of one step that a thread brings in: idx = j * THREADS + tid is also the place in LDS.
template <typename T, bool ACROSS, int ROWS, int THREADS, bool ALIGNED>
struct Stager {
    static constexpr int VEC = VEC_OF<T>, COUNT = (ROWS * 8 + THREADS - 1) / THREADS, PER_K = ROWS / VEC, PER_UNIT = 16 / VEC;
    const T *src[COUNT];        // of the step that is fetched next
    int at[COUNT];              // contraction index of the chunk inside a step
    int left[COUNT];            // across: how many of the chunk's elements exist
    int64_t step;               // elements from one step to the next

    // Whether there is a chunk j for this thread: whole waves have one or not.
    static __device__ bool live(int j) { return ROWS * 8 % THREADS == 0 || j * THREADS + (int)(threadIdx.x & ~63) < ROWS * 8; }

    __device__ void init(const Operand<T> &o, int64_t row0, int64_t k0) {
        const int tid = threadIdx.x;
        step = ACROSS ? STEP_K<T> * o.ld : STEP_K<T>;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const int idx = j * THREADS + tid;
            if constexpr (ACROSS) {
                const int k = idx / PER_K, slot = idx % PER_K;
                const int unit = (slot / PER_UNIT) ^ across_swizzle<T, ROWS>(k);
                int64_t r = row0 + unit * 16 + (slot % PER_UNIT) * VEC;
                at[j] = k;
                const int64_t n = o.extent - r;
                left[j] = n >= VEC ? VEC : n < 0 ? 0 : (int)n;
                if (ALIGNED && n < VEC) r = o.extent - VEC;            // rows that do not exist: any values
                if (!ALIGNED && n <= 0) r = 0;
                src[j] = o.p + (k0 + k) * o.ld + r;
            } else {
                const int r = idx >> 3, chunk = (idx & 7) ^ (r & 7);
                int64_t row = row0 + r;
                if (row >= o.rows) row = o.rows - 1;                      // rows that do not exist: any values
                at[j] = chunk * VEC;
                left[j] = VEC;
                src[j] = o.p + row * o.ld + k0 + chunk * VEC;
            }
        }
    }
    // Brings chunk j of the next step straight into LDS (aligned operands; chunks behind the contraction's end from a zero).
    __device__ void dma(int j, int64_t k_left, char *lds) {
        if (!live(j)) return;
        const void *p = src[j];
        src[j] += step;
        if (k_left < STEP_K<T> && at[j] >= k_left) p = &zero_chunk;
        __builtin_amdgcn_global_load_lds((gptr_t)p, (lptr_t)(lds + (j * THREADS + (threadIdx.x & ~63)) * 16), 16, 0, 0);
    }
    // Chunk j of the next step, which starts k_left elements before the contraction's end; zeros behind the end.
    __device__ detbox_u4 load(int j, int64_t k_left) {
        if (!live(j)) return detbox_u4{0, 0, 0, 0};
        const T *p = src[j];
        src[j] = p + step;
        int n = left[j];
        if (ACROSS) n = at[j] < k_left ? n : 0;
        else if (k_left - at[j] < VEC) n = k_left - at[j] < 0 ? 0 : (int)(k_left - at[j]);
        if (n == VEC) return load_raw<T>(p);
        T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = i < n ? p[i] : (T)0.f;
        detbox_u4 u;
        __builtin_memcpy(&u, e, 16);
        return u;
    }
};

// Fragment of 16 rows and four chunks' worth of contraction: lane l has row l % 16, its elements k of quarter l / 16.
template <typename T, bool ACROSS, int ROWS>
__device__ inline detbox_u4 read_fragment(const char *lds, int row0, int ks) {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    if constexpr (!ACROSS) {
        const int row = row0 + r;
        return *reinterpret_cast<const detbox_u4 *>(lds + (row * 8 + ((ks * 4 + q) ^ (row & 7))) * 16);
    } else if constexpr (sizeof(T) == 2) {
        detbox_u4 u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = ks * 32 + q * 8 + h * 4 + (r >> 2);
            const char *p = lds + k * (ROWS * 2) + (((row0 >> 4) ^ across_swizzle<T, ROWS>(k)) * 32) + (r & 3) * 8;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
            typedef uint32_t u2 __attribute__((ext_vector_type(2)));
            const u2 w = __builtin_bit_cast(u2, v);
            u[2 * h] = w[0];
            u[2 * h + 1] = w[1];
        }
        return u;
    } else {
        detbox_u4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = ks * 16 + q * 4 + j;
            u[j] = *reinterpret_cast<const uint32_t *>(lds + k * (ROWS * 4) + (((row0 >> 4) ^ across_swizzle<T, ROWS>(k)) * 64) + r * 4);
        }
        return u;
    }
}

// acc[n = 4 (l / 16) + i][m = l % 16] += sum over part `t` of the fragments' contraction: all of it for the 16-bit types, a
// quarter for fp32, whose instruction takes one element per lane.
template <typename T> constexpr int PARTS = sizeof(T) == 2 ? 1 : 4;
template <typename T>
__device__ inline f32x4 multiply(detbox_u4 n, detbox_u4 m, f32x4 acc, int t) {
    if constexpr (std::is_same_v<T, __bf16>) {
        typedef __bf16 v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, n), __builtin_bit_cast(v8, m), acc, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, _Float16>) {
        typedef _Float16 v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, n), __builtin_bit_cast(v8, m), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(n[t]), __uint_as_float(m[t]), acc, 0, 0, 0);
    }
}

// Workgroups are dealt to the eight XCDs in turn.  Every XCD gets a run of neighbouring jobs, so that the operands' panels are
// shared in its L2: the tiles of one piece of the contraction one after the other, walked in bands of eight tile rows.
__device__ inline void job_of(int wg, int tiles_m, int tiles_n, int splits, int &tm, int &tn, int &split) {
    const int tiles = tiles_m * tiles_n, total = tiles * splits, per = total / 8, rest = total % 8;
    const int x = wg & 7, i = wg >> 3;
    const int job = x * per + (x < rest ? x : rest) + i;
    split = job / tiles;
    const int t = job - split * tiles;
    const int band = t / (8 * tiles_n), rows = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
    const int in = t - band * 8 * tiles_n;
    tm = band * 8 + in % rows;
    tn = in / rows;
}

// The products of one step, from the buffer `cur` (A's rows first), while the next step comes into `nxt`.  The two pointers
// are restrict: without it the compiler takes every LDS read for one that may want what is still on its way and waits for
// the whole transfer first.  Reads and matrix instructions are interleaved by hand, the second half's reads under the first
// half's products.  8192^3 bf16 forward, short runs: 997 us with staging through registers, 944 with the compiler's order, 860 so;
// over 20 training steps in a row 927-937 on average.
template <typename T, bool AX, bool BX, int BM, int BN, int FM, int FN>
__device__ __forceinline__ void multiply_step(const char *__restrict__ cur, int wm, int wn, f32x4 (&acc)[FM][FN]) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        detbox_u4 fa[FM], fb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[i] = read_fragment<T, AX, BM>(cur, wm + i * 16, ks);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = read_fragment<T, BX, BN>(cur + BM * 128, wn + j * 16, ks);
#pragma unroll
        for (int t = 0; t < PARTS<T>; ++t)                     // neighbouring instructions add to different sums
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = multiply<T>(fb[j], fa[i], acc[i][j], t);
    }
    constexpr int READS = FM * (AX ? 2 : 1) + FN * (BX ? 2 : 1), EACH = FM * FN / READS;
    if constexpr (sizeof(T) == 2 && EACH > 0) {
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
        for (int r = 0; r < READS; ++r) {
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * FM * FN - READS * EACH, 0);
    }
}
template <typename T, bool AX, bool BX, int BM, int BN, int FM, int FN, typename SA, typename SB>
__device__ __forceinline__ void dma_step(const char *__restrict__ cur, char *__restrict__ nxt, SA &sa, SB &sb, bool more,
                                         int64_t k_left, int wm, int wn, f32x4 (&acc)[FM][FN]) {
    if (more) {
#pragma unroll
        for (int j = 0; j < SA::COUNT; ++j) sa.dma(j, k_left, nxt);
#pragma unroll
        for (int j = 0; j < SB::COUNT; ++j) sb.dma(j, k_left, nxt + BM * 128);
    }
    multiply_step<T, AX, BX, BM, BN, FM, FN>(cur, wm, wn, acc);
}

template <typename T, bool AX, bool BX, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void gemm_kernel(GemmArgs<T> g) {
    constexpr int THREADS = (BM / WM) * (BN / WN) * 64, FM = WM / 16, FN = WN / 16;
    constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, PAD = 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
    int tm, tn, split;
    job_of(blockIdx.x, g.tiles_m, g.tiles_n, g.splits, tm, tn, split);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int64_t s0 = split * g.steps_per_split, all = (g.K + STEP_K<T> - 1) / STEP_K<T>;
    const int64_t steps = all - s0 < g.steps_per_split ? all - s0 : g.steps_per_split;

    Stager<T, AX, BM, THREADS, ALIGNED> sa;
    Stager<T, BX, BN, THREADS, ALIGNED> sb;
    const int64_t k0 = s0 * STEP_K<T>;
    sa.init(g.a, m0, k0);
    sb.init(g.b, n0, k0);
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto buffer = [&](int64_t i) { return lds + (i & 1) * (A_BYTES + B_BYTES); };
    const int64_t k_all = g.K - k0;
    if constexpr (ALIGNED) {
        auto issue = [&](int64_t s) {
#pragma unroll
            for (int j = 0; j < sa.COUNT; ++j) sa.dma(j, k_all - s * STEP_K<T>, buffer(s));
#pragma unroll
            for (int j = 0; j < sb.COUNT; ++j) sb.dma(j, k_all - s * STEP_K<T>, buffer(s) + A_BYTES);
        };
        if (steps > 0) issue(0);
        for (int64_t s = 0; s < steps; ++s) {
            __builtin_amdgcn_s_waitcnt(0x0070);              // vmcnt(0) lgkmcnt(0): step s has arrived, what was read is here
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();                    // ... in every wave: the other buffer is free
            asm volatile("" ::: "memory");
            dma_step<T, AX, BX, BM, BN, FM, FN>(buffer(s), buffer(s + 1), sa, sb, s + 1 < steps, k_all - (s + 1) * STEP_K<T>, wm, wn, acc);
        }
        __syncthreads();
    } else {
        // rows that start off 16 bytes or end inside a chunk: through registers
        detbox_u4 ra[sa.COUNT], rb[sb.COUNT];
        auto fetch = [&](int64_t s) {
#pragma unroll
            for (int j = 0; j < sa.COUNT; ++j) ra[j] = sa.load(j, k_all - s * STEP_K<T>);
#pragma unroll
            for (int j = 0; j < sb.COUNT; ++j) rb[j] = sb.load(j, k_all - s * STEP_K<T>);
        };
        auto put = [&](char *to) {
#pragma unroll
            for (int j = 0; j < sa.COUNT; ++j)
                if (sa.live(j)) *reinterpret_cast<detbox_u4 *>(to + (j * THREADS + threadIdx.x) * 16) = ra[j];
#pragma unroll
            for (int j = 0; j < sb.COUNT; ++j)
                if (sb.live(j)) *reinterpret_cast<detbox_u4 *>(to + A_BYTES + (j * THREADS + threadIdx.x) * 16) = rb[j];
        };
        if (steps > 0) {
            fetch(0);
            put(lds);
        }
        __syncthreads();
        for (int64_t s = 0; s < steps; ++s) {
            if (s + 1 < steps) fetch(s + 1);
            multiply_step<T, AX, BX, BM, BN, FM, FN>(buffer(s), wm, wn, acc);
            if (s + 1 < steps) put(buffer(s + 1));
            __syncthreads();
        }
    }

    // The sums go through LDS, 64 rows of the wave's part at a time, so that rows are written (and the residual read) in order.
    constexpr int HALF = WM < 64 ? WM : 64, ROW = WN + PAD, LANES = WN / 4, AT_ONCE = 64 / LANES;
    float *mine = reinterpret_cast<float *>(lds) + wave * (HALF * ROW);
    const int64_t M = g.a.rows, N = g.b.rows, n = n0 + wn + (lane % LANES) * 4;
    const int left = lane >= AT_ONCE * LANES ? 0 : N - n >= 4 ? 4 : N > n ? (int)(N - n) : 0;
    constexpr bool UNSCALE = BX && std::is_same_v<T, _Float16>;               // a product with dz
    float unscale = 1.f;
    if constexpr (UNSCALE)
        if (g.ep.unscale) unscale = *g.ep.unscale;
    const f32x4 bias = g.ep.bias ? load4(g.ep.bias, g.ep.bias_dtype, n, left) : f32x4{0.f, 0.f, 0.f, 0.f};
    // A batch of U turns at a time.  The residual of a batch is on its way while the batch before it is finished (16384 x 4096
    // by 4096 bf16: a residual costs 35 us, 90 where each batch waits for its own).
    constexpr int TURNS = (HALF + AT_ONCE - 1) / AT_ONCE, U = TURNS < 8 ? TURNS : 8;
    const int64_t row0 = m0 + wm + lane / LANES;
    auto alive = [&](int h, int t) { return left > 0 && t * AT_ONCE + lane / LANES < HALF && row0 + h * HALF + t * AT_ONCE < M; };
    detbox_u4 raw[U], next[U];
    auto fetch_residual = [&](detbox_u4 (&to)[U], int h, int t) {
        if (!g.ep.residual || left != 4) return;
        const int64_t by = (int64_t)AT_ONCE * g.ep.ldr, at = (row0 + h * HALF) * g.ep.ldr + n + t * by;
        if (g.ep.out_dtype == DETBOX_F32) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (alive(h, t + u)) to[u] = load_raw<float>(static_cast<const float *>(g.ep.residual) + at + u * by);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (alive(h, t + u)) {
                    const detbox_u2_at2 w = *reinterpret_cast<const detbox_u2_at2 *>(static_cast<const uint16_t *>(g.ep.residual) + at + u * by);
                    to[u][0] = w[0];
                    to[u][1] = w[1];
                }
        }
    };
    if (g.splits == 1) fetch_residual(raw, 0, 0);
#pragma unroll
    for (int h = 0; h < WM / HALF; ++h) {
        if (h) __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < HALF / 16; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                *reinterpret_cast<f32x4 *>(mine + (i * 16 + (lane & 15)) * ROW + j * 16 + (lane >> 4) * 4) = acc[h * (HALF / 16) + i][j];
        __builtin_amdgcn_wave_barrier();
        const int64_t out_at = (row0 + h * HALF) * N + n;
        for (int t = 0; t < TURNS; t += U) {
            if (g.splits == 1) {
                if (t + U < TURNS) fetch_residual(next, h, t + U);
                else if (h + 1 < WM / HALF) fetch_residual(next, h + 1, 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!alive(h, t + u)) continue;
                f32x4 z = *reinterpret_cast<const f32x4 *>(mine + ((t + u) * AT_ONCE + lane / LANES) * ROW + (lane % LANES) * 4);
                const int64_t at = out_at + (int64_t)((t + u) * AT_ONCE) * N;
                if (g.splits > 1) {
                    store4(g.part, DETBOX_F32, (int64_t)split * M * N + at, left, z);
                    continue;
                }
                if constexpr (UNSCALE) z *= unscale;
                z += bias;
                if (g.ep.pre) store4(g.ep.pre, g.ep.pre_dtype, at, left, kept(z, std::is_same_v<T, _Float16>));
                if (g.ep.act != DETBOX_ACTIVATION_NONE) z = act4(z, g.ep.act);
                if (g.ep.residual)
                    z += left == 4 ? widen4(raw[u], g.ep.out_dtype)
                                   : load4(g.ep.residual, g.ep.out_dtype, (row0 + h * HALF + (t + u) * AT_ONCE) * g.ep.ldr + n, left);
                store4(g.ep.out, g.ep.out_dtype, at, left, z);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = next[u];
        }
    }
}

// Adds the pieces of the contraction in a fixed order and applies the epilogue.  SLICES threads share an output: 16 where there
// are many pieces of a small product (256 pieces of 81 x 256: 82 us with one thread per output, 9 us so).
template <int SLICES>
__global__ __launch_bounds__(256) void gemm_join_kernel(const float *__restrict__ part, int splits, int64_t M, int64_t N, Epilogue ep) {
    constexpr int OUT = 256 / SLICES;
    __shared__ f32x4 sums[SLICES > 1 ? 256 : 1];
    const int64_t per = (N + 3) / 4, total = M * per;
    const int slice = threadIdx.x / OUT;
    for (int64_t i0 = (int64_t)blockIdx.x * OUT; i0 < total; i0 += (int64_t)gridDim.x * OUT) {
        const int64_t i = i0 + threadIdx.x % OUT, m = i / per, n = (i % per) * 4;
        const int left = i >= total ? 0 : N - n < 4 ? (int)(N - n) : 4;
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
        if (left > 0) {
#pragma unroll 4
            for (int s = slice; s < splits; s += SLICES) z += load4(part, DETBOX_F32, ((int64_t)s * M + m) * N + n, left);
        }
        if constexpr (SLICES > 1) {
            sums[threadIdx.x] = z;
            __syncthreads();
            if (slice == 0) {
#pragma unroll
                for (int s = 1; s < SLICES; ++s) z += sums[s * OUT + threadIdx.x];
            }
            __syncthreads();
        }
        if (slice == 0 && left > 0) finish4(ep, m * N, m * ep.ldr, (int)n, (int)N, z);
    }
}

// Largest finite |g| of a workgroup's share (0 where there is none), for the scale of an fp16 dz; the slope of no activation is
// above 1.13, so that dz itself need not be computed for it.  A pass over g of its own: HBM bound (480348 x 81 fp32 28 us = 5.6 TB/s).
// Dense gradients are read as one run, four packs in flight; rows with a stride LANES lanes a row.
constexpr int PEAKS = 1024;
__device__ inline float finite_peak(float m, float v) { return fabsf(v) < INFINITY ? fmaxf(m, fabsf(v)) : m; }
// The largest of a workgroup's 256 values, in every thread.
__device__ inline float block_peak(float m) {
    __shared__ float s[4];
    m = group_max<64>(m);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
    __syncthreads();
    return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}
template <typename G>
__global__ __launch_bounds__(256) void linear_peak_dense_kernel(const G *__restrict__ g, int64_t n, float *__restrict__ peaks) {
    constexpr int VEC = VEC_OF<G>, U = 4;
    const int64_t step = (int64_t)gridDim.x * 256 * VEC;
    int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
    float m = 0.f, v[U][VEC];
    for (; i + (U - 1) * step + VEC <= n; i += U * step) {
        detbox_u4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = load_raw<G>(g + i + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            unpack<G>(v[u], raw[u]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) m = finite_peak(m, v[u][j]);
        }
    }
    for (; i < n; i += step) {
        load_pack<G>(v[0], g + i, n - i, 0.f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = finite_peak(m, v[0][j]);
    }
    m = block_peak(m);
    if (threadIdx.x == 0) peaks[blockIdx.x] = m;
}
template <int LANES>
__global__ __launch_bounds__(256) void linear_peak_kernel(const void *g, int gdt, int64_t ldg, int64_t M, int64_t N, float *__restrict__ peaks) {
    constexpr int ROWS = 256 / LANES;
    float m = 0.f;
    for (int64_t c = ((int64_t)blockIdx.x * LANES + threadIdx.x % LANES) * 4; c < N; c += (int64_t)gridDim.x * LANES * 4) {
        const int left = N - c >= 4 ? 4 : (int)(N - c);
        for (int64_t row = (int64_t)blockIdx.y * ROWS + threadIdx.x / LANES; row < M; row += (int64_t)gridDim.y * ROWS) {
            const f32x4 v = load4(g, gdt, row * ldg + c, left);
#pragma unroll
            for (int j = 0; j < 4; ++j) m = finite_peak(m, v[j]);
        }
    }
    m = block_peak(m);
    if (threadIdx.x == 0) peaks[blockIdx.y * gridDim.x + blockIdx.x] = m;
}
// The power of two that brings the largest of `count` <= PEAKS peaks to [2^14, 2^15) (at most 2^126: both it and its inverse are
// normal numbers).  dz then stays below 2^15.2, inside fp16, and what a small dz loses is at most half of fp16's smallest step,
// 2^-39 of the largest gradient.  For all 256 threads of a workgroup.
__device__ inline int scale_exponent(const float *peaks, int count) {
    float m = 0.f;
    for (int i = threadIdx.x; i < count; i += 256) m = fmaxf(m, peaks[i]);
    m = block_peak(m);
    if (m == 0.f) return 0;
    const int e = 14 - ((int)(__float_as_uint(m) >> 23) - 127);
    return e < 126 ? e : 126;
}

// dz = g * act'(pre) in the type of x with rows of ldz elements (zeros behind N), and partial column sums of the unrounded dz
// per row slice.  With peaks, dz is stored times their power of two, the inverse of which goes to *unscale.
// LANES lanes share a row, four columns each; HBM bound (16384 x 4096 bf16 with gelu: 96 us = 4.2 TB/s).
template <typename T, int LANES>
__global__ __launch_bounds__(256) void linear_slope_kernel(const void *g, int gdt, int64_t ldg, const T *__restrict__ pre, int act,
                                                           int64_t M, int64_t N, int64_t ldz, int64_t rows_per_slice,
                                                           T *__restrict__ dz, float *__restrict__ part,
                                                           const float *__restrict__ peaks, int n_peaks, float *__restrict__ unscale) {
    constexpr int DT = sizeof(T) == 4 ? DETBOX_F32 : std::is_same_v<T, __bf16> ? DETBOX_BF16 : DETBOX_F16, ROWS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t c = ((int64_t)blockIdx.x * LANES + lane) * 4;
    const int left = N - c >= 4 ? 4 : N - c > 0 ? (int)(N - c) : 0, room = ldz - c < 4 ? (int)(ldz - c) : 4;
    int up = 0;                             // ldexp, not a product: the products cost 45 us at 16384 x 4096 (98 against 143)
    if constexpr (std::is_same_v<T, _Float16>)
        if (peaks) {
            up = scale_exponent(peaks, n_peaks);
            if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *unscale = __uint_as_float((uint32_t)(127 - up) << 23);
        }
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    const int64_t lo = blockIdx.y * rows_per_slice, hi = lo + rows_per_slice < M ? lo + rows_per_slice : M;
    if (c < ldz) {
        const int64_t row0 = lo + threadIdx.x / LANES, by_g = ROWS * ldg, by_p = ROWS * N, by_z = ROWS * ldz;
        int64_t at_g = row0 * ldg + c, at_p = row0 * N + c, at_z = row0 * ldz + c;
#pragma unroll 1                                                              // more waves hide more than rows in flight do: 96 us against 131 unrolled
        for (int64_t row = row0; row < hi; row += ROWS, at_g += by_g, at_p += by_p, at_z += by_z) {
            f32x4 v = load4(g, gdt, at_g, left);
            if (pre) v *= slope4(load4(pre, DT, at_p, left), act);                // v is 0 behind N
            if (dz) {
                f32x4 d = v;
                if constexpr (std::is_same_v<T, _Float16>) d = f32x4{ldexpf(v[0], up), ldexpf(v[1], up), ldexpf(v[2], up), ldexpf(v[3], up)};
                store4(dz, DT, at_z, room, d);
            }
            a += v;
        }
    }
    if (!part) return;
    __shared__ f32x4 s[256];
    s[threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.x < LANES && left > 0) {
        for (int r = 1; r < ROWS; ++r) a += s[r * LANES + threadIdx.x];
        store4(part, DETBOX_F32, (int64_t)blockIdx.y * N + c, left, a);
    }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------

// At most 16 MT rows of x (serving): the weight is all there is to read, and it goes straight into registers, once.  A workgroup
// owns 16 columns; its eight waves take the contraction's packs in turn and add their sums in LDS in order.  No second launch.
// 4 x 4096 by 4096 bf16: 11.1 us as tiles in pieces and their join, 9.2-9.8 us = 3.4-3.6 TB/s so.
constexpr int64_t FEW_ROWS = 64;
constexpr int FEW_BLOCK = 512, FEW_WAVES = FEW_BLOCK / 64;

template <typename T, int MT>
__global__ __launch_bounds__(FEW_BLOCK) void gemm_few_kernel(const Operand<T> a, const Operand<T> b, int64_t K, Epilogue ep) {
    constexpr int VEC = VEC_OF<T>, KF = 4 * VEC, CHUNK = MT > 2 ? 4 : 8;
    __shared__ f32x4 sums[FEW_WAVES][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int64_t M = a.rows, N = b.rows, kf = (K + KF - 1) / KF;
    for (int64_t n0 = (int64_t)blockIdx.x * 16; n0 < N; n0 += (int64_t)gridDim.x * 16) {
        const int64_t n = n0 + r < N ? n0 + r : N - 1;                       // columns and rows that do not exist: any values
        const T *w = b.p + n * b.ld, *x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = a.p + (i * 16 + r < M ? i * 16 + r : M - 1) * a.ld;
        f32x4 acc[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        int64_t c0 = wave;
        for (; (c0 + (CHUNK - 1) * FEW_WAVES + 1) * KF <= K; c0 += FEW_WAVES * CHUNK) {
            detbox_u4 fw[CHUNK], fx[CHUNK][MT];
#pragma unroll
            for (int c = 0; c < CHUNK; ++c) {
                const int64_t k = (c0 + c * FEW_WAVES) * KF + q * VEC;
                fw[c] = load_raw_nt<T>(w + k);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[c][i] = load_raw<T>(x[i] + k);
            }
#pragma unroll
            for (int c = 0; c < CHUNK; ++c)
#pragma unroll
                for (int t = 0; t < PARTS<T>; ++t)
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[i] = multiply<T>(fw[c], fx[c][i], acc[i], t);
        }
        for (; c0 < kf; c0 += FEW_WAVES) {                                  // the rest, the row's last pack moved down to its place
            const int64_t k = c0 * KF + q * VEC, over = k + VEC - K, at = over <= 0 ? k : K - VEC;     // K >= VEC here
            detbox_u4 fw = load_raw_nt<T>(w + at), fx[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) fx[i] = load_raw<T>(x[i] + at);
            if (over > 0) {
                fw = moved_down<T>(fw, over);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[i] = moved_down<T>(fx[i], over);
            }
#pragma unroll
            for (int t = 0; t < PARTS<T>; ++t)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i] = multiply<T>(fw, fx[i], acc[i], t);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) sums[wave][i][lane] = acc[i];
        __syncthreads();
        if (wave < MT) {
            f32x4 z = sums[0][wave][lane];
#pragma unroll
            for (int v = 1; v < FEW_WAVES; ++v) z += sums[v][wave][lane];
            const int64_t m = wave * 16 + r;
            if (m < M) finish4(ep, m * N, m * ep.ldr, (int)n0 + q * 4, (int)N, z);
        }
        __syncthreads();
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------

bool act_ok(int act) { return act >= DETBOX_ACTIVATION_NONE && act <= DETBOX_ACTIVATION_SIGMOID; }

// How a product is cut.  Tiles of 256 x 256 (eight waves of 128 x 64, one workgroup per CU) where they alone fill the chip and
// have steps enough to hide their start and end; tiles of 128 rows (eight waves; two workgroups per CU at widths of 128 and 96,
// three at 64, by their LDS) otherwise,
// as wide as the columns ask for, with the contraction in pieces where there are fewer than two tiles per CU.  Measured (bf16
// unless it says fp32, us, large / small): 8192^3 860 / 1043, 4096^3 115 / 132, 8192 x 1024 by 8192 149 / 153, 8192 x 512 by
// 8192 103 / 95, 65536 x 256 by 256 24 / 21, 2048^3 (64 large tiles) 59 / 31.  Width (128 / as wide as needed): 480348 x 64 by
// 32 39 / 22, 40000 x 300 by 20 11.7 / 8.6, 120087 x 256 by 81 in fp32, where the matrix instructions count, 87 / 71; 128 / 64
// for few tiles: 4096 x 1024 by 1024 25 / 14, 2048^3 32 / 26, 300 x 1024 by 4096 21 / 14, but 8732 x 1000 by 1208 (690 tiles)
// 41 / 45, 512 x 4096 by 4096 (128 tiles, 64 steps) 30 / 32.
struct Plan { bool big; int width, tiles_m, tiles_n, splits; int64_t steps_per_split; };
Plan plan_of(int dtype, int64_t M, int64_t N, int64_t K, bool across) {
    Plan p;
    const int64_t step = 128 / (int64_t)dtype_size(dtype), steps = (K + step - 1) / step;
    p.big = ((M + 255) / 256) * ((N + 255) / 256) >= 192 && steps > 8;
    const int64_t t = p.big ? 256 : 128;
    // half as wide too where whole tiles would not fill the chip: twice as many take the place of pieces and their join
    const int64_t rows = (M + 127) / 128, whole = rows * ((N + 127) / 128), half = rows * ((N + 63) / 64);
    const bool narrow = whole < 512 && half >= 128 && (half >= 384 || steps < 64);
    p.width = p.big ? 256 : N <= 64 || narrow ? 64 : N <= 96 && !across ? 96 : 128;
    p.tiles_m = (int)((M + t - 1) / t);
    p.tiles_n = (int)((N + p.width - 1) / p.width);
    int64_t splits = 1;
    if (!p.big) {
        splits = 512 / ((int64_t)p.tiles_m * p.tiles_n);
        const int64_t most = steps / 4;                      // at least four steps each
        splits = splits > most ? most : splits;
        splits = splits < 1 ? 1 : splits > 512 ? 512 : splits;
    }
    p.steps_per_split = (steps + splits - 1) / splits;
    p.splits = p.steps_per_split > 0 ? (int)((steps + p.steps_per_split - 1) / p.steps_per_split) : 1;
    if (p.splits < 1) { p.splits = 1; p.steps_per_split = 1; }
    return p;
}
size_t plan_bytes(const Plan &p, int64_t M, int64_t N) {
    return p.splits > 1 ? align_up((size_t)p.splits * M * N * sizeof(float), 256) : 0;
}

template <typename T>
bool whole_chunks(const void *p, int64_t ld, int64_t extent) {
    return (uintptr_t)p % 16 == 0 && ld % VEC_OF<T> == 0 && extent % VEC_OF<T> == 0;
}

template <typename T, bool AX, bool BX, int BM, int BN, int WM, int WN, bool ALIGNED>
int launch_gemm(const GemmArgs<T> &g, hipStream_t s) {
    constexpr int WAVES = (BM / WM) * (BN / WN), HALF = WM < 64 ? WM : 64;
    constexpr int BUFFERS = 2 * (BM + BN) * 128, OUT = WAVES * HALF * (WN + 4) * 4, LDS = BUFFERS > OUT ? BUFFERS : OUT;
    auto kernel = gemm_kernel<T, AX, BX, BM, BN, WM, WN, ALIGNED>;
    DETBOX_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    kernel<<<dim3((unsigned)(g.tiles_m * g.tiles_n * g.splits)), dim3(WAVES * 64), LDS, s>>>(g);
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}

// Measured in bf16 against the tiles (us): 1 x 1000 by 1203 4.5 / 9.9, 64 x 1000 by 1203 6.2 / 12.4, 1 x 4096 by 4096 7.6 / 11.5,
// 16 rows of it 11.7 / 12.9, 32 rows 15.5 / 15.0; with more to read, where every workgroup's copy of x counts, the tiles lead
// (64 x 4096 by 4096 22.7 / 18.6, 1 x 4096 by 32000 56 / 41), and so they do where a long contraction is eight waves' only
// (64 x 4096 by 81 20 / 10).
bool few(int dtype, int64_t M, int64_t N, int64_t K) {
    const int64_t vec = 16 / (int64_t)dtype_size(dtype), tiles = (M + 15) / 16, kf = (K + 4 * vec - 1) / (4 * vec);
    return M <= FEW_ROWS && K >= vec && tiles * N * K <= 20 << 20 && kf <= (tiles > 2 ? 64 : 256);
}

template <typename T>
int gemm_few(const Operand<T> &a, const Operand<T> &b, int64_t K, const Epilogue &ep, hipStream_t s) {
    const int64_t columns = (b.rows + 15) / 16;
    const dim3 grid((unsigned)(columns < 1 << 20 ? columns : 1 << 20)), block(FEW_BLOCK);
    if (a.rows <= 16) gemm_few_kernel<T, 1><<<grid, block, 0, s>>>(a, b, K, ep);
    else if (a.rows <= 32) gemm_few_kernel<T, 2><<<grid, block, 0, s>>>(a, b, K, ep);
    else gemm_few_kernel<T, 4><<<grid, block, 0, s>>>(a, b, K, ep);
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}

template <typename T, bool AX, bool BX>
int gemm(const Operand<T> &a, const Operand<T> &b, int64_t K, int dtype, const Epilogue &ep, void *workspace, hipStream_t s) {
    if constexpr (!AX && !BX) {
        if (few(dtype, a.rows, b.rows, K)) return gemm_few<T>(a, b, K, ep, s);
    }
    const Plan p = plan_of(dtype, a.rows, b.rows, K, BX);
    const GemmArgs<T> g{a, b, K, p.tiles_m, p.tiles_n, p.splits, p.steps_per_split, ep, static_cast<float *>(workspace)};
    const bool aligned = whole_chunks<T>(a.p, a.ld, a.extent) && whole_chunks<T>(b.p, b.ld, b.extent);
    int rc;
    auto launch = [&](auto whole) {
        constexpr bool A = decltype(whole)::value;
        if (p.big) return launch_gemm<T, AX, BX, 256, 256, 128, 64, A>(g, s);
        if (p.width == 64) return launch_gemm<T, AX, BX, 128, 64, 32, 32, A>(g, s);
        if constexpr (!BX)
            if (p.width == 96) return launch_gemm<T, AX, BX, 128, 96, 32, 48, A>(g, s);
        return launch_gemm<T, AX, BX, 128, 128, 64, 32, A>(g, s);
    };
    rc = aligned ? launch(std::true_type{}) : launch(std::false_type{});
    if (rc) return rc;
    if (p.splits > 1) {
        const int64_t outs = a.rows * ((b.rows + 3) / 4);
        if (p.splits >= 16) gemm_join_kernel<16><<<dim3((unsigned)(outs < 16 << 16 ? (outs + 15) / 16 : 65536)), dim3(256), 0, s>>>(g.part, p.splits, a.rows, b.rows, ep);
        else gemm_join_kernel<1><<<dim3((unsigned)(outs < 256 << 16 ? (outs + 255) / 256 : 65536)), dim3(256), 0, s>>>(g.part, p.splits, a.rows, b.rows, ep);
        DETBOX_LAUNCH_CHECK();
    }
    return DETBOX_OK;
}

int check_linear(int dtype, int act, int64_t ldx, int64_t ldw, int64_t M, int64_t N, int64_t K) {
    DETBOX_CHECK_ARG(dtype_ok(dtype), "unknown element type");
    DETBOX_CHECK_ARG(act_ok(act), "unknown activation");
    DETBOX_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31), "bad size");
    DETBOX_CHECK_ARG(ldx >= K && ldw >= K, "row stride below the row length");
    // tiles are counted in 32 bits in each of the three products
    auto tiles = [](int64_t a, int64_t b) { return ((a + 127) / 128) * ((b + 127) / 128); };
    if (tiles(M, N) >= DETBOX_LINEAR_MAX_TILES || tiles(M, K) >= DETBOX_LINEAR_MAX_TILES || tiles(N, K) >= DETBOX_LINEAR_MAX_TILES) {
        set_error("%s: a product of DETBOX_LINEAR_MAX_TILES tiles or more", __func__);
        return DETBOX_ERR_UNSUPPORTED;
    }
    return DETBOX_OK;
}

int workspace_error(const char *who) {
    set_error("%s: workspace missing, misaligned or too small", who);
    return DETBOX_ERR_WORKSPACE;
}

// Row slices of the slope pass: about 2048 workgroups.
struct Slices { int count; int64_t rows; };
Slices slices_of(int64_t M, int64_t N) {
    int64_t n = 2048 / ((N + 255) / 256);
    const int64_t most = (M + 15) / 16;
    n = n > most ? most : n;
    n = n < 1 ? 1 : n;
    const int64_t rows = M > 0 ? (M + n - 1) / n : 1;
    return {(int)(M > 0 ? (M + rows - 1) / rows : 1), rows};
}

}  // namespace

extern "C" size_t detbox_linear_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
    if (!dtype_ok(dtype) || M < 1 || N < 1 || K < 1) return 0;
    return few(dtype, M, N, K) ? 0 : plan_bytes(plan_of(dtype, M, N, K, false), M, N);
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
    const size_t need = detbox_linear_workspace_bytes(dtype, M, N, K);
    if (need && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)) return workspace_error(__func__);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("linear_forward", s);
    const Epilogue ep{bias, bias_dtype, residual, ldr, activation, pre_activation, dtype, y, out_dtype};
    int rc = DETBOX_OK;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        rc = gemm<T, false, false>({static_cast<const T *>(x), ldx, M, K}, {static_cast<const T *>(weight), ldw, N, K}, K, dtype, ep,
                                   workspace, s);
    });
    return rc;
}

extern "C" size_t detbox_linear_backward_workspace_bytes(int dtype, int activation, int grad_dtype, int64_t M, int64_t N, int64_t K) {
    if (!dtype_ok(dtype) || M < 0 || N < 1 || K < 1) return 0;
    // dz has its place in every case: whether g can be used as it lies depends on its address and stride too
    (void)activation; (void)grad_dtype;
    const int64_t vec = 16 / (int64_t)dtype_size(dtype), ldz = (N + vec - 1) / vec * vec;
    size_t b = align_up((size_t)slices_of(M, N).count * (size_t)N * sizeof(float), 256);
    b += align_up((size_t)M * (size_t)ldz * dtype_size(dtype), 256);
    if (dtype == DETBOX_F16) b += align_up((PEAKS + 1) * sizeof(float), 256);
    const size_t px = M ? plan_bytes(plan_of(dtype, M, K, N, true), M, K) : 0, pw = M ? plan_bytes(plan_of(dtype, N, K, M, true), N, K) : 0;
    return b + (px > pw ? px : pw);
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
        workspace_bytes < detbox_linear_backward_workspace_bytes(dtype, activation, grad_dtype, M, N, K))
        return workspace_error(__func__);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("linear_backward", s);
    const Slices sl = slices_of(M, N);
    Carver ws(workspace);
    float *part = ws.take<float>((size_t)sl.count * N);
    int rc = DETBOX_OK;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t padded = (N + VEC_OF<T> - 1) / VEC_OF<T> * VEC_OF<T>;
        T *dz = ws.take<T>((size_t)M * padded);
        float *peaks = dtype == DETBOX_F16 ? ws.take<float>(PEAKS + 1) : nullptr, *unscale = nullptr;
        void *pieces = ws.take<char>(0);
        const bool slope = activation != DETBOX_ACTIVATION_NONE;
        // dz is written out where it is not g itself, or where g's rows start off 16 bytes
        const bool convert = slope || grad_dtype != dtype || !whole_chunks<T>(grad_y, ldg, N);
        // an fp16 dz that has other digits than g (which has its type, and relu keeps or drops it) is scaled into range
        const bool scaled = M && dtype == DETBOX_F16 && (grad_x || grad_weight) &&
                            (grad_dtype != dtype || (slope && activation != DETBOX_ACTIVATION_RELU));
        if (scaled) unscale = peaks + PEAKS;
        if (M && (convert || grad_bias)) {
            auto launch = [&](auto lanes) {
                constexpr int LANES = decltype(lanes)::value;
                int n_peaks = 0;
                if (scaled && (ldg == N || M == 1)) {
                    const int64_t n = M * N, blocks = (n + 1023) / 1024;
                    n_peaks = blocks < PEAKS ? (int)blocks : PEAKS;
                    const dim3 grid((unsigned)n_peaks), block(256);
                    if (grad_dtype == DETBOX_F32) linear_peak_dense_kernel<<<grid, block, 0, s>>>(static_cast<const float *>(grad_y), n, peaks);
                    else linear_peak_dense_kernel<<<grid, block, 0, s>>>(static_cast<const _Float16 *>(grad_y), n, peaks);
                } else if (scaled) {
                    const int64_t by_rows = (M + 256 / LANES - 1) / (256 / LANES), by_columns = (N + LANES * 4 - 1) / (LANES * 4);
                    const int64_t y = by_rows < PEAKS ? by_rows : PEAKS, x = by_columns < PEAKS / y ? by_columns : PEAKS / y;
                    n_peaks = (int)(x * y);
                    linear_peak_kernel<LANES><<<dim3((unsigned)x, (unsigned)y), dim3(256), 0, s>>>(grad_y, grad_dtype, ldg, M, N, peaks);
                }
                linear_slope_kernel<T, LANES><<<dim3((unsigned)((padded + LANES * 4 - 1) / (LANES * 4)), sl.count), dim3(256), 0, s>>>(
                    grad_y, grad_dtype, ldg, slope ? static_cast<const T *>(pre_activation) : nullptr, activation, M, N, padded, sl.rows,
                    convert ? dz : nullptr, grad_bias ? part : nullptr, scaled ? peaks : nullptr, n_peaks, unscale);
            };
            if (padded <= 32) launch(std::integral_constant<int, 8>{});
            else if (padded <= 128) launch(std::integral_constant<int, 32>{});
            else launch(std::integral_constant<int, 64>{});
        }
        const T *z = convert ? dz : static_cast<const T *>(grad_y);
        const int64_t ldz = convert ? padded : ldg, z_end = convert ? padded : N;
        Epilogue ep{nullptr, 0, nullptr, 0, DETBOX_ACTIVATION_NONE, nullptr, 0, grad_x, dtype, unscale};
        // the zeros behind N let the contraction over N run in whole chunks; the weight's rows end there
        if (grad_x && M) rc = gemm<T, false, true>({z, ldz, M, z_end}, {static_cast<const T *>(weight), ldw, K, K}, N, dtype, ep, pieces, s);
        ep.out = grad_weight;
        if (grad_weight && !rc) rc = gemm<T, true, true>({z, ldz, N, z_end}, {static_cast<const T *>(x), ldx, K, K}, M, dtype, ep, pieces, s);
    });
    if (rc) return rc;
    DETBOX_LAUNCH_CHECK();
    if (grad_bias) {
        column_join(part, M ? sl.count : 0, N, N, bias_dtype, grad_bias, nullptr, s);
        DETBOX_LAUNCH_CHECK();
    }
    return DETBOX_OK;
}
