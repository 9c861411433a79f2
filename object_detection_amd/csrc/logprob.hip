// Log probability of a given label, entropy and best alternatives of every row of logits, forward and backward.
//   m = max(x), s = sum exp(x - m), log p_j = (x_j - m) - log s
//   entropy = log s - sum exp(x - m) (x - m) / s;  alternatives: the top_k largest x (lower index first among equals)
//   grad_j = g (1[j = label] - p_j) - h p_j (log p_j + entropy), g and h the incoming gradients of the two
// A row whose label lies outside [0, C) does not take part: log probability 0, g taken as 0.  A row of -inf only has no
// distribution: log probability -inf, entropy 0, alternatives 0 .. top_k-1 with -inf, gradient 0.
//
// Every logit is read once in each direction.  Rows of up to 2048 logits live in the registers of 4, 16 or 64 lanes; longer
// rows are streamed with a running maximum and sums that are rescaled when the maximum grows, by one workgroup per row or,
// when there are few rows, by several whose partial results a second launch joins.  HBM bound: 4096 rows of 131071 bf16 logits
// 188 us forward = 5.7 TB/s, 358 us backward = 6.0 TB/s; 480348 rows of 81 fp32 logits 41 + 67 us.  With alternatives the 16-bit
// form of long rows takes 116-118 registers and 48 bytes of scratch per lane: four waves per SIMD, eight without.
#include "dtype.h"

using namespace detbox;

namespace {

constexpr int LP_BLOCK = 256, LP_WAVES = LP_BLOCK / 64;
// The larger word is the better alternative: by value (NaN above everything, -0 equal to +0), then by the lower index.
__device__ inline uint64_t rank_word(float v, uint32_t i) {
    const uint32_t k = v != v ? 0xffffffffu : okey_from_bits(__float_as_uint(v));
    return ((uint64_t)k << 32) | (uint32_t)~i;
}

// Distances from the largest logit where they are multiplied by their exponential, or by what meets it: no further than this, at
// which (and from -104 on) the exponential is 0 in fp32, so that the product is 0 too and not -inf * 0.  A sum of 2^31 terms or a
// gradient of 2^100 times it stays finite.
constexpr float FAR = -1e4f;

// A row's results from its largest logit (0 where it is -inf) and its sums.
struct RowSums { float ref, sum, dot; };        // sum of e = exp(x - ref), sum of e * (x - ref)
__device__ inline bool no_distribution(float m, float sum) { return m == -INFINITY && sum == 0.f; }

// Merges two running (largest, sum, dot): both sums are brought to the larger of the two references.
__device__ inline void merge_sums(float &m, float &s, float &t, float m2, float s2, float t2) {
    const float n = fmaxf(m, m2);
    const float ref = n == -INFINITY ? 0.f : n;
    const float d1 = m - ref, d2 = m2 - ref;                       // -inf for a side without a finite logit: its sums are 0
    const float e1 = fast_exp(d1), e2 = fast_exp(d2);
    t = e1 * fmaf(s, fmaxf(d1, FAR), t) + e2 * fmaf(s2, fmaxf(d2, FAR), t2);
    s = s * e1 + s2 * e2;
    m = n;
}

struct Outputs {
    float *log_probs, *entropy, *top_lp;
    int64_t *top_ids;
    float *stats;
};

__device__ inline void write_row(const Outputs &o, int64_t row, float m, float s, float t, float label_logit, bool part) {
    const bool none = no_distribution(m, s);
    const float ref = m == -INFINITY ? 0.f : m, ls = logf(s);
    o.log_probs[row] = !part ? 0.f : none ? -INFINITY : (label_logit - ref) - ls;
    if (o.entropy) o.entropy[row] = none ? 0.f : ls - t / s;
    if (o.stats) { o.stats[2 * row] = ref; o.stats[2 * row + 1] = s; }
}
template <typename T>
__device__ inline void write_alternative(const Outputs &o, const T *xr, int64_t row, int top_k, int rank, uint64_t word, float m, float s) {
    const uint32_t i = ~(uint32_t)word;
    o.top_ids[row * top_k + rank] = (int64_t)i;
    o.top_lp[row * top_k + rank] = no_distribution(m, s) ? -INFINITY : ((float)xr[i] - (m == -INFINITY ? 0.f : m)) - logf(s);
}

// ---- rows in registers ---------------------------------------------------------------------------------------------------

// G lanes per row, NV packs per lane: C <= G * NV * VEC.  HBM bound; the reductions over G <= 16 lanes are moves inside the
// vector unit.  The alternatives are taken one by one: every lane offers the best it has left.
template <typename T, int G, int NV>
__global__ __launch_bounds__(LP_BLOCK) void logprob_rows_kernel(const T *__restrict__ x, int64_t ld, const int64_t *__restrict__ labels,
                                                                int64_t rows, int C, int top_k, Outputs o) {
    constexpr int VEC = VEC_OF<T>, PER = LP_BLOCK / G;
    const int lane = threadIdx.x % G;
    for (int64_t row0 = (int64_t)blockIdx.x * PER; row0 < rows; row0 += (int64_t)gridDim.x * PER) {
        const int64_t row = row0 + threadIdx.x / G;
        const bool live = row < rows;
        const T *xr = x + (live ? row : row0) * ld;
        const int64_t label = live ? labels[row] : -1;
        const bool part = label >= 0 && label < C;
        const float at = part ? (float)xr[label] : 0.f;
        float v[NV][VEC];
        float m = -INFINITY;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int c = (q * G + lane) * VEC;
            load_pack<T>(v[q], xr + c, C - c, -INFINITY);
        }
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) m = fmaxf(m, v[q][i]);
        m = group_max<G>(m);
        const float ref = m == -INFINITY ? 0.f : m;
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = v[q][i] - ref, e = fast_exp(d);
                s += e;
                if (o.entropy) t = fmaf(e, fmaxf(d, FAR), t);
            }
        s = group_sum<G>(s);
        if (o.entropy) t = group_sum<G>(t);
        if (live && lane == 0) write_row(o, row, m, s, t, at, part);
        if (top_k) {
            uint64_t last = ~0ull;
            for (int k = 0; k < top_k; ++k) {
                uint64_t best = 0;
#pragma unroll
                for (int q = 0; q < NV; ++q)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const int c = (q * G + lane) * VEC + i;
                        const uint64_t w = rank_word(v[q][i], (uint32_t)c);
                        if (c < C && (w < last || k == 0) && w > best) best = w;
                    }
                best = group_max_u64<G>(best);
                if (live && lane == 0) write_alternative(o, xr, row, top_k, k, best, m, s);
                last = best;
            }
        }
    }
}

// ---- long rows -----------------------------------------------------------------------------------------------------------

// Best words of one wave's share of a row: a buffer in LDS that takes every logit above `bar`, and is cut to the top_k best
// when the next step might not fit.  The bar then is the value of the last one kept: the wave walks its share in index
// order, so a later equal value is not better.  The first bar is the top_k-th largest of the 64 lanes' maxima over the wave's
// first round, which top_k logits of that round reach: on ordinary logits little more than top_k words are ever taken and
// nothing is cut (2048 rows of 49999 fp16, five alternatives: 157 us with a buffer that is filled by the first step and cut,
// 65 us = 3.2 TB/s so).
constexpr int BUF = 640;

struct WaveBest {
    uint64_t *buf;
    int count;
    float bar;              // -inf at first: a class that cannot be is never among the words
};

// Keeps the k largest of count <= 64 * N distinct words.  T grows bit by bit to the largest prefix that k words reach.
template <int N>
__device__ inline void cut_words(WaveBest &b, int k) {
    const int lane = threadIdx.x & 63;
    uint64_t w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = i * 64 + lane < b.count ? b.buf[i * 64 + lane] : 0;
    uint64_t T = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t c = T | (1ull << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popcll(__ballot(w[i] >= c));
        if (n >= k) T = c;
        if (n == k) break;
    }
    int at = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool keep = w[i] >= T && w[i] != 0;
        const unsigned long long mask = __ballot(keep);
        if (keep) b.buf[at + __popcll(mask & ((1ull << lane) - 1))] = w[i];
        at += __popcll(mask);
    }
    b.count = at;
    b.bar = __uint_as_float(bits_from_okey((uint32_t)(T >> 32)));
    __builtin_amdgcn_wave_barrier();
}
__device__ inline void cut_best(WaveBest &b, int k) {
    if (b.count <= k) return;
    if (b.count <= 192) cut_words<3>(b, k);
    else cut_words<BUF / 64>(b, k);
}

// The largest T that k lanes' keys reach (0 where fewer than k lanes have one).
__device__ inline uint32_t kth_key(uint32_t key, int k) {
    uint32_t T = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = T | (1u << bit);
        const int n = __popcll(__ballot(key >= c));
        if (n >= k) T = c;
        if (n == k) break;
    }
    return T;
}
// A bar that every value of at least T's passes (no key lies between those of the negative numbers and +0).
__device__ inline float bar_below(uint32_t T) {
    return __uint_as_float(bits_from_okey(T == 0x80000000u ? 0x7ffffffeu : T - 1u));
}

__device__ inline void offer(WaveBest &b, bool take, uint64_t word) {
    const unsigned long long mask = __ballot(take);
    if (take) b.buf[b.count + __popcll(mask & ((1ull << (threadIdx.x & 63)) - 1))] = word;
    b.count += __popcll(mask);
}

// The workgroup's best of its waves' buffers: words[0 .. n) in LDS, n <= LP_WAVES * 64; rank of a word = how many are larger.
__device__ inline int join_waves(WaveBest &b, int k, uint64_t *words, int *counts) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (b.count > DETBOX_MAX_ALTERNATIVES) cut_best(b, k);
    if (lane == 0) counts[w] = b.count;
    __syncthreads();
    int at = 0, n = 0;
    for (int i = 0; i < LP_WAVES; ++i) { if (i < w) at += counts[i]; n += counts[i]; }
    if (lane < b.count) words[at + lane] = b.buf[lane];
    if (threadIdx.x < 8) words[n + threadIdx.x] = 0;                       // rank_of reads in eights
    __syncthreads();
    return n;
}
constexpr int WORDS = LP_WAVES * DETBOX_MAX_ALTERNATIVES + 8;
__device__ inline int rank_of(uint64_t word, const uint64_t *words, int n) {
    int r = 0;
    for (int i = 0; i < n; i += 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) r += words[i + j] > word;
    return r;
}

// Writes a row's alternatives from the n words of its workgroup (more than top_k of them, or all of the row's logits above
// -inf).  What is missing to top_k are classes at -inf: the lowest indices that are no word's.
template <typename T>
__device__ inline void write_alternatives(const Outputs &o, const T *xr, int64_t row, int top_k, const uint64_t *words, int n, float m, float s) {
    if (threadIdx.x < n) {
        const uint64_t w = words[threadIdx.x];
        const int r = rank_of(w, words, n);
        if (r < top_k) write_alternative(o, xr, row, top_k, r, w, m, s);
    }
    if (n < top_k && threadIdx.x < top_k) {
        const uint32_t i = threadIdx.x;
        int below = 0;
        bool taken = false;
        for (int j = 0; j < n; ++j) {
            const uint32_t at = ~(uint32_t)words[j];
            below += at < i;
            taken |= at == i;
        }
        const int r = n + (int)i - below;
        if (!taken && r < top_k) write_alternative(o, xr, row, top_k, r, (uint64_t)(uint32_t)~i, m, s);
    }
}

// Block-wide merge of every lane's running sums into (m, s, t) of all threads.
__device__ inline void block_sums(float &m, float &s, float &t, float *sm, float *ss, float *st) {
    const float most = group_max<64>(m);
    merge_sums(m, s, t, most, 0.f, 0.f);                                   // to the wave's reference
    s = group_sum<64>(s);
    t = group_sum<64>(t);
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { sm[w] = m; ss[w] = s; st[w] = t; }
    __syncthreads();
    m = sm[0]; s = ss[0]; t = st[0];
#pragma unroll
    for (int i = 1; i < LP_WAVES; ++i) merge_sums(m, s, t, sm[i], ss[i], st[i]);
}

// Alternatives of a row that holds NaN (its sum is NaN): one pass over the row per alternative.  Rare, and the streaming
// pass need not look for NaN among its logits.
template <typename T>
__device__ void slow_alternatives(const Outputs &o, const T *xr, int64_t row, int64_t C, int top_k, float m, float s, uint64_t *words) {
    uint64_t last = ~0ull;
    for (int k = 0; k < top_k; ++k) {
        uint64_t best = 0;
        for (int64_t i = threadIdx.x; i < C; i += LP_BLOCK) {
            const uint64_t w = rank_word((float)xr[i], (uint32_t)i);
            if ((w < last || k == 0) && w > best) best = w;
        }
        best = group_max_u64<64>(best);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = best;
        __syncthreads();
        for (int i = 0; i < LP_WAVES; ++i) best = words[i] > best ? words[i] : best;
        if (threadIdx.x == 0) write_alternative(o, xr, row, top_k, k, best, m, s);
        last = best;
    }
}

// Elements in front of the row's first cache line of 128 bytes (at most 63: one per lane of a wave).
template <typename T>
__device__ inline int head_of(const T *xr, int64_t C) {
    const int h = (int)((0 - (uintptr_t)xr) % 128 / sizeof(T));
    return h < C ? h : (int)C;
}

struct Partial { float m, s, t, unused; };

// One workgroup per (row, piece).  pieces == 1: the row's results are written here; otherwise a Partial and, with TOP, top_k
// words (0 where the piece has fewer) go to the workspace.
template <typename T, bool TOP, bool ENT>
__global__ __launch_bounds__(LP_BLOCK) void logprob_long_kernel(const T *__restrict__ x, int64_t ld, const int64_t *__restrict__ labels,
                                                                int64_t rows, int64_t C, int top_k, int pieces, int64_t piece,
                                                                Outputs o, Partial *__restrict__ partial,
                                                                uint64_t *__restrict__ partial_words) {
    constexpr int VEC = VEC_OF<T>, U = 4, STEP = 64 * VEC;
    static_assert(STEP + DETBOX_MAX_ALTERNATIVES <= BUF, "a step must fit the buffer");
    __shared__ uint64_t s_buf[TOP ? LP_WAVES * BUF : 1];
    __shared__ uint64_t s_words[WORDS];
    __shared__ float s_m[LP_WAVES], s_s[LP_WAVES], s_t[LP_WAVES];
    __shared__ int s_n[LP_WAVES];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t jobs = rows * pieces;
    for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int64_t row = job / pieces, lo = (job % pieces) * piece, hi = lo + piece < C ? lo + piece : C;
        const T *xr = x + row * ld;
        float m = -INFINITY, s = 0.f, t = 0.f;
        WaveBest best{s_buf + (TOP ? wv * BUF : 0), 0, -INFINITY};

        auto take_in = [&](const float (&v)[VEC]) {
            float top = v[0];
#pragma unroll
            for (int i = 1; i < VEC; ++i) top = fmaxf(top, v[i]);
            if (top > m) {
                const float d = m - top, e = fast_exp(d);                  // m == -inf: e = 0 and both sums are 0
                if (ENT) t = e * fmaf(s, fmaxf(d, FAR), t);
                s *= e;
                m = top;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = v[i] - ref, e = fast_exp(d);
                s += e;
                if (ENT) t = fmaf(e, fmaxf(d, FAR), t);
            }
            return top;
        };
        // left: how many of the pack's logits are there
        auto alternatives = [&](const float (&v)[VEC], float top, int64_t c, int left) {
            if (!__any(!(top <= best.bar))) return;
            if (best.count + STEP > BUF) cut_best(best, top_k);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {                                // not in index order inside the step: words are distinct
                const bool take = i < left && !(v[i] <= best.bar);
                if (__any(take)) offer(best, take, rank_word(v[i], (uint32_t)(c + i)));
            }
        };

        // Steps start at cache lines: rows that start off them cost a fifth of the bandwidth (4096 rows of bf16: 131072 logits
        // 186 us, 131071 logits 229 us before, 182 so); the row's first few logits go one per lane of the first wave.  Loads
        // are not kept in the caches: 1.07 GB 163 us against 182; at 268 MB, where the backward pass might have found some of
        // them, forward + backward are 47 + 81 us against 79 + 78, at 134 MB 26 + 43 against 28 + 41.
        const int head = head_of<T>(xr, C);
        if (lo == 0 && head && wv == 0) {
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = -INFINITY;
            if (lane < head) v[0] = (float)xr[lane];
            const float top = take_in(v);
            if (TOP) alternatives(v, top, lane, lane < head);
        }
        const int64_t first = lo + head, end = hi + head < C ? hi + head : C;
        bool fresh = true;
        auto round = [&](const float (&v)[U][VEC], int64_t c, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;                 // all of the round's logits are there
            float tops[U];
#pragma unroll
            for (int u = 0; u < U; ++u) tops[u] = take_in(v[u]);
            if (!TOP) return;
            uint32_t reach = 0;
            if (fresh) {
                float most = tops[0];
#pragma unroll
                for (int u = 1; u < U; ++u) most = fmaxf(most, tops[u]);
                reach = kth_key(WHOLE || c < end ? okey_from_bits(__float_as_uint(most)) : 0u, top_k);
                if (reach > 0x007fffffu) best.bar = bar_below(reach);     // 0x007fffff: the key of -inf
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t left = end - c - u * STEP;
                alternatives(v[u], tops[u], c + u * STEP, WHOLE || left >= VEC ? VEC : left < 0 ? 0 : (int)left);
            }
            const float at = __uint_as_float(bits_from_okey(reach));
            if (fresh && reach > 0x007fffffu && !(at < best.bar)) best.bar = at;
            fresh = false;
        };
        int64_t c = first + (int64_t)wv * STEP * U + lane * VEC;
        for (; c - lane * VEC + STEP * U <= end; c += (int64_t)LP_WAVES * STEP * U) {
            float v[U][VEC];
            detbox_u4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = load_raw_nt<T>(xr + c + u * STEP);
#pragma unroll
            for (int u = 0; u < U; ++u) unpack<T>(v[u], raw[u]);
            round(v, c, std::true_type{});
        }
        if (c - lane * VEC < end) {                                        // the wave's last, partial round
            float v[U][VEC];
            load_packs_to_end<T, U>(v, xr, c, STEP, end, -INFINITY);
            round(v, c, std::false_type{});
        }
        block_sums(m, s, t, s_m, s_s, s_t);
        int n = 0;
        if (TOP) n = join_waves(best, top_k, s_words, s_n);
        if (pieces == 1) {
            if (threadIdx.x == 0) {
                const int64_t label = labels[row];
                const bool part = label >= 0 && label < C;
                write_row(o, row, m, s, t, part ? (float)xr[label] : 0.f, part);
            }
            if (TOP) {
                if (s != s) {
                    __syncthreads();
                    slow_alternatives<T>(o, xr, row, C, top_k, m, s, s_words);
                } else {
                    write_alternatives<T>(o, xr, row, top_k, s_words, n, m, s);
                }
            }
        } else {
            if (threadIdx.x == 0) partial[job] = Partial{m, s, t, 0.f};
            if (TOP) {
                const uint64_t w = threadIdx.x < n ? s_words[threadIdx.x] : 0;
                const int r = threadIdx.x < n ? rank_of(w, s_words, n) : top_k;
                if (r < top_k) partial_words[job * top_k + r] = w;
                if (threadIdx.x < top_k && threadIdx.x >= n) partial_words[job * top_k + threadIdx.x] = 0;
            }
        }
        __syncthreads();
    }
}

// Joins the pieces of a row: one workgroup per row.
template <typename T>
__global__ __launch_bounds__(LP_BLOCK) void logprob_join_kernel(const T *__restrict__ x, int64_t ld, const int64_t *__restrict__ labels,
                                                                int64_t rows, int64_t C, int top_k, int pieces,
                                                                const Partial *__restrict__ partial,
                                                                const uint64_t *__restrict__ partial_words, Outputs o) {
    __shared__ uint64_t s_buf[LP_WAVES * BUF], s_words[WORDS];
    __shared__ float s_m[LP_WAVES], s_s[LP_WAVES], s_t[LP_WAVES];
    __shared__ int s_n[LP_WAVES];
    const int wv = threadIdx.x >> 6;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ld;
        float m = -INFINITY, s = 0.f, t = 0.f;
        for (int i = threadIdx.x; i < pieces; i += LP_BLOCK) {
            const Partial p = partial[row * pieces + i];
            merge_sums(m, s, t, p.m, p.s, p.t);
        }
        block_sums(m, s, t, s_m, s_s, s_t);
        if (threadIdx.x == 0) {
            const int64_t label = labels[row];
            const bool part = label >= 0 && label < C;
            write_row(o, row, m, s, t, part ? (float)xr[label] : 0.f, part);
        }
        if (top_k) {
            if (s != s) {
                slow_alternatives<T>(o, xr, row, C, top_k, m, s, s_words);
            } else {
                WaveBest best{s_buf + wv * BUF, 0, -INFINITY};
                const int total = pieces * top_k;
                for (int i0 = wv * 64; i0 < total; i0 += LP_BLOCK) {
                    const int i = i0 + (threadIdx.x & 63);
                    const uint64_t w = i < total ? partial_words[row * total + i] : 0;
                    if (best.count + 64 > BUF) cut_best(best, top_k);
                    offer(best, w != 0, w);
                }
                const int n = join_waves(best, top_k, s_words, s_n);
                write_alternatives<T>(o, xr, row, top_k, s_words, n, m, s);
            }
        }
        __syncthreads();
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------

// What a row needs of its statistics: grad_j = hit - p (g + h (log p + entropy)) = hit - p (a + h d), d = x - ref
struct RowGrad { float ref, inv, a, h, g; int64_t label; bool zero; };
__device__ inline RowGrad row_grad(int64_t row, int64_t C, const int64_t *labels, const float *stats, const float *entropy,
                                   const float *grad_lp, const float *grad_ent) {
    RowGrad r;
    const float s = stats[2 * row + 1];
    r.ref = stats[2 * row];
    r.label = labels[row];
    const bool part = r.label >= 0 && r.label < C;
    if (!part) r.label = -1;
    r.g = grad_lp && part ? grad_lp[row] : 0.f;
    r.h = grad_ent ? grad_ent[row] : 0.f;
    r.inv = 1.0f / s;
    r.a = grad_ent ? fmaf(r.h, entropy[row] - logf(s), r.g) : r.g;
    r.zero = s == 0.f || !(grad_ent || (part && grad_lp));
    return r;
}
template <int VEC>
__device__ inline void grad_pack(float (&v)[VEC], const RowGrad &r, int64_t c) {
    if (r.zero) {                                     // a row that does not take part has gradient 0 whatever it holds
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 0.f;
        return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const float d = v[i] - r.ref, p = fast_exp(d) * r.inv;
        v[i] = -p * fmaf(r.h, fmaxf(d, FAR), r.a);
    }
    const int64_t at = r.label - c;
    if (at >= 0 && at < VEC) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i == (int)at) v[i] += r.g;
    }
}

// Short rows: the lanes that hold a row in the forward pass.
template <typename T, int G>
__global__ __launch_bounds__(LP_BLOCK) void logprob_rows_grad_kernel(const T *__restrict__ x, int64_t ld, const int64_t *__restrict__ labels,
                                                                     int64_t rows, int C, const float *__restrict__ stats,
                                                                     const float *__restrict__ entropy, const float *__restrict__ grad_lp,
                                                                     const float *__restrict__ grad_ent, T *__restrict__ gx) {
    constexpr int VEC = VEC_OF<T>, PER = LP_BLOCK / G;
    const int lane = threadIdx.x % G;
    for (int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G; row < rows; row += (int64_t)gridDim.x * PER) {
        const RowGrad r = row_grad(row, C, labels, stats, entropy, grad_lp, grad_ent);
        const T *xr = x + row * ld;
        T *gr = gx + row * C;
        for (int c = lane * VEC; c < C; c += G * VEC) {
            float v[VEC];
            load_pack<T>(v, xr + c, C - c, -INFINITY);
            grad_pack<VEC>(v, r, c);
            store_pack<T>(gr + c, C - c, v);
        }
    }
}

// Long rows: a workgroup takes pieces of 4 packs per thread.
template <typename T>
__global__ __launch_bounds__(LP_BLOCK) void logprob_long_grad_kernel(const T *__restrict__ x, int64_t ld, const int64_t *__restrict__ labels,
                                                                     int64_t rows, int64_t C, int64_t pieces,
                                                                     const float *__restrict__ stats, const float *__restrict__ entropy,
                                                                     const float *__restrict__ grad_lp, const float *__restrict__ grad_ent,
                                                                     T *__restrict__ gx) {
    constexpr int VEC = VEC_OF<T>, U = 4;
    for (int64_t job = blockIdx.x; job < rows * pieces; job += gridDim.x) {
        const int64_t row = job / pieces, lo = (job % pieces) * (LP_BLOCK * VEC * U);
        const RowGrad r = row_grad(row, C, labels, stats, entropy, grad_lp, grad_ent);
        const T *xr = x + row * ld;
        T *gr = gx + row * C;
        const int head = head_of<T>(gr, C);                 // the logits start where the gradient does unless they are strided
        const bool at_head = lo == 0 && threadIdx.x < head;
        float front[1] = {at_head ? (float)xr[threadIdx.x] : 0.f};
        const int64_t first = lo + head;
        if (first + LP_BLOCK * VEC * U <= C) {
            float v[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) unpack<T>(v[u], load_raw_nt<T>(xr + first + (u * LP_BLOCK + threadIdx.x) * VEC));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = first + (u * LP_BLOCK + threadIdx.x) * VEC;
                grad_pack<VEC>(v[u], r, c);
                store_pack<T>(gr + c, v[u]);
            }
        } else {
            float v[U][VEC];
            load_packs_to_end<T, U>(v, xr, first + threadIdx.x * VEC, LP_BLOCK * VEC, C, -INFINITY);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = first + (u * LP_BLOCK + threadIdx.x) * VEC;
                grad_pack<VEC>(v[u], r, c);
                store_pack<T>(gr + c, C - c, v[u]);
            }
        }
        if (at_head) {
            grad_pack<1>(front, r, threadIdx.x);
            gr[threadIdx.x] = (T)front[0];
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------

constexpr int64_t SHORT_ROW = 2048;

int check_logprob(int dtype, const void *logits, int64_t ld, const int64_t *labels, int64_t rows, int64_t C) {
    DETBOX_CHECK_ARG(dtype_ok(dtype), "unknown element type");
    DETBOX_CHECK_ARG(rows >= 0 && C >= 1 && rows < (1ll << 40) && C < (1ll << 31), "bad size");
    DETBOX_CHECK_ARG(ld >= C, "row stride below the row length");
    DETBOX_CHECK_ARG(rows == 0 || (logits && labels), "null pointer");
    return DETBOX_OK;
}

// How a long row is cut: into pieces of at least 4096 logits while there are fewer than 1024 workgroups (four per CU).
struct Cut { int pieces; int64_t piece; };
Cut cut_of(int64_t rows, int64_t C) {
    int64_t n = rows < 1 ? 1 : 1024 / rows;
    const int64_t most = (C + 4095) / 4096;
    n = n < 1 ? 1 : n > most ? most : n;
    n = n > 64 ? 64 : n;
    int64_t piece = (C + n - 1) / n;
    piece = (piece + 511) / 512 * 512;
    return {(int)((C + piece - 1) / piece), piece};
}
unsigned grid_of(int64_t jobs) { return (unsigned)(jobs < (1 << 22) ? jobs : (1 << 22)); }

template <typename T, int G, int NV>
void launch_rows(const T *x, int64_t ld, const int64_t *labels, int64_t rows, int64_t C, int top_k, const Outputs &o, hipStream_t s) {
    constexpr int PER = LP_BLOCK / G;
    logprob_rows_kernel<T, G, NV><<<dim3(grid_of((rows + PER - 1) / PER)), dim3(LP_BLOCK), 0, s>>>(x, ld, labels, rows, (int)C, top_k, o);
}

}  // namespace

extern "C" size_t detbox_label_log_probs_workspace_bytes(int64_t rows, int64_t C, int top_k) {
    if (rows < 1 || C <= SHORT_ROW || top_k < 0) return 0;
    const Cut c = cut_of(rows, C);
    if (c.pieces == 1) return 0;
    return align_up((size_t)rows * c.pieces * sizeof(Partial), 256) + align_up((size_t)rows * c.pieces * top_k * sizeof(uint64_t), 256);
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
    const size_t need = detbox_label_log_probs_workspace_bytes(rows, C, top_k);
    if (need && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)) {
        set_error("%s: workspace missing, misaligned or too small", __func__);
        return DETBOX_ERR_WORKSPACE;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    ProfScope ps("label_log_probs_forward", s);
    const Outputs o{log_probs, entropy, top_log_probs, top_ids, stats};
    with_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        constexpr int W = 8 / VEC_OF<T>;                       // packs per eight logits: 1 for the 16-bit types, 2 for fp32
        const T *x = static_cast<const T *>(logits);
        if (C <= 32) launch_rows<T, 4, W>(x, ld, labels, rows, C, top_k, o, s);
        else if (C <= 128) launch_rows<T, 16, W>(x, ld, labels, rows, C, top_k, o, s);
        else if (C <= 256) launch_rows<T, 16, 2 * W>(x, ld, labels, rows, C, top_k, o, s);
        else if (C <= 512) launch_rows<T, 64, W>(x, ld, labels, rows, C, top_k, o, s);
        else if (C <= 1024) launch_rows<T, 64, 2 * W>(x, ld, labels, rows, C, top_k, o, s);
        else if (C <= SHORT_ROW) launch_rows<T, 64, 4 * W>(x, ld, labels, rows, C, top_k, o, s);
        else {
            const Cut cut = cut_of(rows, C);
            Carver ws(workspace);
            Partial *partial = nullptr;
            uint64_t *words = nullptr;
            if (cut.pieces > 1) {
                partial = ws.take<Partial>((size_t)rows * cut.pieces);
                words = ws.take<uint64_t>((size_t)rows * cut.pieces * top_k);
            }
            const dim3 grid(grid_of(rows * cut.pieces)), block(LP_BLOCK);
            auto launch = [&](auto top, auto ent) {
                logprob_long_kernel<T, decltype(top)::value, decltype(ent)::value>
                    <<<grid, block, 0, s>>>(x, ld, labels, rows, C, top_k, cut.pieces, cut.piece, o, partial, words);
            };
            if (top_k) entropy ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
            else entropy ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
            if (cut.pieces > 1)
                logprob_join_kernel<T><<<dim3(grid_of(rows)), block, 0, s>>>(x, ld, labels, rows, C, top_k, cut.pieces, partial, words, o);
        }
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
    with_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        const T *x = static_cast<const T *>(logits);
        T *gx = static_cast<T *>(grad_logits);
        auto rows_grad = [&](auto lanes) {
            constexpr int G = decltype(lanes)::value, PER = LP_BLOCK / G;
            logprob_rows_grad_kernel<T, G><<<dim3(grid_of((rows + PER - 1) / PER)), dim3(LP_BLOCK), 0, s>>>(
                x, ld, labels, rows, (int)C, stats, entropy, grad_log_probs, grad_entropy, gx);
        };
        if (C <= 32) rows_grad(std::integral_constant<int, 4>{});
        else if (C <= 256) rows_grad(std::integral_constant<int, 16>{});
        else if (C <= SHORT_ROW) rows_grad(std::integral_constant<int, 64>{});
        else {
            const int64_t pieces = (C + LP_BLOCK * VEC_OF<T> * 4 - 1) / (LP_BLOCK * VEC_OF<T> * 4);
            logprob_long_grad_kernel<T><<<dim3(grid_of(rows * pieces)), dim3(LP_BLOCK), 0, s>>>(
                x, ld, labels, rows, C, pieces, stats, entropy, grad_log_probs, grad_entropy, gx);
        }
    });
    DETBOX_LAUNCH_CHECK();
    return DETBOX_OK;
}
