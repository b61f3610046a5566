// Objectives on log-probabilities: label log-probs of rows of logits and their
// gradient, a preference loss over paired log ratios, and a clipped policy
// loss with a KL term (group 3 of include/warpgbm_b200.h).
//
// Arithmetic.  A row of logits is reduced to (m, s, t): m = max x, s = sum of
// 2^d and t = sum of 2^d d over d = (x - m) c, c = log2(e) / temperature, all
// in fp32.  Then, in natural units, log s + m / temperature is the
// log-sum-exp, (x_y - m) / temperature - log s the label's log-prob and
// log s - ln2 t / s the entropy.  Sums over tokens are exact: a partial sum
// formed in a fixed order is added to a 128-bit fixed-point number with
// integer atomics (Acc), so no result depends on the order of the atomics.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace wgb {

constexpr float LN2F = 0.693147180559945309f;
constexpr double LOG2E = 1.44269504088896340736;

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 16 bytes of logits as fp32 and back (one rounding to nearest, on the way out)
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    __device__ static void unpack(const uint4 &u, float (&f)[4]) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    __device__ static uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    __device__ static float to(float v) { return v; }
    __device__ static float from(float f) { return f; }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ static void unpack(const uint4 &u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 from(float f) { return __float2bfloat16_rn(f); }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    __device__ static void unpack(const uint4 &u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
    __device__ static uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float to(__half v) { return __half2float(v); }
    __device__ static __half from(float f) { return __float2half_rn(f); }
};

// An index array of 4- or 8-byte integers.
struct Idx {
    const void *p;
    int wide;
    __device__ __forceinline__ long long at(long long i) const {
        return wide ? static_cast<const long long *>(p)[i] : static_cast<const int *>(p)[i];
    }
};

// ------------------------------------------------------------ row sums --
struct RowSum {
    float m, s, t;
};
__device__ __forceinline__ RowSum row_empty() { return RowSum{-INFINITY, 0.0f, 0.0f}; }

// A maximum that is subtracted: a row that is all -inf keeps exponents of -inf.
__device__ __forceinline__ float finite_top(float m) { return m == -INFINITY ? 0.0f : m; }

// d below every exponent that 2^d does not flush to zero, for d * 2^d terms
// that must not be -inf * 0
constexpr float D_FLOOR = -1000.0f;

template <bool ENT>
__device__ __forceinline__ void row_add(RowSum &a, float x, float top, float c) {
    const float d = (x - top) * c;
    const float e = exp2_fast(d);
    a.s += e;
    if (ENT) a.t = fmaf(e, fmaxf(d, D_FLOOR), a.t);
}

// Moves the sums of `a` to the maximum `m` >= a.m.
template <bool ENT>
__device__ __forceinline__ void row_shift(RowSum &a, float m, float c) {
    const float d = (a.m - finite_top(m)) * c;  // -inf where a is empty
    const float f = exp2_fast(d);
    if (ENT) a.t = f * fmaf(a.s, fmaxf(d, D_FLOOR), a.t);
    a.s *= f;
    a.m = m;
}

template <bool ENT>
__device__ __forceinline__ RowSum row_join(RowSum a, RowSum b, float c) {
    const float m = fmaxf(a.m, b.m);
    row_shift<ENT>(a, m, c);
    row_shift<ENT>(b, m, c);
    a.s += b.s;
    if (ENT) a.t += b.t;
    return a;
}

// Sums over the G threads of a group: a warp, or the whole block.
template <int G, bool ENT>
__device__ __forceinline__ RowSum group_join(RowSum a, float c, RowSum *scratch /* >= 33 */) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSum b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.t = ENT ? __shfl_xor_sync(0xffffffffu, a.t, o) : 0.0f;
        a = row_join<ENT>(a, b, c);
    }
    if (G > 32) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        if (lane == 0) scratch[w] = a;
        __syncthreads();
        if (w == 0) {
            RowSum b = lane < G / 32 ? scratch[lane] : row_empty();
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                RowSum t;
                t.m = __shfl_xor_sync(0xffffffffu, b.m, o);
                t.s = __shfl_xor_sync(0xffffffffu, b.s, o);
                t.t = ENT ? __shfl_xor_sync(0xffffffffu, b.t, o) : 0.0f;
                b = row_join<ENT>(b, t, c);
            }
            if (lane == 0) scratch[32] = b;
        }
        __syncthreads();
        a = scratch[32];
        __syncthreads();
    }
    return a;
}

// Row of K elements as: `head` single elements, `vecs` aligned 16-byte words,
// then single elements again.
struct RowCut {
    long long head, vecs;
};
template <typename T>
__device__ __forceinline__ RowCut row_cut(const T *row, long long K) {
    constexpr int N = Vec<T>::N;
    const int off = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % N);
    long long head = off ? N - off : 0;
    if (head > K) head = K;
    return RowCut{head, (K - head) / N};
}

// (m, s, t) of this thread's share of a row.
template <typename T, int G, bool ENT>
__device__ __forceinline__ RowSum row_scan(const T *row, long long K, int tid, float c) {
    constexpr int N = Vec<T>::N;
    RowSum a = row_empty();
    auto single = [&](long long j) {
        const float x = Vec<T>::to(row[j]);
        if (x > a.m) row_shift<ENT>(a, x, c);
        row_add<ENT>(a, x, finite_top(a.m), c);
    };
    if (G <= 32) {
        for (long long j = tid; j < K; j += G) single(j);
        return a;
    }
    const RowCut cut = row_cut(row, K);
    if (tid < cut.head) single(tid);
    const uint4 *v = reinterpret_cast<const uint4 *>(row + cut.head);
    constexpr int U = 4;
    for (long long i = tid; i < cut.vecs; i += (long long)G * U) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + (long long)u * G < cut.vecs) w[u] = v[i + (long long)u * G];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + (long long)u * G >= cut.vecs) break;
            float f[N];
            Vec<T>::unpack(w[u], f);
            float m = f[0];
#pragma unroll
            for (int k = 1; k < N; ++k) m = fmaxf(m, f[k]);
            if (m > a.m) row_shift<ENT>(a, m, c);
            const float top = finite_top(a.m);
#pragma unroll
            for (int k = 0; k < N; ++k) row_add<ENT>(a, f[k], top, c);
        }
    }
    for (long long j = cut.head + cut.vecs * N + tid; j < K; j += G) single(j);
    return a;
}

// What a row's sums say: log-prob of the label, log-sum-exp, entropy.
struct RowStat {
    float logp, lse, ent, logs;
};
template <typename T, bool ENT>
__device__ __forceinline__ RowStat row_stat(const RowSum &a, const T *row, long long K, long long y, float inv_t) {
    RowStat r{-INFINITY, -INFINITY, 0.0f, 0.0f};
    if (a.s == 0.0f) return r;  // every logit is -inf
    r.logs = logf(a.s);
    r.lse = fmaf(a.m, inv_t, r.logs);
    r.logp = y < K ? fmaf(Vec<T>::to(row[y]) - a.m, inv_t, -r.logs) : NAN;
    if (ENT) r.ent = r.logs - LN2F * (a.t / a.s);
    return r;
}

template <typename T, int G, int NT, bool ENT>
__global__ void __launch_bounds__(NT) k_label_logprobs(const T *logits, long long rows, long long K, long long stride,
                                                       Idx labels, float inv_t, float *logp, float *lse, float *ent) {
    __shared__ RowSum scratch[33];
    pdl_wait();
    const int tid = threadIdx.x % G;
    const float c = (float)(LOG2E * inv_t);
    const long long step = (long long)gridDim.x * (NT / G);
    for (long long i = (long long)blockIdx.x * (NT / G) + threadIdx.x / G; i < rows; i += step) {
        const long long y = labels.at(i);
        if (y < 0) {
            if (tid == 0) {
                logp[i] = 0.0f;
                lse[i] = 0.0f;
                if (ENT) ent[i] = 0.0f;
            }
            continue;
        }
        const T *row = logits + i * stride;
        const RowSum a = group_join<G, ENT>(row_scan<T, G, ENT>(row, K, tid, c), c, scratch);
        if (tid == 0) {
            const RowStat r = row_stat<T, ENT>(a, row, K, y, inv_t);
            logp[i] = r.logp;
            lse[i] = r.lse;
            if (ENT) ent[i] = r.ent;
        }
    }
}

// One row of gradient: d x_j = g ([j = y] - p_j) - ge p_j (log p_j + H), with
// log2 p_j = (x_j - top) c - b (subtracting a top near the row's maximum first
// keeps the digits of rows whose logits are all huge); `empty` rows get zeros.
struct RowGrad {
    float top, c, b, g, ge, ent;
    int empty;
};
__device__ __forceinline__ float grad_at(const RowGrad &r, float x) {
    const float d = fmaf(x - r.top, r.c, -r.b);
    const float p = exp2_fast(d);
    const float h = fmaf(fmaxf(d, D_FLOOR), LN2F, r.ent);
    return -p * fmaf(r.ge, h, r.g);
}

template <typename T, int G>
__device__ __forceinline__ void row_grad(const T *row, T *out, long long K, long long y, int tid, const RowGrad &r) {
    constexpr int N = Vec<T>::N;
    auto single = [&](long long j) {
        float v = r.empty ? 0.0f : grad_at(r, Vec<T>::to(row[j]));
        if (j == y && !r.empty) v += r.g;
        out[j] = Vec<T>::from(v);
    };
    const RowCut cut = row_cut(row, K);
    const bool vec = G > 32 && (reinterpret_cast<uintptr_t>(row) - reinterpret_cast<uintptr_t>(out)) % 16 == 0;
    if (!vec) {  // a warp's row, or an output that is aligned otherwise than its input
        for (long long j = tid; j < K; j += G) single(j);
        return;
    }
    if (tid < cut.head) single(tid);
    const uint4 *v = reinterpret_cast<const uint4 *>(row + cut.head);
    uint4 *o = reinterpret_cast<uint4 *>(out + cut.head);
    for (long long i = tid; i < cut.vecs; i += G) {
        float f[N];
        Vec<T>::unpack(v[i], f);
        const long long j0 = cut.head + i * N;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            f[k] = r.empty ? 0.0f : grad_at(r, f[k]);
            if (j0 + k == y && !r.empty) f[k] += r.g;
        }
        o[i] = Vec<T>::pack(f);
    }
    for (long long j = cut.head + cut.vecs * N + tid; j < K; j += G) single(j);
}

// Beyond this |lse| its rounding alone moves every p by more than 2^-16, and
// the row is summed again.
constexpr float LSE_EXACT = 256.0f;

template <typename T, int G, int NT>
__global__ void __launch_bounds__(NT) k_label_logprobs_grad(const T *logits, long long rows, long long K,
                                                            long long stride, Idx labels, float temperature,
                                                            const float *lse, const float *grad_logp, const float *ent,
                                                            const float *grad_ent, T *out, long long out_stride) {
    __shared__ RowSum scratch[33];
    pdl_wait();
    const int tid = threadIdx.x % G;
    const float inv_t = 1.0f / temperature;
    const float c = (float)(LOG2E * inv_t);
    const long long step = (long long)gridDim.x * (NT / G);
    for (long long i = (long long)blockIdx.x * (NT / G) + threadIdx.x / G; i < rows; i += step) {
        const long long y = labels.at(i);
        RowGrad r;
        const T *row = logits + i * stride;
        r.c = c;
        r.top = lse[i] * temperature;
        r.b = 0.0f;
        r.empty = y < 0 || lse[i] == -INFINITY;
        if (!r.empty && fabsf(lse[i]) > LSE_EXACT) {
            const RowSum a = group_join<G, false>(row_scan<T, G, false>(row, K, tid, c), c, scratch);
            r.top = finite_top(a.m);
            r.b = log2f(a.s);
        }
        r.g = y < K ? grad_logp[i] * inv_t : NAN;
        r.ge = grad_ent ? grad_ent[i] * inv_t : 0.0f;
        r.ent = grad_ent ? ent[i] : 0.0f;
        row_grad<T, G>(row, out + i * out_stride, K, y, tid, r);
    }
}

// ------------------------------------------------------- exact totals --
// A sum of real numbers as a 128-bit two's complement number of 2^-64ths, so
// that adding is associative.  A term is cut to a multiple of 2^-64; a term of
// 2^40 or more counts as infinite, and infinities and NaN are kept apart.
struct Acc {
    unsigned long long lo;
    long long hi;
    unsigned long long n;  // terms counted (tokens kept); the top bits hold what is not finite
};
constexpr int ACC_ODD = 61;  // +inf, -inf, NaN in bits 61 to 63 of n
__device__ __forceinline__ unsigned long long acc_count(const Acc &a) { return a.n & ((1ull << ACC_ODD) - 1ull); }

__device__ __forceinline__ void acc_add(Acc *a, double v) {
    const double u = fabs(v);
    if (!(u < 1099511627776.0)) {
        atomicOr(&a->n, (u != u ? 4ull : v > 0 ? 1ull : 2ull) << ACC_ODD);
        return;
    }
    const double whole = floor(u);
    unsigned long long lo = (unsigned long long)((u - whole) * 18446744073709551616.0);
    long long hi = (long long)whole;
    if (v < 0) {
        hi = ~hi + (lo == 0);
        lo = ~lo + 1ull;
    }
    if (lo) {
        const unsigned long long old = atomicAdd(&a->lo, lo);
        hi += old + lo < old;  // carry
    }
    if (hi) atomicAdd(reinterpret_cast<unsigned long long *>(&a->hi), (unsigned long long)hi);
}

__device__ __forceinline__ double acc_value(const Acc &a) {
    if (const unsigned odd = (unsigned)(a.n >> ACC_ODD)) return odd == 1 ? INFINITY : odd == 2 ? -INFINITY : NAN;
    unsigned long long lo = a.lo;
    long long hi = a.hi;
    const bool neg = hi < 0;
    if (neg) {
        hi = ~hi + (lo == 0);
        lo = ~lo + 1ull;
    }
    const double v = (double)hi + (double)lo * 5.42101086242752217e-20;
    return neg ? -v : v;
}

__global__ void k_acc_zero(Acc *a, long long n, unsigned long long *extra, int n_extra) {
    pdl_wait();
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) a[i] = Acc{0ull, 0ll, 0ull};
    if (i < n_extra) extra[i] = 0ull;
}

// ----------------------------------------------------------- sequences --
constexpr int TOK_THREADS = 256;
constexpr int TOK_EACH = 4;
constexpr int TOK_TILE = TOK_THREADS * TOK_EACH;

// First i in [lo, hi) with off[i] > t, else hi; every lane of a warp calls it.
__device__ __forceinline__ long long upper_bound_warp(const Idx &off, long long lo, long long hi, long long t) {
    const int lane = threadIdx.x & 31;
    while (lo < hi) {
        const long long w = (hi - lo + 31) / 32;                       // indices to a lane
        const long long last = lo + (long long)(lane + 1) * w - 1;
        const unsigned above = __ballot_sync(0xffffffffu, last >= hi || off.at(last) > t);
        if (!above) return hi;                                         // the shares end at hi - 1 or later
        const int f = __ffs(above) - 1;
        const long long end = lo + (long long)(f + 1) * w - 1;
        lo += (long long)f * w;
        hi = end < hi ? end : hi;
    }
    return hi;
}
__device__ __forceinline__ long long upper_bound_one(const Idx &off, long long lo, long long hi, long long t) {
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (off.at(mid) > t) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// The sequences that a tile of tokens [t0, t1) can meet: q0 .. q1.
__device__ __forceinline__ void tile_span(const Idx &off, long long S, long long t0, long long t1, long long *span) {
    const int w = threadIdx.x >> 5;
    if (w < 2) {
        const long long u = upper_bound_warp(off, 0, S + 1, w == 0 ? t0 : t1 - 1) - 1;
        if ((threadIdx.x & 31) == 0) span[w] = u;
    }
    __syncthreads();
}
// Sequence of token t of a tile whose span is q0 .. q1, or -1 where none holds it.
__device__ __forceinline__ long long token_seq(const Idx &off, long long S, long long q0, long long q1, long long t) {
    const long long q = upper_bound_one(off, q0 + 1, q1 + 1, t) - 1;
    return q < S ? q : -1;
}

// Adds v (and counts 1) for the lanes of a warp with keep, by sequence q:
// neighbouring lanes of one sequence are summed first.
__device__ __forceinline__ void warp_seq_add(Acc *acc, long long q, double v, int n, bool with_sum) {
    const int lane = threadIdx.x & 31;
    const unsigned full = 0xffffffffu;
    const long long prev = __shfl_up_sync(full, q, 1);
    const unsigned heads = __ballot_sync(full, lane == 0 || prev != q);
    const int head = 31 - __clz(heads & (0xffffffffu >> (31 - lane)));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {  // inclusive sums from each run's first lane
        const double w = __shfl_up_sync(full, v, o);
        const int k = __shfl_up_sync(full, n, o);
        if (lane - o >= head) {
            v += w;
            n += k;
        }
    }
    const bool last = lane == 31 || ((heads >> (lane + 1)) & 1u);
    if (last && q >= 0 && n) {
        if (with_sum) acc_add(acc + q, v);
        atomicAdd(&acc[q].n, (unsigned long long)n);
    }
}

// --------------------------------------------------------- preference --
// Sequence sums of logp - ref over the kept tokens.
__global__ void __launch_bounds__(TOK_THREADS) k_pref_sums(const float *logp, const float *ref, const uint8_t *mask,
                                                           long long T, Idx off, long long S, Acc *acc) {
    __shared__ long long span[2];
    pdl_wait();
    for (long long t0 = (long long)blockIdx.x * TOK_TILE; t0 < T; t0 += (long long)gridDim.x * TOK_TILE) {
        const long long t1 = t0 + TOK_TILE < T ? t0 + TOK_TILE : T;
        tile_span(off, S, t0, t1, span);
        const long long q0 = span[0], q1 = span[1];
#pragma unroll
        for (int e = 0; e < TOK_EACH; ++e) {
            const long long t = t0 + e * TOK_THREADS + threadIdx.x;
            long long q = -1;
            double v = 0.0;
            int n = 0;
            if (t < t1) {
                q = token_seq(off, S, q0, q1, t);
                if (!mask || mask[t]) {
                    v = ref ? (double)(logp[t] - ref[t]) : (double)logp[t];
                    n = 1;
                }
            }
            warp_seq_add(acc, q, v, n, true);
        }
        __syncthreads();
    }
}

struct PairRule {
    int kind;  // 0 sigmoid, 1 hinge, 2 square
    float beta, smoothing;
    int average;
};
struct PairTerm {
    float loss, slope;  // l and dl / dx of one pair with difference x
};
__device__ __forceinline__ PairTerm pair_term(const PairRule &r, float x) {
    PairTerm p;
    const float h = r.beta * x;
    if (r.kind == 0) {
        // -log sigmoid(h) = softplus(-h); sigmoid(-h) = e^-|h| or 1 over 1 + e^-|h|
        const float e = expf(-fabsf(h));
        const float sp = log1pf(e);
        const float inv = 1.0f / (1.0f + e);
        const float up = h >= 0 ? e * inv : inv;    // sigmoid(-h)
        const float down = h >= 0 ? inv : e * inv;  // sigmoid(h)
        p.loss = sp + (h >= 0 ? r.smoothing * h : (r.smoothing - 1.0f) * h);
        p.slope = r.beta * (r.smoothing * down - (1.0f - r.smoothing) * up);
        if (h != h) p.loss = p.slope = h;
        else if (isinf(h) && r.smoothing == 0.0f) p.loss = h > 0 ? 0.0f : INFINITY;
    } else if (r.kind == 1) {
        p.loss = fmaxf(0.0f, 1.0f - h);
        p.slope = h < 1.0f ? -r.beta : 0.0f;
        if (h != h) p.loss = p.slope = h;
    } else {
        const float d = x - 0.5f / r.beta;
        p.loss = d * d;
        p.slope = 2.0f * d;
    }
    return p;
}

// Score of sequence q: its sum (or mean) of log ratios; NaN out of range.
__device__ __forceinline__ double seq_score(const Acc *acc, long long S, long long q, const float *logp,
                                            const float *ref, int average) {
    if (q < 0 || q >= S) return NAN;
    if (!acc) return ref ? (double)(logp[q] - ref[q]) : (double)logp[q];
    const Acc a = acc[q];
    const double v = acc_value(a);
    const unsigned long long n = acc_count(a);
    return average && n ? v / (double)n : v;
}

__device__ __forceinline__ double block_sum(double v, double *scratch /* >= 33 */) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    v = warp_sum(v);
    if (lane == 0) scratch[w] = v;
    __syncthreads();
    if (w == 0) {
        v = warp_sum(lane < nw ? scratch[lane] : 0.0);
        if (lane == 0) scratch[32] = v;
    }
    __syncthreads();
    v = scratch[32];
    __syncthreads();
    return v;
}

constexpr int PAIR_THREADS = 256;
constexpr int PAIR_BLOCKS = 592;  // most blocks, each with one partial loss

// acc null: every row is its own sequence and scores come from logp itself.
__global__ void __launch_bounds__(PAIR_THREADS) k_pref_pairs(const float *logp, const float *ref, const Acc *acc,
                                                             long long S, Idx chosen, Idx rejected, long long P,
                                                             const float *weight, PairRule rule, Acc *gacc,
                                                             float *chosen_reward, float *rejected_reward,
                                                             double *partial) {
    __shared__ double scratch[33];
    pdl_wait();
    double total = 0.0;
    for (long long p = (long long)blockIdx.x * PAIR_THREADS + threadIdx.x; p < P;
         p += (long long)gridDim.x * PAIR_THREADS) {
        const long long c = chosen.at(p), r = rejected.at(p);
        const double dc = seq_score(acc, S, c, logp, ref, rule.average);
        const double dr = seq_score(acc, S, r, logp, ref, rule.average);
        const PairTerm t = pair_term(rule, (float)(dc - dr));
        const double w = weight ? (double)weight[p] : 1.0;
        total += w * (double)t.loss;
        chosen_reward[p] = (float)(rule.beta * dc);
        rejected_reward[p] = (float)(rule.beta * dr);
        const double g = w * (double)t.slope;
        if (c >= 0 && c < S) acc_add(gacc + c, g);
        if (r >= 0 && r < S) acc_add(gacc + r, -g);
    }
    total = block_sum(total, scratch);
    if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// Gradient of every token: its sequence's, where the token is kept.
__global__ void __launch_bounds__(TOK_THREADS) k_pref_grad(const uint8_t *mask, long long T, Idx off, long long S,
                                                           const Acc *acc, const Acc *gacc, long long P, int average,
                                                           const double *partial, int n_partial, float *loss,
                                                           float *grad) {
    __shared__ long long span[2];
    __shared__ double scratch[33];
    pdl_wait();
    const double inv = P ? 1.0 / (double)P : 0.0;
    if (blockIdx.x == 0) {
        double v = 0.0;
        for (int i = threadIdx.x; i < n_partial; i += TOK_THREADS) v += partial[i];
        v = block_sum(v, scratch);
        if (threadIdx.x == 0) *loss = (float)(v * inv);
    }
    for (long long t0 = (long long)blockIdx.x * TOK_TILE; t0 < T; t0 += (long long)gridDim.x * TOK_TILE) {
        const long long t1 = t0 + TOK_TILE < T ? t0 + TOK_TILE : T;
        if (off.p) tile_span(off, S, t0, t1, span);
        const long long q0 = off.p ? span[0] : 0, q1 = off.p ? span[1] : 0;
#pragma unroll
        for (int e = 0; e < TOK_EACH; ++e) {
            const long long t = t0 + e * TOK_THREADS + threadIdx.x;
            if (t >= t1) continue;
            const long long q = off.p ? token_seq(off, S, q0, q1, t) : t;
            float g = 0.0f;
            if (q >= 0 && (!mask || mask[t])) {
                const double v = acc_value(gacc[q]) * inv;
                g = (float)(average ? v / (double)acc_count(acc[q]) : v);
            }
            grad[t] = g;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------- policy --
struct PolicyRule {
    float clip_hi, clip_lo, log_hi, log_lo;  // 1 + high, 1 - low and their logarithms
    float kl_coef, ent_coef, grad_scale;
    int kl_kind;                             // 0 none (no reference), 1, 2, 3
    int by_sequence;                         // mean over sequences of means over tokens
    int adv_by_sequence;
};
struct PolicyTerm {
    float pg, dpg, kl, dkl, cut;
};
__device__ __forceinline__ PolicyTerm policy_term(const PolicyRule &r, float logp, float old, float adv, float ref) {
    PolicyTerm p;
    const float u = logp - old;
    const bool hi = adv > 0 && u > r.log_hi, lo = adv < 0 && u < r.log_lo;
    const float ratio = expf(u);
    p.pg = -adv * (hi ? r.clip_hi : lo ? r.clip_lo : ratio);
    p.dpg = hi || lo ? 0.0f : -adv * ratio;
    p.cut = hi || lo ? 1.0f : 0.0f;
    p.kl = p.dkl = 0.0f;
    if (r.kl_kind) {
        const float d = ref - logp;
        if (r.kl_kind == 1) {
            p.kl = -d;
            p.dkl = 1.0f;
        } else if (r.kl_kind == 2) {
            p.kl = 0.5f * d * d;
            p.dkl = -d;
        } else {
            const float e = expm1f(d);
            // e^d - 1 - d loses its digits near zero: Taylor's series there
            // (the term left out is below 2^-24 of the sum)
            p.kl = fabsf(d) < 0.35f
                       ? 0.5f * d * d *
                             fmaf(d * (1.0f / 3), fmaf(d * 0.25f, fmaf(d * 0.2f, fmaf(d * (1.0f / 6),
                             fmaf(d * (1.0f / 7), fmaf(d, 0.125f, 1.0f), 1.0f), 1.0f), 1.0f), 1.0f), 1.0f)
                       : e - d;
            p.dkl = -e;
        }
    }
    return p;
}

// What the weights of tokens are made from: `total` kept tokens in all, or
// each sequence's own count (acc[q].n) and the number of sequences with any.
struct PolicyCount {
    const unsigned long long *total;  // [0] kept tokens, [1] sequences with kept tokens
    const Acc *acc;
    const int *ids;                   // sequence of each row (rows of logits), else null
};
__device__ __forceinline__ double token_weight(const PolicyRule &r, const PolicyCount &n, long long q) {
    if (!r.by_sequence) return n.total[0] ? 1.0 / (double)n.total[0] : 0.0;
    if (q < 0) return 0.0;
    return 1.0 / ((double)acc_count(n.acc[q]) * (double)n.total[1]);
}

constexpr int POL_STATS = 4;  // policy term, kl, entropy, clipped

// Counts the kept tokens, in all and (acc not null) by sequence; with `ids` also
// writes each token's sequence.  A token is kept where mask and label say so
// and, with offsets, a sequence holds it.
__global__ void __launch_bounds__(TOK_THREADS) k_policy_count(const uint8_t *mask, Idx labels, long long T, Idx off,
                                                              long long S, Acc *acc, unsigned long long *total,
                                                              int *ids) {
    __shared__ long long span[2];
    pdl_wait();
    unsigned mine = 0;
    for (long long t0 = (long long)blockIdx.x * TOK_TILE; t0 < T; t0 += (long long)gridDim.x * TOK_TILE) {
        const long long t1 = t0 + TOK_TILE < T ? t0 + TOK_TILE : T;
        if (off.p) tile_span(off, S, t0, t1, span);
#pragma unroll
        for (int e = 0; e < TOK_EACH; ++e) {
            const long long t = t0 + e * TOK_THREADS + threadIdx.x;
            bool keep = t < t1 && (!mask || mask[t]) && (!labels.p || labels.at(t) >= 0);
            if (off.p) {
                const long long q = t < t1 ? token_seq(off, S, span[0], span[1], t) : -1;
                if (ids && t < t1) ids[t] = (int)q;
                keep = keep && q >= 0;
                if (acc) warp_seq_add(acc, q, 0.0, keep, false);
            }
            mine += keep;
        }
        __syncthreads();
    }
    mine = warp_sum(mine);
    if ((threadIdx.x & 31) == 0 && mine) atomicAdd(total, (unsigned long long)mine);
}
__global__ void k_policy_nonempty(const Acc *acc, long long S, unsigned long long *total) {
    pdl_wait();
    unsigned mine = 0;
    for (long long q = (long long)blockIdx.x * blockDim.x + threadIdx.x; q < S; q += (long long)gridDim.x * blockDim.x)
        mine += acc_count(acc[q]) != 0;
    mine = warp_sum(mine);
    if ((threadIdx.x & 31) == 0 && mine) atomicAdd(total + 1, (unsigned long long)mine);
}

__device__ __forceinline__ void policy_partial(const double (&sum)[POL_STATS], double *scratch, double *partial) {
#pragma unroll
    for (int k = 0; k < POL_STATS; ++k) {
        const double v = block_sum(sum[k], scratch);
        if (threadIdx.x == 0) partial[(long long)blockIdx.x * POL_STATS + k] = v;
    }
}

__global__ void __launch_bounds__(TOK_THREADS) k_policy_tokens(const float *logp, const float *old, const float *adv,
                                                               const float *ref, const uint8_t *mask, long long T,
                                                               Idx off, long long S, PolicyRule rule, PolicyCount cnt,
                                                               float *grad, double *partial) {
    __shared__ long long span[2];
    __shared__ double scratch[33];
    pdl_wait();
    double sum[POL_STATS] = {};
    for (long long t0 = (long long)blockIdx.x * TOK_TILE; t0 < T; t0 += (long long)gridDim.x * TOK_TILE) {
        const long long t1 = t0 + TOK_TILE < T ? t0 + TOK_TILE : T;
        if (off.p) tile_span(off, S, t0, t1, span);
#pragma unroll
        for (int e = 0; e < TOK_EACH; ++e) {
            const long long t = t0 + e * TOK_THREADS + threadIdx.x;
            if (t >= t1) continue;
            const long long q = off.p ? token_seq(off, S, span[0], span[1], t) : -1;
            float g = 0.0f;
            if ((!mask || mask[t]) && (q >= 0 || !(rule.by_sequence || rule.adv_by_sequence))) {
                const double w = token_weight(rule, cnt, q);
                const PolicyTerm p = policy_term(rule, logp[t], old[t], adv[rule.adv_by_sequence ? q : t],
                                                 rule.kl_kind ? ref[t] : 0.0f);
                g = (float)w * (rule.kl_coef != 0.0f ? fmaf(rule.kl_coef, p.dkl, p.dpg) : p.dpg);
                sum[0] += w * p.pg;
                sum[1] += w * p.kl;
                sum[3] += w * p.cut;
            }
            grad[t] = g;
        }
        __syncthreads();
    }
    policy_partial(sum, scratch, partial);
}

// Per-row policy step: sums of the row, the loss's terms, the row's gradient.
template <typename T, int G, int NT>
__global__ void __launch_bounds__(NT) k_policy_rows(const T *logits, long long rows, long long K, long long stride,
                                                    Idx labels, float inv_t, const float *old, const float *adv,
                                                    const float *ref, const uint8_t *mask, PolicyRule rule,
                                                    PolicyCount cnt, float *logp, T *out, long long out_stride,
                                                    double *partial) {
    __shared__ RowSum scratch[33];
    __shared__ double dscratch[33];
    pdl_wait();
    const int tid = threadIdx.x % G;
    const float c = (float)(LOG2E * inv_t);
    const long long step = (long long)gridDim.x * (NT / G);
    double sum[POL_STATS] = {};
    for (long long i = (long long)blockIdx.x * (NT / G) + threadIdx.x / G; i < rows; i += step) {
        const long long y = labels.at(i);
        const long long q = cnt.ids ? cnt.ids[i] : -1;
        const T *row = logits + i * stride;
        RowGrad r{0.0f, c, 0.0f, 0.0f, 0.0f, 0.0f, 1};
        float lp = 0.0f;
        if (y >= 0 && (!mask || mask[i]) && (q >= 0 || !(rule.by_sequence || rule.adv_by_sequence))) {
            const RowSum a = group_join<G, true>(row_scan<T, G, true>(row, K, tid, c), c, scratch);
            const RowStat st = row_stat<T, true>(a, row, K, y, inv_t);
            lp = st.logp;
            const double w = token_weight(rule, cnt, q);
            const PolicyTerm p = policy_term(rule, lp, old[i], adv[rule.adv_by_sequence ? q : i],
                                             rule.kl_kind ? ref[i] : 0.0f);
            const float wg = (float)(w * rule.grad_scale) * inv_t;
            r.g = wg * (rule.kl_coef != 0.0f ? fmaf(rule.kl_coef, p.dkl, p.dpg) : p.dpg);
            r.ge = -wg * rule.ent_coef;
            r.ent = st.ent;
            r.top = finite_top(a.m);
            r.b = log2f(a.s);
            r.empty = a.s == 0.0f;
            if (tid == 0) {
                sum[0] += w * p.pg;
                sum[1] += w * p.kl;
                sum[2] += w * st.ent;
                sum[3] += w * p.cut;
            }
        }
        if (G > 32) __syncthreads();  // in place: the label's logit is read before it is overwritten
        else __syncwarp();
        if (tid == 0) logp[i] = lp;
        row_grad<T, G>(row, out + i * out_stride, K, y, tid, r);
    }
    policy_partial(sum, dscratch, partial);
}

// stats: loss, policy term, kl, entropy, share clipped (weighted means)
__global__ void k_policy_finish(const double *partial, int blocks, PolicyRule rule, float *stats) {
    __shared__ double scratch[33];
    pdl_wait();
    double sum[POL_STATS] = {};
    for (int i = threadIdx.x; i < blocks; i += blockDim.x)
        for (int k = 0; k < POL_STATS; ++k) sum[k] += partial[(long long)i * POL_STATS + k];
    for (int k = 0; k < POL_STATS; ++k) sum[k] = block_sum(sum[k], scratch);
    if (threadIdx.x == 0) {
        double loss = sum[0];
        if (rule.kl_coef != 0.0f) loss += (double)rule.kl_coef * sum[1];
        if (rule.ent_coef != 0.0f) loss -= (double)rule.ent_coef * sum[2];
        stats[0] = (float)loss;
        for (int k = 0; k < POL_STATS; ++k) stats[1 + k] = (float)sum[k];
    }
}

// ---------------------------------------------------------------- host --
static int sm_count() {
    static int n[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!n[dev]) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
        n[dev] = v;
    }
    return n[dev];
}
static inline int grid_of(long long items, long long per_block, int most) {
    const long long b = (items + per_block - 1) / per_block;
    return (int)(b < 1 ? 1 : b < most ? b : most);
}
static inline long long round_up256(long long b) { return (b + 255) & ~255ll; }

static int check_index(const char *name, int bytes) {
    WGB_CHECK_ARG(bytes == 4 || bytes == 8, "%s must be 4- or 8-byte integers", name);
    return WGB_OK;
}
static int check_logits(const void *logits, int dtype, long long rows, long long K, long long stride, float temperature) {
    WGB_CHECK_ARG(dtype >= 0 && dtype <= 2, "logits dtype must be 0 (float32), 1 (bfloat16) or 2 (float16)");
    WGB_CHECK_ARG(rows >= 0 && K >= 1, "logits need at least one class");
    WGB_CHECK_ARG(rows <= 1 || stride >= K, "rows of logits overlap: stride %lld, %lld classes", stride, K);
    WGB_CHECK_ARG(temperature > 0.0f && !isinf(temperature), "temperature must be positive and finite");
    WGB_CHECK_ARG(rows == 0 || logits != nullptr, "logits is null");
    const int size = dtype == 0 ? 4 : 2;
    WGB_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % size == 0, "logits are not aligned to their type");
    return WGB_OK;
}
#define WGB_TRY(...)                      \
    do {                                  \
        const int rc_ = (__VA_ARGS__);    \
        if (rc_ != WGB_OK) return rc_;    \
    } while (0)

// Rows up to this many classes take a warp each, longer ones a block.
constexpr long long WARP_ROW = 1024;
constexpr int ROW_THREADS = 512;

template <typename F>
static int by_dtype(int dtype, F f) {
    return dtype == 0 ? f((float *)nullptr) : dtype == 1 ? f((__nv_bfloat16 *)nullptr) : f((__half *)nullptr);
}

}  // namespace wgb

using namespace wgb;

extern "C" int wgb_label_logprobs(const void *logits, int32_t dtype, int64_t rows, int64_t classes, int64_t row_stride,
                                  const void *labels, int32_t label_bytes, float temperature, float *logp, float *lse,
                                  float *entropy, void *stream) {
    WGB_TRY(check_logits(logits, dtype, rows, classes, row_stride, temperature));
    WGB_TRY(check_index("labels", label_bytes));
    if (rows == 0) return WGB_OK;
    WGB_CHECK_ARG(labels && logp && lse, "labels, logp and lse must not be null");
    cudaStream_t st = as_stream(stream);
    const Idx lab{labels, label_bytes == 8};
    const float inv_t = 1.0f / temperature;
    return by_dtype(dtype, [&](auto *tag) -> int {
        using T = std::remove_pointer_t<decltype(tag)>;
        const T *x = static_cast<const T *>(logits);
        auto go = [&](auto ent) -> int {
            constexpr bool ENT = decltype(ent)::value;
            if (classes <= WARP_ROW)
                WGB_PDL("k_label_logprobs", k_label_logprobs<T, 32, 256, ENT>, dim3(grid_of(rows, 8, sm_count() * 8)),
                        dim3(256), 0, st, x, rows, classes, row_stride, lab, inv_t, logp, lse, entropy);
            else
                WGB_PDL("k_label_logprobs", k_label_logprobs<T, ROW_THREADS, ROW_THREADS, ENT>,
                        dim3(grid_of(rows, 1, sm_count() * 4)), dim3(ROW_THREADS), 0, st, x, rows, classes, row_stride,
                        lab, inv_t, logp, lse, entropy);
            return WGB_OK;
        };
        return entropy ? go(std::true_type{}) : go(std::false_type{});
    });
}

extern "C" int wgb_label_logprobs_grad(const void *logits, int32_t dtype, int64_t rows, int64_t classes,
                                       int64_t row_stride, const void *labels, int32_t label_bytes, float temperature,
                                       const float *lse, const float *grad_logp, const float *entropy,
                                       const float *grad_entropy, void *grad, int64_t grad_stride, void *stream) {
    WGB_TRY(check_logits(logits, dtype, rows, classes, row_stride, temperature));
    WGB_TRY(check_logits(grad, dtype, rows, classes, grad_stride, temperature));
    WGB_TRY(check_index("labels", label_bytes));
    if (rows == 0) return WGB_OK;
    WGB_CHECK_ARG(labels && lse && grad_logp, "labels, lse and grad_logp must not be null");
    WGB_CHECK_ARG(!grad_entropy || entropy, "grad_entropy needs the entropies");
    cudaStream_t st = as_stream(stream);
    const Idx lab{labels, label_bytes == 8};
    return by_dtype(dtype, [&](auto *tag) -> int {
        using T = std::remove_pointer_t<decltype(tag)>;
        const T *x = static_cast<const T *>(logits);
        T *o = static_cast<T *>(grad);
        if (classes <= WARP_ROW)
            WGB_PDL("k_label_logprobs_grad", k_label_logprobs_grad<T, 32, 256>, dim3(grid_of(rows, 8, sm_count() * 8)),
                    dim3(256), 0, st, x, rows, classes, row_stride, lab, temperature, lse, grad_logp, entropy,
                    grad_entropy, o, grad_stride);
        else
            WGB_PDL("k_label_logprobs_grad", k_label_logprobs_grad<T, ROW_THREADS, ROW_THREADS>,
                    dim3(grid_of(rows, 1, sm_count() * 4)), dim3(ROW_THREADS), 0, st, x, rows, classes, row_stride, lab,
                    temperature, lse, grad_logp, entropy, grad_entropy, o, grad_stride);
        return WGB_OK;
    });
}

extern "C" int64_t wgb_preference_ws_bytes(int64_t sequences, int32_t ragged) {
    if (sequences < 0) return 0;
    return round_up256((ragged ? 2 : 1) * sequences * (int64_t)sizeof(Acc)) + PAIR_BLOCKS * (int64_t)sizeof(double);
}

extern "C" int wgb_preference_loss(const float *logp, const float *ref_logp, int64_t tokens, const void *offsets,
                                   int32_t offset_bytes, int64_t sequences, const uint8_t *mask, const void *chosen,
                                   const void *rejected, int32_t index_bytes, int64_t pairs, const float *weight,
                                   int32_t kind, float beta, float smoothing, int32_t average, void *ws,
                                   int64_t ws_bytes, float *loss, float *grad_logp, float *chosen_reward,
                                   float *rejected_reward, void *stream) {
    WGB_CHECK_ARG(tokens >= 0 && sequences >= 0 && pairs >= 0, "bad sizes");
    WGB_CHECK_ARG(kind >= 0 && kind <= 2, "loss kind must be 0 (sigmoid), 1 (hinge) or 2 (square)");
    WGB_CHECK_ARG(beta > 0.0f && !isinf(beta), "beta must be positive and finite");
    WGB_CHECK_ARG(smoothing >= 0.0f && smoothing < 0.5f, "label smoothing must be in [0, 0.5)");
    WGB_CHECK_ARG(smoothing == 0.0f || kind == 0, "label smoothing is for the sigmoid loss");
    WGB_TRY(check_index("pair indices", index_bytes));
    if (offsets) WGB_TRY(check_index("offsets", offset_bytes));
    WGB_CHECK_ARG(offsets || (sequences == tokens && !mask && !average),
                  "without offsets every row is a sequence: no mask, no average, as many sequences as rows");
    WGB_CHECK_ARG(tokens == 0 || (logp && grad_logp), "logp and grad_logp must not be null");
    WGB_CHECK_ARG(pairs == 0 || (chosen && rejected && chosen_reward && rejected_reward), "pair arrays must not be null");
    WGB_CHECK_ARG(loss != nullptr, "loss must not be null");
    WGB_CHECK_ARG(ws && ws_bytes >= wgb_preference_ws_bytes(sequences, offsets != nullptr), "workspace too small");
    WGB_CHECK_ARG(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "workspace is not aligned to 16 bytes");
    cudaStream_t st = as_stream(stream);
    Acc *gacc = static_cast<Acc *>(ws);
    Acc *acc = offsets ? gacc + sequences : nullptr;
    const long long n_acc = (offsets ? 2 : 1) * sequences;
    double *partial = reinterpret_cast<double *>(static_cast<char *>(ws) + round_up256(n_acc * (long long)sizeof(Acc)));
    const Idx off{offsets, offset_bytes == 8}, ci{chosen, index_bytes == 8}, ri{rejected, index_bytes == 8};
    const PairRule rule{kind, beta, smoothing, average};
    const int tok_grid = grid_of(tokens, TOK_TILE, sm_count() * 8);
    if (n_acc)
        WGB_PDL("k_acc_zero", k_acc_zero, dim3((unsigned)((n_acc + 255) / 256)), dim3(256), 0, st, gacc, n_acc,
                (unsigned long long *)nullptr, 0);
    if (offsets && tokens)
        WGB_PDL("k_pref_sums", k_pref_sums, dim3(tok_grid), dim3(TOK_THREADS), 0, st, logp, ref_logp, mask, tokens, off,
                sequences, acc);
    const int pair_grid = grid_of(pairs, PAIR_THREADS, PAIR_BLOCKS);
    WGB_PDL("k_pref_pairs", k_pref_pairs, dim3(pair_grid), dim3(PAIR_THREADS), 0, st, logp, ref_logp,
            (const Acc *)acc, sequences, ci, ri, pairs, weight, rule, gacc, chosen_reward, rejected_reward, partial);
    WGB_PDL("k_pref_grad", k_pref_grad, dim3(tok_grid), dim3(TOK_THREADS), 0, st, mask, tokens, off, sequences,
            (const Acc *)acc, (const Acc *)gacc, pairs, average, (const double *)partial, pair_grid, loss, grad_logp);
    return WGB_OK;
}

namespace wgb {
constexpr int POL_BLOCKS_PER_SM = 8;
struct PolicyWs {
    unsigned long long *total;
    double *partial;
    Acc *acc;
    int *ids;
    long long bytes;
};
static PolicyWs policy_ws(void *ws, long long tokens, long long sequences, bool ids) {
    PolicyWs w;
    char *p = static_cast<char *>(ws);
    w.total = reinterpret_cast<unsigned long long *>(p);
    w.partial = reinterpret_cast<double *>(p + 256);
    long long at = 256 + round_up256((long long)sm_count() * POL_BLOCKS_PER_SM * POL_STATS * sizeof(double));
    w.acc = reinterpret_cast<Acc *>(p + at);
    at += round_up256(sequences * (long long)sizeof(Acc));
    w.ids = ids ? reinterpret_cast<int *>(p + at) : nullptr;
    w.bytes = at + (ids ? round_up256(tokens * 4) : 0);
    return w;
}

struct PolicyArgs {
    float clip_low, clip_high, kl_coef, ent_coef, grad_scale;
    int kl_kind, by_sequence, adv_by_sequence;
};
static int policy_rule(const PolicyArgs &a, const float *ref, long long tokens, PolicyRule &r) {
    WGB_CHECK_ARG(a.clip_low >= 0.0f && a.clip_low < 1.0f, "clip_low must be in [0, 1)");
    WGB_CHECK_ARG(a.clip_high >= 0.0f && !isinf(a.clip_high), "clip_high must be non-negative and finite");
    WGB_CHECK_ARG(isfinite(a.kl_coef) && isfinite(a.ent_coef) && isfinite(a.grad_scale),
                  "kl_coef, entropy_coef and grad_scale must be finite");
    WGB_CHECK_ARG(a.kl_kind >= 1 && a.kl_kind <= 3, "kl must be 1 (k1), 2 (k2) or 3 (k3)");
    WGB_CHECK_ARG(a.kl_coef == 0.0f || ref || tokens == 0, "kl_coef needs ref_logp");
    r.clip_hi = 1.0f + a.clip_high;
    r.clip_lo = 1.0f - a.clip_low;
    r.log_hi = (float)log1p((double)a.clip_high);
    r.log_lo = (float)log1p(-(double)a.clip_low);
    r.kl_coef = a.kl_coef;
    r.ent_coef = a.ent_coef;
    r.grad_scale = a.grad_scale;
    r.kl_kind = ref ? a.kl_kind : 0;
    r.by_sequence = a.by_sequence;
    r.adv_by_sequence = a.adv_by_sequence;
    return WGB_OK;
}

// Zeroes and counts what the weights need.
static int policy_counts(const PolicyWs &w, const uint8_t *mask, Idx labels, long long tokens, Idx off,
                         long long sequences, const PolicyRule &rule, cudaStream_t st) {
    const long long n = rule.by_sequence ? sequences : 0;
    WGB_PDL("k_acc_zero", k_acc_zero, dim3((unsigned)((n + 255) / 256 + (n == 0))), dim3(256), 0, st, w.acc, n, w.total, 2);
    WGB_PDL("k_policy_count", k_policy_count, dim3(grid_of(tokens, TOK_TILE, sm_count() * 8)), dim3(TOK_THREADS), 0, st,
            mask, labels, tokens, off, sequences, rule.by_sequence ? w.acc : nullptr, w.total, w.ids);
    if (rule.by_sequence)
        WGB_PDL("k_policy_nonempty", k_policy_nonempty, dim3(grid_of(sequences, 256, sm_count())), dim3(256), 0, st,
                (const Acc *)w.acc, sequences, w.total);
    return WGB_OK;
}
}  // namespace wgb

extern "C" int64_t wgb_policy_ws_bytes(int64_t tokens, int64_t sequences, int32_t rows_of_logits) {
    if (tokens < 0 || sequences < 0) return 0;
    return policy_ws(nullptr, tokens, sequences, rows_of_logits != 0).bytes;
}

extern "C" int wgb_policy_loss(const float *logp, const float *old_logp, const float *advantages, const float *ref_logp,
                               int64_t tokens, const uint8_t *mask, const void *offsets, int32_t offset_bytes,
                               int64_t sequences, int32_t adv_by_sequence, int32_t by_sequence, float clip_low,
                               float clip_high, int32_t kl_kind, float kl_coef, void *ws, int64_t ws_bytes,
                               float *stats, float *grad_logp, void *stream) {
    WGB_CHECK_ARG(tokens >= 0 && sequences >= 0, "bad sizes");
    PolicyRule rule;
    WGB_TRY(policy_rule(PolicyArgs{clip_low, clip_high, kl_coef, 0.0f, 1.0f, kl_kind, by_sequence, adv_by_sequence},
                        ref_logp, tokens, rule));
    if (offsets) WGB_TRY(check_index("offsets", offset_bytes));
    WGB_CHECK_ARG(offsets || (!by_sequence && !adv_by_sequence), "a mean or advantages by sequence need offsets");
    WGB_CHECK_ARG(tokens == 0 || (logp && old_logp && advantages && grad_logp),
                  "logp, old_logp, advantages and grad_logp must not be null");
    WGB_CHECK_ARG(stats != nullptr, "stats must not be null");
    WGB_CHECK_ARG(ws && ws_bytes >= wgb_policy_ws_bytes(tokens, sequences, 0), "workspace too small");
    WGB_CHECK_ARG(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "workspace is not aligned to 16 bytes");
    cudaStream_t st = as_stream(stream);
    const PolicyWs w = policy_ws(ws, tokens, sequences, false);
    const bool seqs = by_sequence || adv_by_sequence;
    const Idx off{seqs ? offsets : nullptr, offset_bytes == 8};
    WGB_TRY(policy_counts(w, mask, Idx{nullptr, 0}, tokens, off, sequences, rule, st));
    const int grid = grid_of(tokens, TOK_TILE, sm_count() * POL_BLOCKS_PER_SM);
    WGB_PDL("k_policy_tokens", k_policy_tokens, dim3(grid), dim3(TOK_THREADS), 0, st, logp, old_logp, advantages,
            ref_logp, mask, tokens, off, sequences, rule, PolicyCount{w.total, w.acc, nullptr}, grad_logp, w.partial);
    WGB_PDL("k_policy_finish", k_policy_finish, dim3(1), dim3(256), 0, st, (const double *)w.partial, grid, rule, stats);
    return WGB_OK;
}

extern "C" int wgb_policy_loss_logits(const void *logits, int32_t dtype, int64_t rows, int64_t classes,
                                      int64_t row_stride, const void *labels, int32_t label_bytes, float temperature,
                                      const float *old_logp, const float *advantages, const float *ref_logp,
                                      const uint8_t *mask, const void *offsets, int32_t offset_bytes, int64_t sequences,
                                      int32_t adv_by_sequence, int32_t by_sequence, float clip_low, float clip_high,
                                      int32_t kl_kind, float kl_coef, float entropy_coef, float grad_scale, void *ws,
                                      int64_t ws_bytes, float *stats, float *logp, void *grad, int64_t grad_stride,
                                      void *stream) {
    WGB_TRY(check_logits(logits, dtype, rows, classes, row_stride, temperature));
    WGB_TRY(check_logits(grad, dtype, rows, classes, grad_stride, temperature));
    WGB_TRY(check_index("labels", label_bytes));
    WGB_CHECK_ARG(sequences >= 0 && sequences < (1ll << 31), "too many sequences");
    PolicyRule rule;
    WGB_TRY(policy_rule(
        PolicyArgs{clip_low, clip_high, kl_coef, entropy_coef, grad_scale, kl_kind, by_sequence, adv_by_sequence},
        ref_logp, rows, rule));
    if (offsets) WGB_TRY(check_index("offsets", offset_bytes));
    WGB_CHECK_ARG(offsets || (!by_sequence && !adv_by_sequence), "a mean or advantages by sequence need offsets");
    WGB_CHECK_ARG(rows == 0 || (labels && old_logp && advantages && logp),
                  "labels, old_logp, advantages and logp must not be null");
    WGB_CHECK_ARG(stats != nullptr, "stats must not be null");
    const bool seqs = by_sequence || adv_by_sequence;
    WGB_CHECK_ARG(ws && ws_bytes >= wgb_policy_ws_bytes(rows, sequences, 1), "workspace too small");
    WGB_CHECK_ARG(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "workspace is not aligned to 16 bytes");
    cudaStream_t st = as_stream(stream);
    const PolicyWs w = policy_ws(ws, rows, sequences, seqs);
    const Idx off{seqs ? offsets : nullptr, offset_bytes == 8}, lab{labels, label_bytes == 8};
    WGB_TRY(policy_counts(w, mask, lab, rows, off, sequences, rule, st));
    const PolicyCount cnt{w.total, w.acc, w.ids};
    const float inv_t = 1.0f / temperature;
    int grid = 1;
    WGB_TRY(by_dtype(dtype, [&](auto *tag) -> int {
        using T = std::remove_pointer_t<decltype(tag)>;
        const T *x = static_cast<const T *>(logits);
        T *o = static_cast<T *>(grad);
        if (classes <= WARP_ROW) {
            grid = grid_of(rows, 8, sm_count() * POL_BLOCKS_PER_SM);
            WGB_PDL("k_policy_rows", k_policy_rows<T, 32, 256>, dim3(grid), dim3(256), 0, st, x, rows, classes,
                    row_stride, lab, inv_t, old_logp, advantages, ref_logp, mask, rule, cnt, logp, o, grad_stride,
                    w.partial);
        } else {
            grid = grid_of(rows, 1, sm_count() * 4);
            WGB_PDL("k_policy_rows", k_policy_rows<T, ROW_THREADS, ROW_THREADS>, dim3(grid), dim3(ROW_THREADS), 0, st,
                    x, rows, classes, row_stride, lab, inv_t, old_logp, advantages, ref_logp, mask, rule, cnt, logp, o,
                    grad_stride, w.partial);
        }
        return WGB_OK;
    }));
    WGB_PDL("k_policy_finish", k_policy_finish, dim3(1), dim3(256), 0, st, (const double *)w.partial, grid, rule, stats);
    return WGB_OK;
}
