// Objectives on per-token log-probabilities: a preference loss over paired log
// ratios and a clipped policy loss with a KL term (group 3 of
// include/warpgbm_b200.h; the calls that take rows of logits are in
// wgb_logits.cu).
//
// Sums over the tokens of a sequence and over the pairs of a sequence are
// exact: a partial sum formed in a fixed order is added to a 128-bit
// fixed-point number with integer atomics (Acc), so no result depends on the
// order of the atomics.
#include <type_traits>

namespace wgb {

// An index array of 4- or 8-byte integers.
struct Idx {
    const void *p;
    int wide;
    __device__ __forceinline__ long long at(long long i) const {
        return wide ? static_cast<const long long *>(p)[i] : static_cast<const int *>(p)[i];
    }
};

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
// In fp32: one rounding of a count and one of the quotient.
__device__ __forceinline__ float token_weight(const PolicyCount &n) {
    return n.total[0] ? 1.0f / (float)n.total[0] : 0.0f;
}
__device__ __forceinline__ float seq_weight(const PolicyCount &n, long long q) {
    return 1.0f / ((float)acc_count(n.acc[q]) * (float)n.total[1]);
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
    const float w_all = rule.by_sequence ? 0.0f : token_weight(cnt);
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
                const float w = rule.by_sequence ? seq_weight(cnt, q) : w_all;
                const PolicyTerm p = policy_term(rule, logp[t], old[t], adv[rule.adv_by_sequence ? q : t],
                                                 rule.kl_kind ? ref[t] : 0.0f);
                g = w * (rule.kl_coef != 0.0f ? fmaf(rule.kl_coef, p.dkl, p.dpg) : p.dpg);
                sum[0] += (double)w * p.pg;
                sum[1] += (double)w * p.kl;
                sum[3] += (double)w * p.cut;
            }
            grad[t] = g;
        }
        __syncthreads();
    }
    policy_partial(sum, scratch, partial);
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
#define WGB_TRY(...)                      \
    do {                                  \
        const int rc_ = (__VA_ARGS__);    \
        if (rc_ != WGB_OK) return rc_;    \
    } while (0)

}  // namespace wgb

using namespace wgb;

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
constexpr int POL_BLOCKS_PER_SM = 16;
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

