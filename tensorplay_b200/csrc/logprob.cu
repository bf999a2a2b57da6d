// Objectives on logits: log-probabilities of given tokens and their gradient, the clipped policy loss
// with a KL term, and the preference loss on pairs of sequences, behind tpb200_token_logprobs*,
// tpb200_policy_loss and tpb200_preference_loss.
//
// Mathematics.  For a row x of V logits and its token y, in base 2 with c = log2(e):
//     m = max_j x_j,   s = sum_j 2^(c (x_j - m)),   lse = m + log2(s) / c,   logp = x_y - lse
//     d logp / d x_j = [j = y] - p_j,   p_j = 2^(c (x_j - m)) / s
// so every loss that depends on x through logp alone has the gradient coef * ([j = y] - p_j) with one
// number `coef` per row.  x - m is formed before it is multiplied: a single fused multiply-add c x - c m
// would save an instruction but loses every digit where the logits themselves are huge, as rows of a
// type's lowest value are.  c is the float32 nearest to log2(e) and is divided out again in 64 bits.
//   * s is kept in float32 per thread (a few hundred terms) and joined in float64;
//   * the per-row scalars (log2 s, logp, differences of log-probabilities) are formed in float64 from an
//     exponent and a mantissa, the gradient at the token itself is coef * -expm1(logp), which keeps its
//     digits where p_y is near 1.
// A token with a negative label or a weight of zero takes no part: its row is not read, its outputs and
// its gradient are zero.  A label of V or more gives NaN, never an access outside the row.
#define TPB_FILE_ID 7
#include "host_util.h"
#include "lowp.cuh"

#include <algorithm>

namespace tpb {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A float32 (or label) for every token (a, b), at a * s0 + b * s1; strides of 0 broadcast.
template <class U>
struct PerToken {
    const U* p;
    long long s0, s1;
    __device__ __forceinline__ U at(long long a, long long b) const { return *TPB_CK(&p[a * s0 + b * s1]); }
};

template <class T>
struct Logits {
    const T* x;
    long long s0, s1, inner;
    int vocab;
};

// Running (maximum, sum of 2^(c (x - maximum))) of a set of values; the empty set is (-inf, 0).
struct ExpSum {
    float m, s;
    __device__ __forceinline__ void init() { m = -INFINITY; s = 0.0f; }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N]) {
        float top = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);     // NaN is never the maximum; it reaches the sum below
        if (top > m) {
            s *= ex2((m - top) * kLog2e);
            m = top;
        }
        float t = 0.0f;
        if (m == -INFINITY) {   // only -inf (and NaN) so far: nothing to add but a NaN
#pragma unroll
            for (int i = 0; i < N; ++i) t += v[i];
            if (t != t) s = NAN;
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) t += ex2((v[i] - m) * kLog2e);
        s += t;
    }
};

struct RowStats { float m; double s; };

// The pairs of all threads of the CTA as one; every thread gets it.
__device__ __forceinline__ RowStats join_block(const ExpSum& e, float* red_m, double* red_s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    float m = e.m;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
    if (lane == 0) red_m[warp] = m;
    __syncthreads();
    m = lane < nw ? red_m[lane] : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
    // a thread that saw nothing but -inf passes its sum (0 or NaN) as it is
    double s = warp_add((double)(e.m == -INFINITY ? e.s : e.s * ex2((e.m - m) * kLog2e)));
    if (lane == 0) red_s[warp] = s;
    __syncthreads();
    s = warp_add(lane < nw ? red_s[lane] : 0.0);
    return RowStats{m, s};
}

// log2 of a positive double: exponent and the float32 logarithm of a mantissa in [1/sqrt 2, sqrt 2)
__device__ __forceinline__ double log2_split(double s) {
    if (!(s > 0.0) || s > 1e300) return (double)log2f((float)s);   // 0, NaN, inf
    int e = (int)((__double_as_longlong(s) >> 52) & 0x7ff) - 1023;
    double f = __longlong_as_double((__double_as_longlong(s) & 0x000fffffffffffffLL) | 0x3ff0000000000000LL);
    if (f > 1.4142135623730951) { f *= 0.5; ++e; }
    return (double)e + (double)(log1pf((float)(f - 1.0)) * kLog2e);
}

__device__ __forceinline__ double lse_of(const RowStats& r) { return (double)r.m + log2_split(r.s) / (double)kLog2e; }

// ---------------------------------------------------------------- sweeps over one row --------
// A row is a head up to the first 16-byte boundary, vectors, and a tail.
template <class T>
struct Span {
    int head, nvec, tail;
    __device__ __forceinline__ Span(const T* p, int len) {
        constexpr int N = Elem<T>::N;
        head = (int)((N - (((uintptr_t)p / sizeof(T)) % N)) % N);
        if (head > len) head = len;
        nvec = (len - head) / N;
        tail = len - head - nvec * N;
    }
};

template <class T>
__device__ __forceinline__ void sweep_stats(const T* p, int len, ExpSum& acc) {
    constexpr int N = Elem<T>::N;
    const Span<T> sp(p, len);
    const int tid = threadIdx.x, nthr = blockDim.x;
    const T* q = p + sp.head;
    int i = tid;
    for (; i + 3 * nthr < sp.nvec; i += 4 * nthr) {
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = ld_once16(q + (size_t)(i + u * nthr) * N);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float v[N];
            Elem<T>::unpack(raw[u], v);
            acc.add(v);
        }
    }
    for (; i < sp.nvec; i += nthr) {
        float v[N];
        Elem<T>::unpack(ld_once16(q + (size_t)i * N), v);
        acc.add(v);
    }
    if (tid < sp.head) {
        float v[1] = {Elem<T>::get(*TPB_CK(&p[tid]))};
        acc.add(v);
    }
    if (tid < sp.tail) {
        float v[1] = {Elem<T>::get(*TPB_CK(&p[len - 1 - tid]))};
        acc.add(v);
    }
}

// What the gradient of one row needs: g_j = k * 2^(c (x_j - m)), and `at_label` in the token's place.
struct RowGrad {
    float m, k, at_label;
    int label;
};
__device__ __forceinline__ float grad_at(float x, int j, const RowGrad& g) {
    return j == g.label ? g.at_label : g.k * ex2((x - g.m) * kLog2e);
}

template <class T>
__device__ __forceinline__ void sweep_grad(const T* p, T* o, int len, const RowGrad& g) {
    constexpr int N = Elem<T>::N;
    const int tid = threadIdx.x, nthr = blockDim.x;
    if ((((uintptr_t)p ^ (uintptr_t)o) & 15) == 0) {
        const Span<T> sp(p, len);
        for (int i = tid; i < sp.nvec; i += nthr) {
            const int j0 = sp.head + i * N;
            float v[N];
            Elem<T>::unpack(ld_once16(p + j0), v);
#pragma unroll
            for (int c = 0; c < N; ++c) v[c] = grad_at(v[c], j0 + c, g);
            st_out16(o + j0, Elem<T>::pack(v));
        }
        if (tid < sp.head) *TPB_CK(&o[tid]) = Elem<T>::put(grad_at(Elem<T>::get(*TPB_CK(&p[tid])), tid, g));
        if (tid < sp.tail) {
            const int j = len - 1 - tid;
            *TPB_CK(&o[j]) = Elem<T>::put(grad_at(Elem<T>::get(*TPB_CK(&p[j])), j, g));
        }
    } else {
        for (int j = tid; j < len; j += nthr) *TPB_CK(&o[j]) = Elem<T>::put(grad_at(Elem<T>::get(*TPB_CK(&p[j])), j, g));
    }
}

template <class T>
__device__ __forceinline__ void sweep_zero(T* o, int len) {
    const Span<T> sp(o, len);
    const int tid = threadIdx.x, nthr = blockDim.x;
    for (int i = tid; i < sp.nvec; i += nthr) st_out16(o + sp.head + (size_t)i * Elem<T>::N, make_uint4(0, 0, 0, 0));
    if (tid < sp.head) *TPB_CK(&o[tid]) = Elem<T>::put(0.0f);
    if (tid < sp.tail) *TPB_CK(&o[len - 1 - tid]) = Elem<T>::put(0.0f);
}

// ---------------------------------------------------------------- log-probabilities ----------
// The range of rows that belong to a sequence (all of them without offsets).
struct RowLimits {
    const long long* offsets;   // NULL: every row
    long long last;             // index of the last offset
    __device__ __forceinline__ bool inside(long long r) const {
        return !offsets || (r >= *TPB_CK(&offsets[0]) && r < *TPB_CK(&offsets[last]));
    }
};

// logp and lse of every row; `keep` (a workspace, may be NULL) gets (m, 1 / s) for the gradient.
template <class T>
__global__ void __launch_bounds__(512)
score_kernel(Logits<T> in, PerToken<long long> labels, RowLimits limits, float* __restrict__ logp, float* __restrict__ lse,
             float2* __restrict__ keep) {
    __shared__ float red_m[32];
    __shared__ double red_s[32];
    const long long r = blockIdx.x, a = r / in.inner, b = r - a * in.inner;
    const long long y = labels.at(a, b);
    if (y < 0 || !limits.inside(r)) {
        if (threadIdx.x == 0) {
            *TPB_CK(&logp[r]) = 0.0f;
            if (lse) *TPB_CK(&lse[r]) = 0.0f;
            if (keep) *TPB_CK(&keep[r]) = make_float2(0.0f, 0.0f);
        }
        return;
    }
    const T* p = in.x + a * in.s0 + b * in.s1;
    ExpSum acc;
    acc.init();
    sweep_stats(p, in.vocab, acc);
    const RowStats st = join_block(acc, red_m, red_s);
    if (threadIdx.x == 0) {
        const double n = lse_of(st);
        *TPB_CK(&logp[r]) = y < in.vocab ? (float)((double)Elem<T>::get(*TPB_CK(&p[y])) - n) : NAN;
        if (lse) *TPB_CK(&lse[r]) = (float)n;
        if (keep) *TPB_CK(&keep[r]) = make_float2(st.m, (float)(1.0 / st.s));
    }
}

// ---------------------------------------------------------------- gradient from saved statistics
// coef of every row from the caller's grad_logp (with lse), or from a workspace (with keep).
template <class T>
__global__ void __launch_bounds__(512)
score_grad_kernel(Logits<T> in, PerToken<long long> labels, PerToken<float> grad_logp, const float* __restrict__ lse,
                  const float2* __restrict__ keep, const float* __restrict__ coefs, const float* __restrict__ logp,
                  T* __restrict__ out) {
    const long long r = blockIdx.x, a = r / in.inner, b = r - a * in.inner;
    T* o = out + r * (long long)in.vocab;
    const long long y = labels.at(a, b);
    const float coef = y < 0 ? 0.0f : (coefs ? *TPB_CK(&coefs[r]) : grad_logp.at(a, b));
    if (coef == 0.0f) {
        sweep_zero(o, in.vocab);
        return;
    }
    const T* p = in.x + a * in.s0 + b * in.s1;
    RowGrad g;
    float lp;
    if (keep) {
        const float2 k = *TPB_CK(&keep[r]);
        g.m = k.x;
        g.k = -coef * k.y;
        lp = *TPB_CK(&logp[r]);
    } else {
        // p = 2^(c (x - lse))
        const double L = (double)*TPB_CK(&lse[r]);
        g.m = (float)L;
        g.k = -coef;
        lp = y < in.vocab ? (float)((double)Elem<T>::get(*TPB_CK(&p[y])) - L) : NAN;
    }
    if (y >= in.vocab) g.k = NAN;
    g.label = y < in.vocab ? (int)y : -1;
    g.at_label = coef * -expm1f(lp);
    sweep_grad(p, o, in.vocab, g);
}

// ---------------------------------------------------------------- clipped policy loss ---------
struct PolicyTerms {
    PerToken<float> old_logp, advantage, weight, ref;   // ref.p may be NULL
    float low, high, kl_coef, grad_scale;
};
struct PolicyOut {
    float* logp;
    float* ratio;
    float* kl;
    double* part;   // weight * loss of every row, for the sum
};

// e^d - d - 1 without cancellation for small d
__device__ __forceinline__ float kl_term(float d) {
    if (fabsf(d) < 0.5f) {
        float t = 1.0f / 3628800.0f;      // Taylor: d^2 (1/2! + d/3! + ... + d^8/10!)
        t = fmaf(t, d, 1.0f / 362880.0f);
        t = fmaf(t, d, 1.0f / 40320.0f);
        t = fmaf(t, d, 1.0f / 5040.0f);
        t = fmaf(t, d, 1.0f / 720.0f);
        t = fmaf(t, d, 1.0f / 120.0f);
        t = fmaf(t, d, 1.0f / 24.0f);
        t = fmaf(t, d, 1.0f / 6.0f);
        t = fmaf(t, d, 0.5f);
        return t * d * d;
    }
    return expm1f(d) - d;
}

// The row's outputs and its coefficient d loss / d logp:
//   l = -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef (e^d - d - 1),  r = e^(logp - old), d = ref - logp
//   dl / d logp = -r A (where the unclipped branch is the smaller one) + kl_coef (1 - e^d)
__device__ __forceinline__ float policy_row(const PolicyTerms& t, const PolicyOut& out, long long r, long long a, long long b,
                                            double logp, float w) {
    const float adv = t.advantage.at(a, b);
    const float ratio = expf((float)(logp - (double)t.old_logp.at(a, b)));
    const float free_gain = ratio * adv;
    const float held = fminf(fmaxf(ratio, 1.0f - t.low), 1.0f + t.high) * adv;
    // not (held < free): NaN keeps the unclipped branch, and with it the NaN
    const bool clipped = held < free_gain;
    float loss = -(clipped ? held : free_gain), slope = clipped ? 0.0f : -free_gain, kl = 0.0f;
    if (t.ref.p) {
        const float d = (float)((double)t.ref.at(a, b) - logp);
        kl = kl_term(d);
        loss = fmaf(t.kl_coef, kl, loss);
        slope = fmaf(t.kl_coef, -expm1f(d), slope);
    }
    *TPB_CK(&out.logp[r]) = (float)logp;
    *TPB_CK(&out.ratio[r]) = ratio;
    *TPB_CK(&out.kl[r]) = kl;
    *TPB_CK(&out.part[r]) = (double)w * (double)loss;
    return w * slope * t.grad_scale;
}

template <class T>
__global__ void __launch_bounds__(512)
policy_kernel(Logits<T> in, PerToken<long long> labels, PolicyTerms terms, PolicyOut out, T* __restrict__ grad) {
    __shared__ float red_m[32];
    __shared__ double red_s[32];
    __shared__ RowGrad sh;
    const long long r = blockIdx.x, a = r / in.inner, b = r - a * in.inner;
    const long long y = labels.at(a, b);
    const float w = terms.weight.at(a, b);
    T* o = grad ? grad + r * (long long)in.vocab : nullptr;
    if (y < 0 || w == 0.0f) {
        if (threadIdx.x == 0) {
            *TPB_CK(&out.logp[r]) = 0.0f;
            *TPB_CK(&out.ratio[r]) = 0.0f;
            *TPB_CK(&out.kl[r]) = 0.0f;
            *TPB_CK(&out.part[r]) = 0.0;
        }
        if (o) sweep_zero(o, in.vocab);
        return;
    }
    const T* p = in.x + a * in.s0 + b * in.s1;
    ExpSum acc;
    acc.init();
    sweep_stats(p, in.vocab, acc);
    const RowStats st = join_block(acc, red_m, red_s);
    if (threadIdx.x == 0) {
        const double logp = y < in.vocab ? (double)Elem<T>::get(*TPB_CK(&p[y])) - lse_of(st) : (double)NAN;
        const float coef = policy_row(terms, out, r, a, b, logp, w);
        sh.m = st.m;
        sh.k = (float)(-(double)coef / st.s);
        sh.label = y < in.vocab ? (int)y : -1;
        sh.at_label = coef * -expm1f((float)logp);
    }
    if (!o) return;
    __syncthreads();
    const RowGrad g = sh;
    sweep_grad(p, o, in.vocab, g);
}

// ---------------------------------------------------------------- sums and pairs --------------
// Sum of n doubles in a fixed order by one CTA, times `factor`, rounded to float32.
__global__ void __launch_bounds__(1024)
loss_sum_kernel(const double* __restrict__ part, long long n, double factor, float* __restrict__ out) {
    __shared__ double red[32];
    double s = 0.0;
    for (long long i = threadIdx.x; i < n; i += blockDim.x) s += *TPB_CK(&part[i]);
    s = warp_add(s);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = warp_add(red[threadIdx.x]);
        if (threadIdx.x == 0) *TPB_CK(out) = (float)(s * factor);
    }
}

// One CTA per pair: sums of logp - ref over both sequences, the pair's loss, and the rows' coefficients.
//   margin = beta (s_chosen - s_rejected);  loss = -(1 - e) log sig(margin) - e log sig(-margin)
//   d loss / d margin = e sig(margin) - (1 - e) sig(-margin)
__global__ void __launch_bounds__(256)
pair_kernel(PerToken<long long> labels, PerToken<float> ref, const float* __restrict__ logp, const long long* __restrict__ offsets,
            long long rows, long long inner, long long pairs, double beta, double smoothing, double grad_scale,
            float* __restrict__ rewards, double* __restrict__ part, float* __restrict__ coefs) {
    __shared__ double red[8];
    __shared__ double sums[2];
    const long long pair = blockIdx.x;
    long long lo[2], hi[2];
    bool ordered = true;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const long long q = 2 * pair + j;
        lo[j] = offsets ? *TPB_CK(&offsets[q]) : q * inner;
        hi[j] = offsets ? *TPB_CK(&offsets[q + 1]) : (q + 1) * inner;
        if (lo[j] < 0 || hi[j] < lo[j] || hi[j] > rows) {   // no such rows: nothing is read, the loss is NaN
            ordered = false;
            lo[j] = hi[j] = 0;
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        double s = 0.0;
        for (long long r = lo[j] + threadIdx.x; r < hi[j]; r += blockDim.x) {
            const long long a = r / inner, b = r - a * inner;
            if (labels.at(a, b) >= 0) s += (double)*TPB_CK(&logp[r]) - (double)ref.at(a, b);
        }
        s = warp_add(s);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            s = 0.0;
            for (int w = 0; w < 8; ++w) s += red[w];
            sums[j] = ordered ? s : (double)NAN;
        }
        __syncthreads();
    }
    const double margin = beta * (sums[0] - sums[1]);
    const double e = exp(-fabs(margin));                       // sig(|m|) = 1 / (1 + e), sig(-|m|) = e / (1 + e)
    const double won = (margin >= 0.0 ? 1.0 : e) / (1.0 + e), lost = (margin >= 0.0 ? e : 1.0) / (1.0 + e);
    if (threadIdx.x == 0) {
        // -log sig(m) = log(1 + e^-|m|) + max(-m, 0)
        const double l = log1p(e);
        const double win = (1.0 - smoothing) * (l + fmax(-margin, 0.0));
        *TPB_CK(&part[pair]) = smoothing > 0.0 ? win + smoothing * (l + fmax(margin, 0.0)) : win;   // 0 * inf must not appear
        *TPB_CK(&rewards[2 * pair]) = (float)(beta * sums[0]);
        *TPB_CK(&rewards[2 * pair + 1]) = (float)(beta * sums[1]);
    }
    if (!coefs) return;
    const double slope = grad_scale * beta * (smoothing * won - (1.0 - smoothing) * lost) / (double)pairs;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        for (long long r = lo[j] + threadIdx.x; r < hi[j]; r += blockDim.x) *TPB_CK(&coefs[r]) = (float)(j == 0 ? slope : -slope);
}

__global__ void __launch_bounds__(256) fill_kernel(float* __restrict__ p, long long n, float v) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) *TPB_CK(&p[i]) = v;
}

// ---------------------------------------------------------------- host side -------------------
template <class T>
Logits<T> logits_of(const void* x, int64_t inner, int64_t vocab, const int64_t* strides) {
    return Logits<T>{(const T*)x, strides[0], strides[1], inner, (int)vocab};
}
inline PerToken<float> per_token(const float* p, const int64_t* strides) {
    return PerToken<float>{p, strides ? strides[0] : 0, strides ? strides[1] : 0};
}

#define TPB_BY_TYPE(dtype, call)                              \
    do {                                                      \
        if ((dtype) == TPB200_F32) { using T = float; call; } \
        else if ((dtype) == TPB200_BF16) { using T = __nv_bfloat16; call; } \
        else { using T = __half; call; }                      \
    } while (0)

int check_logits(const char* what, int dtype, int64_t outer, int64_t inner, int64_t vocab, const void* logits, const int64_t* strides,
                 const int64_t* labels, const int64_t* label_strides) {
    TPB_TRY_ROWS(what, dtype, outer, inner, vocab);
    if (!strides || !label_strides) return fail(TPB200_ERR_INVALID, "%s: strides must not be NULL", what);
    if (outer * inner > 0) {
        if (vocab == 0) return fail(TPB200_ERR_INVALID, "%s: the vocabulary is empty", what);
        if (!logits || !labels) return fail(TPB200_ERR_INVALID, "%s: NULL pointer argument", what);
    }
    return TPB200_OK;
}

}  // namespace tpb

using namespace tpb;

extern "C" int tpb200_token_logprobs(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t vocab,
                                     const int64_t* strides, const int64_t* labels, const int64_t* label_strides, float* logp,
                                     float* lse, void* stream) {
    const int rc = check_logits("token_logprobs", dtype, outer, inner, vocab, logits, strides, labels, label_strides);
    if (rc != TPB200_OK) return rc;
    const int64_t rows = outer * inner;
    if (rows == 0) return TPB200_OK;
    if (!logp || !lse) return fail(TPB200_ERR_INVALID, "token_logprobs: NULL pointer argument");
    cudaStream_t st = (cudaStream_t)stream;
    TPB_CHECK_RANGES(st, rows_range(logits, outer, inner, vocab, strides, dtype_bytes(dtype)), rows_range(labels, outer, inner, 1, label_strides, 8),
                     HostRange{logp, (size_t)rows * 4}, HostRange{lse, (size_t)rows * 4});
    const PerToken<long long> lab{(const long long*)labels, label_strides[0], label_strides[1]};
    TPB_BY_TYPE(dtype, TPB_LAUNCH("score_kernel", score_kernel<T>, dim3((unsigned)rows), 512, 0, st,
                                  logits_of<T>(logits, inner, vocab, strides), lab, RowLimits{nullptr, 0}, logp, lse, nullptr));
    return TPB200_OK;
}

extern "C" int tpb200_token_logprobs_backward(const float* grad_logp, const int64_t* grad_strides, const void* logits, int dtype,
                                              int64_t outer, int64_t inner, int64_t vocab, const int64_t* strides,
                                              const int64_t* labels, const int64_t* label_strides, const float* lse,
                                              void* grad_logits, void* stream) {
    const int rc = check_logits("token_logprobs_backward", dtype, outer, inner, vocab, logits, strides, labels, label_strides);
    if (rc != TPB200_OK) return rc;
    const int64_t rows = outer * inner;
    if (rows == 0) return TPB200_OK;
    if (!grad_logp || !grad_strides || !lse || !grad_logits) return fail(TPB200_ERR_INVALID, "token_logprobs_backward: NULL pointer argument");
    cudaStream_t st = (cudaStream_t)stream;
    TPB_CHECK_RANGES(st, rows_range(logits, outer, inner, vocab, strides, dtype_bytes(dtype)), rows_range(labels, outer, inner, 1, label_strides, 8),
                     rows_range(grad_logp, outer, inner, 1, grad_strides, 4), HostRange{lse, (size_t)rows * 4},
                     HostRange{grad_logits, (size_t)(rows * vocab * dtype_bytes(dtype))});
    const PerToken<long long> lab{(const long long*)labels, label_strides[0], label_strides[1]};
    TPB_BY_TYPE(dtype, TPB_LAUNCH("score_grad_kernel", score_grad_kernel<T>, dim3((unsigned)rows), 512, 0, st,
                                  logits_of<T>(logits, inner, vocab, strides), lab, per_token(grad_logp, grad_strides), lse, nullptr, nullptr,
                                  nullptr, (T*)grad_logits));
    return TPB200_OK;
}

extern "C" size_t tpb200_policy_loss_workspace_bytes(int64_t outer, int64_t inner) {
    return outer > 0 && inner > 0 ? (size_t)(outer * inner) * sizeof(double) : 0;
}

extern "C" int tpb200_policy_loss(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t vocab, const int64_t* strides,
                                  const int64_t* labels, const int64_t* label_strides, const float* old_logp,
                                  const int64_t* old_strides, const float* advantages, const int64_t* advantage_strides,
                                  const float* weights, const int64_t* weight_strides, const float* ref_logp,
                                  const int64_t* ref_strides, double clip_low, double clip_high, double kl_coef, double grad_scale,
                                  float* loss, void* grad_logits, float* logp, float* ratio, float* kl, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    int rc = check_logits("policy_loss", dtype, outer, inner, vocab, logits, strides, labels, label_strides);
    if (rc != TPB200_OK) return rc;
    if (!(clip_low >= 0.0 && clip_low <= 1.0) || !(clip_high >= 0.0)) return fail(TPB200_ERR_INVALID, "policy_loss: clip_low must lie in [0, 1] and clip_high must not be negative");
    if (!(kl_coef >= 0.0)) return fail(TPB200_ERR_INVALID, "policy_loss: kl_coef must not be negative");
    if (kl_coef > 0.0 && !ref_logp && outer * inner > 0) return fail(TPB200_ERR_INVALID, "policy_loss: kl_coef needs ref_logp");
    if (!loss) return fail(TPB200_ERR_INVALID, "policy_loss: NULL pointer argument");
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t rows = outer * inner;
    if (rows > 0) {
        if (!old_logp || !advantages || !weights || !old_strides || !advantage_strides || !weight_strides || (ref_logp && !ref_strides) || !logp || !ratio || !kl)
            return fail(TPB200_ERR_INVALID, "policy_loss: NULL pointer argument");
        if (!workspace || workspace_bytes < tpb200_policy_loss_workspace_bytes(outer, inner))
            return fail(TPB200_ERR_WORKSPACE, "policy_loss: workspace missing or too small (%zu of %zu bytes)", workspace_bytes, tpb200_policy_loss_workspace_bytes(outer, inner));
    }
    TPB_CHECK_RANGES(st, rows_range(logits, outer, inner, vocab, strides, dtype_bytes(dtype)), rows_range(labels, outer, inner, 1, label_strides, 8),
                     rows_range(old_logp, outer, inner, 1, old_strides, 4), rows_range(advantages, outer, inner, 1, advantage_strides, 4),
                     rows_range(weights, outer, inner, 1, weight_strides, 4), rows_range(ref_logp, outer, inner, 1, ref_strides, 4),
                     HostRange{loss, 4}, HostRange{grad_logits, grad_logits ? (size_t)(rows * vocab * dtype_bytes(dtype)) : 0},
                     HostRange{logp, (size_t)rows * 4}, HostRange{ratio, (size_t)rows * 4}, HostRange{kl, (size_t)rows * 4},
                     HostRange{workspace, (size_t)rows * 8});
    if (rows > 0) {
        const PerToken<long long> lab{(const long long*)labels, label_strides[0], label_strides[1]};
        const PolicyTerms terms{per_token(old_logp, old_strides), per_token(advantages, advantage_strides), per_token(weights, weight_strides),
                                per_token(ref_logp, ref_strides), (float)clip_low, (float)clip_high, (float)kl_coef, (float)grad_scale};
        const PolicyOut out{logp, ratio, kl, (double*)workspace};
        TPB_BY_TYPE(dtype, TPB_LAUNCH("policy_kernel", policy_kernel<T>, dim3((unsigned)rows), 512, 0, st,
                                      logits_of<T>(logits, inner, vocab, strides), lab, terms, out, (T*)grad_logits));
    }
    TPB_LAUNCH("loss_sum_kernel", loss_sum_kernel, dim3(1), 1024, 0, st, (const double*)workspace, (long long)rows, 1.0, loss);
    return TPB200_OK;
}

// workspace of the preference loss: (m, 1 / s) and the coefficient of every row, the loss of every pair
extern "C" size_t tpb200_preference_loss_workspace_bytes(int64_t outer, int64_t inner, int64_t pairs) {
    if (outer < 0 || inner < 0 || pairs < 0) return 0;
    return (size_t)(outer * inner) * (sizeof(float2) + 8) + (size_t)pairs * sizeof(double);
}

extern "C" int tpb200_preference_loss(const void* logits, int dtype, int64_t outer, int64_t inner, int64_t vocab,
                                      const int64_t* strides, const int64_t* labels, const int64_t* label_strides,
                                      const float* ref_logp, const int64_t* ref_strides, const int64_t* offsets, int64_t pairs,
                                      double beta, double label_smoothing, double grad_scale, float* loss, void* grad_logits,
                                      float* rewards, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_logits("preference_loss", dtype, outer, inner, vocab, logits, strides, labels, label_strides);
    if (rc != TPB200_OK) return rc;
    if (pairs < 1 || pairs > 0x3fffffffLL) return fail(TPB200_ERR_INVALID, "preference_loss: at least one pair is needed");
    if (!(label_smoothing >= 0.0 && label_smoothing < 0.5)) return fail(TPB200_ERR_INVALID, "preference_loss: label_smoothing must lie in [0, 0.5)");
    if (offsets ? outer != 1 : outer != 2 * pairs)
        return fail(TPB200_ERR_INVALID, "preference_loss: offsets go with packed rows (outer = 1); without them there are two sequences per pair (outer = 2 * pairs)");
    if (!loss || !rewards) return fail(TPB200_ERR_INVALID, "preference_loss: NULL pointer argument");
    const int64_t rows = outer * inner;
    if (rows > 0 && (!ref_logp || !ref_strides || !logp)) return fail(TPB200_ERR_INVALID, "preference_loss: NULL pointer argument");
    const size_t need = tpb200_preference_loss_workspace_bytes(outer, inner, pairs);
    if (!workspace || workspace_bytes < need)
        return fail(TPB200_ERR_WORKSPACE, "preference_loss: workspace missing or too small (%zu of %zu bytes)", workspace_bytes, need);
    cudaStream_t st = (cudaStream_t)stream;
    TPB_CHECK_RANGES(st, rows_range(logits, outer, inner, vocab, strides, dtype_bytes(dtype)), rows_range(labels, outer, inner, 1, label_strides, 8),
                     rows_range(ref_logp, outer, inner, 1, ref_strides, 4), HostRange{offsets, offsets ? (size_t)(2 * pairs + 1) * 8 : 0},
                     HostRange{loss, 4}, HostRange{grad_logits, grad_logits ? (size_t)(rows * vocab * dtype_bytes(dtype)) : 0},
                     HostRange{rewards, (size_t)pairs * 8}, HostRange{logp, (size_t)rows * 4}, HostRange{workspace, need});
    double* part = (double*)workspace;
    float2* keep = (float2*)(part + pairs);
    float* coefs = (float*)(keep + rows);
    const PerToken<long long> lab{(const long long*)labels, label_strides[0], label_strides[1]};
    const RowLimits limits{(const long long*)offsets, 2 * pairs};
    if (rows > 0) {
        if (grad_logits) TPB_LAUNCH("fill_kernel", fill_kernel, dim3((unsigned)ceil_div(rows, 256)), 256, 0, st, coefs, (long long)rows, 0.0f);
        TPB_BY_TYPE(dtype, TPB_LAUNCH("score_kernel", score_kernel<T>, dim3((unsigned)rows), 512, 0, st,
                                      logits_of<T>(logits, inner, vocab, strides), lab, limits, logp, nullptr, keep));
    }
    TPB_LAUNCH("pair_kernel", pair_kernel, dim3((unsigned)pairs), 256, 0, st, lab, per_token(ref_logp, ref_strides), (const float*)logp,
               (const long long*)offsets, (long long)rows, (long long)std::max<int64_t>(inner, 1), (long long)pairs, beta, label_smoothing, grad_scale,
               rewards, part, grad_logits ? coefs : nullptr);
    TPB_LAUNCH("loss_sum_kernel", loss_sum_kernel, dim3(1), 1024, 0, st, (const double*)part, (long long)pairs, 1.0 / (double)pairs, loss);
    if (rows > 0 && grad_logits)
        TPB_BY_TYPE(dtype, TPB_LAUNCH("score_grad_kernel", score_grad_kernel<T>, dim3((unsigned)rows), 512, 0, st,
                                      logits_of<T>(logits, inner, vocab, strides), lab, PerToken<float>{nullptr, 0, 0}, (const float*)nullptr,
                                      (const float2*)keep, (const float*)coefs, (const float*)logp, (T*)grad_logits));
    return TPB200_OK;
}
