// Objectives on logits: log-probabilities of given tokens and their gradient, the clipped policy loss
// with a KL term, and the preference loss on pairs of sequences, behind tpb200_token_logprobs*,
// tpb200_policy_loss and tpb200_preference_loss.
//
// Mathematics.  For a row x of V logits and its token y, in base 2 with c = log2(e):
//     m = max_j x_j,   s = sum over j != y of 2^(c (x_j - m)),   g = (x_y - m) - log2(s) / c
//     logp = -log(1 + e^-g),   1 - p_y = 1 / (1 + e^g),   p_j = (1 - p_y) 2^(c (x_j - m)) / s,   d logp / d x_j = [j = y] - p_j
// so every loss that depends on x through logp alone has the gradient coef * ([j = y] - p_j) with one
// number `coef` per row.  The token's own term stays out of the sum: g, the log of its odds against all others,
// holds the digits of 1 - p_y however near p_y is to 1 (most tokens of a trained model), where a sum of all would hold
// p_y alone, and the rows of the gradient add up to zero.  m may be any reference near the maximum.
//   * Sums go by an integer E near c m, c x - E, so that sums of threads and CTAs are joined by exact powers of two, and by
//     c to 1e-10 of itself (FixedSum): a base that is off by d shifts every log s to the same side, by d times the mean
//     distance of the logits, and a reward adds that up over its sequence.  (With c a float32 rewards of [3001,151936]
//     were 1.2e-6 of themselves off.)  The gradient, whose entries stand by themselves, takes one multiply-add
//     with the float32 c.
//   * Where |m| >= 2^15 (rows of a type's lowest value are such rows) x - m is formed first.
//   * s is kept in float32, a few hundred terms per thread at most, and joined by trees;
//   * the per-row scalars (log s, g, logp, differences of log-probabilities) are formed in float64 from an
//     exponent and a mantissa; the gradient at the token itself is coef * (1 - p_y).
// A token with a negative label or a weight of zero takes no part: its row is not read, its outputs and
// its gradient are zero.  A label of V or more gives NaN, never an access outside the row.
#define TPB_FILE_ID 7
#include "host_util.h"
#include "lowp.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace tpb {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
// log2(e) = kStep + kRest to 1.2e-10 of itself; kStep has five bits, so that kStep x - E is exact for 16-bit types
constexpr float kStep = 1.4375f, kRest = 1.4426950408889634 - 1.4375;
// e^v = 2^(kLog2e v) times e^(kLow c v): what the float32 c leaves out
constexpr float kLow = (1.4426950408889634 - (double)kLog2e) / 1.4426950408889634 * kLn2;
// ex2.approx is low by this on average over an octave of negative arguments (2^22 of them measured, each off by at most
// 1.5e-7); a sum of many terms is low by as much, always to the same side
constexpr double kExLow = 5.0e-8;
constexpr float kFar = 32768.0f;         // |reference| from which x - m is formed first: log-probabilities of [2048,50016] bf16 44 us, there 85
constexpr float kAbove = 6.0f;           // octaves of E above the reference, so that no argument of ex2 is above 1

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two float32 operations per instruction (sm_100a): differences, products and sums of the sweeps.
struct __align__(8) Two { float a, b; };
__device__ __forceinline__ unsigned long long bits_of(float a, float b) {
    return (unsigned long long)__float_as_uint(a) | ((unsigned long long)__float_as_uint(b) << 32);
}
__device__ __forceinline__ Two two_of(unsigned long long v) {
    return Two{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}
__device__ __forceinline__ unsigned long long add2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

__device__ __forceinline__ unsigned long long fma2(unsigned long long x, unsigned long long y, unsigned long long z) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}

// v[i] := 2^(c v[i] - E), 2^(kLog2e v[i] - M), or 2^(c (v[i] - m)), for an even number of values
template <int N>
__device__ __forceinline__ void exps_fine(float (&v)[N], float E) {
    const unsigned long long neg = bits_of(-E, -E), step = bits_of(kStep, kStep), rest = bits_of(kRest, kRest);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const unsigned long long x = bits_of(v[i], v[i + 1]);
        const Two t = two_of(fma2(x, rest, fma2(x, step, neg)));
        v[i] = ex2(t.a);
        v[i + 1] = ex2(t.b);
    }
}
template <int N>
__device__ __forceinline__ void exps_fma(float (&v)[N], float M) {
    const unsigned long long neg = bits_of(-M, -M), c = bits_of(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const Two t = two_of(fma2(bits_of(v[i], v[i + 1]), c, neg));
        v[i] = ex2(t.a);
        v[i + 1] = ex2(t.b);
    }
}
template <int N>
__device__ __forceinline__ void exps(float (&v)[N], float m) {
    const unsigned long long neg = bits_of(-m, -m), c = bits_of(kLog2e, kLog2e);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const Two t = two_of(mul2(add2(bits_of(v[i], v[i + 1]), neg), c));
        v[i] = ex2(t.a);
        v[i + 1] = ex2(t.b);
    }
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

// What the sums of a reference m are relative to: 2^E, an integer E near c m, or, for a far one, e^m.
__device__ __forceinline__ bool near(float m) { return fabsf(m) < kFar; }
__device__ __forceinline__ float base_of(float m) { return rintf(m * kLog2e) + kAbove; }
// a sum that is relative to `own` as one relative to m >= own
__device__ __forceinline__ float rebase(float own, float m) {
    if (own == m) return 1.0f;
    if (near(own) && near(m)) {
        const float d = base_of(own) - base_of(m);
        return d > -126.0f ? __int_as_float(((int)d + 127) << 23) : 0.0f;
    }
    const float r = near(own) ? fmaf(own, -kLog2e, base_of(own)) : 0.0f, t = near(m) ? fmaf(m, -kLog2e, base_of(m)) : 0.0f;
    return ex2((own - m) * kLog2e + (r - t));      // own = -inf: 0
}

// log(s) of a row's sum: the exponent and the logarithm of a mantissa in [1/sqrt 2, sqrt 2), so that the float32 part is
// below 0.35.  No float64 division on the way: one costs a row some 0.5 us.
__device__ __forceinline__ double log_sum(float s) {
    if (!(s >= 1.17549435e-38f && s < INFINITY)) return (double)logf(s);   // 0, NaN, inf
    int e = (int)(__float_as_uint(s) >> 23) - 127;
    float f = __uint_as_float((__float_as_uint(s) & 0x007fffffu) | 0x3f800000u);
    if (f > 1.41421356f) { f *= 0.5f; ++e; }
    return fma((double)e, kLn2, (double)log1pf(f - 1.0f));
}

// What a row's sum over the other entries says of its token.  e^-|g| is rounded to float32, 2^-23 of itself, logarithms are
// float32 below 0.7: logp is within 2^-22 of itself, or 1e-7 where it is large.
struct Score {
    double logp, lse;
    float gap, e;                // g, NaN for a label beyond the vocabulary, and e^-|g|
    // 1 - p_y
    __device__ __forceinline__ float rest() const { return gap != gap ? NAN : __fdividef(gap >= 0.0f ? e : 1.0f, 1.0f + e); }
};
// x_y, and (reference, sum) of the others; `known`: the label lies in the vocabulary
__device__ __forceinline__ Score score_of(bool known, float own, float m, float s) {
    Score o;
    const double log_s = log_sum(s) + kExLow, base = near(m) ? (double)base_of(m) * kLn2 : (double)m;
    // the difference from the base first: base + log s would not hold log s where |m| is large (rows of a type's lowest value)
    const double gap = ((double)own - base) - log_s;
    o.gap = known && own < INFINITY ? (float)gap : NAN;
    const float low = (float)(gap - (double)o.gap);           // NaN where gap is infinite: e is 0 then
    o.e = expf(-fabsf(o.gap));
    if (o.e > 0.0f) o.e = fmaf(o.e, o.gap < 0.0f ? low : -low, o.e);
    const float l = log1pf(o.e);
    if (o.gap >= 0.0f) {
        o.logp = (double)(0.0f - l);
        o.lse = (double)(own + l);
    } else {                                                  // NaN too
        o.logp = (o.gap != o.gap ? (double)NAN : gap) - (double)l;
        o.lse = known ? (base + log_s) + (double)l : base + log_s;
    }
    return o;
}
// The reference, and `unit` such that p_j = unit * 2^(c x_j - E) for the others (far: unit * e^(x_j - m)).  Where there are none (a vocabulary
// of one, or all of them -inf) they have no share.
__device__ __forceinline__ float2 unit_of(const Score& y, float own, float m, float s) {
    const float rest = y.rest();
    return s == 0.0f ? make_float2(own, rest) : make_float2(m, __fdividef(rest, s));
}

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

// What the gradient of one row needs: g_j = k * 2^(kLog2e x_j - M), M = E, or k * 2^(c (x_j - m)) for a far row, and
// `at_label` in the token's place.  k holds what the float32 c leaves out at x = m; 1.3e-8 of x_j - m remain.
struct RowGrad {
    float m, M, k, at_label;
    int label, far;
    // from the reference, `unit` and 1 - p_y of the row's score, and the coefficient
    __device__ __forceinline__ void set(float reference, float unit, float rest, float coef, int at) {
        m = reference;
        far = !near(m);
        M = far ? 0.0f : base_of(m);
        k = -coef * unit;
        if (!far) k = fmaf(k, kLow * M, k);
        at_label = coef * rest;
        label = at;
    }
    __device__ __forceinline__ float value(float x) const { return k * ex2(far ? (x - m) * kLog2e : fmaf(x, kLog2e, -M)); }
};
__device__ __forceinline__ float grad_at(float x, int j, const RowGrad& g) { return j == g.label ? g.at_label : g.value(x); }

// k * 2^(c x - M) of a vector
template <class T>
__device__ __forceinline__ uint4 grad_vector(const uint4& raw, const RowGrad& g, bool far) {
    constexpr int N = Elem<T>::N;
    float v[N];
    Elem<T>::unpack(raw, v);
    if (far) exps(v, g.m);
    else exps_fma(v, g.M);
    const unsigned long long k = bits_of(g.k, g.k);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const Two t = two_of(mul2(bits_of(v[i], v[i + 1]), k));
        v[i] = t.a;
        v[i + 1] = t.b;
    }
    return Elem<T>::pack(v);
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
    const float e = expm1f(d);
    return e == INFINITY ? e : e - d;     // inf - inf at d = inf
}

// A token's inputs, fetched before the row is swept, asynchronously into shared memory: the sweep has no register to
// spare for them ([4096,151936] bf16: 545 us with them in registers, 534 so).
struct PolicyToken { float old_logp, advantage, weight, ref; };
__device__ __forceinline__ void copy_async4(float* dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(TPB_CK(src)) : "memory");
}
__device__ __forceinline__ void fetch_token(const PolicyTerms& t, long long a, long long b, float w, PolicyToken* k) {
    copy_async4(&k->old_logp, t.old_logp.p + a * t.old_logp.s0 + b * t.old_logp.s1);
    copy_async4(&k->advantage, t.advantage.p + a * t.advantage.s0 + b * t.advantage.s1);
    k->weight = w;
    if (t.ref.p) copy_async4(&k->ref, t.ref.p + a * t.ref.s0 + b * t.ref.s1);
}

// The row's outputs and its coefficient d loss / d logp, in float32 from differences of float64 log-probabilities: the outputs
// are float32, each is a few roundings of 2^-24 off (measured against 64 bits: ratio 6e-8, kl 2e-7 of their norms), and
// float64 exponentials by one thread would lengthen every row.  The sum over the rows is float64.
//   l = -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef (e^d - d - 1),  r = e^(logp - old), d = ref - logp
//   dl / d logp = -r A (where the unclipped branch is the smaller one) + kl_coef (1 - e^d)
struct PolicyRow { float ratio, kl, coef; double part; };
__device__ __forceinline__ PolicyRow policy_row(const PolicyTerms& t, const PolicyToken& k, double logp) {
    PolicyRow o;
    o.ratio = expf((float)(logp - (double)k.old_logp));
    const float free_gain = o.ratio * k.advantage;
    const float held = fminf(fmaxf(o.ratio, 1.0f - t.low), 1.0f + t.high) * k.advantage;
    // not (held < free): NaN keeps the unclipped branch, and with it the NaN
    const bool clipped = held < free_gain;
    float loss = -(clipped ? held : free_gain), slope = clipped ? 0.0f : -free_gain;
    o.kl = 0.0f;
    if (t.ref.p) {
        const float d = (float)((double)k.ref - logp);
        o.kl = kl_term(d);
        if (t.kl_coef > 0.0f) {                  // 0 * inf must not appear: a KL that is only watched may be infinite
            loss = fmaf(t.kl_coef, o.kl, loss);
            slope = fmaf(t.kl_coef, -expm1f(d), slope);
        }
    }
    o.part = (double)k.weight * (double)loss;
    o.coef = k.weight * slope * t.grad_scale;
    return o;
}
__device__ __forceinline__ void store_policy(const PolicyOut& out, long long r, double logp, const PolicyRow& o) {
    *TPB_CK(&out.logp[r]) = (float)logp;
    *TPB_CK(&out.ratio[r]) = o.ratio;
    *TPB_CK(&out.kl[r]) = o.kl;
    *TPB_CK(&out.part[r]) = o.part;
}

// ---------------------------------------------------------------- sweeps of a part of a row ---
// The part of a row that CTA `rank` of `C` takes: `n` vectors from vector `first` behind the head.
template <class T>
struct Part {
    int head, tail, nvec, first, n;
    __device__ __forceinline__ Part(const T* p, int len, int rank, int C) {
        const Span<T> sp(p, len);
        head = sp.head;
        tail = sp.tail;
        nvec = sp.nvec;
        const int each = (nvec + C - 1) / C;
        first = min(rank * each, nvec);
        n = min(each, nvec - first);
    }
    // the element outside of the vectors that this thread takes (the CTA has at least 32 threads), or -1
    __device__ __forceinline__ int edge(int tid, int len, int rank, int C) const {
        if (rank == 0 && tid < head) return tid;
        if (rank == C - 1 && tid >= 16 && tid - 16 < tail) return len - 1 - (tid - 16);
        return -1;
    }
};

template <class T>
__device__ __forceinline__ void zero_part(T* o, const Part<T>& z, int len, int rank, int C) {
    constexpr int N = Elem<T>::N;
    const int tid = threadIdx.x;
    for (int i = tid; i < z.n; i += blockDim.x) st_out16(o + z.head + (size_t)(z.first + i) * N, make_uint4(0, 0, 0, 0));
    const int e = z.edge(tid, len, rank, C);
    if (e >= 0) *TPB_CK(&o[e]) = Elem<T>::put(0.0f);
}

// Maximum of a vector's elements and `m`, on packed pairs for the 16-bit types; NaN is never the maximum.
template <class T> struct VecMax;
template <> struct VecMax<float> {
    float m = -INFINITY;
    __device__ __forceinline__ void add(const uint4& v) {
        m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
    }
    __device__ __forceinline__ float get() const { return m; }
};
template <> struct VecMax<__nv_bfloat16> {
    __nv_bfloat162 m = __nv_bfloat162{__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80)};
    static __device__ __forceinline__ __nv_bfloat162 of(uint32_t w) { __nv_bfloat162 r; memcpy(&r, &w, 4); return r; }
    __device__ __forceinline__ void add(const uint4& v) { m = __hmax2(m, __hmax2(__hmax2(of(v.x), of(v.y)), __hmax2(of(v.z), of(v.w)))); }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <> struct VecMax<__half> {
    __half2 m = __half2{__ushort_as_half(0xfc00), __ushort_as_half(0xfc00)};
    static __device__ __forceinline__ __half2 of(uint32_t w) { __half2 r; memcpy(&r, &w, 4); return r; }
    __device__ __forceinline__ void add(const uint4& v) { m = __hmax2(m, __hmax2(__hmax2(of(v.x), of(v.y)), __hmax2(of(v.z), of(v.w)))); }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};

__device__ __forceinline__ unsigned lanes_below(int n) { return n >= 32 ? kFull : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ float lanes_max(float v, unsigned mask) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(mask));
    return r;
}

// -inf in place of element e of VECS vectors
template <class T, int VECS>
__device__ __forceinline__ void leave_out(uint4 (&raw)[VECS], int e) {
    constexpr int per = 4 / (int)sizeof(T);     // elements of a word
#pragma unroll
    for (int u = 0; u < VECS; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t& x = w == 0 ? raw[u].x : w == 1 ? raw[u].y : w == 2 ? raw[u].z : raw[u].w;
            if (e / per == u * 4 + w) x = per == 1 ? Elem<T>::kNegInf : __byte_perm(x, Elem<T>::kNegInf, e & 1 ? 0x5410 : 0x3254);
        }
}

// Running sum of 2^(c x - E) of one thread over a row, two vectors at a time, against a reference that is fixed
// after the first step, the maximum of what the warp has met there: no maximum and no rescaling per element.  A step
// whose sum is not below 2 -- values well above the reference, infinities, NaN, far rows (their E is NaN) -- is done
// again the careful way, which raises the reference.  The exponent is kRest x + (kStep x - E): two roundings, of 2^-22 at
// most below 8 octaves, the first of them none for a 16-bit type and up to 2^-32 |x| for a float32 above 1500.  Nine thread instructions per
// element in all ([2048,50016] bf16, counted by the profiler), of which one is ex2 on a pipe of 16 a cycle.
template <class T>
struct FixedSum {
    static constexpr int N = Elem<T>::N;
    float ref, E, s;      // ref = -inf: nothing but -inf and NaN so far; E = NaN then, and for a far reference
    __device__ __forceinline__ void init() { ref = -INFINITY; E = NAN; s = 0.0f; }
    __device__ __forceinline__ void refer(float high) {
        ref = high;
        E = near(ref) ? base_of(ref) : NAN;
    }
    static __device__ __noinline__ FixedSum careful(FixedSum f, uint4 raw) {
        VecMax<T> top;
        top.add(raw);
        const float high = top.get();
        if (high > f.ref) {
            f.s *= rebase(f.ref, high);     // 0 * 0 at the start
            f.refer(high);
        }
        float t = 0.0f, v[N];
        Elem<T>::unpack(raw, v);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (f.E == f.E) t += ex2(fmaf(v[i], kRest, fmaf(v[i], kStep, -f.E)));
            else t += f.ref == -INFINITY ? (v[i] != v[i] ? NAN : 0.0f) : ex2((v[i] - f.ref) * kLog2e);
        }
        f.s += t;
        return f;
    }
    // `first`: this thread's first step, which the lanes of `mask()` take together
    template <int VECS, class Mask>
    __device__ __forceinline__ void add(const uint4 (&raw)[VECS], bool first, const Mask& mask) {
        if (first) {
            VecMax<T> top;
#pragma unroll
            for (int u = 0; u < VECS; ++u) top.add(raw[u]);
            refer(lanes_max(top.get(), mask()));
        }
        unsigned long long t2 = 0;
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
            float v[N];
            Elem<T>::unpack(raw[u], v);
            exps_fine(v, E);
#pragma unroll
            for (int i = 0; i < N; i += 2) t2 = add2(t2, bits_of(v[i], v[i + 1]));
        }
        const Two h = two_of(t2);
        const float t = h.a + h.b;
        if (t < 2.0f) {
            s += t;
        } else {
#pragma unroll
            for (int u = 0; u < VECS; ++u) *this = careful(*this, raw[u]);
        }
    }
};

// Where the output's 16-byte boundaries lie `k` elements (1 .. N - 1) behind those of the input: the vector that
// ends at the boundary inside a lane's own vector, from the last N - k elements of the vector before it and
// the first k of its own.
template <class T>
__device__ __forceinline__ uint4 straddle(const uint4& before, const uint4& own, int k) {
    const int bits = k * (int)sizeof(T) * 8;      // the same for the whole row
    uint32_t w[8] = {before.x, before.y, before.z, before.w, own.x, own.y, own.z, own.w};
    if (bits & 64) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (bits & 32) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int sh = bits & 31;
    return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh), __funnelshift_r(w[2], w[3], sh),
                      __funnelshift_r(w[3], w[4], sh));
}

// The gradient of one CTA's part of a row.  FAR and the alignment of the output are the same for the whole row.
template <class T>
__device__ __forceinline__ void grad_part(const T* p, T* o, const Part<T>& part, const RowGrad& g, int edge, float edge_x) {
    constexpr int N = Elem<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, nthr = blockDim.x;
    const T* q = p + part.head + (size_t)part.first * N;
    T* t = o + part.head + (size_t)part.first * N;
    const int shift = (int)(((16 - ((uintptr_t)t & 15)) & 15) / sizeof(T));    // elements up to a 16-byte boundary
    int lo = tid, hi = part.n, step = nthr;         // this thread's vectors: lo, lo + step, ... below hi
    if (shift == 0 && !g.far) {
        for (int i = lo; i < hi; i += step) st_out16(t + (size_t)i * N, grad_vector<T>(ld_once16(q + (size_t)i * N), g, false));
    } else if (shift == 0) {
        for (int i = lo; i < hi; i += step) st_out16(t + (size_t)i * N, grad_vector<T>(ld_once16(q + (size_t)i * N), g, true));
    } else {
        // a run of consecutive vectors for every warp; what is left over at its two ends goes out one by one
        const int run = (part.n + nthr - 1) / nthr * 32;
        lo = min((tid >> 5) * run, part.n) + lane;
        hi = min(lo - lane + run, part.n);
        step = 32;
        uint4 last = make_uint4(0, 0, 0, 0);
        for (int i = lo; i - lane < hi; i += 32) {
            const uint4 v = grad_vector<T>(i < hi ? ld_once16(q + (size_t)i * N) : make_uint4(0, 0, 0, 0), g, g.far);
            const uint4 give = lane == 31 ? last : v;       // lane 0 follows lane 31 of the step before
            uint4 before;
            before.x = __shfl_sync(kFull, give.x, (lane + 31) & 31);
            before.y = __shfl_sync(kFull, give.y, (lane + 31) & 31);
            before.z = __shfl_sync(kFull, give.z, (lane + 31) & 31);
            before.w = __shfl_sync(kFull, give.w, (lane + 31) & 31);
            T* at = t + (size_t)i * N;
            const bool first = i == lo && lane == 0, end = i == hi - 1;
            if (i < hi && !first) st_out16(at + shift - N, straddle<T>(before, v, shift));
            if ((first && i < hi) || end) {
                union { uint4 u; T e[N]; } x;
                x.u = v;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e < shift ? first : end) *TPB_CK(&at[e]) = x.e[e];
            }
            last = v;
        }
    }
    if (edge >= 0) *TPB_CK(&o[edge]) = Elem<T>::put(grad_at(edge_x, edge, g));
    // the token's own entry, over what this warp has just stored there
    __syncwarp();
    if (g.label >= part.head && g.label < part.head + part.nvec * N) {
        const int i = (g.label - part.head) / N - part.first;
        if (i >= lo && i < hi && (i - lo) % step == 0) *TPB_CK(&o[g.label]) = Elem<T>::put(g.at_label);
    }
}

// The mean of up to kFewPairs losses by one warp; a CTA of the gradient's kernel does it beside its rows.
constexpr int kFewPairs = 4096;
struct PairSum {
    const double* part;   // NULL: nothing to add up
    int n;
    float* loss;
    __device__ __forceinline__ void run() const {
        if (!part || threadIdx.x >= 32) return;
        double s = 0.0;
        for (int i = threadIdx.x; i < n; i += 32) s += *TPB_CK(&part[i]);
        s = warp_add(s);
        if (threadIdx.x == 0) *TPB_CK(loss) = (float)(s / (double)n);
    }
};
__global__ void __launch_bounds__(32) pair_sum_kernel(PairSum sum) { sum.run(); }

struct ScoreOut {
    float *logp, *lse;   // all but logp may be NULL
    float2* keep;        // (reference, unit)
    double* exact;       // logp before it is rounded
    float* coef;         // set to zero: rows of no sequence keep that
};

// The gradient of logp that the caller has, and lse as the forward call rounded it.
struct BackwardIn {
    PerToken<float> grad;
    const float* lse;
};

// (sum, reference) pairs of the lanes as one
__device__ __forceinline__ void join_warp(float& s, float& m) {
    const float own = m;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
    s = warp_add(s * rebase(own, m));
}

constexpr int kRowThreads = 512;
#ifdef TPB200_CHECKED
constexpr int kRowCtas = 3;      // on an SM; the checker's own function needs 38 registers
#else
constexpr int kRowCtas = 4;
#endif
constexpr int kRowCluster = 8;

// Log-probabilities, the whole policy loss, or the gradient of log-probabilities: a cluster of C CTAs per row, each with 1/C of the
// row's 16-byte vectors.  The first sweep sums, the CTAs' (sum, reference) pairs cross the cluster through
// distributed shared memory, and the second sweep writes the gradient; it reads the row again, from L2,
// because C is chosen so that the rows in flight take half of it (row_shape), and because loads and stores say
// what may be evicted.  Bytes from and to memory are then near one read and one write.  What bounds the losses: two
// ex2 per element, 16 a cycle on an SM (249 of 360 us on [4096,151936] bf16 with 90 % of the rows counted; the pipe is 62 %
// busy, the issue slots 56 %), and the second read through L2; 2048 threads on an SM hide their latencies.
// Measured, of one read and one write: [4096,50016] bf16 4.90 TB/s (C = 1), [1024,151936] bf16 4.38 (C = 3),
// f32 4.59 (C = 6); the backward call, most rows by lse: 6.11, 5.98 (C = 3).  An earlier form, without the exact sums and
// at 4.97, 4.46 and 4.83, was the base of these comparisons: two CTAs of 512 on an SM instead of four 4.0, 4.0
// and 4.3; separate kernels for sum and gradient 3.8 and 3.8; the row kept in shared memory (a ring of bulk copies,
// persistent CTAs), which left 16 to 26 warps on an SM to hide the latencies, 4.6, 4.0 and 3.2.
enum Mode { kScores, kPolicy, kBackward };
template <class T, int MODE>
__global__ void __launch_bounds__(kRowThreads, kRowCtas)
row_kernel(Logits<T> in, PerToken<long long> labels, RowLimits limits, PolicyTerms terms, PolicyOut out, ScoreOut score, BackwardIn back,
           T* __restrict__ grad, int C, float* __restrict__ loss) {
    constexpr int N = Elem<T>::N;
    constexpr bool POLICY = MODE == kPolicy, BACKWARD = MODE == kBackward;
    __shared__ float red_s[kRowThreads / 32], red_m[kRowThreads / 32];
    __shared__ float2 pair[kRowCluster];     // (sum, reference) of every CTA of the cluster
    __shared__ RowGrad sh;
    __shared__ PolicyToken token;            // of thread 0 alone
    __shared__ int skipped[kRowThreads / 32];   // the place of the token's entry in its vector, for every warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthr = blockDim.x;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = C > 1 ? (int)cluster.block_rank() : 0;
    const unsigned r = blockIdx.x / (unsigned)C, a = r / (unsigned)in.inner, b = r - a * (unsigned)in.inner;
    long long label = labels.at(a, b);
    float weight = 0.0f;                    // BACKWARD: the caller's gradient of logp
    if (POLICY || BACKWARD) {
        weight = POLICY ? terms.weight.at(a, b) : back.grad.at(a, b);
        if (weight == 0.0f) label = -1;
    } else if (!limits.inside(r)) {
        label = -1;
    }
    T* o = MODE != kScores && grad ? grad + (long long)r * in.vocab : nullptr;
    if (label < 0) {
        if (!BACKWARD && tid == 0 && rank == 0) {
            if (POLICY) {
                store_policy(out, r, 0.0, PolicyRow{0.0f, 0.0f, 0.0f, 0.0});
                if (loss) *TPB_CK(loss) = 0.0f;
            } else {
                *TPB_CK(&score.logp[r]) = 0.0f;
                if (score.lse) *TPB_CK(&score.lse[r]) = 0.0f;
                if (score.keep) *TPB_CK(&score.keep[r]) = make_float2(0.0f, 0.0f);
                if (score.exact) *TPB_CK(&score.exact[r]) = 0.0;
                if (score.coef) *TPB_CK(&score.coef[r]) = 0.0f;
            }
        }
        if (MODE != kScores && o) zero_part(o, Part<T>(o, in.vocab, rank, C), in.vocab, rank, C);
        return;                             // all CTAs of the cluster alike
    }
    const T* p = in.x + (long long)a * in.s0 + (long long)b * in.s1;
    const Part<T> part(p, in.vocab, rank, C);
    const int at = label < in.vocab ? (int)label : -1;
    const int edge = part.edge(tid, in.vocab, rank, C);
    const float edge_x = edge >= 0 ? Elem<T>::get(*TPB_CK(&p[edge])) : -INFINITY;
    float at_label = 0.0f;
    if (BACKWARD) {
        if (at >= 0) at_label = Elem<T>::get(*TPB_CK(&p[at]));
        const float lse = *TPB_CK(&back.lse[r]);
        // The float32 lse is up to 2^-24 |lse| off, and so is every p.  It serves while that is under 2^-20 and the token has
        // less than half of the probability (it goes by 1 - p); else the row is summed again (all CTAs alike).
        if (at < 0 || (fabsf(lse) < 32.0f && at_label - lse < -0.7f)) {
            RowGrad g;
            // p = 2^(c x - E) 2^(E - c lse)
            const float unit = ex2(fmaf(lse, -kLog2e, base_of(lse)) - lse * (float)(1.4426950408889634 - (double)kLog2e));
            g.set(lse, unit, at < 0 ? NAN : -expm1f((float)((double)at_label - (double)lse)), weight, at);
            if (at < 0) g.k = NAN;
            grad_part(p, o, part, g, edge, edge_x);
            return;
        }
    } else if (tid == 0) {
        if (POLICY) fetch_token(terms, a, b, weight, &token);
        if (at >= 0) at_label = Elem<T>::get(*TPB_CK(&p[at]));
    }
    if (C > 1) cluster_arrive();

    // ---- the sum of all but the token's own term
    const int skip = at >= part.head && at < in.vocab - part.tail ? (at - part.head) / N - part.first : -1;   // the vector with the token's entry
    if (lane == 0) skipped[warp] = (at - part.head) & (N - 1);
    __syncwarp();
    const T* q = p + part.head + (size_t)part.first * N;
    FixedSum<T> sum;
    sum.init();
    {
        // a row that is swept twice stays in L2 until then
        const unsigned long long policy = MODE != kScores && o ? l2_last() : l2_first();
        // the lanes of this warp whose first step has two vectors, or one
        const auto pairs = [&] { return lanes_below(part.n - nthr - (tid & ~31)); };
        const auto singles = [&] { return lanes_below(part.n - (tid & ~31)) & ~pairs(); };
        int i = tid;
        for (; i + nthr < part.n; i += 2 * nthr) {
            uint4 raw[2] = {ld_policy16(q + (size_t)i * N, policy), ld_policy16(q + (size_t)(i + nthr) * N, policy)};
            const int d = skip - i;
            if (d == 0 || d == nthr) leave_out<T>(raw, (d == 0 ? 0 : N) + skipped[warp]);
            sum.add(raw, i == tid, pairs);
        }
        if (i < part.n) {
            uint4 raw[1] = {ld_policy16(q + (size_t)i * N, policy)};
            if (i == skip) leave_out<T>(raw, skipped[warp]);
            sum.add(raw, i == tid, singles);
        }
        if (edge >= 0 && edge != at) {      // as a vector with one element
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = e == 0 ? edge_x : -INFINITY;
            const uint4 raw[1] = {Elem<T>::pack(v)};
            sum.add(raw, false, [] { return 0u; });
        }
    }
    float m = sum.ref, s = sum.s;
    join_warp(s, m);
    if (nthr > 32) {
        if (lane == 0) {
            red_s[warp] = s;
            red_m[warp] = m;
        }
        __syncthreads();
        if (warp == 0) {                    // the others have no use for the sum
            const int nw = nthr >> 5;
            s = lane < nw ? red_s[lane] : 0.0f;
            m = lane < nw ? red_m[lane] : -INFINITY;
            join_warp(s, m);
        }
    }
    if (C > 1) {
        cluster_wait();                     // all CTAs of the cluster have started
        if (tid < C) *cluster.map_shared_rank(&pair[rank], (unsigned)tid) = make_float2(s, m);
        cluster.sync();
        if (warp == 0) {
            const float2 v = lane < C ? pair[lane & (kRowCluster - 1)] : make_float2(0.0f, -INFINITY);
            s = v.x;
            m = v.y;
            join_warp(s, m);                // the same order in every CTA
        }
    }
    if (tid == 0) {
        const Score y = score_of(at >= 0, at_label, m, s);
        if (POLICY) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            const PolicyRow row = policy_row(terms, token, y.logp);
            const float2 k = unit_of(y, at_label, m, s);
            sh.set(k.x, k.y, y.rest(), row.coef, at);
            if (rank == 0) {
                store_policy(out, r, y.logp, row);
                if (loss) *TPB_CK(loss) = (float)row.part;
            }
        } else if (BACKWARD) {
            const float2 k = unit_of(y, at_label, m, s);
            sh.set(k.x, k.y, y.rest(), weight, at);
        } else if (rank == 0) {
            *TPB_CK(&score.logp[r]) = (float)y.logp;
            if (score.lse) *TPB_CK(&score.lse[r]) = (float)y.lse;
            if (score.keep) *TPB_CK(&score.keep[r]) = unit_of(y, at_label, m, s);
            if (score.exact) *TPB_CK(&score.exact[r]) = y.logp;
            if (score.coef) *TPB_CK(&score.coef[r]) = 0.0f;
        }
    }
    if (MODE == kScores || !o) return;
    __syncthreads();
    const RowGrad g = sh;
    grad_part(p, o, part, g, edge, edge_x);
}

// ---------------------------------------------------------------- gradient from saved statistics
// The preference loss's second part, by the (reference, unit) of every row and its coefficient.
template <class T>
__global__ void __launch_bounds__(kRowThreads, kRowCtas)
score_grad_kernel(Logits<T> in, PerToken<long long> labels, const float2* __restrict__ keep, const float* __restrict__ coefs,
                  const float* __restrict__ logp, T* __restrict__ out, unsigned rows, int C, PairSum sum) {
    if (blockIdx.x == 0) sum.run();
    // the rows go backwards: the last ones that the sums read are still in L2
    const unsigned from = blockIdx.x / (unsigned)C, r = rows - 1 - from;
    const int rank = (int)(blockIdx.x - from * (unsigned)C);
    const unsigned a = r / (unsigned)in.inner, b = r - a * (unsigned)in.inner;
    T* o = out + (long long)r * in.vocab;
    const long long y = labels.at(a, b);
    const float coef = y < 0 ? 0.0f : *TPB_CK(&coefs[r]);
    if (coef == 0.0f) {
        zero_part(o, Part<T>(o, in.vocab, rank, C), in.vocab, rank, C);
        return;
    }
    const T* p = in.x + (long long)a * in.s0 + (long long)b * in.s1;
    const Part<T> part(p, in.vocab, rank, C);
    const int edge = part.edge(threadIdx.x, in.vocab, rank, C);
    const float edge_x = edge >= 0 ? Elem<T>::get(*TPB_CK(&p[edge])) : -INFINITY;
    RowGrad g;
    const float2 k = *TPB_CK(&keep[r]);
    g.set(k.x, k.y, -expm1f(*TPB_CK(&logp[r])), coef, y < in.vocab ? (int)y : -1);
    if (y >= in.vocab) g.k = NAN;
    grad_part(p, o, part, g, edge, edge_x);
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
pair_kernel(PerToken<long long> labels, PerToken<float> ref, const double* __restrict__ logp, const long long* __restrict__ offsets,
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
            if (labels.at(a, b) >= 0) s += *TPB_CK(&logp[r]) - (double)ref.at(a, b);
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

// Threads of a CTA and CTAs per row.  Short rows get as many threads as they have pairs of vectors.  More than one
// CTA per row: with a second sweep, so that the rows in flight (four CTAs on every SM) take at most 60 MB, half
// of L2; and while all CTAs fit the GPU at once and a CTA still has a vector per thread.  Policy loss on [1024,151936],
// bf16, C = 1, 2, 3, 4, 6: 4.11, 4.30, 4.36, 4.23, 3.85 TB/s; f32: 4.13, 4.18, 4.37, 4.34, 4.59; on [4096,50016] bf16, C = 1, 2:
// 4.90, 4.11.  Scores of [256,151936] f32, C = 1, 2 (512 CTAs of 592), 3, 4: 34.6, 29.0, 36.8, 34.5 us; of [1,151936] bf16,
// C = 1, 4, 8: 12.6, 7.4, 6.0 us.  The backward call goes by the rule of two sweeps, though it mostly needs one:
// [1024,151936] bf16, C = 1, 2, 3, 4: 107, 106, 105, 104 us.
struct RowShape { int threads, C; };
inline RowShape row_shape(int64_t rows, int64_t vocab, int64_t elem, bool twice) {
    const int64_t vectors = vocab * elem / 16, room = 4LL * sm_count();
    RowShape s{(int)std::max<int64_t>(32, std::min<int64_t>(kRowThreads, round_up(ceil_div(vectors, 2), 32))), 1};
    if (s.threads < kRowThreads) return s;
    int64_t C = 1;
    if (twice) C = std::min<int64_t>(kRowCluster, ceil_div(std::min(rows, room) * vocab * elem, 60LL << 20));
    while (C < kRowCluster && rows * (C + 1) <= room && vectors >= (C + 1) * kRowThreads) ++C;
    int forced = 0;      // experiment and test switch: that many CTAs per row (tests run every kernel at 1 to 8)
    if (env_int("TPB200_ROW_CTAS", &forced) && forced >= 1 && forced <= kRowCluster) C = forced;
    if (rows * C > 0x7fffffffLL) C = 1;
    s.C = (int)C;
    return s;
}

template <class T, int MODE>
int row_run(const Logits<T>& in, const PerToken<long long>& lab, const RowLimits& limits, const PolicyTerms& terms, const PolicyOut& out,
            const ScoreOut& score, const BackwardIn& back, T* grad, int64_t rows, float* loss, cudaStream_t st) {
    const RowShape s = row_shape(rows, in.vocab, sizeof(T), grad != nullptr);
    const cudaError_t e = launch_ex(row_kernel<T, MODE>, dim3((unsigned)(rows * s.C)), s.threads, 0, st, s.C, false, in, lab, limits, terms, out, score, back,
                                    grad, s.C, rows == 1 ? loss : nullptr);
    return e == cudaSuccess ? TPB200_OK : cuda_fail(e, "row_kernel");
}
template <class T>
int score_run(const Logits<T>& in, const PerToken<long long>& lab, const RowLimits& limits, float* logp, float* lse, float2* keep,
              double* exact, float* coef, int64_t rows, cudaStream_t st) {
    return row_run<T, kScores>(in, lab, limits, PolicyTerms{}, PolicyOut{}, ScoreOut{logp, lse, keep, exact, coef}, BackwardIn{}, (T*)nullptr, rows, nullptr, st);
}
template <class T>
int score_grad_run(const Logits<T>& in, const PerToken<long long>& lab, const float2* keep, const float* coefs, const float* logp, T* out,
                   int64_t rows, const PairSum& sum, cudaStream_t st) {
    const RowShape s = row_shape(rows, in.vocab, sizeof(T), false);
    TPB_LAUNCH("score_grad_kernel", score_grad_kernel<T>, dim3((unsigned)(rows * s.C)), s.threads, 0, st, in, lab, keep, coefs, logp, out, (unsigned)rows,
               s.C, sum);
    return TPB200_OK;
}

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
    TPB_BY_TYPE(dtype, return score_run<T>(logits_of<T>(logits, inner, vocab, strides), lab, RowLimits{nullptr, 0}, logp, lse, nullptr, nullptr, nullptr, rows, st));
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
    const BackwardIn back{per_token(grad_logp, grad_strides), lse};
    TPB_BY_TYPE(dtype, return (row_run<T, kBackward>(logits_of<T>(logits, inner, vocab, strides), lab, RowLimits{nullptr, 0}, PolicyTerms{}, PolicyOut{},
                                                     ScoreOut{}, back, (T*)grad_logits, rows, nullptr, st)));
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
        TPB_BY_TYPE(dtype, rc = (row_run<T, kPolicy>(logits_of<T>(logits, inner, vocab, strides), lab, RowLimits{nullptr, 0}, terms, out,
                                                  ScoreOut{}, BackwardIn{}, (T*)grad_logits, rows, loss, st)));
        if (rc != TPB200_OK || rows == 1) return rc;     // a single row has written the loss itself
    }
    TPB_LAUNCH("loss_sum_kernel", loss_sum_kernel, dim3(1), 1024, 0, st, (const double*)workspace, (long long)rows, 1.0, loss);
    return TPB200_OK;
}

// workspace of the preference loss: logp in 64 bits, (reference, unit) and the coefficient of every row, the loss of every pair
extern "C" size_t tpb200_preference_loss_workspace_bytes(int64_t outer, int64_t inner, int64_t pairs) {
    if (outer < 0 || inner < 0 || pairs < 0) return 0;
    return (size_t)(outer * inner) * (sizeof(double) + sizeof(float2) + sizeof(float)) + (size_t)pairs * sizeof(double);
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
    double* exact = part + pairs;
    float2* keep = (float2*)(exact + rows);
    float* coefs = (float*)(keep + rows);
    const PerToken<long long> lab{(const long long*)labels, label_strides[0], label_strides[1]};
    const RowLimits limits{(const long long*)offsets, 2 * pairs};
    if (rows > 0) {
        TPB_BY_TYPE(dtype, rc = score_run<T>(logits_of<T>(logits, inner, vocab, strides), lab, limits, logp, nullptr, keep, exact, grad_logits ? coefs : nullptr, rows, st));
        if (rc != TPB200_OK) return rc;
    }
    TPB_LAUNCH("pair_kernel", pair_kernel, dim3((unsigned)pairs), 256, 0, st, lab, per_token(ref_logp, ref_strides), (const double*)exact,
               (const long long*)offsets, (long long)rows, (long long)std::max<int64_t>(inner, 1), (long long)pairs, beta, label_smoothing, grad_scale,
               rewards, part, grad_logits ? coefs : nullptr);
    const bool few = pairs <= kFewPairs, beside = few && rows > 0 && grad_logits;
    const PairSum sum{few ? part : nullptr, few ? (int)pairs : 0, loss};
    if (!few) TPB_LAUNCH("loss_sum_kernel", loss_sum_kernel, dim3(1), 1024, 0, st, (const double*)part, (long long)pairs, 1.0 / (double)pairs, loss);
    else if (!beside) TPB_LAUNCH("pair_sum_kernel", pair_sum_kernel, dim3(1), 32, 0, st, sum);
    if (rows > 0 && grad_logits)
        TPB_BY_TYPE(dtype, return score_grad_run<T>(logits_of<T>(logits, inner, vocab, strides), lab, keep, coefs, logp, (T*)grad_logits, rows, beside ? sum : PairSum{}, st));
    return TPB200_OK;
}
