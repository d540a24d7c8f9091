// Losses over the log-probability of given labels: label_logp and its gradient, the clipped policy loss, the preference loss.
//
//   lse_r = log sum_c exp z_rc        logp_r = z_r,label - lse_r        d logp_r / d z_rc = [c = label] - exp(z_rc - lse_r)
//
// Rows whose label is outside [0, C), and rows of weight 0, take no part: logp 0, gradient 0, whatever their logits hold.
// Logits and gradients are f32 or bf16, rows of ldl >= C elements, of which the gradient's last ldl - C are zero; all arithmetic is f32,
// sums over rows are f64, every reduction has a fixed order.
#include <math.h>

#include "common.h"

namespace {

using namespace emadapt;

// 16 bytes of a row, kept as they are loaded: any element alignment (gfx950 loads and stores dwordx4 at any address the element type allows).
typedef unsigned Raw __attribute__((ext_vector_type(4)));
template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T> __device__ __forceinline__ void unpack(Raw r, float (&v)[Vec<T>::N]);
template <> __device__ __forceinline__ void unpack<float>(Raw r, float (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = __uint_as_float(r[k]);
}
template <> __device__ __forceinline__ void unpack<__bf16>(Raw r, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[2 * k] = __uint_as_float(r[k] << 16);
        v[2 * k + 1] = __uint_as_float(r[k] & 0xFFFF0000u);
    }
}
typedef unsigned U4 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef unsigned U2 __attribute__((ext_vector_type(2), aligned(2), may_alias));
// ONCE: read for the last time (nontemporal: what is in the cache stays there)
template <bool ONCE, typename T> __device__ __forceinline__ Raw load16(const T *p) {
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const U4 *>(p)) : *reinterpret_cast<const U4 *>(p);
}
template <typename T> __device__ __forceinline__ Raw pack_raw(const T (&t)[Vec<T>::N]) {
    Raw r;
    __builtin_memcpy(&r, t, 16);
    return r;
}
// Vector at element i of a row of C elements (ldl with the padding); what is not one of the C is -inf: no weight in any sum of exponentials.
template <bool ONCE, typename T> __device__ __forceinline__ Raw load_row(const T *z, int i, int C, int ldl) {
    constexpr int N = Vec<T>::N;
    T t[N];
    if (i + N <= C) return load16<ONCE>(z + i);
    if (i + N <= ldl) {
        __builtin_memcpy(t, z + i, 16);
#pragma unroll
        for (int k = 0; k < N; k++) t[k] = i + k < C ? t[k] : (T)-INFINITY;
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) t[k] = i + k < C ? z[i + k] : (T)-INFINITY;
    }
    return pack_raw<T>(t);
}
// (the empty asm keeps the compiler from making one plain store of the two)
template <typename U> __device__ __forceinline__ void put(char *p, const char *t, bool once) {
    U r;
    __builtin_memcpy(&r, t, sizeof(r));
    if (once) {
        asm volatile("");
        __builtin_nontemporal_store(r, reinterpret_cast<U *>(p));
        asm volatile("");
    } else
        *reinterpret_cast<U *>(p) = r;
}
template <typename T, int N> __device__ __forceinline__ void store_row(T *d, int i, int ldl, const float (&v)[N], bool once) {
    T t[N];
#pragma unroll
    for (int k = 0; k < N; k++) t[k] = (T)v[k];
    char *p = reinterpret_cast<char *>(d + i);
    const char *q = reinterpret_cast<const char *>(t);
    if (i + N <= ldl) {
        if constexpr (sizeof(t) == 8) put<U2>(p, q, once);
        else {
#pragma unroll
            for (int k = 0; k < (int)sizeof(t); k += 16) put<U4>(p + k, q + k, once);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (i + k < ldl) d[i + k] = t[k];
    }
}
// d logits of one vector: [c = label] f - exp(z - base) fs, where base is the row's maximum and fs = f / sum (or its log-sum-exp, and fs = f);
// at = label - first element of the vector
template <typename T> __device__ __forceinline__ void grad_vec(Raw r, float base, float fs, float f, int at, float (&v)[Vec<T>::N]) {
    unpack<T>(r, v);
#pragma unroll
    for (int k = 0; k < Vec<T>::N; k++) v[k] = -__expf(v[k] - base) * fs;
    if ((unsigned)at < (unsigned)Vec<T>::N) {   // (one vector of a row)
#pragma unroll
        for (int k = 0; k < Vec<T>::N; k++) v[k] = at == k ? v[k] + f : v[k];
    }
}

__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

// running maximum and sum of exponentials of a part of a row
struct MaxSum {
    float m, s;
};
// the label's log-probability in a row with this maximum and sum (64 bits: the differences are exact, the sum's logarithm is what is rounded)
__device__ __forceinline__ double logp_of(float z, MaxSum row) { return ((double)z - (double)row.m) - (double)logf(row.s); }
// over a workgroup of W waves, from each wave's pair: one barrier, sh is free again at the next one
template <int W> __device__ __forceinline__ MaxSum block_join(MaxSum wave, MaxSum *sh) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = wave;
    __syncthreads();
    const MaxSum t = sh[threadIdx.x & (W - 1)];   // (W lanes hold all pairs)
    MaxSum r;
    r.m = group_max<W>(t.m);
    r.s = group_sum<W>(t.s * __expf(t.m - finite_or_0(r.m)));
    return r;
}
// of a row's kSplits parts, by every kSplits lanes that call it together
constexpr int kSplits = 32;   // parts of a row where rows are few
__device__ __forceinline__ MaxSum join_parts(const MaxSum *parts) {
    const MaxSum t = parts[threadIdx.x % kSplits];
    MaxSum r;
    r.m = group_max<kSplits>(t.m);
    r.s = group_sum<kSplits>(t.s * __expf(t.m - finite_or_0(r.m)));
    return r;
}
struct Rows {
    const void *logits;
    const long long *labels;
    long long ldl, M;
    int C;
    bool once;   // the gradient is too large to stay in the cache: it is not left there
    bool last;   // nor are the logits, which are read for the last time
};

// An f32 log-sum-exp of this size and more keeps too little of the sum (2^-12 of a probability is rounding here, and of a row masked as a whole with
// the type's lowest value the log C is gone): one wave takes the rows' maxima and sums anew, one row after the other, for its lanes.  False: no such
// row, or its lse is not its own (of a part of the classes, say).
constexpr float kFar = 4096.f;
template <typename T>
__device__ bool sum_anew(const Rows &a, long long row, bool far, float lse, MaxSum &own) {
    bool anew = false;
    for (unsigned long long left = __ballot(far); left;) {
        const long long r = __shfl(row, __ffsll((long long)left) - 1);
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        float m = -INFINITY, s = 0.f;
#pragma unroll 1
        for (int i = threadIdx.x & 63; i < a.C; i += 64) m = fmaxf(m, (float)z[i]);
        m = group_max<64>(m);
#pragma unroll 1
        for (int i = threadIdx.x & 63; i < a.C; i += 64) s += __expf((float)z[i] - m);
        s = group_sum<64>(s);
        const bool mine = far && row == r;
        if (mine && fabsf(m + logf(s) - lse) <= 0x1p-22f * fabsf(lse)) {
            own = {m, s};
            anew = true;
        }
        left &= ~__ballot(mine);
    }
    return anew;
}

// dz = [c = label] coef - exp(z - base) coef / sum (base, sum: the row's maximum and sum; without SUM base is the log-sum-exp): every thread kUnroll
// vectors of the flattened [M][vectors per row], all in flight.  A workgroup's vectors lie behind one another; their rows come from one 64-bit
// division for the workgroup and a 32-bit one for each vector.  HBM bounds it (4001 x 32768 bf16 behind its statistics 77.5 us, 6.8 TB/s of 4.8 to
// 6.7 that a copy reaches: a part of the logits is still in the cache).  Rows far from zero are written again at the end (looked at in front of the store
// they cost the others 4 to 9 % of the time).
template <typename T, typename TD, int kUnroll, bool SUM>
__global__ void __launch_bounds__(256) row_grad_kernel(Rows a, const float *__restrict__ base, const float *__restrict__ sum, const float *__restrict__ coef, TD *__restrict__ dlogits,
                                                      unsigned nvec, long long total) {
    constexpr int N = Vec<T>::N;
    const long long b = (long long)(gridDim.x - 1 - blockIdx.x) * (256 * kUnroll);   // (the rows that were read last come first: some are still in the cache)
    const long long r0 = b / nvec;
    const unsigned i0 = (unsigned)(b - r0 * nvec);
    struct Place {
        long long row;   // -1: past the end
        int at;
    };
    auto place = [&](int q) {
        const unsigned o = i0 + q * 256 + threadIdx.x, dr = o / nvec;
        return Place{b + q * 256 + threadIdx.x < total ? r0 + dr : -1, (int)(o - dr * nvec) * N};
    };
    Raw raw[kUnroll];
    Place to[kUnroll];
    int hit[kUnroll];
    float l[kUnroll], f[kUnroll], fs[kUnroll];
#pragma unroll
    for (int q = 0; q < kUnroll; q++) {
        to[q] = place(q);
        const long long row = to[q].row;
        if (row < 0) continue;
        raw[q] = load_row<false>(static_cast<const T *>(a.logits) + row * a.ldl, to[q].at, a.C, (int)a.ldl);
        const long long lab = a.labels[row];
        const bool used = lab >= 0 && lab < a.C;
        hit[q] = used ? (int)lab : -(1 << 30);
        l[q] = base[row];
        f[q] = used ? coef[row] : 0.f;
        fs[q] = SUM ? f[q] * __builtin_amdgcn_rcpf(sum[row]) : f[q];
    }
    unsigned far = 0u;
#pragma unroll
    for (int q = 0; q < kUnroll; q++) {
        const long long row = to[q].row;
        if (row < 0) continue;
        if (!SUM) far |= f[q] != 0.f && fabsf(l[q]) >= kFar && fabsf(l[q]) < INFINITY ? 1u << q : 0u;
        float v[N];
        grad_vec<T>(raw[q], l[q], fs[q], f[q], hit[q] - to[q].at, v);
        if (f[q] == 0.f) {   // (a row that takes no part: 0, also where 0 * NaN is not)
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = 0.f;
        }
        store_row<TD>(dlogits + row * a.ldl, to[q].at, (int)a.ldl, v, a.once);
    }
    if (SUM || !__any(far != 0u)) return;
#pragma unroll 1
    for (int q = 0; q < kUnroll; q++) {
        const bool mine = far >> q & 1u;
        const Place t = place(q);
        MaxSum own = {0.f, 1.f};
        if (!sum_anew<T>(a, t.row, mine, mine ? base[t.row] : 0.f, own)) continue;
        const float c = coef[t.row];
        float v[N];
        grad_vec<T>(load_row<false>(static_cast<const T *>(a.logits) + t.row * a.ldl, t.at, a.C, (int)a.ldl), own.m, c / own.s, c, (int)a.labels[t.row] - t.at, v);
        store_row<TD>(dlogits + t.row * a.ldl, t.at, (int)a.ldl, v, false);
    }
}

// ------------------------------------------------------------------------------------------
// the clipped policy loss
// ------------------------------------------------------------------------------------------
struct Policy {
    const float *old_logp, *ref_logp, *adv, *weight;
    double low, high;   // the ratio's borders, 1 - clip_low and 1 + clip_high
    double log_low, log_high;
    float kl, scale, tol;
};
struct PolicyTerms {
    double loss, surrogate, kl, clipped;
};

// exp(q) - 1 to a few roundings of itself: by its series where the subtraction would lose bits (q^9 / 9! is below 2^-24 q for |q| < 0.6)
__device__ __forceinline__ float exp_minus_1(float q) {
    const float series = q * (1.f + q * (1.f / 2 + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720 + q * (1.f / 5040 + q * (1.f / 40320))))))));
    return fabsf(q) < 0.5f ? series : __expf(q) - 1.f;
}
// What one row adds to the sums before its weight, and its d loss / d logp.
template <typename F> struct PolicyRow {
    F loss, part, k, c;
};
__device__ __forceinline__ void policy_add(PolicyTerms &t, double w, double loss, double part, double k, bool clipped) {
    t.loss += w * loss;
    t.surrogate += w * part;
    t.kl += w * k;
    t.clipped += clipped ? w : 0.0;
}
// in f32, as far as its intermediates go (fits)
__device__ __forceinline__ PolicyRow<float> policy_row(float log_ratio, float q, bool has_ref, float adv, float w, const Policy &p, bool clipped) {
    const float free = adv == 0.f && log_ratio == log_ratio ? 0.f : -adv * __expf(log_ratio);   // (without an advantage nothing, however large the ratio)
    const float e = has_ref ? exp_minus_1(q) : 0.f;
    PolicyRow<float> r;
    r.part = clipped ? -adv * (float)(adv > 0.f ? p.high : p.low) : free;
    // exp(q) - 1 - q: from q^2 / 2 on where the rest cancels
    r.k = !has_ref ? 0.f
          : fabsf(q) < 0.5f ? q * q * (1.f / 2 + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720 + q * (1.f / 5040 + q * (1.f / 40320)))))))
                            : e - q;
    r.loss = p.kl != 0.f ? r.part + p.kl * r.k : r.part;
    r.c = w * p.scale * ((clipped ? 0.f : free) - (p.kl != 0.f ? p.kl * e : 0.f));   // (e may have overflowed: no term, not 0 * inf)
    return r;
}
__device__ __forceinline__ bool fits(const PolicyRow<float> &r) { return fabsf(r.loss) < INFINITY && fabsf(r.c) < INFINITY; }
// exp(x) where f32 may not hold it, as the eighth power of an f32 exponential.  Held at e^600: beyond what f32 factors bring back, and still finite, so
// that a factor of 0 gives 0.
__device__ __forceinline__ double wide_exp(float x) {
    if (!(x > 80.f)) return (double)__expf(x);   // (NaN too)
    double e = (double)__expf((x < 600.f ? x : 600.f) * 0.125f);
    e *= e;
    e *= e;
    return e * e;
}
// exp(q) - 1 - q beyond f32 (q may be infinite)
__device__ __forceinline__ double wide_k(float q) { return wide_exp(q) - 1.0 - (double)(q < 600.f ? q : 600.f); }
// A row's coefficient: what f32 cannot hold is held to its largest finite value.  (An infinite one gives NaN at every class whose probability underflows.)
__device__ __forceinline__ double held_to_f32(double c) {
    constexpr double kMost = 0x1.fffffep127;
    return c > kMost ? kMost : c < -kMost ? -kMost : c;   // (NaN stays)
}
// in 64 bits, of every row that is looked at again: an exponential beyond f32 (of an action that the old policy held for impossible, of a reference far
// away) counts as what its factors make of it.
__device__ __forceinline__ PolicyRow<double> policy_row_wide(float log_ratio, float q, bool has_ref, double adv, double w, const Policy &p, bool clipped) {
    const double free = -adv * wide_exp(log_ratio);
    const bool small = fabsf(q) < 0.5f;
    const double e = !has_ref ? 0.0 : small ? (double)exp_minus_1(q) : wide_exp(q) - 1.0;
    PolicyRow<double> r;
    r.part = clipped ? -adv * (adv > 0.0 ? p.high : p.low) : free;
    r.k = !has_ref ? 0.0
          : small ? (double)(q * q * (1.f / 2 + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720 + q * (1.f / 5040 + q * (1.f / 40320))))))))
                  : wide_k(q);
    r.loss = p.kl != 0.f ? r.part + (double)p.kl * r.k : r.part;
    r.c = held_to_f32(w * (double)p.scale * ((clipped ? 0.0 : free) - (p.kl != 0.f ? (double)p.kl * e : 0.0)));
    return r;
}
// is the log of the ratio past the border that its advantage's sign puts up?
__device__ __forceinline__ bool past_border(double log_ratio, float adv, const Policy &p) {
    return adv > 0.f ? log_ratio > p.log_high : (adv < 0.f ? log_ratio < p.log_low : false);
}
// The log ratio from an f32 sum of exponentials (z, maximum and old_logp are taken in 64 bits) is off by less than tol: with h = 2^-24, 3 h for each
// of the `steps` additions and rescalings behind one another and 30 h for the trees, 2 h |z - m| + 2 h for an exponential -- whose mean over the
// softmax is at most log C --, and 2 h log C for the logarithm; half as much again.
__host__ __device__ inline float border_tol(int steps, int C) { return 1.5f * 0x1p-24f * (3.f * steps + 40.f + 5.f * logf((float)C)); }
__device__ __forceinline__ bool near_border(double log_ratio, float adv, const Policy &p) {
    const double border = adv > 0.f ? p.log_high : p.log_low;
    return adv != 0.f && fabs(log_ratio - border) < (double)p.tol;
}
// sum over elements `first`, first + step, .. of the row of exp(z - its maximum) in 64 bits; the label's log-probability from the whole sum.
// LONG: four loads in flight (one workgroup's way through the row is all that such a row costs), for registers that short rows had better keep.
template <bool LONG, typename T>
__device__ double exact_part(const T *z, int C, float top, int first, int step) {
    double s = 0.0;
    int i = first;
#pragma unroll 1
    for (; LONG && i + 3 * step < C; i += 4 * step) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)z[i + k * step];
#pragma unroll
        for (int k = 0; k < 4; k++) s += exp((double)v[k] - (double)top);
    }
#pragma unroll 1
    for (; i < C; i += step) s += exp((double)(float)z[i] - (double)top);
    return s;
}
__device__ __forceinline__ double exact_logp(float z, float top, double sum) { return ((double)z - (double)top) - log(sum); }

// ------------------------------------------------------------------------------------------
// rows that stay in registers: one pass over the logits
// ------------------------------------------------------------------------------------------
enum { kLogp = 0, kPolicy = 1, kPolicyGrad = 2 };
struct Outputs {
    float *logp, *lse;          // kLogp: any of these may be null
    float *base, *sum, *zero;   // kLogp: the rows' maximum and sum of exponentials; a value per row set to 0 (kPolicyGrad: base of the near rows)
    void *dlogits;
    double *partial;            // a workgroup's sums, [gridDim.x][4]
    unsigned char *near;        // rows to be looked at again in 64 bits from their maximum in base (policy_finish_kernel)
    unsigned *ticket;           // its ticket, to be zeroed
    MaxSum *parts;              // [M][gridDim.y] of rows in several parts
    float *sums;                // of a grid of one workgroup
};

// A row's part of the policy loss once its log-sum-exp is known, as f32 sees it; near: to be looked at in 64 bits, since exact arithmetic may cut the ratio
// where f32 does not, or since f32 does not hold the row's terms.
struct PolicyInputs {
    float oldp, adv, w, refp;
    bool has_ref;
};
__device__ __forceinline__ PolicyInputs policy_inputs(const Policy &p, long long r) {
    return {p.old_logp[r], p.adv[r], p.weight ? p.weight[r] : 1.f, p.ref_logp ? p.ref_logp[r] : 0.f, p.ref_logp != nullptr};
}
__device__ __forceinline__ float policy_of_row(const Policy &p, const PolicyInputs &x, float z, MaxSum row, bool count, float &lp, bool &near, PolicyTerms &t) {
    const double lp64 = logp_of(z, row), lr = lp64 - (double)x.oldp, q = (double)x.refp - lp64;
    lp = (float)lp64;
    const bool clipped = past_border(lr, x.adv, p);
    const PolicyRow<float> r = policy_row((float)lr, (float)q, x.has_ref, x.adv, x.w, p, clipped);
    near = near_border(lr, x.adv, p);
    if (!fits(r)) near |= lr == lr && q == q && x.adv == x.adv && x.w == x.w;   // (what is NaN stays so)
    if (count && !near) policy_add(t, (double)x.w, (double)r.loss, (double)r.part, r.k < INFINITY ? (double)r.k : wide_k((float)q), clipped);   // (a KL part without a coefficient)
    return r.c;
}
__device__ __forceinline__ float policy_of_exact(const Policy &p, const PolicyInputs &x, double lp64, bool count, float &lp, PolicyTerms &t) {
    const double lr = lp64 - (double)x.oldp;
    lp = (float)lp64;
    const bool clipped = past_border(lr, x.adv, p);
    const PolicyRow<double> r = policy_row_wide((float)lr, (float)((double)x.refp - lp64), x.has_ref, (double)x.adv, (double)x.w, p, clipped);
    if (count) policy_add(t, (double)x.w, r.loss, r.part, r.k, clipped);
    return (float)r.c;
}

constexpr int kInlineLanes = 16;
// L lanes to a row, NV vectors of the padded row to a lane: few lanes, so that what is done once a row (logarithm, loss) is done for many rows by
// a wave's instruction (1.6 M rows of 24 f32: 54 us with a vector to a lane, 39 with three).  One pass: logits in, and with the policy loss their
// gradient out; HBM bounds it from some 100000 rows on (logp of those rows 28.6 us in the kernel, 5.8 TB/s; 195312 rows of 1024 f32 65 us, 6.1),
// below that the launches.  Narrow policy rows stay at 3 to 4 TB/s.  With the gradient its stores bound them, of which one covers 32 of every 96 bytes
// (1.67 M rows of 24 f32: 118 us, 63 without the stores, 121 with them and without the loss's arithmetic), without it each row's arithmetic (58 us,
// 35 without).
// The bound: 4 waves to a SIMD, where the rows' 64-bit path would take the registers of one (40 M bf16 in rows of 128: 53.1 us with the bound, 58.7 without).
template <typename T, typename TD, int L, int NV, int MODE>
__global__ void __launch_bounds__(256, MODE == kPolicyGrad ? 4 : 1) group_kernel(Rows a, Policy p, Outputs out) {
    constexpr int N = Vec<T>::N;
    // Rows to be looked at again (near) here, or in policy_finish_kernel: 64-bit exponentials here double the registers of all rows (200 M bf16 in rows of 1000:
    // 252 us and 198), but find the row's inputs at hand (26896 rows of 24 f32, two of them near a border: 10.8 us and 20.5; none of them: 9.7 and 12.5;
    // 1.67 M rows: 118 and 137, of 24 bf16 46 and 58)
    constexpr bool kInline = L <= kInlineLanes;
    __shared__ double sh[4];
    const int lane = threadIdx.x % L;
    const long long per_grid = (long long)gridDim.x * (256 / L);
    PolicyTerms t = {0, 0, 0, 0};
    if (MODE != kLogp && !kInline && blockIdx.x == 0 && threadIdx.x == 0) *out.ticket = 0u;
    for (long long r = (long long)blockIdx.x * (256 / L) + threadIdx.x / L; r < a.M; r += per_grid) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        const long long lab = a.labels[r];
        PolicyInputs x = {0.f, 0.f, 1.f, 0.f, false};
        if (MODE != kLogp) x = policy_inputs(p, r);   // (in front of the row: their way to memory is the row's)
        const bool used = lab >= 0 && lab < a.C && x.w != 0.f;
        const float zl = (float)z[used ? lab : 0];
        Raw raw[NV];
        if (a.last) {
            asm volatile("");
#pragma unroll
            for (int k = 0; k < NV; k++) raw[k] = load_row<true>(z, (lane + k * L) * N, a.C, (int)a.ldl);
            asm volatile("");
        } else {
#pragma unroll
            for (int k = 0; k < NV; k++) raw[k] = load_row<false>(z, (lane + k * L) * N, a.C, (int)a.ldl);
        }
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float v[N];
            unpack<T>(raw[k], v);
#pragma unroll
            for (int e = 0; e < N; e++) m = fmaxf(m, v[e]);
        }
        m = group_max<L>(m);
        const float m0 = finite_or_0(m);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float v[N];
            unpack<T>(raw[k], v);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = __expf(v[e] - m0);
#pragma unroll
            for (int w = N / 2; w > 0; w /= 2)
#pragma unroll
                for (int e = 0; e < w; e++) v[e] += v[e + w];
            s += v[0];
        }
        s = group_sum<L>(s);
        float lp = 0.f, f = 0.f;
        bool near = false;
        if (used) {
            if (MODE == kLogp) lp = (float)logp_of(zl, MaxSum{m, s});
            else {
                f = policy_of_row(p, x, zl, MaxSum{m, s}, lane == 0, lp, near, t);
                if (kInline && near) {
                    double e = exact_part<false>(z, a.C, m, lane, L);
                    for (int o = L / 2; o > 0; o >>= 1) e += __shfl_xor(e, o);
                    f = policy_of_exact(p, x, exact_logp(zl, m, e), lane == 0, lp, t);
                }
            }
        }
        if (lane == 0) {
            if (MODE != kLogp || out.logp) out.logp[r] = lp;
            if (MODE == kLogp) {
                if (out.lse) out.lse[r] = m + logf(s);
                if (out.base) { out.base[r] = m; out.sum[r] = s; }
                if (out.zero) out.zero[r] = 0.f;
            } else if (!kInline) {
                out.near[r] = near;
                if (near) out.base[r] = m;
            }
        }
        if (MODE == kPolicyGrad) {
            const float fs = f * __builtin_amdgcn_rcpf(s);
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int i = (lane + k * L) * N;
                if (i >= a.ldl) continue;
                float v[N];
                grad_vec<T>(raw[k], m, fs, f, used ? (int)lab - i : -1, v);
                if (f == 0.f) {
#pragma unroll
                    for (int e = 0; e < N; e++) v[e] = 0.f;
                }
                store_row<TD>(static_cast<TD *>(out.dlogits) + r * a.ldl, i, (int)a.ldl, v, a.once && L >= 32);
            }
        }
    }
    if (MODE != kLogp) {
        const double sum[4] = {t.loss, t.surrogate, t.kl, t.clipped};
        for (int k = 0; k < 4; k++) {
            const double v = block_sum_f64(sum[k], sh);
            if (threadIdx.x != 0) continue;
            if (out.sums) out.sums[k] = (float)v;
            else out.partial[(long long)blockIdx.x * 4 + k] = v;
        }
    }
}

// One more 16 bytes into a thread's running maximum and sum of exponentials.  (exp2 of one fma, v log2 e - m log2 e, would save an instruction an
// element, but m log2 e overflows where a row is masked with the type's lowest value.)
template <int N> __device__ __forceinline__ void take(const float (&v)[N], float &m, float &s) {
    float top = m;
#pragma unroll
    for (int e = 0; e < N; e++) top = fmaxf(top, v[e]);
    const float m0 = finite_or_0(top);
    float x[N];
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = __expf(v[e] - m0);
#pragma unroll
    for (int w = N / 2; w > 0; w /= 2)   // (a tree: the rounding of the sum, and with it near_border's width, goes by the vectors)
#pragma unroll
        for (int e = 0; e < w; e++) x[e] += x[e + w];
    s = __builtin_fmaf(s, __expf(m - m0), x[0]);
    m = top;
}

// The policy loss with its gradient by a workgroup of W waves to a row, NV whole vectors to a thread, and the C % N last elements one to a thread.  HBM bounds it, each logit read and
// each gradient written once: 4096 x 65536 bf16 199 us, 5.4 TB/s of the 4.8 to 5.3 that a copy of that size reaches (330 us where statistics and
// gradient each read the logits).
template <typename T, typename TD, int W, int NV>
__global__ void __launch_bounds__(64 * W, 4) block_kernel(Rows a, Policy p, Outputs out) {
    constexpr int N = Vec<T>::N, kThreads = 64 * W;
    __shared__ MaxSum pair[2][W];
    __shared__ PolicyTerms terms;   // (thread 0's: registers are short here)
    if (threadIdx.x == 0) {
        terms = {0, 0, 0, 0};
        if (blockIdx.x == 0) *out.ticket = 0u;
    }
    const int nfull = a.C / N;
    int turn = 0;
    for (long long r = blockIdx.x; r < a.M; r += gridDim.x, turn ^= 1) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        unsigned tid = threadIdx.x;
        asm volatile("" : "+v"(tid));   // (or the row loop's registers go to the addresses and comparisons of all NV vectors, made once in front of it)
        const int last = nfull * N + (int)tid;
        const long long lab = a.labels[r];
        const PolicyInputs x = policy_inputs(p, r);   // (in front of the row: their way to memory is the row's)
        const bool used = lab >= 0 && lab < a.C && x.w != 0.f;
        const float zl = (float)z[used ? lab : 0];
        Raw raw[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {   // (all of them load, the ones past the row its last vector: the waits below can then count the loads)
            const int i = (int)tid + k * kThreads, j = i < nfull ? i : nfull - 1;
            raw[k] = load16<true>(reinterpret_cast<const T *>(reinterpret_cast<const char *>(z) + (unsigned)j * 16u));
        }
        float m = last < a.C ? (float)z[last] : -INFINITY;
        float s = last < a.C ? __expf(m - finite_or_0(m)) : 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++)
            if ((int)tid + k * kThreads < nfull) {
                float v[N];
                unpack<T>(raw[k], v);
                take(v, m, s);
                // (what is kept is the 16 bytes, not the numbers unpacked from them)
                asm volatile("" : "+v"(raw[k]));
            }
        const float mw = group_max<64>(m);
        s = group_sum<64>(s * __expf(m - finite_or_0(mw)));
        const MaxSum row = block_join<W>(MaxSum{mw, s}, pair[turn]);   // (two buffers: a wave may be a row ahead)
        float lp = 0.f, f = 0.f;
        bool near = false;
        if (used) {
            PolicyTerms one = {0, 0, 0, 0};
            f = policy_of_row(p, x, zl, row, threadIdx.x == 0, lp, near, one);
            if (threadIdx.x == 0) {
                terms.loss += one.loss; terms.surrogate += one.surrogate; terms.kl += one.kl; terms.clipped += one.clipped;
            }
        }
        if (threadIdx.x == 0) {
            out.logp[r] = lp;
            out.near[r] = near;
            if (near) out.base[r] = row.m;
        }
        TD *d = static_cast<TD *>(out.dlogits) + r * a.ldl;
        const int hit = used ? (int)lab : -(1 << 30);
        const float fs = f * __builtin_amdgcn_rcpf(row.s);
        for (int i = last; i < a.ldl; i += kThreads)   // the last elements and the padding
            d[i] = (TD)(f != 0.f && i < a.C ? (i == hit ? f : 0.f) - __expf((float)z[i] - row.m) * fs : 0.f);
        if (f == 0.f) {   // (a row that takes no part)
#pragma unroll 1
            for (int i = tid; i < nfull; i += kThreads) {
                const float v[N] = {};
                store_row<TD>(d, i * N, nfull * N, v, a.once);
            }
            continue;
        }
        asm volatile("" : "+v"(tid));
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int i = (int)tid + k * kThreads;
            if (i < nfull) {
                float v[N];
                grad_vec<T>(raw[k], row.m, fs, f, hit - i * N, v);
                store_row<TD>(reinterpret_cast<TD *>(reinterpret_cast<char *>(d) + (unsigned)i * (unsigned)(N * sizeof(TD))), 0, N, v, a.once);
            }
        }
    }
    if (threadIdx.x == 0) {
        double *o = out.partial + (long long)blockIdx.x * 4;
        o[0] = terms.loss; o[1] = terms.surrogate; o[2] = terms.kl; o[3] = terms.clipped;
    }
}

// One workgroup to a row of any length, read once: a running maximum and sum for every thread, kAhead vectors in flight.  Bound by HBM: 1500 x 100003
// f32 90 us in the kernel, 6.65 TB/s.
template <typename T, int W, bool ONCE>
__global__ void __launch_bounds__(64 * W) stream_stats_kernel(Rows a, Outputs out) {
    constexpr int N = Vec<T>::N, kThreads = 64 * W, kAhead = 4;
    __shared__ MaxSum pair[2][W];
    int turn = 0;
    for (long long r = blockIdx.x; r < a.M; r += gridDim.x, turn ^= 1) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        const long long lab = a.labels[r];
        float m = -INFINITY, s = 0.f;
        // (part y of the row: whole vectors, the last part with the rest)
        const int per = ((a.C + (int)gridDim.y * N - 1) / ((int)gridDim.y * N)) * N, begin = per * (int)blockIdx.y;
        const int end = begin + per < a.C ? begin + per : a.C;
        int i0 = begin + threadIdx.x * N;
        for (; i0 + (kAhead - 1) * kThreads * N + N <= end; i0 += kThreads * N * kAhead) {
            Raw raw[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) raw[k] = load16<ONCE>(z + i0 + k * kThreads * N);
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                float v[N];
                unpack<T>(raw[k], v);
                take(v, m, s);
            }
        }
        for (; i0 < end; i0 += kThreads * N) {   // (one at a time: all of the rest in flight costs 16 waves the second workgroup on a CU, 31 -> 39 us for 3000 x 32768)
            float v[N];
            unpack<T>(load_row<ONCE>(z, i0, end, end), v);
            take(v, m, s);
        }
        const float mw = group_max<64>(m);
        s = group_sum<64>(s * __expf(m - finite_or_0(mw)));
        const MaxSum row = block_join<W>(MaxSum{mw, s}, pair[turn]);
        if (threadIdx.x != 0) continue;
        if (out.parts) out.parts[r * gridDim.y + blockIdx.y] = row;
        else {
            if (out.lse) out.lse[r] = row.m + logf(row.s);
            if (out.base) { out.base[r] = row.m; out.sum[r] = row.s; }
            if (out.logp) out.logp[r] = lab >= 0 && lab < a.C ? (float)logp_of((float)z[lab], row) : 0.f;
            if (out.zero) out.zero[r] = 0.f;
        }
    }
}

// The rows' terms where the log-sum-exp comes from a launch of its own: as the rows' maximum and sum, or (PARTS) in kSplits parts of each row.
// By workgroup `block` of `blocks`; a single one also writes the sums.
template <typename T, bool PARTS>
__device__ void policy_rows(const Rows &a, const Policy &p, const MaxSum *__restrict__ parts, const float *__restrict__ base, const float *__restrict__ sum,
                            float *__restrict__ logp, float *__restrict__ coef, double *__restrict__ partial, float *__restrict__ sums, unsigned block, unsigned blocks) {
    __shared__ double sh[4];
    __shared__ unsigned long long mask[4];
    __shared__ MaxSum whole[PARTS ? 256 : 1];
    PolicyTerms t = {0, 0, 0, 0};
    for (long long r0 = (long long)block * 256; r0 < a.M; r0 += (long long)blocks * 256) {
        const long long r = r0 + threadIdx.x;
        bool again = false;
        if (PARTS) {   // a lane to a part
            for (int q = threadIdx.x / kSplits; q < 256 && r0 + q < a.M; q += 256 / kSplits) {
                const MaxSum row = join_parts(parts + (r0 + q) * kSplits);
                if (threadIdx.x % kSplits == 0) whole[q] = row;
            }
            __syncthreads();
        }
        if (r < a.M) {
            const long long lab = a.labels[r];
            const float w = p.weight ? p.weight[r] : 1.f;
            const MaxSum row = PARTS ? whole[threadIdx.x] : MaxSum{base[r], sum[r]};
            float lp = 0.f, f = 0.f;
            if (lab >= 0 && lab < a.C && w != 0.f)
                f = policy_of_row(p, policy_inputs(p, r), (float)(static_cast<const T *>(a.logits) + r * a.ldl)[lab], row, true, lp, again, t);
            logp[r] = lp;
            if (!PARTS) coef[r] = f;
        }
        // rows to be looked at again, in the order of their index
        const unsigned long long b = __ballot(again);
        if ((threadIdx.x & 63) == 0) mask[threadIdx.x >> 6] = b;
        __syncthreads();
        for (int q = 0; q < 4; q++)
            for (unsigned long long left = mask[q]; left; left &= left - 1) {
                const int k = q * 64 + (__ffsll((long long)left) - 1);
                const long long rr = r0 + k;
                const T *z = static_cast<const T *>(a.logits) + rr * a.ldl;
                const float top = PARTS ? whole[k].m : base[rr];
                const double lp64 = exact_logp((float)z[a.labels[rr]], top, block_sum_f64(exact_part<true>(z, a.C, top, threadIdx.x, 256), sh));
                if (threadIdx.x == 0) {
                    float lp;
                    const float f = policy_of_exact(p, policy_inputs(p, rr), lp64, true, lp, t);
                    logp[rr] = lp;
                    if (!PARTS) coef[rr] = f;
                }
            }
        __syncthreads();
    }
    const double s[4] = {t.loss, t.surrogate, t.kl, t.clipped};
    for (int k = 0; k < 4; k++) {
        const double v = block_sum_f64(s[k], sh);
        if (threadIdx.x == 0) {
            if (blocks == 1) sums[k] = (float)v;
            else partial[(long long)block * 4 + k] = v;
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(256) policy_row_kernel(Rows a, Policy p, const float *__restrict__ base, const float *__restrict__ sum, float *__restrict__ logp,
                                                        float *__restrict__ coef, double *__restrict__ partial, float *__restrict__ sums) {
    policy_rows<T, false>(a, p, nullptr, base, sum, logp, coef, partial, sums, blockIdx.x, gridDim.x);
}
// Few long rows, whose statistics came in parts: the first workgroup writes logp and the sums, the others the gradient of 256 kUnroll vectors of
// one row each (per: workgroups to a row), whose term each of them takes from the parts by itself -- a launch less than with the terms in one of
// their own (7 rows of 128001 bf16: 20.9 us and 17.5, 128 rows: 35 and 26).  In a row to be looked at again each of them goes through it.
template <typename T, typename TD, int kUnroll>
__global__ void __launch_bounds__(256) policy_few_kernel(Rows a, Policy p, const MaxSum *__restrict__ parts, float *__restrict__ logp, float *__restrict__ sums,
                                                        TD *__restrict__ dlogits, unsigned per) {
    constexpr int N = Vec<T>::N;
    __shared__ double sh[4];
    if (blockIdx.x == 0) {
        policy_rows<T, true>(a, p, parts, nullptr, nullptr, logp, nullptr, nullptr, sums, 0, 1);
        return;
    }
    const long long r = (blockIdx.x - 1) / per;
    const int first = (int)((blockIdx.x - 1) % per * (256 * kUnroll) + threadIdx.x);
    const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
    Raw raw[kUnroll];
#pragma unroll
    for (int q = 0; q < kUnroll; q++) raw[q] = load_row<true>(z, (first + q * 256) * N, a.C, (int)a.ldl);   // (past the row: reads nothing)
    const MaxSum row = join_parts(parts + r * kSplits);
    const PolicyInputs x = policy_inputs(p, r);
    const long long lab = a.labels[r];
    const bool used = lab >= 0 && lab < a.C && x.w != 0.f;
    float f = 0.f, lp;
    bool near = false;
    PolicyTerms none = {0, 0, 0, 0};
    if (used) f = policy_of_row(p, x, (float)z[lab], row, false, lp, near, none);
    if (near) f = policy_of_exact(p, x, exact_logp((float)z[lab], row.m, block_sum_f64(exact_part<true>(z, a.C, row.m, threadIdx.x, 256), sh)), false, lp, none);
    const float fs = f * __builtin_amdgcn_rcpf(row.s);
#pragma unroll
    for (int q = 0; q < kUnroll; q++) {
        const int i = (first + q * 256) * N;
        if (i >= a.ldl) continue;
        float v[N];
        grad_vec<T>(raw[q], row.m, fs, f, used ? (int)lab - i : -1, v);
        if (f == 0.f) {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = 0.f;
        }
        store_row<TD>(dlogits + r * a.ldl, i, (int)a.ldl, v, false);
    }
}

constexpr int kFinishRows = 16 * 1024;   // to a workgroup
// The sums of the launch before, and its rows to be looked at again (near, of a launch that wrote a gradient; or null) in 64 bits: most workgroups find none.
// Their terms were left out there; logp and the gradient are written again.  The last workgroup adds everything up in a fixed order.
template <typename T, typename TD>
__global__ void __launch_bounds__(1024) policy_finish_kernel(Rows a, Policy p, Outputs out, int nparts, double *__restrict__ fixed, float *__restrict__ sums) {
    __shared__ double sh[16][4];
    __shared__ double one[16];
    __shared__ unsigned long long mask[16];
    __shared__ bool last;
    PolicyTerms t = {0, 0, 0, 0};
    bool hit = false;
    if (out.near) {
        // 16 rows to a thread at a look, and 1024 to the workgroup where there are any
        for (long long r0 = (long long)blockIdx.x * kFinishRows, look = r0; r0 < a.M; r0 = look) {
            if (r0 % kFinishRows == 0) {
                const long long at = r0 + threadIdx.x * 16;
                const Raw some = at < a.M ? *reinterpret_cast<const Raw *>(out.near + at) : Raw{0, 0, 0, 0};
                if (!__syncthreads_or(some[0] | some[1] | some[2] | some[3])) {
                    look = r0 + (long long)gridDim.x * kFinishRows;
                    continue;
                }
            }
            look = r0 + 1024;
            if (look % kFinishRows == 0) look += (long long)(gridDim.x - 1) * kFinishRows;
            const long long mine = r0 + threadIdx.x;
            const unsigned long long b = __ballot(mine < a.M && out.near[mine]);
            hit = true;
            // one row, by `step` threads of which this is number `first`
            auto exact_row = [&](long long r, int first, int step, auto &&sum_of) {
                const long long lab = a.labels[r];
                const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
                const float top = out.base[r];
                const double sum = sum_of(exact_part<true>(z, a.C, top, first, step)), lp64 = exact_logp((float)z[lab], top, sum);
                float lp;
                const float f = policy_of_exact(p, policy_inputs(p, r), lp64, first == 0, lp, t);
                if (first == 0) out.logp[r] = lp;
                TD *d = static_cast<TD *>(out.dlogits) + r * a.ldl;
                const float over = (float)((double)f / sum);
#pragma unroll 1
                for (int i = first; i < a.C; i += step) d[i] = (TD)(f == 0.f ? 0.f : (i == (int)lab ? f : 0.f) - __expf((float)z[i] - top) * over);
            };
            if (a.C <= 4096) {   // each wave its own rows
                for (unsigned long long left = b; left; left &= left - 1)
                    exact_row(r0 + (threadIdx.x & ~63u) + (__ffsll((long long)left) - 1), threadIdx.x & 63, 64, [](double v) {
                        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
                        return v;
                    });
                continue;
            }
            if ((threadIdx.x & 63) == 0) mask[threadIdx.x >> 6] = b;
            __syncthreads();
            for (int q = 0; q < 16; q++)
                for (unsigned long long left = mask[q]; left; left &= left - 1)
                    exact_row(r0 + q * 64 + (__ffsll((long long)left) - 1), threadIdx.x, 1024, [&](double v) { return block_sum_f64(v, one); });
            __syncthreads();
        }
        double own[4] = {t.loss, t.surrogate, t.kl, t.clipped};
        if (hit)
            for (int k = 0; k < 4; k++) own[k] = block_sum_f64(own[k], one);
        // (a ticket among few workgroups; the part is where every CU sees it before the ticket counts it)
        if (threadIdx.x == 0) {
            for (int k = 0; k < 4; k++) __hip_atomic_store(&fixed[(long long)blockIdx.x * 4 + k], own[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __builtin_amdgcn_s_waitcnt(0);
            last = __hip_atomic_fetch_add(out.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        }
        __syncthreads();
        if (!last) return;
    }
    double s[4] = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < nparts; i += 1024)
        for (int k = 0; k < 4; k++) s[k] += out.partial[(long long)i * 4 + k];
    if (out.near)
        for (int i = threadIdx.x; i < (int)gridDim.x; i += 1024)
            for (int k = 0; k < 4; k++) s[k] += __hip_atomic_load(&fixed[(long long)i * 4 + k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int o = 32; o > 0; o >>= 1)
        for (int k = 0; k < 4; k++) s[k] += __shfl_xor(s[k], o);
    if ((threadIdx.x & 63) == 0)
        for (int k = 0; k < 4; k++) sh[threadIdx.x >> 6][k] = s[k];
    __syncthreads();
    if (threadIdx.x < 4) {
        double v = 0.0;
        for (int w = 0; w < 16; w++) v += sh[w][threadIdx.x];
        sums[threadIdx.x] = (float)v;
    }
}

// ------------------------------------------------------------------------------------------
// the preference loss: one workgroup to a pair of sequences, or (SPLIT) gridDim.x of them where pairs are long.  A sequence's sum has to be known
// before its first gradient, so the logits are read twice around it; the launch itself (6 us for 12 pairs of 3362 rows) waits for its chain of loads,
// sums and 64-bit exponentials.
// ------------------------------------------------------------------------------------------
struct Preference {
    const float *logp;
    const long long *seq_start;
    const float *ref;
    long long M;
    float beta, smooth, scale;
    float *loss, *seq_logp, *coef;   // coef: or null
    double *part;                    // SPLIT: [2 pairs][gridDim.x] sums of parts of the sequences
};
// rows of part x of n of sequence s (a start outside the rows, or before the one in front of it, reads and writes nothing)
__device__ __forceinline__ void part_of(const Preference &a, long long s, unsigned x, unsigned n, long long &begin, long long &end) {
    const long long lo = min(max(a.seq_start[s], 0ll), a.M), hi = min(max(a.seq_start[s + 1], 0ll), a.M), per = hi > lo ? (hi - lo + n - 1) / n : 0;
    begin = lo + x * per;
    end = min(begin + per, hi);
}
__device__ __forceinline__ double part_sum(const Preference &a, long long begin, long long end, double *sh) {
    double v = 0.0;
    for (long long r = begin + threadIdx.x; r < end; r += 1024) v += (double)a.logp[r];
    return block_sum_f64(v, sh);
}
__global__ void __launch_bounds__(1024) preference_part_kernel(Preference a) {   // sequence blockIdx.y
    __shared__ double sh[16];
    long long begin, end;
    part_of(a, blockIdx.y, blockIdx.x, gridDim.x, begin, end);
    const double v = part_sum(a, begin, end, sh);
    if (threadIdx.x == 0) a.part[(long long)blockIdx.y * gridDim.x + blockIdx.x] = v;
}
template <bool SPLIT> __global__ void __launch_bounds__(1024) preference_pair_kernel(Preference a) {
    __shared__ double sh[16];
    const long long pair = SPLIT ? blockIdx.y : blockIdx.x;
    const unsigned x = SPLIT ? blockIdx.x : 0, n = SPLIT ? gridDim.x : 1;
    long long begin[2], end[2];
    double s[2];
    for (int q = 0; q < 2; q++) {
        part_of(a, 2 * pair + q, x, n, begin[q], end[q]);
        if (SPLIT) {
            double v = 0.0;
            for (unsigned i = threadIdx.x; i < n; i += 1024) v += a.part[(2 * pair + q) * n + i];
            s[q] = block_sum_f64(v, sh);
        } else s[q] = part_sum(a, begin[q], end[q], sh);
    }
    const double h = (double)a.beta * ((s[0] - (double)a.ref[2 * pair]) - (s[1] - (double)a.ref[2 * pair + 1]));
    if (threadIdx.x == 0 && x == 0) {
        const double soft = log1p(exp(-fabs(h)));   // softplus(h) = soft + max(h, 0)
        a.loss[pair] = (float)((1.0 - (double)a.smooth) * (soft - fmin(h, 0.0)) + (double)a.smooth * (soft + fmax(h, 0.0)));
        a.seq_logp[2 * pair] = (float)s[0];
        a.seq_logp[2 * pair + 1] = (float)s[1];
    }
    if (!a.coef) return;
    const float g = (float)held_to_f32((double)a.scale * (double)a.beta * ((double)a.smooth - 1.0 / (1.0 + exp(h))));
    for (int q = 0; q < 2; q++)
        for (long long r = begin[q] + threadIdx.x; r < end[q]; r += 1024) a.coef[r] = q ? -g : g;
}
// Parts of a pair: 8192 rows each, where it has 32768 and more on average (all launches of the loss over f32 rows of 24, a workgroup to a pair and
// parts: 2 pairs of 16384 rows 19.1 us and 21.2, of 32768 21.7 and 21.2, 8 of 206081 154 and 101).
inline int64_t pair_parts(int64_t M, int64_t pairs) {
    const int64_t want = M / pairs < 32768 || pairs > 16384 ? 1 : ceil_div(M, pairs * 8192);   // (2 pairs go into a grid's second dimension)
    return want < 256 ? want : 256;
}
inline bool is_dt(int dt) { return dt == EMADAPT_DT_F32 || dt == EMADAPT_DT_BF16; }
inline size_t dt_size(int dt) { return dt == EMADAPT_DT_BF16 ? 2 : 4; }
inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}
inline unsigned grid_of(int64_t n, int64_t cap) { return (unsigned)(n < 1 ? 1 : (n < cap ? n : cap)); }

// what every entry asks of the rows; `grad` may be null
int check_rows(const void *logits, int dtype, int64_t ldl, const int64_t *labels, int64_t M, int64_t C, const void *grad, int grad_dtype) {
    if (!is_dt(dtype) || (grad && !is_dt(grad_dtype)) || M < 0 || C <= 0 || ldl < C) return EMADAPT_ERR_INVALID;
    if (ldl > (int64_t)1 << 30 || M > ((int64_t)1 << 48) / ldl) return EMADAPT_ERR_UNSUPPORTED;
    // (a grid has fewer than 2^32 threads, of which each writes the gradient of at most four vectors, in whole workgroups to each of a few rows)
    if (grad && M * ceil_div(ldl, 16 / (int64_t)dt_size(dtype)) > ((int64_t)1 << 34) - (1 << 20)) return EMADAPT_ERR_UNSUPPORTED;
    if (M == 0) return EMADAPT_OK;
    if (!logits || !labels || !aligned(logits, dt_size(dtype)) || !aligned(labels, 8) || (grad && !aligned(grad, dt_size(grad_dtype)))) return EMADAPT_ERR_INVALID;
    // (the rows are read again after other rows' gradients are written)
    if (grad && overlap(logits, (size_t)M * ldl * dt_size(dtype), grad, (size_t)M * ldl * dt_size(grad_dtype))) return EMADAPT_ERR_INVALID;
    return EMADAPT_OK;
}
constexpr double kCache = 256e6;   // bytes of the last cache before the memory
Rows rows_of(const void *logits, int64_t ldl, const int64_t *labels, int64_t M, int64_t C, size_t grad_size = 0) {
    return Rows{logits, reinterpret_cast<const long long *>(labels), (long long)ldl, (long long)M, (int)C, (double)M * ldl * grad_size > kCache / 4, false};
}

// Rows of up to 64 vectors, three or four of them to a lane; up to 8 where that still beats a workgroup to a row.  False: longer rows.
//   statistics  512 vectors (200 M bf16, rows of 520: 105 us against 375; of 4096: 68 against 84), 384 where nothing is left in the cache (of 4000:
//               117 against 88)
//   gradient    384 vectors (rows of 520: 278 us against 688, of 2047 217 against 282, of 2900 204 against 208, of 4000 230 against 170)
//   loss alone  16 vectors, behind them statistics and rows' terms in two launches (f32 rows of 24: 52 us against 75 for 1.6 M, of 64: 106 against
//               121, of 130: 135 against 114)
template <int MODE, typename T, typename TD>
bool launch_short(const Rows &a, const Policy &p, Outputs out, int cap, int *blocks, hipStream_t stream) {
    const int64_t nvec = ceil_div(a.ldl, Vec<T>::N);
    if (nvec > (MODE == kLogp ? (a.last ? 384 : 512) : MODE == kPolicyGrad ? 384 : 16)) return false;
    int L = 1;
    while (L * 4 < nvec && L < 64) L *= 2;
    const bool three = nvec <= 3 * L;
    *blocks = (int)grid_of(ceil_div(a.M, 256 / L), cap);
    if (MODE != kLogp && L <= kInlineLanes && a.M <= 1024 / L) *blocks = 1;   // (its sums are the whole ones, a launch less: 500 rows of 24 f32 16.6 us and 13.3)
    if (*blocks > 1 || L > kInlineLanes) out.sums = nullptr;
#define EMADAPT_GROUP(L, NV) hipLaunchKernelGGL((group_kernel<T, TD, L, NV, MODE>), dim3(*blocks), dim3(256), 0, stream, a, p, out)
    switch (L) {
        case 1: if (three) EMADAPT_GROUP(1, 3); else EMADAPT_GROUP(1, 4); break;
        case 2: if (three) EMADAPT_GROUP(2, 3); else EMADAPT_GROUP(2, 4); break;
        case 4: if (three) EMADAPT_GROUP(4, 3); else EMADAPT_GROUP(4, 4); break;
    }
    if constexpr (MODE != kPolicy) switch (L) {
        case 8: if (three) EMADAPT_GROUP(8, 3); else EMADAPT_GROUP(8, 4); break;
        case 16: if (three) EMADAPT_GROUP(16, 3); else EMADAPT_GROUP(16, 4); break;
        case 32: if (three) EMADAPT_GROUP(32, 3); else EMADAPT_GROUP(32, 4); break;
        case 64:
            if (three) EMADAPT_GROUP(64, 3);
            else if (nvec <= 256) EMADAPT_GROUP(64, 4);
            else if (nvec <= 384) EMADAPT_GROUP(64, 6);
            else if constexpr (MODE == kLogp) EMADAPT_GROUP(64, 8);
    }
#undef EMADAPT_GROUP
    return true;
}
// Rows of up to 16384 vectors in the registers of a workgroup.
template <typename T, typename TD>
bool launch_block(const Rows &a, const Policy &p, const Outputs &out, int cap, int *blocks, hipStream_t stream) {
    const int64_t nvec = a.C / Vec<T>::N;
    if (nvec < 1 || nvec > 16384) return false;   // (a thread without a vector of its own loads the row's last whole one: there has to be one)
    *blocks = (int)grid_of(a.M, cap);
    const dim3 grid(*blocks);
#define EMADAPT_BLOCK(W, NV) hipLaunchKernelGGL((block_kernel<T, TD, W, NV>), grid, dim3(64 * W), 0, stream, a, p, out)
    if (nvec <= 512) EMADAPT_BLOCK(1, 8);
    else if (nvec <= 1024) EMADAPT_BLOCK(1, 16);
    else if (nvec <= 2048) EMADAPT_BLOCK(2, 16);
    else if (nvec <= 4096) EMADAPT_BLOCK(4, 16);
    else if (nvec <= 8192) EMADAPT_BLOCK(8, 16);
    else EMADAPT_BLOCK(16, 16);
#undef EMADAPT_BLOCK
    return true;
}
// Waves to a row: 16 where the row fills a round of their loads, enough in flight for a CU's share of the memory's rate (bf16, with 4 waves and with
// 16: 4000 x 27000 33.7 and 38.8 us, 4001 x 32768 with the gradient behind it 126.6 and 122.5, 2000 x 65536 42.6 and 39.9).
template <typename T> int stats_width(int C) { return C < 16 * 64 * 4 * Vec<T>::N ? 4 : 16; }
// again: the rows are read once more afterwards
template <typename T>
int launch_stats_t(Rows a, const Outputs &out, int splits, bool again, hipStream_t stream) {
    int blocks;
    a.last = !again;
    if (splits > 1 || !launch_short<kLogp, T, T>(a, Policy(), out, 1 << 16, &blocks, stream)) {
        const dim3 grid(grid_of(a.M, 1 << 16), splits);
        const bool narrow = splits > 1 || stats_width<T>(a.C) == 4;
        if (narrow && again) hipLaunchKernelGGL((stream_stats_kernel<T, 4, false>), grid, dim3(256), 0, stream, a, out);
        else if (narrow) hipLaunchKernelGGL((stream_stats_kernel<T, 4, true>), grid, dim3(256), 0, stream, a, out);
        else if (again) hipLaunchKernelGGL((stream_stats_kernel<T, 16, false>), grid, dim3(1024), 0, stream, a, out);
        else hipLaunchKernelGGL((stream_stats_kernel<T, 16, true>), grid, dim3(1024), 0, stream, a, out);
    }
    return launch_status();
}
int launch_stats(const Rows &a, int dtype, const Outputs &out, bool again, hipStream_t stream) {
    return dtype == EMADAPT_DT_BF16 ? launch_stats_t<__bf16>(a, out, 1, again, stream) : launch_stats_t<float>(a, out, 1, again, stream);
}
template <typename T>
int launch_grad_t(const Rows &a, const float *base, const float *sum, const float *coef, void *d, int ddt, hipStream_t stream) {
    const int64_t nvec = ceil_div(a.ldl, Vec<T>::N), total = nvec * a.M;
    // four vectors to a thread, or one where that leaves CUs without a workgroup (40344 rows of 24 f32: 7.7 us and 4.1)
    const bool four = total >= 4 * 256 * 1024;
    const int64_t blocks = ceil_div(total, four ? 1024 : 256);   // (check_rows: not more threads than a grid has)
#define EMADAPT_GRAD(TD, U, SUM) \
    hipLaunchKernelGGL((row_grad_kernel<T, TD, U, SUM>), dim3((unsigned)blocks), dim3(256), 0, stream, a, base, sum, coef, static_cast<TD *>(d), (unsigned)nvec, (long long)total)
#define EMADAPT_GRAD_OF(SUM)                                             \
    if (ddt == EMADAPT_DT_BF16) {                                        \
        if (four) EMADAPT_GRAD(__bf16, 4, SUM); else EMADAPT_GRAD(__bf16, 1, SUM); \
    } else {                                                             \
        if (four) EMADAPT_GRAD(float, 4, SUM); else EMADAPT_GRAD(float, 1, SUM);   \
    }
    if (sum) {
        EMADAPT_GRAD_OF(true)
    } else {
        EMADAPT_GRAD_OF(false)
    }
#undef EMADAPT_GRAD_OF
#undef EMADAPT_GRAD
    return launch_status();
}
int launch_grad(const Rows &a, int dtype, const float *base, const float *sum, const float *coef, void *d, int ddt, hipStream_t stream) {
    return dtype == EMADAPT_DT_BF16 ? launch_grad_t<__bf16>(a, base, sum, coef, d, ddt, stream) : launch_grad_t<float>(a, base, sum, coef, d, ddt, stream);
}
constexpr int kPolicyBlocks = 2048, kFinishBlocks = 512;

// Where the policy loss keeps what its launches hand on.
struct PolicySpace {
    float *base, *sum, *coef;   // [M] each
    MaxSum *parts;              // [kFewRows][kSplits]
    double *partial, *fixed;    // [kPolicyBlocks][4], [kFinishBlocks][4]
    unsigned *ticket;
    unsigned char *near;        // [M]
    size_t bytes;
};
constexpr int64_t kFewRows = 128;   // (33000 bf16: 128 rows 16.3 us in parts, 17 with a workgroup to a row; 192 rows 22.7 and 15.6)
PolicySpace policy_space(void *workspace, int64_t M) {
    PolicySpace s;
    size_t at = 0;
    auto take = [&](size_t n) {
        char *p = static_cast<char *>(workspace) + at;
        at += align_up(n, 256);
        return p;
    };
    s.base = reinterpret_cast<float *>(take((size_t)M * 12));
    s.sum = s.base + M;
    s.coef = s.sum + M;
    s.parts = reinterpret_cast<MaxSum *>(take(kFewRows * kSplits * sizeof(MaxSum)));
    s.partial = reinterpret_cast<double *>(take((size_t)kPolicyBlocks * 32));
    s.fixed = reinterpret_cast<double *>(take((size_t)kFinishBlocks * 32));
    s.ticket = reinterpret_cast<unsigned *>(take(4));
    s.near = reinterpret_cast<unsigned char *>(take((size_t)M + 16));   // (looked at 16 at a time)
    s.bytes = at;
    return s;
}

template <typename T, typename TD>
int launch_few(const Rows &a, const Policy &p, const MaxSum *parts, float *logp, float *sums, TD *d, hipStream_t stream) {
    const int64_t nvec = ceil_div(a.ldl, Vec<T>::N);
    const bool four = nvec * a.M >= 4 * 256 * 1024;   // (as in launch_grad_t)
    const unsigned per = (unsigned)ceil_div(nvec, four ? 1024 : 256), blocks = d ? 1 + (unsigned)a.M * per : 1;
    if (four) hipLaunchKernelGGL((policy_few_kernel<T, TD, 4>), dim3(blocks), dim3(256), 0, stream, a, p, parts, logp, sums, d, per);
    else hipLaunchKernelGGL((policy_few_kernel<T, TD, 1>), dim3(blocks), dim3(256), 0, stream, a, p, parts, logp, sums, d, per);
    return launch_status();
}

template <typename T, typename TD>
int policy_t(Rows a, Policy p, float *sums, float *logp, void *dlogits, int ddt, void *workspace, hipStream_t stream) {
    const PolicySpace w = policy_space(workspace, a.M);
    Outputs out = {logp, nullptr, nullptr, nullptr, nullptr, dlogits, w.partial, nullptr, w.ticket, nullptr, sums};
    int blocks = 0;
    unsigned finish = 1;
    if (a.M) {
        const int64_t nvec = a.C / Vec<T>::N;
        const bool few = a.M <= kFewRows && nvec > 4096;   // (a CU to a row leaves the others idle)
        bool done;
        a.last = a.once;
        p.tol = border_tol(16, (int)a.C);   // (short rows: none; a row in registers: 16 vectors to a thread)
        out.near = w.near;
        out.base = w.base;
        if (!dlogits) done = launch_short<kPolicy, T, T>(a, p, out, kPolicyBlocks, &blocks, stream);
        else {
            done = launch_short<kPolicyGrad, T, TD>(a, p, out, kPolicyBlocks, &blocks, stream);
            if (!done && !few) done = launch_block<T, TD>(a, p, out, kPolicyBlocks, &blocks, stream);
        }
        const bool in_place = done && ceil_div(a.ldl, Vec<T>::N) <= kInlineLanes * 4;
        if (in_place && blocks == 1) return launch_status();
        if (done && !in_place) finish = grid_of(ceil_div(a.M, kFinishRows), kFinishBlocks);
        else out.near = nullptr;
        if (int rc = launch_status()) return rc;
        if (!done) {   // rows that no workgroup's registers hold, that are only read, or too few: log-sum-exp, the rows' terms, the gradient
            Outputs st = {};
            p.tol = border_tol((int)ceil_div(a.C, few ? kSplits * 256 * Vec<T>::N : stats_width<T>(a.C) * 64 * Vec<T>::N) + (few ? kSplits : 0), (int)a.C);
            if (few) st.parts = w.parts;
            else { st.base = w.base; st.sum = w.sum; }
            if (int rc = launch_stats_t<T>(a, st, few ? kSplits : 1, dlogits != nullptr, stream)) return rc;
            if (few) return launch_few<T, TD>(a, p, w.parts, logp, sums, static_cast<TD *>(dlogits), stream);
            blocks = (int)grid_of(ceil_div(a.M, 256), kPolicyBlocks);
            hipLaunchKernelGGL(policy_row_kernel<T>, dim3(blocks), dim3(256), 0, stream, a, p, w.base, w.sum, logp, w.coef, w.partial, sums);
            if (int rc = launch_status()) return rc;
            if (dlogits)
                if (int rc = launch_grad_t<T>(a, w.base, w.sum, w.coef, dlogits, ddt, stream)) return rc;
            if (blocks == 1) return EMADAPT_OK;
        }
    }
    hipLaunchKernelGGL((policy_finish_kernel<T, TD>), dim3(finish), dim3(1024), 0, stream, a, p, out, blocks, w.fixed, sums);
    return launch_status();
}
template <typename T>
int policy_any(const Rows &a, const Policy &p, float *sums, float *logp, void *dlogits, int ddt, void *workspace, hipStream_t stream) {
    return ddt == EMADAPT_DT_BF16 ? policy_t<T, __bf16>(a, p, sums, logp, dlogits, ddt, workspace, stream) : policy_t<T, float>(a, p, sums, logp, dlogits, ddt, workspace, stream);
}

}  // namespace

extern "C" {

int emadapt_label_logp(const void *logits, int dtype, int64_t ldl, const int64_t *labels, int64_t M, int64_t C, float *logp, float *lse, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, nullptr, 0)) return rc;
    if (M == 0) return EMADAPT_OK;
    if (!logp && !lse) return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + 16.0), stream);
    // (whether a gradient follows is not known here: of up to twice the cache a second reader still finds a good part -- 4001 x 32768 bf16 with
    // the gradient 123 us, 140 where the first reader leaves nothing; 1500 x 100003 f32 alone 100 and 92)
    const bool again = (double)M * C * dt_size(dtype) < 2 * kCache;
    return launch_stats(rows_of(logits, ldl, labels, M, C), dtype, Outputs{logp, lse}, again, stream);
}

int emadapt_label_logp_bwd(const void *logits, int dtype, int64_t ldl, const int64_t *labels, const float *lse, const float *dlogp, int64_t M, int64_t C,
                           void *dlogits, int dlogits_dtype, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, dlogits, dlogits_dtype)) return rc;
    if (M == 0) return EMADAPT_OK;
    if (!lse || !dlogp || !dlogits) return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + (double)ldl * dt_size(dlogits_dtype) + 16.0), stream);
    return launch_grad(rows_of(logits, ldl, labels, M, C, dt_size(dlogits_dtype)), dtype, lse, nullptr, dlogp, dlogits, dlogits_dtype, stream);
}

size_t emadapt_policy_loss_workspace_bytes(int64_t M, int64_t C) {
    (void)C;
    return policy_space(nullptr, M > 0 ? M : 0).bytes;
}

int emadapt_policy_loss(const void *logits, int dtype, int64_t ldl, const int64_t *actions, const float *old_logp, const float *ref_logp, const float *advantages,
                        const float *weights, int64_t M, int64_t C, double clip_low, double clip_high, float kl_coef, float grad_scale, float *sums, float *logp,
                        void *dlogits, int dlogits_dtype, void *workspace, size_t workspace_bytes, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, actions, M, C, dlogits, dlogits_dtype)) return rc;
    if (!sums || !(clip_low >= 0.0 && clip_low <= 1.0) || !(clip_high >= 0.0) || !isfinite(kl_coef) || !isfinite(grad_scale)) return EMADAPT_ERR_INVALID;
    if (M && (!old_logp || !advantages || !logp)) return EMADAPT_ERR_INVALID;
    if (!workspace || !aligned(workspace, 8) || workspace_bytes < emadapt_policy_loss_workspace_bytes(M, C)) return EMADAPT_ERR_WORKSPACE;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + (dlogits ? (double)ldl * dt_size(dlogits_dtype) : 0.0) + 28.0), stream);
    const Rows a = rows_of(logits, ldl, actions, M, C, dt_size(dlogits_dtype));
    const Policy p = {old_logp, ref_logp, advantages, weights, 1.0 - clip_low, 1.0 + clip_high, log1p(-clip_low), log1p(clip_high), kl_coef, grad_scale, 0.f};
    return dtype == EMADAPT_DT_BF16 ? policy_any<__bf16>(a, p, sums, logp, dlogits, dlogits_dtype, workspace, stream)
                                    : policy_any<float>(a, p, sums, logp, dlogits, dlogits_dtype, workspace, stream);
}

size_t emadapt_preference_loss_workspace_bytes(int64_t M, int64_t C) {
    (void)C;
    // (four floats a row; parts of long pairs: at most M / 8192 + pairs of them, pairs <= M / 32768, two sums each)
    const size_t rows = M > 0 ? (size_t)M : 1;
    return align_up(rows * 16, 256) + rows / 8192 * 24 + 64;
}

int emadapt_preference_loss(const void *logits, int dtype, int64_t ldl, const int64_t *labels, const int64_t *seq_start, int64_t pairs, const float *ref_logp,
                            int64_t M, int64_t C, float beta, float label_smoothing, float grad_scale, float *loss, float *seq_logp, void *dlogits,
                            int dlogits_dtype, void *workspace, size_t workspace_bytes, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, dlogits, dlogits_dtype)) return rc;
    if (pairs < 0 || !(label_smoothing >= 0.f && label_smoothing <= 1.f) || !isfinite(beta) || !isfinite(grad_scale)) return EMADAPT_ERR_INVALID;
    if (pairs > 0x7FFFFFFF) return EMADAPT_ERR_UNSUPPORTED;
    if (pairs && (!seq_start || !aligned(seq_start, 8) || !ref_logp || !loss || !seq_logp)) return EMADAPT_ERR_INVALID;
    if (M && (!workspace || !aligned(workspace, 8) || workspace_bytes < emadapt_preference_loss_workspace_bytes(M, C))) return EMADAPT_ERR_WORKSPACE;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * (2.0 * C * dt_size(dtype) + (dlogits ? (double)ldl * dt_size(dlogits_dtype) : 0.0) + 24.0), stream);
    float *logp = static_cast<float *>(workspace), *base = logp + M, *sum = base + M, *coef = sum + M;
    const Rows a = rows_of(logits, ldl, labels, M, C, dt_size(dlogits_dtype));
    if (M)   // (rows of no sequence have no gradient: their coefficient starts at 0)
        if (int rc = launch_stats(a, dtype, Outputs{logp, nullptr, dlogits ? base : nullptr, sum, dlogits ? coef : nullptr}, dlogits != nullptr, stream)) return rc;
    if (pairs) {
        const Preference p = {logp, reinterpret_cast<const long long *>(seq_start), ref_logp, (long long)M, beta, label_smoothing, grad_scale, loss, seq_logp,
                              dlogits ? coef : nullptr, reinterpret_cast<double *>(static_cast<char *>(workspace) + align_up((size_t)M * 16, 256))};
        const int64_t parts = pair_parts(M, pairs);
        if (parts > 1) {
            hipLaunchKernelGGL(preference_part_kernel, dim3((unsigned)parts, (unsigned)(2 * pairs)), dim3(1024), 0, stream, p);
            hipLaunchKernelGGL(preference_pair_kernel<true>, dim3((unsigned)parts, (unsigned)pairs), dim3(1024), 0, stream, p);
        } else {
            constexpr int64_t kMost = 0xFFFFFFFFll / 1024;   // (a grid has fewer than 2^32 threads)
            for (int64_t at = 0; at < pairs; at += kMost) {
                Preference some = p;
                some.seq_start += 2 * at;
                some.ref += 2 * at;
                some.loss += at;
                some.seq_logp += 2 * at;
                hipLaunchKernelGGL(preference_pair_kernel<false>, dim3((unsigned)(pairs - at < kMost ? pairs - at : kMost)), dim3(1024), 0, stream, some);
            }
        }
        if (int rc = launch_status()) return rc;
    }
    if (M && dlogits) return launch_grad(a, dtype, base, sum, coef, dlogits, dlogits_dtype, stream);
    return EMADAPT_OK;
}

}  // extern "C"
