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
template <typename T> __device__ __forceinline__ Raw pack_raw(const T (&t)[Vec<T>::N]) {
    Raw r;
    __builtin_memcpy(&r, t, 16);
    return r;
}
// Vector at element i of a row of C elements (ldl with the padding); what is not one of the C is -inf: no weight in any sum of exponentials.
template <typename T> __device__ __forceinline__ Raw load_row(const T *z, int i, int C, int ldl) {
    constexpr int N = Vec<T>::N;
    T t[N];
    if (i + N <= C) {
        Raw r;
        __builtin_memcpy(&r, z + i, 16);
        return r;
    }
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
template <typename T, int N> __device__ __forceinline__ void store_row(T *d, int i, int ldl, const float (&v)[N]) {
    T t[N];
#pragma unroll
    for (int k = 0; k < N; k++) t[k] = (T)v[k];
    if (i + N <= ldl) __builtin_memcpy(d + i, t, sizeof(t));
    else {
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
struct Rows {
    const void *logits;
    const long long *labels;
    long long ldl, M;
    int C;
};

// dz = [c = label] coef - exp(z - base) coef / sum (base, sum: the row's maximum and sum; without sum the log-sum-exp): every thread its vectors of the flattened [M][vectors per row], kUnroll of them in flight.  A
// workgroup's vectors lie behind one another; their rows come from one 64-bit division for the workgroup and a 32-bit one for each vector.
constexpr int kUnroll = 4;
template <typename T, typename TD>
__global__ void __launch_bounds__(256) row_grad_kernel(Rows a, const float *__restrict__ base, const float *__restrict__ sum, const float *__restrict__ coef, TD *__restrict__ dlogits,
                                                      unsigned nvec, long long total) {
    constexpr int N = Vec<T>::N;
    const long long b = (long long)(gridDim.x - 1 - blockIdx.x) * (256 * kUnroll);   // (the rows that were read last come first: some are still in the cache)
    const long long r0 = b / nvec;
    const unsigned i0 = (unsigned)(b - r0 * nvec);
    Raw raw[kUnroll];
    long long row[kUnroll];
    int at[kUnroll], hit[kUnroll];
    float l[kUnroll], f[kUnroll], fs[kUnroll];
#pragma unroll
    for (int q = 0; q < kUnroll; q++) {
        const unsigned o = i0 + q * 256 + threadIdx.x, dr = o / nvec;
        row[q] = b + q * 256 + threadIdx.x < total ? r0 + dr : -1;
        if (row[q] < 0) continue;
        at[q] = (int)(o - dr * nvec) * N;
        raw[q] = load_row(static_cast<const T *>(a.logits) + row[q] * a.ldl, at[q], a.C, (int)a.ldl);
        const long long lab = a.labels[row[q]];
        const bool used = lab >= 0 && lab < a.C;
        hit[q] = used ? (int)lab : -(1 << 30);
        l[q] = base[row[q]];
        f[q] = used ? coef[row[q]] : 0.f;
        fs[q] = sum ? f[q] * __builtin_amdgcn_rcpf(sum[row[q]]) : f[q];
    }
#pragma unroll
    for (int q = 0; q < kUnroll; q++) {
        if (row[q] < 0) continue;
        float v[N];
        grad_vec<T>(raw[q], l[q], fs[q], f[q], hit[q] - at[q], v);
        if (f[q] == 0.f) {   // (a row that takes no part: 0, also where 0 * NaN is not)
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = 0.f;
        }
        store_row<TD>(dlogits + row[q] * a.ldl, at[q], (int)a.ldl, v);
    }
}

// ------------------------------------------------------------------------------------------
// the clipped policy loss
// ------------------------------------------------------------------------------------------
struct Policy {
    const float *old_logp, *ref_logp, *adv, *weight;
    double low, high;   // the ratio's borders, 1 - clip_low and 1 + clip_high
    double log_low, log_high;
    float kl, scale;
};
struct PolicyTerms {
    double loss, surrogate, kl, clipped;
};

// exp(q) - 1 to a few roundings of itself: by its series where the subtraction would lose bits (q^9 / 9! is below 2^-24 q for |q| < 0.6)
__device__ __forceinline__ float exp_minus_1(float q) {
    const float series = q * (1.f + q * (1.f / 2 + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720 + q * (1.f / 5040 + q * (1.f / 40320))))))));
    return fabsf(q) < 0.5f ? series : __expf(q) - 1.f;
}
// d loss / d logp of one row, and (count) what it adds to the sums.
__device__ __forceinline__ float policy_row(float log_ratio, float q, bool has_ref, float adv, float w, const Policy &p, bool clipped, bool count,
                                            PolicyTerms &t) {
    const float free = -adv * __expf(log_ratio);
    const float e = has_ref ? exp_minus_1(q) : 0.f;
    if (count) {
        const float part = clipped ? -adv * (float)(adv > 0.f ? p.high : p.low) : free;
        // exp(q) - 1 - q: from q^2 / 2 on where the rest cancels
        const float k = !has_ref ? 0.f
                        : fabsf(q) < 0.5f ? q * q * (1.f / 2 + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720 + q * (1.f / 5040 + q * (1.f / 40320)))))))
                                          : e - q;
        t.loss += (double)w * (double)(part + p.kl * k);
        t.surrogate += (double)w * (double)part;
        t.kl += (double)w * (double)k;
        t.clipped += clipped ? (double)w : 0.0;
    }
    return w * p.scale * ((clipped ? 0.f : free) - p.kl * e);
}
// is the log of the ratio past the border that its advantage's sign puts up?
__device__ __forceinline__ bool past_border(double log_ratio, float adv, const Policy &p) {
    return adv > 0.f ? log_ratio > p.log_high : (adv < 0.f ? log_ratio < p.log_low : false);
}
// f32's log ratio is off by less than this: rounding of the sum over a row (at most 2^-15 of it), of exponents and of the differences
__device__ __forceinline__ bool near_border(float log_ratio, float magnitude, float adv, const Policy &p) {
    const float tol = 1e-4f + 4.8e-7f * magnitude;
    const float border = adv > 0.f ? (float)p.log_high : (float)p.log_low;
    return adv != 0.f && fabsf(log_ratio - border) < tol;
}
// sum over elements `first`, first + step, .. of the row of exp(z - z_label) in 64 bits
template <typename T>
__device__ double exact_part(const T *z, int C, long long lab, int first, int step) {
    const double at = (double)(float)z[lab];
    double s = 0.0;
#pragma unroll 1
    for (int i = first; i < C; i += step) s += exp((double)(float)z[i] - at);
    return s;
}

// ------------------------------------------------------------------------------------------
// rows that stay in registers: one pass over the logits
// ------------------------------------------------------------------------------------------
enum { kLogp = 0, kPolicy = 1, kPolicyGrad = 2 };
struct Outputs {
    float *logp, *lse;          // kLogp: any of these may be null
    float *base, *sum, *zero;   // kLogp: the rows' maximum and sum of exponentials; a value per row set to 0
    void *dlogits;
    double *partial;            // [gridDim.x][4]
};

// A row's part of the policy loss once its log-sum-exp is known.  The ratio is cut where exact arithmetic on the inputs cuts it: for a row near
// a border `exact` gives logp in 64 bits.  The sums are taken by one thread of the row's (count).
template <typename E>
__device__ __forceinline__ float policy_of_row(const Policy &p, long long r, float z, MaxSum row, bool count, E exact, float &lp, PolicyTerms &t) {
    const float oldp = p.old_logp[r], adv = p.adv[r], w = p.weight ? p.weight[r] : 1.f, refp = p.ref_logp ? p.ref_logp[r] : 0.f;
    const float log_sum = logf(row.s);
    lp = (z - row.m) - log_sum;
    float lr = lp - oldp;
    bool clipped = past_border(lr, adv, p);
    if (near_border(lr, fabsf(z - row.m) + log_sum + fabsf(oldp), adv, p)) {
        const double lp64 = exact();
        lp = (float)lp64;
        lr = (float)(lp64 - (double)oldp);
        clipped = past_border(lp64 - (double)oldp, adv, p);
    }
    return policy_row(lr, refp - lp, p.ref_logp != nullptr, adv, w, p, clipped, count, t);
}

// L lanes to a row, a vector of the padded row to a lane.
template <typename T, typename TD, int L, int MODE>
__global__ void __launch_bounds__(256) group_kernel(Rows a, Policy p, Outputs out) {
    constexpr int N = Vec<T>::N;
    __shared__ double sh[4];
    const int lane = threadIdx.x % L;
    const long long per_grid = (long long)gridDim.x * (256 / L);
    PolicyTerms t = {0, 0, 0, 0};
    for (long long r = (long long)blockIdx.x * (256 / L) + threadIdx.x / L; r < a.M; r += per_grid) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        const long long lab = a.labels[r];
        bool used = lab >= 0 && lab < a.C;
        if (MODE != kLogp && p.weight) used = used && p.weight[r] != 0.f;
        const int i = lane * N;
        const Raw raw = load_row(z, i, a.C, (int)a.ldl);
        float v[N], m = -INFINITY, s = 0.f;
        unpack<T>(raw, v);
#pragma unroll
        for (int e = 0; e < N; e++) m = fmaxf(m, v[e]);
        m = group_max<L>(m);
        const float m0 = finite_or_0(m);
#pragma unroll
        for (int e = 0; e < N; e++) s += __expf(v[e] - m0);
        s = group_sum<L>(s);
        float lp = 0.f, f = 0.f;
        if (used) {
            const float zl = (float)z[lab];
            if (MODE == kLogp) lp = (zl - m) - logf(s);
            else
                f = policy_of_row(p, r, zl, MaxSum{m, s}, lane == 0, [&] {
                    double e = exact_part(z, a.C, lab, lane, L);
                    for (int o = L / 2; o > 0; o >>= 1) e += __shfl_xor(e, o);
                    return -log(e);
                }, lp, t);
        }
        if (lane == 0) {
            if (MODE != kLogp || out.logp) out.logp[r] = lp;
            if (MODE == kLogp) {
                if (out.lse) out.lse[r] = m + logf(s);
                if (out.base) { out.base[r] = m; out.sum[r] = s; }
                if (out.zero) out.zero[r] = 0.f;
            }
        }
        if (MODE == kPolicyGrad && i < a.ldl) {
            grad_vec<T>(raw, m, f * __builtin_amdgcn_rcpf(s), f, used ? (int)lab - i : -1, v);
            if (f == 0.f) {
#pragma unroll
                for (int e = 0; e < N; e++) v[e] = 0.f;
            }
            store_row<TD>(static_cast<TD *>(out.dlogits) + r * a.ldl, i, (int)a.ldl, v);
        }
    }
    if (MODE != kLogp) {
        const double sum[4] = {t.loss, t.surrogate, t.kl, t.clipped};
        for (int k = 0; k < 4; k++) {
            const double v = block_sum_f64(sum[k], sh);
            if (threadIdx.x == 0) out.partial[(long long)blockIdx.x * 4 + k] = v;
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
    s *= __expf(m - m0);
#pragma unroll
    for (int e = 0; e < N; e++) s += __expf(v[e] - m0);
    m = top;
}

// A workgroup of W waves to a row, NV whole vectors to a thread, and the C % N last elements one to a thread.
template <typename T, typename TD, int W, int NV, int MODE>
__global__ void __launch_bounds__(64 * W) block_kernel(Rows a, Policy p, Outputs out) {
    constexpr int N = Vec<T>::N, kThreads = 64 * W;
    __shared__ MaxSum pair[2][W];
    __shared__ double sh[W];
    __shared__ PolicyTerms terms;   // (thread 0's: registers are short here)
    if (threadIdx.x == 0) terms = {0, 0, 0, 0};
    const int nfull = a.C / N, last = nfull * N + threadIdx.x;
    int turn = 0;
    for (long long r = blockIdx.x; r < a.M; r += gridDim.x, turn ^= 1) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        const long long lab = a.labels[r];
        bool used = lab >= 0 && lab < a.C;
        if (p.weight) used = used && p.weight[r] != 0.f;
        Raw raw[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int i = threadIdx.x + k * kThreads;
            if (i < nfull) __builtin_memcpy(&raw[k], z + i * N, 16);
        }
        float m = last < a.C ? (float)z[last] : -INFINITY;
        float s = last < a.C ? __expf(m - finite_or_0(m)) : 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++)
            if ((int)threadIdx.x + k * kThreads < nfull) {
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
        if (used) {   // (the same in every thread: the barriers inside are met by all)
            PolicyTerms one = {0, 0, 0, 0};
            f = policy_of_row(p, r, (float)z[lab], row, threadIdx.x == 0, [&] { return -log(block_sum_f64(exact_part(z, a.C, lab, threadIdx.x, kThreads), sh)); }, lp, one);
            if (threadIdx.x == 0) {
                terms.loss += one.loss; terms.surrogate += one.surrogate; terms.kl += one.kl; terms.clipped += one.clipped;
            }
        }
        if (threadIdx.x == 0) out.logp[r] = lp;
        TD *d = static_cast<TD *>(out.dlogits) + r * a.ldl;
        const int hit = used ? (int)lab : -(1 << 30);
        const float fs = f * __builtin_amdgcn_rcpf(row.s);
        for (int i = last; i < a.ldl; i += kThreads)   // the last elements and the padding
            d[i] = (TD)(f != 0.f && i < a.C ? (i == hit ? f : 0.f) - __expf((float)z[i] - row.m) * fs : 0.f);
        if (f == 0.f) {   // (a row that takes no part)
#pragma unroll 1
            for (int i = threadIdx.x; i < nfull; i += kThreads) {
                const float v[N] = {};
                store_row<TD>(d, i * N, nfull * N, v);
            }
            continue;
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int i = threadIdx.x + k * kThreads;
            if (i < nfull) {
                float v[N];
                grad_vec<T>(raw[k], row.m, fs, f, hit - i * N, v);
                store_row<TD>(d, i * N, nfull * N, v);
            }
        }
    }
    if (threadIdx.x == 0) {
        double *o = out.partial + (long long)blockIdx.x * 4;
        o[0] = terms.loss; o[1] = terms.surrogate; o[2] = terms.kl; o[3] = terms.clipped;
    }
}

// One workgroup to a row of any length, read once: a running maximum and sum for every thread, kAhead vectors in flight.
template <typename T, int W>
__global__ void __launch_bounds__(64 * W) stream_stats_kernel(Rows a, Outputs out) {
    constexpr int N = Vec<T>::N, kThreads = 64 * W, kAhead = 4;
    __shared__ MaxSum pair[2][W];
    int turn = 0;
    for (long long r = blockIdx.x; r < a.M; r += gridDim.x, turn ^= 1) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        const long long lab = a.labels[r];
        float m = -INFINITY, s = 0.f;
        for (int i0 = threadIdx.x * N; i0 < a.C; i0 += kThreads * N * kAhead) {
            Raw raw[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) raw[k] = load_row(z, i0 + k * kThreads * N, a.C, (int)a.ldl);
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                float v[N];
                unpack<T>(raw[k], v);
                take(v, m, s);
            }
        }
        const float mw = group_max<64>(m);
        s = group_sum<64>(s * __expf(m - finite_or_0(mw)));
        const MaxSum row = block_join<W>(MaxSum{mw, s}, pair[turn]);
        if (threadIdx.x == 0) {
            const float log_sum = logf(row.s);
            if (out.lse) out.lse[r] = row.m + log_sum;
            if (out.base) { out.base[r] = row.m; out.sum[r] = row.s; }
            if (out.logp) out.logp[r] = lab >= 0 && lab < a.C ? ((float)z[lab] - row.m) - log_sum : 0.f;
            if (out.zero) out.zero[r] = 0.f;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) policy_row_kernel(Rows a, Policy p, const float *__restrict__ base, const float *__restrict__ sum, float *__restrict__ logp, float *__restrict__ coef,
                                                        double *__restrict__ partial) {
    __shared__ double sh[4];
    __shared__ unsigned long long mask[4];
    PolicyTerms t = {0, 0, 0, 0};
    for (long long r0 = (long long)blockIdx.x * 256; r0 < a.M; r0 += (long long)gridDim.x * 256) {
        const long long r = r0 + threadIdx.x;
        bool again = false;
        if (r < a.M) {
            const long long lab = a.labels[r];
            const float w = p.weight ? p.weight[r] : 1.f;
            float lp = 0.f, f = 0.f;
            if (lab >= 0 && lab < a.C && w != 0.f) {
                const float z = (float)(static_cast<const T *>(a.logits) + r * a.ldl)[lab], m = base[r], log_sum = logf(sum[r]), oldp = p.old_logp[r], adv = p.adv[r];
                lp = (z - m) - log_sum;
                const float lr = lp - oldp;
                again = near_border(lr, fabsf(z - m) + log_sum + fabsf(oldp), adv, p);
                if (!again) f = policy_row(lr, p.ref_logp ? p.ref_logp[r] - lp : 0.f, p.ref_logp != nullptr, adv, w, p, past_border(lr, adv, p), true, t);
            }
            logp[r] = lp;
            coef[r] = f;
        }
        // rows near a border, in the order of their index
        const unsigned long long b = __ballot(again);
        if ((threadIdx.x & 63) == 0) mask[threadIdx.x >> 6] = b;
        __syncthreads();
        for (int q = 0; q < 4; q++)
            for (unsigned long long left = mask[q]; left; left &= left - 1) {
                const long long rr = r0 + q * 64 + (__ffsll((long long)left) - 1);
                const long long lab = a.labels[rr];
                const double lp = -log(block_sum_f64(exact_part(static_cast<const T *>(a.logits) + rr * a.ldl, a.C, lab, threadIdx.x, 256), sh));
                if (threadIdx.x == 0) {
                    const float adv = p.adv[rr], lpf = (float)lp;
                    const double lr = lp - (double)p.old_logp[rr];
                    logp[rr] = lpf;
                    coef[rr] = policy_row((float)lr, p.ref_logp ? p.ref_logp[rr] - lpf : 0.f, p.ref_logp != nullptr, adv, p.weight ? p.weight[rr] : 1.f, p,
                                          past_border(lr, adv, p), true, t);
                }
            }
        __syncthreads();
    }
    const double s[4] = {t.loss, t.surrogate, t.kl, t.clipped};
    for (int k = 0; k < 4; k++) {
        const double v = block_sum_f64(s[k], sh);
        if (threadIdx.x == 0) partial[(long long)blockIdx.x * 4 + k] = v;
    }
}

__global__ void __launch_bounds__(256) policy_sums_kernel(const double *__restrict__ partial, int n, float *__restrict__ sums) {
    __shared__ double sh[4];
    for (int k = 0; k < 4; k++) {
        double s = 0.0;
        for (int i = threadIdx.x; i < n; i += 256) s += partial[(long long)i * 4 + k];
        s = block_sum_f64(s, sh);
        if (threadIdx.x == 0) sums[k] = (float)s;
    }
}

// ------------------------------------------------------------------------------------------
// the preference loss: one workgroup to a pair of sequences
// ------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) preference_pair_kernel(const float *__restrict__ logp, const long long *__restrict__ seq_start, const float *__restrict__ ref,
                                                             long long M, float beta, float smooth, float scale, float *__restrict__ loss,
                                                             float *__restrict__ seq_logp, float *__restrict__ coef) {
    __shared__ double sh[16];
    const long long pair = blockIdx.x;
    long long at[3];
    for (int k = 0; k < 3; k++) {   // (a start outside the rows, or before the one in front of it, reads and writes nothing)
        const long long v = seq_start[2 * pair + k];
        at[k] = v < 0 ? 0 : (v > M ? M : v);
    }
    double s[2];
    for (int q = 0; q < 2; q++) {
        double v = 0.0;
        for (long long r = at[q] + threadIdx.x; r < at[q + 1]; r += 1024) v += (double)logp[r];
        s[q] = block_sum_f64(v, sh);
    }
    const double h = (double)beta * ((s[0] - (double)ref[2 * pair]) - (s[1] - (double)ref[2 * pair + 1]));
    const double soft = log1p(exp(-fabs(h)));   // softplus(h) = soft + max(h, 0)
    if (threadIdx.x == 0) {
        loss[pair] = (float)((1.0 - (double)smooth) * (soft - fmin(h, 0.0)) + (double)smooth * (soft + fmax(h, 0.0)));
        seq_logp[2 * pair] = (float)s[0];
        seq_logp[2 * pair + 1] = (float)s[1];
    }
    if (!coef) return;
    const float g = (float)((double)scale * (double)beta * ((double)smooth - 1.0 / (1.0 + exp(h))));
    for (int q = 0; q < 2; q++)
        for (long long r = at[q] + threadIdx.x; r < at[q + 1]; r += 1024) coef[r] = q ? -g : g;
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
    if (ldl > (int64_t)1 << 30 || M > (int64_t)1 << 40) return EMADAPT_ERR_UNSUPPORTED;
    if (M == 0) return EMADAPT_OK;
    if (!logits || !labels || !aligned(logits, dt_size(dtype)) || !aligned(labels, 8) || (grad && !aligned(grad, dt_size(grad_dtype)))) return EMADAPT_ERR_INVALID;
    // (the rows are read again after other rows' gradients are written)
    if (grad && overlap(logits, (size_t)M * ldl * dt_size(dtype), grad, (size_t)M * ldl * dt_size(grad_dtype))) return EMADAPT_ERR_INVALID;
    return EMADAPT_OK;
}
Rows rows_of(const void *logits, int64_t ldl, const int64_t *labels, int64_t M, int64_t C) {
    return Rows{logits, reinterpret_cast<const long long *>(labels), (long long)ldl, (long long)M, (int)C};
}

// Rows of up to 64 vectors: as many lanes as vectors.  false: longer rows.
template <int MODE, typename T, typename TD>
bool launch_short(const Rows &a, const Policy &p, const Outputs &out, int cap, int *blocks, hipStream_t stream) {
    const int64_t nvec = ceil_div(a.ldl, Vec<T>::N);
    if (nvec > 64) return false;
    int L = 1;
    while (L < nvec) L *= 2;
    *blocks = (int)grid_of(ceil_div(a.M, 256 / L), cap);
    const dim3 grid(*blocks), block(256);
    switch (L) {
        case 1: hipLaunchKernelGGL((group_kernel<T, TD, 1, MODE>), grid, block, 0, stream, a, p, out); break;
        case 2: hipLaunchKernelGGL((group_kernel<T, TD, 2, MODE>), grid, block, 0, stream, a, p, out); break;
        case 4: hipLaunchKernelGGL((group_kernel<T, TD, 4, MODE>), grid, block, 0, stream, a, p, out); break;
        case 8: hipLaunchKernelGGL((group_kernel<T, TD, 8, MODE>), grid, block, 0, stream, a, p, out); break;
        case 16: hipLaunchKernelGGL((group_kernel<T, TD, 16, MODE>), grid, block, 0, stream, a, p, out); break;
        case 32: hipLaunchKernelGGL((group_kernel<T, TD, 32, MODE>), grid, block, 0, stream, a, p, out); break;
        default: hipLaunchKernelGGL((group_kernel<T, TD, 64, MODE>), grid, block, 0, stream, a, p, out);
    }
    return true;
}
// Rows of up to 16384 vectors in the registers of a workgroup.
template <int MODE, typename T, typename TD>
bool launch_block(const Rows &a, const Policy &p, const Outputs &out, int cap, int *blocks, hipStream_t stream) {
    const int64_t nvec = a.C / Vec<T>::N;
    if (nvec > 16384) return false;
    *blocks = (int)grid_of(a.M, cap);
    const dim3 grid(*blocks);
    if (nvec <= 128) hipLaunchKernelGGL((block_kernel<T, TD, 1, 2, MODE>), grid, dim3(64), 0, stream, a, p, out);
    else if (nvec <= 256) hipLaunchKernelGGL((block_kernel<T, TD, 1, 4, MODE>), grid, dim3(64), 0, stream, a, p, out);
    else if (nvec <= 1024) hipLaunchKernelGGL((block_kernel<T, TD, 4, 4, MODE>), grid, dim3(256), 0, stream, a, p, out);
    else if (nvec <= 2048) hipLaunchKernelGGL((block_kernel<T, TD, 4, 8, MODE>), grid, dim3(256), 0, stream, a, p, out);
    else if (nvec <= 4096) hipLaunchKernelGGL((block_kernel<T, TD, 8, 8, MODE>), grid, dim3(512), 0, stream, a, p, out);
    else if (nvec <= 8192) hipLaunchKernelGGL((block_kernel<T, TD, 16, 8, MODE>), grid, dim3(1024), 0, stream, a, p, out);
    else hipLaunchKernelGGL((block_kernel<T, TD, 16, 16, MODE>), grid, dim3(1024), 0, stream, a, p, out);
    return true;
}
template <typename T>
int launch_stats_t(const Rows &a, const Outputs &out, hipStream_t stream) {
    int blocks;
    if (!launch_short<kLogp, T, T>(a, Policy(), out, 1 << 16, &blocks, stream)) {
        // a workgroup wide enough to hold what a CU's share of the memory's rate needs in flight
        const dim3 grid(grid_of(a.M, 1 << 16));
        if (a.C <= 16384) hipLaunchKernelGGL((stream_stats_kernel<T, 4>), grid, dim3(256), 0, stream, a, out);
        else hipLaunchKernelGGL((stream_stats_kernel<T, 16>), grid, dim3(1024), 0, stream, a, out);
    }
    return launch_status();
}
int launch_stats(const Rows &a, int dtype, const Outputs &out, hipStream_t stream) {
    return dtype == EMADAPT_DT_BF16 ? launch_stats_t<__bf16>(a, out, stream) : launch_stats_t<float>(a, out, stream);
}
template <typename T>
int launch_grad_t(const Rows &a, const float *base, const float *sum, const float *coef, void *d, int ddt, hipStream_t stream) {
    const int64_t nvec = ceil_div(a.ldl, Vec<T>::N), total = nvec * a.M, blocks = ceil_div(total, 256 * kUnroll);
    if (blocks > 0x7FFFFFFF) return EMADAPT_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks);
    if (ddt == EMADAPT_DT_BF16) hipLaunchKernelGGL((row_grad_kernel<T, __bf16>), grid, dim3(256), 0, stream, a, base, sum, coef, static_cast<__bf16 *>(d), (unsigned)nvec, (long long)total);
    else hipLaunchKernelGGL((row_grad_kernel<T, float>), grid, dim3(256), 0, stream, a, base, sum, coef, static_cast<float *>(d), (unsigned)nvec, (long long)total);
    return launch_status();
}
int launch_grad(const Rows &a, int dtype, const float *base, const float *sum, const float *coef, void *d, int ddt, hipStream_t stream) {
    return dtype == EMADAPT_DT_BF16 ? launch_grad_t<__bf16>(a, base, sum, coef, d, ddt, stream) : launch_grad_t<float>(a, base, sum, coef, d, ddt, stream);
}
constexpr int kPolicyBlocks = 2048;

template <typename T>
int policy_t(const Rows &a, const Policy &p, float *sums, float *logp, void *dlogits, int ddt, void *workspace, hipStream_t stream) {
    float *base = static_cast<float *>(workspace), *sum = base + a.M, *coef = sum + a.M;
    double *partial = reinterpret_cast<double *>(static_cast<char *>(workspace) + align_up((size_t)a.M * 12, 256));
    const Outputs out = {logp, nullptr, nullptr, nullptr, nullptr, dlogits, partial};
    int blocks = 0;
    if (a.M) {
        bool done;
        if (!dlogits) done = launch_short<kPolicy, T, T>(a, p, out, kPolicyBlocks, &blocks, stream);
        else if (ddt == EMADAPT_DT_BF16)
            done = launch_short<kPolicyGrad, T, __bf16>(a, p, out, kPolicyBlocks, &blocks, stream) || launch_block<kPolicyGrad, T, __bf16>(a, p, out, kPolicyBlocks, &blocks, stream);
        else
            done = launch_short<kPolicyGrad, T, float>(a, p, out, kPolicyBlocks, &blocks, stream) || launch_block<kPolicyGrad, T, float>(a, p, out, kPolicyBlocks, &blocks, stream);
        if (int rc = launch_status()) return rc;
        if (!done) {   // rows that no workgroup's registers hold, or that are only read: log-sum-exp, the rows' terms, the gradient
            if (int rc = launch_stats_t<T>(a, Outputs{nullptr, nullptr, base, sum, nullptr, nullptr, nullptr}, stream)) return rc;
            blocks = (int)grid_of(ceil_div(a.M, 256), kPolicyBlocks);
            hipLaunchKernelGGL(policy_row_kernel<T>, dim3(blocks), dim3(256), 0, stream, a, p, base, sum, logp, coef, partial);
            if (int rc = launch_status()) return rc;
            if (dlogits)
                if (int rc = launch_grad_t<T>(a, base, sum, coef, dlogits, ddt, stream)) return rc;
        }
    }
    hipLaunchKernelGGL(policy_sums_kernel, dim3(1), dim3(256), 0, stream, partial, blocks, sums);
    return launch_status();
}

}  // namespace

extern "C" {

size_t emadapt_label_logp_workspace_bytes(int64_t M, int64_t C) {
    (void)M; (void)C;
    return 0;
}

int emadapt_label_logp(const void *logits, int dtype, int64_t ldl, const int64_t *labels, int64_t M, int64_t C, float *logp, float *lse, void *workspace,
                       size_t workspace_bytes, void *stream_) {
    (void)workspace; (void)workspace_bytes;
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, nullptr, 0)) return rc;
    if (M == 0) return EMADAPT_OK;
    if (!logp && !lse) return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + 16.0), stream);
    return launch_stats(rows_of(logits, ldl, labels, M, C), dtype, Outputs{logp, lse, nullptr, nullptr, nullptr, nullptr, nullptr}, stream);
}

int emadapt_label_logp_bwd(const void *logits, int dtype, int64_t ldl, const int64_t *labels, const float *lse, const float *dlogp, int64_t M, int64_t C,
                           void *dlogits, int dlogits_dtype, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, dlogits, dlogits_dtype)) return rc;
    if (M == 0) return EMADAPT_OK;
    if (!lse || !dlogp || !dlogits) return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + (double)ldl * dt_size(dlogits_dtype) + 16.0), stream);
    return launch_grad(rows_of(logits, ldl, labels, M, C), dtype, lse, nullptr, dlogp, dlogits, dlogits_dtype, stream);
}

size_t emadapt_policy_loss_workspace_bytes(int64_t M, int64_t C) {
    (void)C;
    return align_up((size_t)(M > 0 ? M : 0) * 12, 256) + (size_t)kPolicyBlocks * 4 * sizeof(double);
}

int emadapt_policy_loss(const void *logits, int dtype, int64_t ldl, const int64_t *actions, const float *old_logp, const float *ref_logp, const float *advantages,
                        const float *weights, int64_t M, int64_t C, double clip_low, double clip_high, float kl_coef, float grad_scale, float *sums, float *logp,
                        void *dlogits, int dlogits_dtype, void *workspace, size_t workspace_bytes, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, actions, M, C, dlogits, dlogits_dtype)) return rc;
    if (!sums || !(clip_low >= 0.0 && clip_low <= 1.0) || !(clip_high >= 0.0)) return EMADAPT_ERR_INVALID;
    if (M && (!old_logp || !advantages || !logp)) return EMADAPT_ERR_INVALID;
    if (!workspace || !aligned(workspace, 8) || workspace_bytes < emadapt_policy_loss_workspace_bytes(M, C)) return EMADAPT_ERR_WORKSPACE;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + (dlogits ? (double)ldl * dt_size(dlogits_dtype) : 0.0) + 28.0), stream);
    const Rows a = rows_of(logits, ldl, actions, M, C);
    const Policy p = {old_logp, ref_logp, advantages, weights, 1.0 - clip_low, 1.0 + clip_high, log1p(-clip_low), log1p(clip_high), kl_coef, grad_scale};
    return dtype == EMADAPT_DT_BF16 ? policy_t<__bf16>(a, p, sums, logp, dlogits, dlogits_dtype, workspace, stream)
                                    : policy_t<float>(a, p, sums, logp, dlogits, dlogits_dtype, workspace, stream);
}

size_t emadapt_preference_loss_workspace_bytes(int64_t M, int64_t C) {
    (void)C;
    return (size_t)(M > 0 ? M : 1) * 16;
}

int emadapt_preference_loss(const void *logits, int dtype, int64_t ldl, const int64_t *labels, const int64_t *seq_start, int64_t pairs, const float *ref_logp,
                            int64_t M, int64_t C, float beta, float label_smoothing, float grad_scale, float *loss, float *seq_logp, void *dlogits,
                            int dlogits_dtype, void *workspace, size_t workspace_bytes, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, dlogits, dlogits_dtype)) return rc;
    if (pairs < 0 || !(label_smoothing >= 0.f && label_smoothing <= 1.f)) return EMADAPT_ERR_INVALID;
    if (pairs > 0x7FFFFFFF) return EMADAPT_ERR_UNSUPPORTED;
    if (pairs && (!seq_start || !aligned(seq_start, 8) || !ref_logp || !loss || !seq_logp)) return EMADAPT_ERR_INVALID;
    if (M && (!workspace || !aligned(workspace, 4) || workspace_bytes < emadapt_preference_loss_workspace_bytes(M, C))) return EMADAPT_ERR_WORKSPACE;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * (2.0 * C * dt_size(dtype) + (dlogits ? (double)ldl * dt_size(dlogits_dtype) : 0.0) + 24.0), stream);
    float *logp = static_cast<float *>(workspace), *base = logp + M, *sum = base + M, *coef = sum + M;
    const Rows a = rows_of(logits, ldl, labels, M, C);
    if (M)   // (rows of no sequence have no gradient: their coefficient starts at 0)
        if (int rc = launch_stats(a, dtype, Outputs{logp, nullptr, dlogits ? base : nullptr, sum, dlogits ? coef : nullptr, nullptr, nullptr}, stream)) return rc;
    if (pairs) {
        hipLaunchKernelGGL(preference_pair_kernel, dim3((unsigned)pairs), dim3(1024), 0, stream, logp, reinterpret_cast<const long long *>(seq_start), ref_logp, (long long)M,
                           beta, label_smoothing, grad_scale, loss, seq_logp, dlogits ? coef : nullptr);
        if (int rc = launch_status()) return rc;
    }
    if (M && dlogits) return launch_grad(a, dtype, base, sum, coef, dlogits, dlogits_dtype, stream);
    return EMADAPT_OK;
}

}  // extern "C"
