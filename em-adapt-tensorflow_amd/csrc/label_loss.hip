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

// 16 bytes of a row: any element alignment (gfx950 loads and stores dwordx4 at any address the element type allows).
template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T> __device__ __forceinline__ void load_vec(const T *p, float (&v)[Vec<T>::N]) {
    T t[Vec<T>::N];
    __builtin_memcpy(t, p, 16);
#pragma unroll
    for (int k = 0; k < Vec<T>::N; k++) v[k] = (float)t[k];
}
template <typename T, int N> __device__ __forceinline__ void store_vec(T *p, const float (&v)[N]) {
    T t[N];
#pragma unroll
    for (int k = 0; k < N; k++) t[k] = (T)v[k];
    __builtin_memcpy(p, t, sizeof(t));
}

// running maximum and sum of exponentials of a part of a row
struct MaxSum {
    float m, s;
};
__device__ __forceinline__ float exp_from(float z, float m) { return __expf(z - (m == -INFINITY ? 0.f : m)); }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
    MaxSum r;
    r.m = fmaxf(a.m, b.m);
    r.s = a.s * exp_from(a.m, r.m) + b.s * exp_from(b.m, r.m);
    return r;
}
__device__ __forceinline__ MaxSum wave_join(MaxSum v, int width) {
    for (int o = width / 2; o > 0; o >>= 1) {
        MaxSum b;
        b.m = __shfl_xor(v.m, o);
        b.s = __shfl_xor(v.s, o);
        v = join(v, b);
    }
    return v;
}
__device__ __forceinline__ MaxSum block_join(MaxSum v, MaxSum *sh) {
    v = wave_join(v, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    MaxSum r = sh[0];
    for (int k = 1; k < (int)(blockDim.x >> 6); k++) r = join(r, sh[k]);
    __syncthreads();
    return r;
}
__device__ __forceinline__ double block_sum_f64(double v, double *sh) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
    for (int k = 0; k < (int)(blockDim.x >> 6); k++) r += sh[k];
    __syncthreads();
    return r;
}

struct Rows {
    const void *logits;
    const long long *labels;
    long long ldl, M;
    int C;
};

// one workgroup to a row (grid-stride): log-sum-exp and the label's log-probability
template <typename T>
__global__ void __launch_bounds__(256) row_stats_kernel(Rows a, float *__restrict__ logp, float *__restrict__ lse) {
    __shared__ MaxSum sh[4];
    constexpr int N = Vec<T>::N;
    for (long long r = blockIdx.x; r < a.M; r += gridDim.x) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        MaxSum t = {-INFINITY, 0.f};
        for (int i = threadIdx.x * N; i < a.C; i += 256 * N) {
            if (i + N <= a.C) {
                float v[N];
                load_vec(z + i, v);
                float top = v[0];
#pragma unroll
                for (int k = 1; k < N; k++) top = fmaxf(top, v[k]);
                const float m = fmaxf(t.m, top);
                float s = t.s * exp_from(t.m, m);
#pragma unroll
                for (int k = 0; k < N; k++) s += exp_from(v[k], m);
                t = {m, s};
            } else
                for (int k = i; k < a.C; k++) t = join(t, MaxSum{(float)z[k], (float)z[k] == -INFINITY ? 0.f : 1.f});
        }
        t = block_join(t, sh);
        if (threadIdx.x == 0) {
            const float l = t.m + logf(t.s);
            const long long lab = a.labels[r];
            if (lse) lse[r] = l;
            if (logp) logp[r] = (lab >= 0 && lab < a.C) ? (float)z[lab] - l : 0.f;
        }
    }
}

// dz = ([c = label] - exp(z - lse)) coef, one workgroup to a row
template <typename T, typename TD>
__global__ void __launch_bounds__(256) row_grad_kernel(Rows a, const float *__restrict__ lse, const float *__restrict__ coef, TD *__restrict__ dlogits) {
    constexpr int N = Vec<T>::N;
    for (long long r = blockIdx.x; r < a.M; r += gridDim.x) {
        const T *z = static_cast<const T *>(a.logits) + r * a.ldl;
        TD *d = dlogits + r * a.ldl;
        const long long lab = a.labels[r];
        const bool used = lab >= 0 && lab < a.C;
        const float l = lse[r], f = used ? coef[r] : 0.f;
        for (int i = threadIdx.x * N; i < a.ldl; i += 256 * N) {
            float v[N];
            if (i + N <= a.C) {
                load_vec(z + i, v);
#pragma unroll
                for (int k = 0; k < N; k++) v[k] = ((i + k == (int)lab ? 1.f : 0.f) - __expf(v[k] - l)) * f;
            } else
                for (int k = 0; k < N; k++) v[k] = i + k < a.C ? ((i + k == (int)lab ? 1.f : 0.f) - __expf((float)z[i + k] - l)) * f : 0.f;
            if (!used || f == 0.f) {   // (0 * NaN of a masked row)
#pragma unroll
                for (int k = 0; k < N; k++) v[k] = 0.f;
            }
            if (i + N <= a.ldl) store_vec(d + i, v);
            else
                for (int k = 0; k < N; k++)
                    if (i + k < a.ldl) d[i + k] = (TD)v[k];
        }
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

// What one row adds to the sums, and its d loss / d logp.  The ratio is cut where exact arithmetic on the inputs cuts it: near a border
// (`near`) the caller comes again with logp in 64 bits.
__device__ __forceinline__ float policy_row(double logp, double oldp, float refp, bool has_ref, float adv, float w, const Policy &p, bool clipped,
                                            PolicyTerms &t) {
    const float ratio = expf((float)(logp - oldp));
    const float free = -adv * ratio;
    const float part = clipped ? -adv * (float)(adv > 0.f ? p.high : p.low) : free;
    float k = 0.f, kslope = 0.f;
    if (has_ref) {
        const float q = (float)((double)refp - logp), e = expm1f(q);
        k = e - q;
        kslope = -p.kl * e;
    }
    t.loss += (double)w * (double)(part + p.kl * k);
    t.surrogate += (double)w * (double)part;
    t.kl += (double)w * (double)k;
    t.clipped += clipped ? (double)w : 0.0;
    return w * p.scale * ((clipped ? 0.f : free) + kslope);
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
// sum over the row of exp(z - z_label) in 64 bits, by one workgroup
template <typename T>
__device__ double exact_logp(const T *z, int C, long long lab, double *sh) {
    const double at = (double)(float)z[lab];
    double s = 0.0;
    for (int i = threadIdx.x; i < C; i += blockDim.x) s += exp((double)(float)z[i] - at);
    return -log(block_sum_f64(s, sh));
}

template <typename T>
__global__ void __launch_bounds__(256) policy_row_kernel(Rows a, Policy p, const float *__restrict__ lse, float *__restrict__ logp, float *__restrict__ coef,
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
                const float z = (float)(static_cast<const T *>(a.logits) + r * a.ldl)[lab], l = lse[r], oldp = p.old_logp[r], adv = p.adv[r];
                lp = z - l;
                const float lr = lp - oldp;
                again = near_border(lr, fabsf(z) + fabsf(l) + fabsf(oldp), adv, p);
                if (!again) f = policy_row(lp, oldp, p.ref_logp ? p.ref_logp[r] : 0.f, p.ref_logp != nullptr, adv, w, p, past_border(lr, adv, p), t);
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
                const double lp = exact_logp(static_cast<const T *>(a.logits) + rr * a.ldl, a.C, lab, sh);
                if (threadIdx.x == 0) {
                    const float adv = p.adv[rr];
                    logp[rr] = (float)lp;
                    coef[rr] = policy_row(lp, (double)p.old_logp[rr], p.ref_logp ? p.ref_logp[rr] : 0.f, p.ref_logp != nullptr, adv,
                                          p.weight ? p.weight[rr] : 1.f, p, past_border(lp - (double)p.old_logp[rr], adv, p), t);
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
__global__ void __launch_bounds__(256) preference_pair_kernel(const float *__restrict__ logp, const long long *__restrict__ seq_start, const float *__restrict__ ref,
                                                             long long M, float beta, float smooth, float scale, float *__restrict__ loss,
                                                             float *__restrict__ seq_logp, float *__restrict__ coef) {
    __shared__ double sh[4];
    const long long pair = blockIdx.x;
    long long at[3];
    for (int k = 0; k < 3; k++) {   // (a start outside the rows, or before the one in front of it, reads and writes nothing)
        const long long v = seq_start[2 * pair + k];
        at[k] = v < 0 ? 0 : (v > M ? M : v);
    }
    double s[2];
    for (int q = 0; q < 2; q++) {
        double v = 0.0;
        for (long long r = at[q] + threadIdx.x; r < at[q + 1]; r += 256) v += (double)logp[r];
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
        for (long long r = at[q] + threadIdx.x; r < at[q + 1]; r += 256) coef[r] = q ? -g : g;
}
__global__ void __launch_bounds__(256) fill_kernel(float *__restrict__ p, long long n, float v) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = v;
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

int launch_stats(const Rows &a, int dtype, float *logp, float *lse, hipStream_t stream) {
    const dim3 grid(grid_of(a.M, 1 << 20));
    if (dtype == EMADAPT_DT_BF16) hipLaunchKernelGGL(row_stats_kernel<__bf16>, grid, dim3(256), 0, stream, a, logp, lse);
    else hipLaunchKernelGGL(row_stats_kernel<float>, grid, dim3(256), 0, stream, a, logp, lse);
    return launch_status();
}
template <typename T>
int launch_grad_t(const Rows &a, const float *lse, const float *coef, void *d, int ddt, hipStream_t stream) {
    const dim3 grid(grid_of(a.M, 1 << 20));
    if (ddt == EMADAPT_DT_BF16) hipLaunchKernelGGL((row_grad_kernel<T, __bf16>), grid, dim3(256), 0, stream, a, lse, coef, static_cast<__bf16 *>(d));
    else hipLaunchKernelGGL((row_grad_kernel<T, float>), grid, dim3(256), 0, stream, a, lse, coef, static_cast<float *>(d));
    return launch_status();
}
int launch_grad(const Rows &a, int dtype, const float *lse, const float *coef, void *d, int ddt, hipStream_t stream) {
    return dtype == EMADAPT_DT_BF16 ? launch_grad_t<__bf16>(a, lse, coef, d, ddt, stream) : launch_grad_t<float>(a, lse, coef, d, ddt, stream);
}
constexpr int kPolicyBlocks = 1024;

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
    return launch_stats(rows_of(logits, ldl, labels, M, C), dtype, logp, lse, stream);
}

int emadapt_label_logp_bwd(const void *logits, int dtype, int64_t ldl, const int64_t *labels, const float *lse, const float *dlogp, int64_t M, int64_t C,
                           void *dlogits, int dlogits_dtype, void *stream_) {
    if (int rc = check_rows(logits, dtype, ldl, labels, M, C, dlogits, dlogits_dtype)) return rc;
    if (M == 0) return EMADAPT_OK;
    if (!lse || !dlogp || !dlogits) return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)M * ((double)C * dt_size(dtype) + (double)ldl * dt_size(dlogits_dtype) + 16.0), stream);
    return launch_grad(rows_of(logits, ldl, labels, M, C), dtype, lse, dlogp, dlogits, dlogits_dtype, stream);
}

size_t emadapt_policy_loss_workspace_bytes(int64_t M, int64_t C) {
    (void)C;
    return align_up((size_t)(M > 0 ? M : 0) * 8, 256) + (size_t)kPolicyBlocks * 4 * sizeof(double);
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
    float *lse = static_cast<float *>(workspace), *coef = lse + M;
    double *partial = reinterpret_cast<double *>(static_cast<char *>(workspace) + align_up((size_t)M * 8, 256));
    const Rows a = rows_of(logits, ldl, actions, M, C);
    const Policy p = {old_logp, ref_logp, advantages, weights, 1.0 - clip_low, 1.0 + clip_high, log1p(-clip_low), log1p(clip_high), kl_coef, grad_scale};
    int blocks = 0;
    if (M) {
        if (int rc = launch_stats(a, dtype, nullptr, lse, stream)) return rc;
        blocks = (int)grid_of(ceil_div(M, 256), kPolicyBlocks);
        if (dtype == EMADAPT_DT_BF16) hipLaunchKernelGGL(policy_row_kernel<__bf16>, dim3(blocks), dim3(256), 0, stream, a, p, lse, logp, coef, partial);
        else hipLaunchKernelGGL(policy_row_kernel<float>, dim3(blocks), dim3(256), 0, stream, a, p, lse, logp, coef, partial);
        if (int rc = launch_status()) return rc;
        if (dlogits)
            if (int rc = launch_grad(a, dtype, lse, coef, dlogits, dlogits_dtype, stream)) return rc;
    }
    hipLaunchKernelGGL(policy_sums_kernel, dim3(1), dim3(256), 0, stream, partial, blocks, sums);
    return launch_status();
}

size_t emadapt_preference_loss_workspace_bytes(int64_t M, int64_t C) {
    (void)C;
    return (size_t)(M > 0 ? M : 1) * 12;
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
    float *logp = static_cast<float *>(workspace), *lse = logp + M, *coef = lse + M;
    const Rows a = rows_of(logits, ldl, labels, M, C);
    if (M) {
        if (int rc = launch_stats(a, dtype, logp, lse, stream)) return rc;
        if (dlogits) {   // rows of no sequence have no gradient
            hipLaunchKernelGGL(fill_kernel, dim3(grid_of(ceil_div(M, 256), 1024)), dim3(256), 0, stream, coef, (long long)M, 0.f);
            if (int rc = launch_status()) return rc;
        }
    }
    if (pairs) {
        hipLaunchKernelGGL(preference_pair_kernel, dim3((unsigned)pairs), dim3(256), 0, stream, logp, reinterpret_cast<const long long *>(seq_start), ref_logp, (long long)M,
                           beta, label_smoothing, grad_scale, loss, seq_logp, dlogits ? coef : nullptr);
        if (int rc = launch_status()) return rc;
    }
    if (M && dlogits) return launch_grad(a, dtype, lse, coef, dlogits, dlogits_dtype, stream);
    return EMADAPT_OK;
}

}  // extern "C"
