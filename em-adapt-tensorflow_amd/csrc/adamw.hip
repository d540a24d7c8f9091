// AdamW over many tensors in one launch, with moments in 32 or in 8 bits, and the global norm of the gradients.
//
//   g <- c g,  c = grad_scale * min(1, max_norm / |grad_scale * all gradients|)
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2        u = sqrt(v)
//   w <- (w - lr ls wd w) - (lr / (1 - b1^t)) ls * m / (u / sqrt(1 - b2^t) + eps)
//
// Every product and sum of the moments and of w is rounded on its own (no contraction): the stored moments are then a function of the
// inputs that any implementation with IEEE arithmetic reproduces bit for bit, and so are the 8-bit codes cut from them.
//
// The 8-bit form.  m is held as sign + 4 exponent + 3 mantissa bits, u (not v: the root halves the range to cover) as 4 exponent + 4
// mantissa bits; 64 elements share a power of two 2^k for each, chosen so that the block's largest value lies in the uppermost binade.
// A float's bits do the coding: x * 2^(15 - k) has an fp32 exponent field of at most 15, fields below 1 are fp32's own subnormals, and the
// code is its 7 (8) bits from bit 20 (19) up.  Rounding is stochastic: a moment moves by about (1 - b) of itself per step, far below half a
// step of a 3- or 4-bit mantissa, so rounding to nearest would freeze it, while floor(x + random) moves on average as the 32-bit form does.
// The random bits come from the package's counter-based generator at (seed, step, element).  A root above zero is never stored as zero:
// m / u would run away where m's code survived.
//
// Bound: HBM bytes.  32-bit 28 bytes per parameter (g 4, w 8, m 8, v 8), 8-bit 16.06 (g 4, w 8, codes 4, powers 0.06).
#include <math.h>
#include <string.h>

#include "common.h"

namespace {

using namespace emadapt;

// One workgroup's share: at most kChunk elements of one tensor, with direct pointers (a uniform 64-byte scalar load).
struct AdamwChunk {
    float *w;
    void *g;
    void *m, *v;          // f32 moments, or the uint8 codes of m and u
    unsigned char *e;     // 8-bit: the powers of two, (m, u) byte pairs per 64 elements
    unsigned long long unit;   // index of the first element in the state buffers: the random generator's counter
    int n;
    float wd, ls;
    int pad;
};
static_assert(sizeof(AdamwChunk) == 64, "one cache line half, one uniform load");
constexpr int kChunk = 4096, kBlock = 64, kParts = 2048;

// The control block on the device.  steps persists; the rest is what one step's kernels hand to the next.
struct AdamwControl {
    long long steps;
    float norm, coef, rate, root2;
    unsigned go, pad;
    double sum[kParts];
};

struct AdamwArgs {
    float b1, omb1, b2, omb2, eps;
    double lr;
    unsigned seed;
    int zero_grads;
};

template <typename T> __device__ __forceinline__ void load4(const T *p, float (&v)[4]);
template <> __device__ __forceinline__ void load4<float>(const float *p, float (&v)[4]) { __builtin_memcpy(v, p, 16); }
template <> __device__ __forceinline__ void load4<__bf16>(const __bf16 *p, float (&v)[4]) {
    __bf16 t[4];
    __builtin_memcpy(t, p, 8);
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = (float)t[k];
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

// Sum of squares of all gradients, in 64 bits: the products of 24-bit numbers are exact, so the norm and with it the clip's factor are
// the ones of exact arithmetic whatever the split (the double adds run beside the loads).
template <typename TG>
__global__ void __launch_bounds__(256) adamw_norm_kernel(const AdamwChunk *__restrict__ table, long long nchunks, AdamwControl *__restrict__ ctl) {
    __shared__ double sh[4];
    double s = 0.0;
    for (long long c = blockIdx.x; c < nchunks; c += gridDim.x) {
        const TG *g = static_cast<const TG *>(table[c].g);
        const int n = table[c].n;
        for (int i = threadIdx.x * 4; i < n; i += 1024) {
            float v[4];
            if (i + 4 <= n) load4(g + i, v);
            else
                for (int k = 0; k < 4; k++) v[k] = i + k < n ? (float)g[i + k] : 0.f;
            for (int k = 0; k < 4; k++) s += (double)v[k] * (double)v[k];
        }
    }
    s = block_sum_f64(s, sh);
    if (threadIdx.x == 0) ctl->sum[blockIdx.x] = s;
}

// Everything that is the same for all elements: the clip's factor, the bias corrections of step t, whether the step happens at all.
__global__ void __launch_bounds__(256) adamw_control_kernel(AdamwControl *__restrict__ ctl, int nparts, double lr, double b1, double b2,
                                                          float grad_scale, double max_norm, unsigned *__restrict__ status, int ignore_status) {
    __shared__ double sh[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += ctl->sum[i];
    s = block_sum_f64(s, sh);
    if (threadIdx.x != 0) return;
    bool go = ignore_status || !status_raised(status);
    float coef = grad_scale;
    if (nparts > 0) {
        const double norm = fabs((double)grad_scale) * sqrt(s);
        ctl->norm = (float)norm;
        if (!(norm <= 1.7976931348623157e308)) {
            if (go) status_raise(status, EMADAPT_STATUS_NAN_GRADIENT);
            go = false;
        } else if (norm > max_norm) coef = (float)((double)grad_scale * (max_norm / norm));
    }
    ctl->go = go ? 1u : 0u;
    if (!go) return;
    const long long t = ctl->steps + 1;
    ctl->steps = t;
    ctl->coef = coef;
    ctl->rate = (float)(lr / (1.0 - pow(b1, (double)t)));
    ctl->root2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
}

// One element (m, v in, m, u, w out), every operation rounded on its own.  false: the gradient took a moment out of the finite numbers.
__device__ __forceinline__ bool adamw_element(float g, float &m, float &v, float &u, float &w, float coef, float fade, float rate, float root2,
                                              const AdamwArgs &a) {
#pragma clang fp contract(off)
    const float gs = g * coef;
    const float m1 = m * a.b1 + gs * a.omb1;
    const float v1 = v * a.b2 + (gs * gs) * a.omb2;
    const bool ok = fabsf(m1) < INFINITY && v1 < INFINITY;
    const float u1 = sqrtf(v1);
    const float w1 = (w - fade * w) - rate * (m1 / (u1 * root2 + a.eps));
    m = ok ? m1 : m;
    v = ok ? v1 : v;
    u = ok ? u1 : u;
    w = ok ? w1 : w;
    return ok;
}

template <typename TG>
__global__ void __launch_bounds__(256) adamw_f32_kernel(const AdamwChunk *__restrict__ table, const AdamwControl *__restrict__ ctl, AdamwArgs a,
                                                       unsigned *__restrict__ status) {
    if (!ctl->go) return;
    const AdamwChunk c = table[blockIdx.x];
    const float coef = ctl->coef, root2 = ctl->root2;
    const float rate = mul_rn(ctl->rate, c.ls), fade = (float)(a.lr * (double)c.ls * (double)c.wd);
    TG *gp = static_cast<TG *>(c.g);
    float *mp = static_cast<float *>(c.m), *vp = static_cast<float *>(c.v);
    bool bad = false;
    for (int i = threadIdx.x * 4; i < c.n; i += 1024) {
        float g[4], w[4], m[4], v[4], u;
        if (i + 4 <= c.n) {
            load4(gp + i, g); load4(c.w + i, w); load4(mp + i, m); load4(vp + i, v);
#pragma unroll
            for (int k = 0; k < 4; k++) bad |= !adamw_element(g[k], m[k], v[k], u, w[k], coef, fade, rate, root2, a);
            __builtin_memcpy(c.w + i, w, 16); __builtin_memcpy(mp + i, m, 16); __builtin_memcpy(vp + i, v, 16);
            if (a.zero_grads) __builtin_memset(gp + i, 0, 4 * sizeof(TG));
        } else {
            for (int k = i; k < c.n; k++) {
                float wk = c.w[k], mk = mp[k], vk = vp[k];
                bad |= !adamw_element((float)gp[k], mk, vk, u, wk, coef, fade, rate, root2, a);
                c.w[k] = wk; mp[k] = mk; vp[k] = vk;
                if (a.zero_grads) gp[k] = (TG)0.f;
            }
        }
    }
    if (bad) status_raise(status, EMADAPT_STATUS_NAN_GRADIENT);
}

// ---- the 8-bit formats.  BITS mantissa bits; kShift = the lowest code bit's place in the fp32 pattern.
template <int BITS> __device__ __forceinline__ int block_power(float top) {   // top >= 0, the block's largest magnitude
    const unsigned e = (__float_as_uint(top) + (1u << (23 - BITS)) - 1u) >> 23;   // (past the largest code of its binade: one binade up)
    return (int)(e < 254u ? e : 254u);
}
template <int BITS> __device__ __forceinline__ unsigned code_of(float x, int e, unsigned draw) {   // x >= 0; draw < 2^(23 - BITS)
    constexpr unsigned kTop = (16u << BITS) - 1u;
    const unsigned c = (__float_as_uint(__builtin_amdgcn_ldexpf(x, 15 - e)) + draw) >> (23 - BITS);
    return c < kTop ? c : kTop;
}
template <int BITS> __device__ __forceinline__ float value_of(unsigned code, int e) {
    return __builtin_amdgcn_ldexpf(__uint_as_float(code << (23 - BITS)), e - 15);
}
__device__ __forceinline__ float m_value(unsigned code, int e) {
    const float x = value_of<3>(code & 0x7Fu, e);
    return (code & 0x80u) ? -x : x;
}
__device__ __forceinline__ unsigned m_code(float m, int e, unsigned draw) {
    return code_of<3>(fabsf(m), e, draw) | ((__float_as_uint(m) >> 24) & 0x80u);
}
__device__ __forceinline__ unsigned u_code(float u, int e, unsigned draw) {
    const unsigned c = code_of<4>(u, e, draw);
    return c == 0u && u > 0.f ? 1u : c;
}
// largest of a row of 16 lanes (a block of 64 elements, 4 to a lane), in all of them
__device__ __forceinline__ float row_max(float x) {
    for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

template <typename TG>
__global__ void __launch_bounds__(256) adamw_u8_kernel(const AdamwChunk *__restrict__ table, const AdamwControl *__restrict__ ctl, AdamwArgs a,
                                                      unsigned *__restrict__ status) {
    if (!ctl->go) return;
    const AdamwChunk c = table[blockIdx.x];
    const float coef = ctl->coef, root2 = ctl->root2;
    const float rate = mul_rn(ctl->rate, c.ls), fade = (float)(a.lr * (double)c.ls * (double)c.wd);
    const DropKey key = drop_key(((unsigned long long)a.seed << 32) + (unsigned)ctl->steps);
    TG *gp = static_cast<TG *>(c.g);
    unsigned char *mp = static_cast<unsigned char *>(c.m), *up = static_cast<unsigned char *>(c.v);
    const int rounded = (c.n + kBlock - 1) / kBlock * kBlock;   // (whole rows of lanes: the codes' buffers reach that far)
    bool bad = false;
    for (int i = threadIdx.x * 4; i < rounded; i += 1024) {
        float g[4] = {0.f, 0.f, 0.f, 0.f}, w[4] = {0.f, 0.f, 0.f, 0.f}, m[4], u[4];
        if (i + 4 <= c.n) {
            load4(gp + i, g); load4(c.w + i, w);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < c.n) { g[k] = (float)gp[i + k]; w[k] = c.w[i + k]; }
        }
        const unsigned mc = *reinterpret_cast<const unsigned *>(mp + i), uc = *reinterpret_cast<const unsigned *>(up + i);
        const unsigned ee = *reinterpret_cast<const unsigned short *>(c.e + i / kBlock * 2);
        const int em = ee & 0xFF, eu = ee >> 8;
        float mtop = 0.f, utop = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            m[k] = m_value(mc >> (8 * k) & 0xFFu, em);
            u[k] = value_of<4>(uc >> (8 * k) & 0xFFu, eu);
            float v = mul_rn(u[k], u[k]);
            if (i + k < c.n) bad |= !adamw_element(g[k], m[k], v, u[k], w[k], coef, fade, rate, root2, a);
            mtop = fmaxf(mtop, fabsf(m[k]));
            utop = fmaxf(utop, u[k]);
        }
        const int em1 = block_power<3>(row_max(mtop)), eu1 = block_power<4>(row_max(utop));
        unsigned mo = 0, uo = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const unsigned h = drop_hash(key, c.unit + (unsigned)(i + k));
            mo |= m_code(m[k], em1, (h & 0xFFFFu) << 4) << (8 * k);
            uo |= u_code(u[k], eu1, (h >> 16) << 3) << (8 * k);
        }
        *reinterpret_cast<unsigned *>(mp + i) = mo;
        *reinterpret_cast<unsigned *>(up + i) = uo;
        if ((threadIdx.x & 15) == 0) *reinterpret_cast<unsigned short *>(c.e + i / kBlock * 2) = (unsigned short)(em1 | eu1 << 8);
        if (i + 4 <= c.n) {
            __builtin_memcpy(c.w + i, w, 16);
            if (a.zero_grads) __builtin_memset(gp + i, 0, 4 * sizeof(TG));
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < c.n) { c.w[i + k] = w[k]; if (a.zero_grads) gp[i + k] = (TG)0.f; }
        }
    }
    if (bad) status_raise(status, EMADAPT_STATUS_NAN_GRADIENT);
}

// codes <-> values, for checkpoints: four elements to a thread, rounding to nearest on the way in
template <typename TO>
__global__ void __launch_bounds__(256) adamw_unpack_kernel(const unsigned char *__restrict__ mp, const unsigned char *__restrict__ up,
                                                          const unsigned char *__restrict__ e, long long n4, TO *__restrict__ m, TO *__restrict__ u) {
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < n4; q += (long long)gridDim.x * 256) {
        const unsigned mc = reinterpret_cast<const unsigned *>(mp)[q], uc = reinterpret_cast<const unsigned *>(up)[q];
        const unsigned ee = reinterpret_cast<const unsigned short *>(e)[q / (kBlock / 4)];
        TO mo[4], uo[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            mo[k] = (TO)m_value(mc >> (8 * k) & 0xFFu, ee & 0xFF);
            uo[k] = (TO)value_of<4>(uc >> (8 * k) & 0xFFu, ee >> 8);
        }
        __builtin_memcpy(m + q * 4, mo, sizeof(mo));
        __builtin_memcpy(u + q * 4, uo, sizeof(uo));
    }
}
__global__ void __launch_bounds__(256) adamw_pack_kernel(const float *__restrict__ m, const float *__restrict__ u, long long n4,
                                                        unsigned char *__restrict__ mp, unsigned char *__restrict__ up, unsigned char *__restrict__ e) {
    // (n4 is a multiple of 16: a row of lanes is in the range as a whole or not at all)
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < n4; q += (long long)gridDim.x * 256) {
        float mv[4], uv[4], mtop = 0.f, utop = 0.f;
        load4(m + q * 4, mv); load4(u + q * 4, uv);
#pragma unroll
        for (int k = 0; k < 4; k++) { uv[k] = fmaxf(uv[k], 0.f); mtop = fmaxf(mtop, fabsf(mv[k])); utop = fmaxf(utop, uv[k]); }
        const int em = block_power<3>(row_max(mtop)), eu = block_power<4>(row_max(utop));
        unsigned mo = 0, uo = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            mo |= m_code(mv[k], em, 1u << 19) << (8 * k);
            uo |= u_code(uv[k], eu, 1u << 18) << (8 * k);
        }
        reinterpret_cast<unsigned *>(mp)[q] = mo;
        reinterpret_cast<unsigned *>(up)[q] = uo;
        if ((threadIdx.x & 15) == 0) reinterpret_cast<unsigned short *>(e)[q / (kBlock / 4)] = (unsigned short)(em | eu << 8);
    }
}

inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool is_dt(int dt) { return dt == EMADAPT_DT_F32 || dt == EMADAPT_DT_BF16; }

}  // namespace

extern "C" {

int64_t emadapt_adamw_chunks(int count, const emadapt_adamw_tensor *tensors) {
    if (count < 0 || (count && !tensors)) return EMADAPT_ERR_INVALID;
    int64_t chunks = 0;
    for (int k = 0; k < count; k++) {
        if (tensors[k].n < 0) return EMADAPT_ERR_INVALID;
        chunks += ceil_div(tensors[k].n, kChunk);
    }
    return chunks;
}

size_t emadapt_adamw_table_bytes(int64_t chunks) { return (size_t)(chunks > 0 ? chunks : 1) * sizeof(AdamwChunk); }
size_t emadapt_adamw_control_bytes(void) { return sizeof(AdamwControl); }

int emadapt_adamw_table(int count, const emadapt_adamw_tensor *tensors, int grad_dtype, int state, void *table_host, size_t table_bytes) {
    if (!is_dt(grad_dtype) || (state != EMADAPT_ADAMW_F32 && state != EMADAPT_ADAMW_U8)) return EMADAPT_ERR_INVALID;
    const int64_t chunks = emadapt_adamw_chunks(count, tensors);
    if (chunks < 0) return (int)chunks;
    if (chunks == 0) return EMADAPT_OK;
    if (!table_host || table_bytes < emadapt_adamw_table_bytes(chunks)) return EMADAPT_ERR_WORKSPACE;
    AdamwChunk *out = static_cast<AdamwChunk *>(table_host);
    const size_t gs = grad_dtype == EMADAPT_DT_BF16 ? 2 : 4, ss = state == EMADAPT_ADAMW_U8 ? 1 : 4;
    for (int k = 0; k < count; k++) {
        const emadapt_adamw_tensor &t = tensors[k];
        if (t.n == 0) continue;
        if (!t.w || !t.g || !t.m || !t.v || !aligned(t.w, 4) || !aligned(t.g, gs) || t.unit < 0) return EMADAPT_ERR_INVALID;
        // (codes are read four at a time and the powers of two by pairs; f32 moments at their own alignment)
        if (state == EMADAPT_ADAMW_U8 ? (!t.e || !aligned(t.m, 4) || !aligned(t.v, 4) || !aligned(t.e, 2)) : (!aligned(t.m, 4) || !aligned(t.v, 4)))
            return EMADAPT_ERR_INVALID;
        for (int64_t at = 0; at < t.n; at += kChunk, out++) {
            AdamwChunk c;
            memset(&c, 0, sizeof(c));
            c.w = t.w + at;
            c.g = static_cast<char *>(t.g) + at * gs;
            c.m = static_cast<char *>(t.m) + at * ss;
            c.v = static_cast<char *>(t.v) + at * ss;
            c.e = t.e ? static_cast<unsigned char *>(t.e) + at / kBlock * 2 : nullptr;
            c.unit = (unsigned long long)(t.unit + at);
            c.n = (int)(t.n - at < kChunk ? t.n - at : kChunk);
            c.wd = t.weight_decay;
            c.ls = t.lr_scale;
            memcpy(out, &c, sizeof(c));
        }
    }
    return EMADAPT_OK;
}

int emadapt_adamw_step(const void *table, int64_t chunks, int grad_dtype, int state, void *control, size_t control_bytes, double lr, double beta1,
                       double beta2, double eps, float grad_scale, double max_norm, unsigned seed, int zero_grads, void *stream_) {
    if (!is_dt(grad_dtype) || (state != EMADAPT_ADAMW_F32 && state != EMADAPT_ADAMW_U8)) return EMADAPT_ERR_INVALID;
    if (chunks < 0 || (chunks && !table) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 1e-30) || !(max_norm >= 0.0))
        return EMADAPT_ERR_INVALID;
    if (!control || control_bytes < sizeof(AdamwControl)) return EMADAPT_ERR_WORKSPACE;
    if (chunks > 0x7FFFFFFF) return EMADAPT_ERR_UNSUPPORTED;
    hipStream_t stream = as_stream(stream_);
    const AdamwChunk *tab = static_cast<const AdamwChunk *>(table);
    AdamwControl *ctl = static_cast<AdamwControl *>(control);
    unsigned *status = status_word();
    const bool bf = grad_dtype == EMADAPT_DT_BF16;
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)chunks * kChunk * ((bf ? 2.0 : 4.0) + 8.0 + (state == EMADAPT_ADAMW_U8 ? 4.06 : 16.0)), stream);
    int nparts = 0;
    if (max_norm > 0.0) {
        nparts = (int)(chunks < kParts ? (chunks ? chunks : 1) : kParts);
        if (bf) hipLaunchKernelGGL(adamw_norm_kernel<__bf16>, dim3(nparts), dim3(256), 0, stream, tab, (long long)chunks, ctl);
        else hipLaunchKernelGGL(adamw_norm_kernel<float>, dim3(nparts), dim3(256), 0, stream, tab, (long long)chunks, ctl);
        if (int rc = launch_status()) return rc;
    }
    hipLaunchKernelGGL(adamw_control_kernel, dim3(1), dim3(256), 0, stream, ctl, nparts, lr, beta1, beta2, grad_scale, max_norm, status, status_collective());
    if (int rc = launch_status()) return rc;
    if (!chunks) return EMADAPT_OK;
    const AdamwArgs a = {(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, lr, seed, zero_grads};
    const dim3 grid((unsigned)chunks), block(256);
    if (state == EMADAPT_ADAMW_F32) {
        if (bf) hipLaunchKernelGGL(adamw_f32_kernel<__bf16>, grid, block, 0, stream, tab, ctl, a, status);
        else hipLaunchKernelGGL(adamw_f32_kernel<float>, grid, block, 0, stream, tab, ctl, a, status);
    } else {
        if (bf) hipLaunchKernelGGL(adamw_u8_kernel<__bf16>, grid, block, 0, stream, tab, ctl, a, status);
        else hipLaunchKernelGGL(adamw_u8_kernel<float>, grid, block, 0, stream, tab, ctl, a, status);
    }
    return launch_status();
}

int emadapt_adamw_unpack(const void *m_codes, const void *u_codes, const void *powers, int64_t n, void *m, void *u, int dtype, void *stream_) {
    if (!is_dt(dtype) || n < 0 || n % kBlock) return EMADAPT_ERR_INVALID;
    if (n == 0) return EMADAPT_OK;
    if (!m_codes || !u_codes || !powers || !m || !u || !aligned(m_codes, 4) || !aligned(u_codes, 4) || !aligned(powers, 2) || !aligned(m, 16) || !aligned(u, 16))
        return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)n * (2.06 + (dtype == EMADAPT_DT_BF16 ? 4.0 : 8.0)), stream);
    const unsigned char *mc = static_cast<const unsigned char *>(m_codes), *uc = static_cast<const unsigned char *>(u_codes), *e = static_cast<const unsigned char *>(powers);
    const long long n4 = n / 4, want = ceil_div(n4, 256);
    const dim3 grid((unsigned)(want < 8192 ? want : 8192));
    if (dtype == EMADAPT_DT_BF16) hipLaunchKernelGGL(adamw_unpack_kernel<__bf16>, grid, dim3(256), 0, stream, mc, uc, e, n4, static_cast<__bf16 *>(m), static_cast<__bf16 *>(u));
    else hipLaunchKernelGGL(adamw_unpack_kernel<float>, grid, dim3(256), 0, stream, mc, uc, e, n4, static_cast<float *>(m), static_cast<float *>(u));
    return launch_status();
}

int emadapt_adamw_pack(const float *m, const float *u, int64_t n, void *m_codes, void *u_codes, void *powers, void *stream_) {
    if (n < 0 || n % kBlock) return EMADAPT_ERR_INVALID;
    if (n == 0) return EMADAPT_OK;
    if (!m_codes || !u_codes || !powers || !m || !u || !aligned(m_codes, 4) || !aligned(u_codes, 4) || !aligned(powers, 2) || !aligned(m, 16) || !aligned(u, 16))
        return EMADAPT_ERR_INVALID;
    hipStream_t stream = as_stream(stream_);
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)n * 10.06, stream);
    const long long n4 = n / 4, want = ceil_div(n4, 256);
    hipLaunchKernelGGL(adamw_pack_kernel, dim3((unsigned)(want < 8192 ? want : 8192)), dim3(256), 0, stream, m, u, n4, static_cast<unsigned char *>(m_codes),
                       static_cast<unsigned char *>(u_codes), static_cast<unsigned char *>(powers));
    return launch_status();
}

}  // extern "C"
