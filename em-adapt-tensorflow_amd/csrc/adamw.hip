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
constexpr int kRounds = 4, kChunk = 1024 * kRounds, kBlock = 64, kParts = 2048;   // (four elements to a thread and round)

// The control block on the device: steps and norm are the caller's to read, the rest is what one step's launches hand on.
struct AdamwControl {
    long long steps;
    float norm, coef, rate, root2;   // of this step: the clip's factor and the bias corrections
    unsigned go, ticket;             // what happens (kNothing ..); the norm's workgroups that are done (0 between launches)
    double sum[kParts];
};

enum { kNothing = 0, kStep = 1, kClean = 2 };   // kClean: no update, but the gradients are zeroed where the step was asked to

struct AdamwArgs {
    float b1, omb1, b2, omb2, eps;
    double lr;
    unsigned seed;
    int zero_grads;
};

// The tensors' addresses come out of memory: said to be global here, or every access would be a flat one (which waits for the LDS as well).
#define EMADAPT_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ EMADAPT_GLOBAL T *global(void *p) { return (EMADAPT_GLOBAL T *)p; }

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 h4 __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void load4(const EMADAPT_GLOBAL float *p, float (&v)[4]) {
    const f4 t = *(const EMADAPT_GLOBAL f4 *)p;
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ void load4(const EMADAPT_GLOBAL __bf16 *p, float (&v)[4]) {
    const h4 t = *(const EMADAPT_GLOBAL h4 *)p;
    v[0] = (float)t.x; v[1] = (float)t.y; v[2] = (float)t.z; v[3] = (float)t.w;
}
__device__ __forceinline__ void zero4(EMADAPT_GLOBAL float *p) { *(EMADAPT_GLOBAL f4 *)p = f4{0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ void zero4(EMADAPT_GLOBAL __bf16 *p) { *(EMADAPT_GLOBAL h4 *)p = h4{(__bf16)0.f, (__bf16)0.f, (__bf16)0.f, (__bf16)0.f}; }
// 16 bytes that are not read again soon
__device__ __forceinline__ void load4_once(const EMADAPT_GLOBAL float *p, float (&v)[4]) {
    const f4 t = __builtin_nontemporal_load((const EMADAPT_GLOBAL f4 *)p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ void store4_once(EMADAPT_GLOBAL float *p, const float (&v)[4]) {
    const f4 t = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(t, (EMADAPT_GLOBAL f4 *)p);
}

struct AdamwScalars {
    double lr, beta1, beta2, max_norm;
    float grad_scale;
    int clip, ignore_status;
};
// What is the same for all elements of a step, by one wave: whether it happens, the clip's factor, the bias corrections (a power to a lane).
__device__ void adamw_control(AdamwControl *ctl, const AdamwScalars &a, double sum, unsigned *status) {
    const long long t = ctl->steps + 1;
    const double bias = 1.0 - pow(threadIdx.x & 1 ? a.beta2 : a.beta1, (double)t), bias1 = __shfl(bias, 0), bias2 = __shfl(bias, 1);
    if (threadIdx.x != 0) return;
    unsigned go = a.ignore_status || !status_raised(status) ? kStep : kNothing;
    float coef = a.grad_scale;
    if (a.clip) {
        const double norm = fabs((double)a.grad_scale) * sqrt(sum);
        ctl->norm = (float)norm;
        if (!(norm <= 1.7976931348623157e308)) {
            if (go) {   // (an accumulator would keep what is not finite for good)
                status_raise(status, EMADAPT_STATUS_NAN_GRADIENT);
                go = kClean;
            }
        } else if (norm > a.max_norm) coef = (float)((double)a.grad_scale * (a.max_norm / norm));
    }
    ctl->go = go;
    if (go != kStep) return;
    ctl->steps = t;
    ctl->coef = coef;
    ctl->rate = (float)(a.lr / bias1);
    ctl->root2 = (float)(1.0 / sqrt(bias2));
}
__global__ void adamw_control_kernel(AdamwControl *ctl, AdamwScalars a, unsigned *__restrict__ status) { adamw_control(ctl, a, 0.0, status); }

// Sum of squares of all gradients, in 64 bits: the products of 24-bit numbers are exact, so the norm and with it the clip's factor are
// the ones of exact arithmetic whatever the split (the double adds run beside the loads).  The last workgroup adds the parts up in their
// order and does the control kernel's work.  The ticket is a relaxed atomic behind a wait for the part's own store: a release of every
// workgroup writes the XCD's L2 back each time (410 -> 611 us for the step of 65.1 M parameters).  Only here, where 2048 workgroups
// have one: they come at 3.6 ns each.
template <typename TG>
__global__ void __launch_bounds__(256) adamw_norm_kernel(const AdamwChunk *__restrict__ table, long long nchunks, AdamwControl *ctl, AdamwScalars a,
                                                        unsigned *__restrict__ status) {
    __shared__ double sh[4];
    __shared__ bool last;
    double s = 0.0;
    constexpr int N = 16 / (int)sizeof(TG), kLoads = kChunk / (256 * N);   // 16 bytes to a load: 4 loads of f32, 2 of bf16
    typedef TG Piece __attribute__((ext_vector_type(16 / sizeof(TG)), aligned(sizeof(TG))));
    for (long long c = blockIdx.x; c < nchunks; c += gridDim.x) {
        const EMADAPT_GLOBAL TG *g = global<TG>(table[c].g);
        const int n = table[c].n;
        Piece v[kLoads];
        if (n == kChunk) {
#pragma unroll
            for (int q = 0; q < kLoads; q++) v[q] = *(const EMADAPT_GLOBAL Piece *)(g + (q * 256 + threadIdx.x) * N);
        } else {
#pragma unroll
            for (int q = 0; q < kLoads; q++)
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const int i = (q * 256 + threadIdx.x) * N + k;
                    v[q][k] = i < n ? g[i] : (TG)0.f;
                }
        }
#pragma unroll
        for (int q = 0; q < kLoads; q++)
#pragma unroll
            for (int k = 0; k < N; k++) s = __builtin_fma((double)(float)v[q][k], (double)(float)v[q][k], s);
    }
    s = block_sum_f64(s, sh);
    if (threadIdx.x == 0) {
        __hip_atomic_store(&ctl->sum[blockIdx.x], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0);
        last = atomicInc(&ctl->ticket, gridDim.x - 1) == gridDim.x - 1;   // (back to 0 by itself)
    }
    __syncthreads();
    if (!last) return;
    s = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) s += __hip_atomic_load(&ctl->sum[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum_f64(s, sh);
    if (threadIdx.x >= 64) return;
    adamw_control(ctl, a, s, status);
}

// a / b to one rounding or next to it (b a normal number of ordinary size): a reciprocal and one correction by the remainder
__device__ __forceinline__ float quotient(float a, float b) {
    const float r = __builtin_amdgcn_rcpf(b), q = a * r;
    return __builtin_fmaf(__builtin_fmaf(-b, q, a), r, q);
}
// sqrt(x) to nearest for x >= 2^-120 (below, next to it): the instruction's value or a neighbour, by the remainders' signs
__device__ __forceinline__ float root(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float lo = __uint_as_float(__float_as_uint(s) - 1u), hi = __uint_as_float(__float_as_uint(s) + 1u);
    const float t = __builtin_fmaf(-lo, s, x) <= 0.f ? lo : s;   // (0 and inf: the neighbours' remainders are NaN or 0, s stays)
    return __builtin_fmaf(-hi, s, x) > 0.f ? hi : t;
}
// One element: new moments, the root of the second and the new weight, every operation rounded on its own.
struct Element {
    float m, v, u, w;
};
__device__ __forceinline__ Element adamw_element(float g, float m, float v, float w, float coef, float fade, float rate, float root2, const AdamwArgs &a) {
#pragma clang fp contract(off)
    Element e;
    const float gs = g * coef;
    e.m = m * a.b1 + gs * a.omb1;
    e.v = v * a.b2 + (gs * gs) * a.omb2;
    e.u = root(e.v);
    e.w = (w - fade * w) - rate * quotient(e.m, e.u * root2 + a.eps);
    return e;
}
__device__ __forceinline__ bool finite(const Element &e) { return fabsf(e.m) < INFINITY && e.v < INFINITY; }

// the clean op alone, on element i of a chunk and every `step`-th after it
template <typename TG> __device__ __forceinline__ void zero_chunk(const AdamwChunk &c, int i, int step) {
    EMADAPT_GLOBAL TG *g = global<TG>(c.g);
    for (; i < c.n; i += step) g[i] = (TG)0.f;
}

// A workgroup to a chunk: of a whole one all 16 loads are in flight before the first is used.  (Fewer workgroups that walk several chunks each are
// slower: 351 us with 2048 of them against 323 for 65.1 M parameters.)  Last chunks first: the norm has just read their gradients.  Everything
// else is read and written once and told so (nontemporal), so that the gradients stay in the cache from the norm to here: 403 -> 329 us.
template <typename TG>
__global__ void __launch_bounds__(256) adamw_f32_kernel(const AdamwChunk *__restrict__ table, const AdamwControl *__restrict__ ctl, AdamwArgs a,
                                                       unsigned *__restrict__ status) {
    const unsigned go = ctl->go;
    if (!go) return;
    const AdamwChunk c = table[gridDim.x - 1 - blockIdx.x];
    if (go == kClean) {
        if (a.zero_grads) zero_chunk<TG>(c, threadIdx.x, 256);
        return;
    }
    const float rate = mul_rn(ctl->rate, c.ls), fade = (float)(a.lr * (double)c.ls * (double)c.wd), coef = ctl->coef, root2 = ctl->root2;
    EMADAPT_GLOBAL TG *gp = global<TG>(c.g);
    EMADAPT_GLOBAL float *wp = global<float>(c.w), *mp = global<float>(c.m), *vp = global<float>(c.v);
    bool bad = false;
    auto round4 = [&](int i, float (&g)[4], float (&w)[4], float (&m)[4], float (&v)[4]) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const Element e = adamw_element(g[k], m[k], v[k], w[k], coef, fade, rate, root2, a);
            const bool ok = finite(e);   // (else the gradient took a moment out of the finite numbers: the element is left alone)
            bad |= !ok;
            m[k] = ok ? e.m : m[k];
            v[k] = ok ? e.v : v[k];
            w[k] = ok ? e.w : w[k];
        }
        store4_once(wp + i, w); store4_once(mp + i, m); store4_once(vp + i, v);
        if (a.zero_grads) zero4(gp + i);
    };
    if (c.n == kChunk) {
        float g[kRounds][4], w[kRounds][4], m[kRounds][4], v[kRounds][4];
#pragma unroll
        for (int q = 0; q < kRounds; q++) {
            const int i = (q * 256 + threadIdx.x) * 4;
            load4(gp + i, g[q]); load4_once(wp + i, w[q]); load4_once(mp + i, m[q]); load4_once(vp + i, v[q]);
        }
#pragma unroll
        for (int q = 0; q < kRounds; q++) round4((q * 256 + threadIdx.x) * 4, g[q], w[q], m[q], v[q]);
    } else {
        int i = threadIdx.x * 4;
        for (; i + 4 <= c.n; i += 1024) {
            float g[4], w[4], m[4], v[4];
            load4(gp + i, g); load4_once(wp + i, w); load4_once(mp + i, m); load4_once(vp + i, v);
            round4(i, g, w, m, v);
        }
        for (; i < c.n; i++) {   // (fewer than four, of one thread)
            const Element e = adamw_element((float)gp[i], mp[i], vp[i], wp[i], coef, fade, rate, root2, a);
            if (finite(e)) { wp[i] = e.w; mp[i] = e.m; vp[i] = e.v; }
            else bad = true;
            if (a.zero_grads) gp[i] = (TG)0.f;
        }
    }
    if (bad) status_raise(status, EMADAPT_STATUS_NAN_GRADIENT);
}

// ---- the 8-bit formats.  BITS mantissa bits; kShift = the lowest code bit's place in the fp32 pattern.
// largest pattern of a row of 16 lanes (patterns of numbers >= 0 are in their order), in all of them
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned x) {
    const unsigned y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
    return x > y ? x : y;
}
__device__ __forceinline__ unsigned row_top(float x) { return dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(__float_as_uint(x))))); }
template <int BITS> __device__ __forceinline__ int block_power(unsigned top) {   // pattern of the block's largest magnitude
    const unsigned e = (top + (1u << (23 - BITS)) - 1u) >> 23;   // (past the largest code of its binade: one binade up)
    return (int)(e < 254u ? e : 254u);
}
// x >= 0 and at most the largest code of a block with this power; draw < 2^(23 - BITS): never above the largest code
template <int BITS> __device__ __forceinline__ unsigned code_of(float x, int e, unsigned draw) {
    return (__float_as_uint(__builtin_amdgcn_ldexpf(x, 15 - e)) + draw) >> (23 - BITS);
}
template <int BITS> __device__ __forceinline__ float value_of(unsigned code, int e) {
    return __builtin_amdgcn_ldexpf(__uint_as_float(code << (23 - BITS)), e - 15);
}
__device__ __forceinline__ float m_value(unsigned code, int e) {   // code: 8 bits
    return __builtin_amdgcn_ldexpf(__uint_as_float((code << 24 & 0x80000000u) | (code & 0x7Fu) << 20), e - 15);
}
__device__ __forceinline__ unsigned m_code(float m, int e, unsigned draw) {
    return code_of<3>(fabsf(m), e, draw) | ((__float_as_uint(m) >> 24) & 0x80u);
}
__device__ __forceinline__ unsigned u_code(float u, int e, unsigned draw) {
    const unsigned c = code_of<4>(u, e, draw), least = __float_as_uint(u) < 1u ? __float_as_uint(u) : 1u;
    return c > least ? c : least;
}
// the formats' largest values at the uppermost power: what pack() is given is held to them (a step's moments are finite sums of what is there)
constexpr float kMostM = 0x1.Ep127f, kMostU = 0x1.Fp127f;

// One thread's four elements, 16 lanes to a block of 64: from the stored codes to the new ones.  n4: how many of them are the tensor's.
struct Codes {
    unsigned m, u, e;   // four codes each; the block's two powers
};
__device__ __forceinline__ bool adamw_codes(Codes &c, const float (&g)[4], float (&w)[4], int n4, unsigned long long unit, const DropKey key, float coef, float fade,
                                            float rate, float root2, const AdamwArgs &a) {
    float m[4], u[4], w1[4], mtop = 0.f, utop = 0.f, all = 0.f;
    const int em = c.e & 0xFF, eu = c.e >> 8;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float uk = value_of<4>(c.u >> (8 * k) & 0xFFu, eu);
        const Element e = adamw_element(g[k], m_value(c.m >> (8 * k) & 0xFFu, em), mul_rn(uk, uk), w[k], coef, fade, rate, root2, a);
        m[k] = e.m; u[k] = e.u; w1[k] = e.w;
        all += fabsf(e.m) + e.v;
    }
    bool ok = true;
    if (!(all < INFINITY)) {   // (a sum of finite ones may overflow too: looked at one by one)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float uk = value_of<4>(c.u >> (8 * k) & 0xFFu, eu), mk = m_value(c.m >> (8 * k) & 0xFFu, em);
            if (!finite(adamw_element(g[k], mk, mul_rn(uk, uk), w[k], coef, fade, rate, root2, a))) {
                m[k] = mk; u[k] = uk; w1[k] = w[k];
                ok = false;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (k >= n4) m[k] = u[k] = 0.f;   // (past the tensor's end)
        w[k] = w1[k];
        mtop = fmaxf(mtop, fabsf(m[k]));
        utop = fmaxf(utop, u[k]);
    }
    const int em1 = block_power<3>(row_top(mtop)), eu1 = block_power<4>(row_top(utop));
    c.m = c.u = 0;
    const unsigned line = drop_line(unit);   // (unit % 4 == 0: the four are behind one another)
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const unsigned h = drop_mix(key, line + (unsigned)k * kDropStep);
        c.m |= m_code(m[k], em1, (h & 0xFFFFu) << 4) << (8 * k);
        c.u |= u_code(u[k], eu1, (h >> 16) << 3) << (8 * k);
    }
    c.e = (unsigned)(em1 | eu1 << 8);
    return ok;
}

// A workgroup to a round of a chunk, four elements to a thread: with the norm's and unpack()'s launches 262 us for 65.1 M parameters (f32 gradients)
// against 281 where a workgroup has the chunk's four rounds in flight.  Some 85 vector-ALU slots to an element (generator 17, root 12, quotient
// 7, both formats 25) are 140 us of the 190 that 65.1 M elements take, their 16.06 bytes 160: the two overlap.
template <typename TG>
__global__ void __launch_bounds__(256) adamw_u8_kernel(const AdamwChunk *__restrict__ table, const AdamwControl *__restrict__ ctl, AdamwArgs a,
                                                      unsigned *__restrict__ status) {
    const unsigned go = ctl->go, at = gridDim.x - 1 - blockIdx.x;
    if (!go) return;
    const AdamwChunk c = table[at / kRounds];
    if (go == kClean) {
        if (a.zero_grads) zero_chunk<TG>(c, (int)(at % kRounds) * 256 + threadIdx.x, 256 * kRounds);
        return;
    }
    const int i = (int)(at % kRounds) * 256 + threadIdx.x, n4 = c.n - i * 4;   // (n4: the thread's elements, may be more than 4)
    if (n4 + (int)(threadIdx.x & 15) * 4 <= 0) return;                          // (whole rows of lanes: the codes' buffers reach that far)
    const float rate = mul_rn(ctl->rate, c.ls), fade = (float)(a.lr * (double)c.ls * (double)c.wd);
    const DropKey key = drop_key(((unsigned long long)a.seed << 32) + (unsigned)ctl->steps);
    EMADAPT_GLOBAL TG *gp = global<TG>(c.g) + i * 4;
    EMADAPT_GLOBAL float *wp = global<float>(c.w) + i * 4;
    EMADAPT_GLOBAL unsigned *mp = global<unsigned>(c.m) + i, *up = global<unsigned>(c.v) + i;
    EMADAPT_GLOBAL unsigned short *ep = global<unsigned short>(c.e) + i / 16;
    float g[4], w[4];
    Codes o;
    o.m = __builtin_nontemporal_load(mp); o.u = __builtin_nontemporal_load(up); o.e = *ep;
    if (n4 >= 4) {
        load4(gp, g); load4_once(wp, w);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            g[k] = k < n4 ? (float)gp[k] : 0.f;
            w[k] = k < n4 ? wp[k] : 0.f;
        }
    }
    const bool ok = adamw_codes(o, g, w, n4, c.unit + (unsigned)(i * 4), key, ctl->coef, fade, rate, ctl->root2, a);
    __builtin_nontemporal_store(o.m, mp);
    __builtin_nontemporal_store(o.u, up);
    if ((threadIdx.x & 15) == 0) *ep = (unsigned short)o.e;
    if (n4 >= 4) {
        store4_once(wp, w);
        if (a.zero_grads) zero4(gp);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k < n4) { wp[k] = w[k]; if (a.zero_grads) gp[k] = (TG)0.f; }
    }
    if (!ok) status_raise(status, EMADAPT_STATUS_NAN_GRADIENT);
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
        load4((const EMADAPT_GLOBAL float *)m + q * 4, mv); load4((const EMADAPT_GLOBAL float *)u + q * 4, uv);
#pragma unroll
        for (int k = 0; k < 4; k++) {   // (NaN: 0)
            mv[k] = mv[k] == mv[k] ? fminf(fmaxf(mv[k], -kMostM), kMostM) : 0.f;
            uv[k] = fminf(fmaxf(uv[k], 0.f), kMostU);
            mtop = fmaxf(mtop, fabsf(mv[k]));
            utop = fmaxf(utop, uv[k]);
        }
        const int em = block_power<3>(row_top(mtop)), eu = block_power<4>(row_top(utop));
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
        if (!t.w || !t.g || !t.m || !t.v || !aligned(t.w, 4) || !aligned(t.g, gs) || t.unit < 0 || t.unit % 4) return EMADAPT_ERR_INVALID;
        if (!isfinite(t.weight_decay) || !isfinite(t.lr_scale)) return EMADAPT_ERR_INVALID;
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
    if (chunks < 0 || (chunks && !table) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 1e-16) || !(max_norm >= 0.0) ||
        !isfinite(lr) || !isfinite(grad_scale))
        return EMADAPT_ERR_INVALID;
    if (!control || control_bytes < sizeof(AdamwControl)) return EMADAPT_ERR_WORKSPACE;
    if (chunks > 0x7FFFFFFF / kRounds) return EMADAPT_ERR_UNSUPPORTED;   // (2 T elements)
    hipStream_t stream = as_stream(stream_);
    const AdamwChunk *tab = static_cast<const AdamwChunk *>(table);
    AdamwControl *ctl = static_cast<AdamwControl *>(control);
    unsigned *status = status_word();
    const bool bf = grad_dtype == EMADAPT_DT_BF16;
    ProfScope prof(EMADAPT_K_OTHER, 0.0, (double)chunks * kChunk * ((bf ? 2.0 : 4.0) + 8.0 + (state == EMADAPT_ADAMW_U8 ? 4.06 : 16.0)), stream);
    const AdamwScalars sc = {lr, beta1, beta2, max_norm, grad_scale, max_norm > 0.0 ? 1 : 0, status_collective()};
    if (max_norm > 0.0) {
        const dim3 parts((unsigned)(chunks < 1 ? 1 : (chunks < kParts ? chunks : kParts)));
        if (bf) hipLaunchKernelGGL(adamw_norm_kernel<__bf16>, parts, dim3(256), 0, stream, tab, (long long)chunks, ctl, sc, status);
        else hipLaunchKernelGGL(adamw_norm_kernel<float>, parts, dim3(256), 0, stream, tab, (long long)chunks, ctl, sc, status);
    } else
        hipLaunchKernelGGL(adamw_control_kernel, dim3(1), dim3(64), 0, stream, ctl, sc, status);
    if (int rc = launch_status()) return rc;
    if (!chunks) return EMADAPT_OK;
    const AdamwArgs a = {(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, lr, seed, zero_grads};
    // (a grid has fewer than 2^32 threads: one launch up to 2^24 chunks, 2^22 in 8 bits; last chunks first, as in the kernels)
    const int64_t rounds = state == EMADAPT_ADAMW_U8 ? kRounds : 1, most = 0xFFFFFFFFll / (256 * rounds);
    for (int64_t left = chunks; left > 0;) {
        const int64_t n = left < most ? left : most;
        left -= n;
        const dim3 grid((unsigned)(n * rounds)), block(256);
        const AdamwChunk *from = tab + left;
        if (state == EMADAPT_ADAMW_F32) {
            if (bf) hipLaunchKernelGGL(adamw_f32_kernel<__bf16>, grid, block, 0, stream, from, ctl, a, status);
            else hipLaunchKernelGGL(adamw_f32_kernel<float>, grid, block, 0, stream, from, ctl, a, status);
        } else {
            if (bf) hipLaunchKernelGGL(adamw_u8_kernel<__bf16>, grid, block, 0, stream, from, ctl, a, status);
            else hipLaunchKernelGGL(adamw_u8_kernel<float>, grid, block, 0, stream, from, ctl, a, status);
        }
        if (int rc = launch_status()) return rc;
    }
    return EMADAPT_OK;
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
