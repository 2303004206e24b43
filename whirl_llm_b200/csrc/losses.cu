// Log-probabilities of given tokens, the clipped policy loss and the preference loss, with their gradients down to the
// logits (formulas: include/whirl_b200.h).
//
// Every row needs its softmax statistics before any of its gradient can be written.  The statistics are one online pass: a
// thread keeps the largest logit it has met, the sum of exp((x - about that) * inv_t) and (for the entropy) the sum of the
// exponentials times their exponents, and brings them to a new reference when a larger logit comes along; partial results merge
// the same way.  The gradient is one elementwise pass over the row.
//
//   forward_kernel     statistics of long rows, a cluster of 1 to 16 CTAs each      1024 x 262144 f32: 165 us, 6.5 TB/s; bf16: 93 us, 5.8 TB/s
//   grad_kernel        gradient of long rows from given statistics                  1024 x 262144 bf16: 175 us, 6.1 TB/s
//   fused_kernel       policy loss: both at once, the row held in shared memory     4096 x 151936 bf16, a third masked: 503 us, 4.1 TB/s
//   small_rows_kernel, small_grad_kernel   the same for short rows, a warp each     60000 x 2000 bf16: 76, 181 and 88 us
//
// All are bound by memory in principle (a logit costs about 7 instructions for the statistics, 5 for the gradient, and one
// exponential of the special function unit for each).  The preference loss needs its sequences' sums before any gradient: forward_kernel,
// pairs_kernel, grad_kernel, two reads and one write.
#include "../../include/whirl_b200.h"

#include <algorithm>
#include <atomic>
#include <cfloat>

#include "common.cuh"
#include "kernels.h"

namespace wb {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// pairs of floats: two results per instruction (add / mul / fma .f32x2)
// ---------------------------------------------------------------------------------------------------------------

struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 split(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// ---------------------------------------------------------------------------------------------------------------
// softmax statistics
// ---------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// c = inv_t log2 e in two floats, hi rounded down so that lo > 0 (a logit of -inf keeps its sign in both products).  With one float
// the exponents of a whole row are off in the same direction, by up to 6e-8 of their size: a bias of some 3e-7 in every
// log-probability, which sums over a sequence do not average out.  hi has 16 bits: with 24, x lo is less than half a step of the exponent that it
// is added to, and the same rounding takes it away in term after term (measured: 3e-8 to 8e-8 in the sum).
// most: logits are clamped to +-most where a reference is made of them.  The terms of logits below -most vanish then (a thread that has met
// masks of -1e30 alone keeps a sum of 0); a row whose own maximum lies beyond is a far row.
// From 2^18 on an exponent m c, less its reference, keeps a rest of m lo that takes bits from the result.
constexpr float kFarExponent = 262144.f;
struct Scale {
    float hi, lo, most;
};
__device__ __forceinline__ Scale scale_of(float inv_t) {
    const double c = fmin(double(inv_t) * 1.4426950408889634, 3e38);  // (at the largest inv_t hi + lo stays finite: only the maxima count there)
    Scale r;
    r.hi = __uint_as_float(__float_as_uint(__double2float_rd(c)) & 0xffffff00u);
    r.lo = fmaxf(float(c - double(r.hi)), fmaxf(r.hi * 1e-12f, 1e-45f));  // (at the smallest inv_t too it may not outweigh hi)
    r.most = fminf(kFarExponent / r.hi, FLT_MAX);
    return r;
}
// The reference exponent of a maximum: a whole number, so that moving a sum from one reference to another scales it by a power of two, exactly
// (ex2.approx is low by 5e-8 on average: three moves of every partial sum would show in the log-probability).  It lies kAbove above the maximum's
// own exponent, so that every term's is below -1: there ex2.approx has the same mean error at every exponent (mended).
// (hi + lo: off the chain of dependent instructions, which in short rows one lane or another of a warp goes through at most of its vectors.
// With two multiply-adds 20000 x 4200 bf16 took 69 us, with one 62.)
constexpr float kAbove = 2.f;
__device__ __forceinline__ float ref_of(float m, const Scale& c) {
    const float x = fminf(fmaxf(m, -c.most), c.most);
    return rintf(fmaf(x, c.hi + c.lo, kAbove));
}

// Partial statistics of a set of logits: m their maximum (-inf without one), e = ref_of(m), s - k = sum 2^(x c - e) (k: what
// Kahan's sum owes), q = sum of the same terms times their exponent.  The exponent is two fused multiply-adds from the logit (first hi: the
// difference to e is small, and rounded as such, before lo comes to it; both roundings fall anywhere); that e is not
// the maximum's own exponent shifts all terms of a row by the same factor (shift_of).
// A plain float sum is not enough: in the thread that meets the row's peak every later term is rounded to the peak's last
// bits, 300 times in a row of 151936, all of it landing in the log-probability (measured: 4e-7).
struct Soft {
    float m, e, s, k, q;
};
__device__ __forceinline__ Soft soft_empty(const Scale& c) { return Soft{-INFINITY, ref_of(-INFINITY, c), 0.f, 0.f, 0.f}; }

template <bool ENT>
__device__ __forceinline__ void raise(Soft& a, float m, const Scale& c) {  // moves a's reference to that of m >= a.m
    const float e = ref_of(m, c), t = a.e - e, f = ex2_approx(t);
    if (ENT) a.q = f * fmaf(fmaxf(t, -1000.f), a.s, a.q);
    a.s *= f, a.k *= f;
    a.m = m, a.e = e;
}
// N logits: their terms are summed as a tree, the tree's sum goes into the thread's by Kahan's rule
template <bool ENT, int N>
__device__ __forceinline__ void add_many(Soft& a, const float (&x)[N], const Scale& c) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) m = max3(m, x[i], x[i + 1]);
    if (N % 2 == 0) m = fmaxf(m, x[N - 1]);
    if (m > a.m) raise<ENT>(a, m, c);
    float sum, qs = 0.f;
    if (N == 1) {
        const float t = fmaf(x[0], c.lo, fmaf(x[0], c.hi, -a.e));
        sum = ex2_approx(t);
        if (ENT) qs = sum * fmaxf(t, -1000.f);
    } else {
        const F2 ne = f2(-a.e, -a.e), hi = f2(c.hi, c.hi), lo = f2(c.lo, c.lo);
        F2 w[N / 2 > 0 ? N / 2 : 1], q = f2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const F2 v = f2(x[2 * i], x[2 * i + 1]);
            const float2 t = split(fma2(v, lo, fma2(v, hi, ne)));
            w[i] = f2(ex2_approx(t.x), ex2_approx(t.y));
            if (ENT) q = fma2(w[i], f2(fmaxf(t.x, -1000.f), fmaxf(t.y, -1000.f)), q);  // (0 * -inf is not what a forbidden token adds)
        }
#pragma unroll
        for (int k = N / 4; k >= 1; k /= 2)
#pragma unroll
            for (int i = 0; i < k; ++i) w[i] = add2(w[i], w[i + k]);
        const float2 p = split(w[0]), v = split(q);
        sum = p.x + p.y;
        if (ENT) qs = v.x + v.y;
    }
    const float y = __fsub_rn(sum, a.k), t = __fadd_rn(a.s, y);
    a.k = __fsub_rn(__fsub_rn(t, a.s), y);
    a.s = t;
    if (ENT) a.q += qs;
}

// The statistics of all threads of the CTA, then of all CTAs of the cluster; the result is valid in warp 0 of every CTA.
struct ReduceShared {
    float m[32];
    float2 sq[32];
    float4 part[2][16];  // one per CTA of the cluster; a second set for a far row's second reduction
};
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float warp_max_f(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <bool ENT>
__device__ __forceinline__ Soft reduce(Soft a, const Scale& c, ReduceShared& sh, int ctas, int turn) {
    const int w = threadIdx.x >> 5, nw = blockDim.x >> 5, lane = lane_id();
    a.s -= a.k, a.k = 0.f;
    float m = warp_max_f(a.m);
    if (lane == 0) sh.m[w] = m;
    __syncthreads();
    m = warp_max_f(lane < nw ? sh.m[lane] : -INFINITY);
    raise<ENT>(a, m, c);
    a.s = warp_sum_f(a.s);
    if (ENT) a.q = warp_sum_f(a.q);
    if (lane == 0) sh.sq[w] = make_float2(a.s, a.q);
    __syncthreads();
    if (w == 0) {
        const float2 v = lane < nw ? sh.sq[lane] : make_float2(0.f, 0.f);
        a.s = warp_sum_f(v.x);
        a.q = ENT ? warp_sum_f(v.y) : 0.f;
    }
    if (ctas > 1) {
        if (w == 0 && lane < ctas) {  // lane i tells CTA i
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&sh.part[turn][cluster_rank()])), "r"(lane));
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(m), "f"(a.s), "f"(a.q), "f"(0.f) : "memory");
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (w == 0) {
            const float4 p = lane < ctas ? sh.part[turn][lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
            a.m = p.x, a.e = ref_of(p.x, c), a.s = p.y, a.q = p.z;
            m = warp_max_f(a.m);
            raise<ENT>(a, m, c);
            a.s = warp_sum_f(a.s);
            if (ENT) a.q = warp_sum_f(a.q);
        }
    }
    return a;
}

// the same for a far row's thread sums, all relative to the row's maximum m
template <bool ENT>
__device__ __forceinline__ Soft reduce_far(Soft a, float m, ReduceShared& sh, int ctas) {
    Scale one{1.f, 0.f, FLT_MAX};
    a.m = 0.f, a.e = ref_of(0.f, one);  // (references alike: nothing is scaled)
    a = reduce<ENT>(a, one, sh, ctas, 1);
    a.m = m;
    return a;
}

// A row whose maximum (of any sign: rows of the type's lowest value or of -1e30 alone, temperatures near zero) is beyond the references:
// its exponents are made of the differences to the maximum, which is known by then.  One rule, from the maximum alone, for the
// statistics and for a gradient that starts from given ones.
__device__ __forceinline__ bool is_far(float m, const Scale& c) { return fabsf(m) <= FLT_MAX && fabsf(m) * c.hi >= kFarExponent; }
// the exponent of a far row's logit
__device__ __forceinline__ float far_exponent(float x, float m, float hi, float lo) {
    const float d = x - m;
    return fmaf(d, lo, d * hi);
}

// ---------------------------------------------------------------------------------------------------------------
// reading and writing logits
// ---------------------------------------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ float load_one(const T* p) {
    return sizeof(T) == 4 ? *reinterpret_cast<const float*>(p) : bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
}
// round to nearest even, NaN kept (cvt.rn.bf16x2)
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ void store_one(T* p, float v) {
    if (sizeof(T) == 4) *reinterpret_cast<float*>(p) = v;
    else *reinterpret_cast<uint16_t*>(p) = uint16_t(pack_bf16(v, 0.f));
}
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[16 / sizeof(T)]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
        else x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&x)[16 / sizeof(T)]) {
    if (sizeof(T) == 4) return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
// elements before the first 16-byte boundary at or after p
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
    const int h = int((16u - (uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u)) & 15u) / int(sizeof(T));
    return h < n ? h : n;
}

// ---------------------------------------------------------------------------------------------------------------
// one row's scalars
// ---------------------------------------------------------------------------------------------------------------

constexpr double kLn2 = 0.6931471805599453;

// The row's scalars are one warp's work per row, in the time that the others need for a slice: single-precision functions of the hardware
// with one correction each, and 64 bits where a last bit would add up over a sequence.  (The library's log, exp and expm1 in 64
// bits, and the divisions around them, took 2.7 us a row.)
// log of a sum > 0 (NaN without one): 2^k f with f in [sqrt 1/2, sqrt 2), log f = 2 atanh z, z = (f - 1) / (f + 1), |z| < 0.172; the
// first term left out, 2 z^15 / 15, is below 5e-13.  (lg2.approx and a step of Newton's method with ex2.approx is low by 4e-8.)
__device__ __forceinline__ double ln_of(double d) {
    if (!(d > 1e-300 && d < 1e300)) return NAN;
    const int hi = __double2hiint(d), k = (hi - 0x3fe6a09e) >> 20;
    const double f = __hiloint2double(hi - (k << 20), __double2loint(d)), b = f + 1.0;
    double r = double(__frcp_rn(float(b)));
    r = r * (2.0 - b * r);
    const double z = (f - 1.0) * r, y = z * z;
    double t = 1.0 / 13.0;
    t = fma(t, y, 1.0 / 11.0), t = fma(t, y, 1.0 / 9.0), t = fma(t, y, 1.0 / 7.0), t = fma(t, y, 1.0 / 5.0), t = fma(t, y, 1.0 / 3.0);
    return fma(double(k), kLn2, 2.0 * z * fma(t, y, 1.0));
}
// exp of |d| <= 20 (shifted: of 0.35), the exponent's rounding errors taken out; what is left is ex2.approx's own, up to 1.4e-7 of the result.  The
// ratio of a policy row and its kl are made of it: as exact as the f32 outputs that they become.
__device__ __forceinline__ float exp_of(float d) {
    const float hi = d * kLog2e, lo = fmaf(d, kLog2e, -hi) + d * 1.92596299e-8f;  // (log2 e = kLog2e + 1.926e-8)
    const float e = ex2_approx(hi);
    return fmaf(e, lo * float(kLn2), e);
}
// exp k - k - 1, by its series where the terms cancel
__device__ __forceinline__ float kl_of(float k) {
    if (!(fabsf(k) <= 1.f)) return exp_of(k) - 1.f - k;
    float t = 1.f / 39916800.f;
    t = fmaf(t, k, 1.f / 3628800.f), t = fmaf(t, k, 1.f / 362880.f), t = fmaf(t, k, 1.f / 40320.f), t = fmaf(t, k, 1.f / 5040.f);
    t = fmaf(t, k, 1.f / 720.f), t = fmaf(t, k, 1.f / 120.f), t = fmaf(t, k, 1.f / 24.f), t = fmaf(t, k, 1.f / 6.f);
    return k * k * fmaf(t, k, 0.5f);
}

// The natural logarithm of what the reference e of a row with maximum m puts into its sum, ln 2 (e - m c).  64 bits: m c has to be exact
// to the last bits of e.
__device__ __forceinline__ double shift_of(float m, float e, float inv_t) { return kLn2 * (double(e) - double(m) * (double(inv_t) * 1.4426950408889634)); }
__device__ __forceinline__ float shifted(float s, double y) {  // s e^y; the whole powers of two apart, they are exact
    const float k = rintf(float(y) * kLog2e);
    return s * exp_of(float(y - kLn2 * double(k))) * ex2_approx(k);
}
// A row's sum s, relative to its reference e, less the errors of ex2.approx that show.  That of the maximum's own term is taken out exactly (it is all that
// stands between a near-certain token's log-probability and 0).  The others are low by 5e-8 on average: measured over exponents of -24 to -1, each
// power of two between 4.9e-8 and 5.1e-8, a sixteenth of one between 3.3e-8 and 6.2e-8, a single term up to 1.4e-7.  So a row of
// many terms keeps some 1e-9, a row of two or three up to 1e-7 of what stands beside the maximum.
__device__ __forceinline__ double mended(float s, float m, float e, const Scale& c, double shift) {
    const double y = double(kAbove) * kLn2 - shift;  // ln 2 (m c - e + kAbove), within ln 2 / 2
    if (!(fabs(y) < 0.36)) return double(s);
    double t = 1.0 / 3628800.0;
    t = fma(t, y, 1.0 / 362880.0), t = fma(t, y, 1.0 / 40320.0), t = fma(t, y, 1.0 / 5040.0), t = fma(t, y, 1.0 / 720.0), t = fma(t, y, 1.0 / 120.0);
    t = fma(t, y, 1.0 / 24.0), t = fma(t, y, 1.0 / 6.0), t = fma(t, y, 0.5), t = fma(t, y, 1.0), t = fma(t, y, 1.0);
    const double top = double(ex2_approx(fmaf(m, c.lo, fmaf(m, c.hi, -e))));  // as it went into the sum
    return t * 0.25 + (double(s) - top) * (1.0 + 5e-8);                       // (2^-kAbove)
}

// The row's gradient: dx_j = w_j * (a + b * t_j), + d on the token, with t_j = x_j c - e (far: (x_j - m) c) and w_j = 2^t_j, whose sum
// over the row is s:
//   -inv_t g p_j - inv_t h p_j (log p_j + H),  p_j = w_j / s,  log p_j = ln 2 t_j - log s
//   => a = -(inv_t / s) (g + h (H - log s)),  b = -(inv_t / s) h ln 2
struct GradRow {
    float e, c, c_lo, a, b, d;
    int token, far;
};
__device__ __forceinline__ GradRow grad_row(float m, bool far, float s, float ln_s, const Scale& c, float inv_t, int token, float g, float h, float entropy) {
    GradRow q;
    q.far = far, q.e = far ? m : ref_of(m, c), q.c = c.hi, q.c_lo = c.lo, q.token = token;
    float k = 1.f / s;
    if (!far) k = fmaf(k, 5e-8f, k);  // (what ex2.approx is low by: see mended)
    q.d = inv_t * g;                  // (first: inv_t / s may be too large for a float)
    const float hh = inv_t * h;
    q.a = -k * (h == 0.f ? q.d : q.d + hh * (entropy - ln_s));
    q.b = -k * hh * float(kLn2);
    return q;
}
// (The scale's second float is needed for results of 8 bits too: it is worth x c_lo in the exponent, 0.8 % of p at a logit of 1e5.)
template <bool ENT>
__device__ __forceinline__ float grad_of(const GradRow& q, float x) {
    const float t0 = fmaf(x, q.c, -q.e), t = q.far ? far_exponent(x, q.e, q.c, q.c_lo) : fmaf(x, q.c_lo, t0), w = ex2_approx(t);
    return ENT ? w * fmaf(q.b, fmaxf(t, -1000.f), q.a) : w * q.a;
}
template <bool ENT, int N>
__device__ __forceinline__ void grad_many(const GradRow& q, float (&x)[N]) {  // (not for a far row)
    const F2 ne = f2(-q.e, -q.e), c = f2(q.c, q.c), lo = f2(q.c_lo, q.c_lo), a = f2(q.a, q.a), b = f2(q.b, q.b);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const F2 v = f2(x[i], x[i + 1]);
        const float2 t = split(fma2(v, lo, fma2(v, c, ne)));
        const F2 w = f2(ex2_approx(t.x), ex2_approx(t.y));
        const float2 r = split(ENT ? mul2(w, fma2(b, f2(fmaxf(t.x, -1000.f), fmaxf(t.y, -1000.f)), a)) : mul2(w, a));
        x[i] = r.x, x[i + 1] = r.y;
    }
}
// one vector of a row's gradient
template <typename T, bool ENT>
__device__ __forceinline__ uint4 grad_vec(const GradRow& q, uint4 v) {
    float e[16 / sizeof(T)];
    unpack<T>(v, e);
    grad_many<ENT, 16 / sizeof(T)>(q, e);
    return pack<T>(e);
}

// ---------------------------------------------------------------------------------------------------------------
// rows: statistics, what a call wants of them, and (with GRAD) the gradient
// ---------------------------------------------------------------------------------------------------------------

constexpr int kRowThreads = 256;
constexpr int kSharedMost = 225 * 1024;  // bytes of dynamic shared memory that a CTA may ask for

// A row as a user's call describes it, and whether it counts.
struct RowOf {
    int token;
    float inv_t, weight;
    float adv, old_logp, ref_logp;  // (policy loss; the preference loss has ref_logp)
    float scale;                    // row_scale, where it was known when the row was read
    bool live;
};
// Read by a warp, one word per lane, so that a row costs one trip to memory (row_word); every lane then gets the whole (row_from).
template <int EPI>
__device__ __forceinline__ uint32_t row_word(const LossArgs& a, int row, bool with_scale) {
    const int lane = lane_id();
    const void* p = nullptr;
    if (lane == 0) p = a.token + row;
    else if (lane == 1 && a.inv_t_rows) p = a.inv_t_rows + row;
    else if (lane == 2 && a.weight) p = a.weight + row;
    else if (lane == 3 && EPI == EPI_POLICY) p = a.adv + row;
    else if (lane == 4 && EPI == EPI_POLICY && a.old_logp) p = a.old_logp + row;
    else if (lane == 5 && EPI != EPI_NONE && a.ref_logp) p = a.ref_logp + row;
    else if (lane == 6 && EPI == EPI_POLICY && with_scale) p = a.row_scale + row;
    else if (lane == 7 && EPI == EPI_PREF) p = a.seq_start;
    else if (lane == 8 && EPI == EPI_PREF) p = a.seq_start + a.seqs;
    return p ? *static_cast<const uint32_t*>(p) : 0u;
}
template <int EPI>
__device__ __forceinline__ RowOf row_from(const LossArgs& a, int row, uint32_t got) {
    auto word = [&](int l) { return __shfl_sync(0xffffffffu, got, l); };
    auto real = [&](int l) { return __uint_as_float(word(l)); };
    RowOf r;
    r.token = int(word(0));
    const float it = real(1), wt = real(2);
    r.inv_t = a.inv_t_rows ? it : a.inv_t, r.weight = a.weight ? wt : 1.f;
    r.adv = real(3), r.old_logp = real(4), r.ref_logp = real(5), r.scale = real(6);
    r.live = unsigned(r.token) < unsigned(a.n) && r.weight > 0.f;
    if (EPI == EPI_PREF) r.live = r.live && row >= int(word(7)) && row < int(word(8));  // (the policy loss leaves such rows s = 0)
    return r;
}
template <int EPI>
__device__ __forceinline__ RowOf row_of(const LossArgs& a, int row, bool with_scale) { return row_from<EPI>(a, row, row_word<EPI>(a, row, with_scale)); }

// The policy loss of one row.
struct PolicyRow {
    float loss, kl, dlogp;
};
__device__ __forceinline__ PolicyRow policy_row(const LossArgs& a, const RowOf& w, double logp, float entropy) {
    PolicyRow p;
    const float adv = w.adv;
    float ratio = 1.f;
    bool free_d = true;
    if (a.old_logp) {
        const float d = float(logp - double(w.old_logp));
        free_d = !(d <= -20.f || d >= 20.f);
        ratio = exp_of(d < -20.f ? -20.f : (d > 20.f ? 20.f : d));
    }
    const float lo = 1.f - a.clip_low, hi = 1.f + a.clip_high;
    const float plain = ratio * adv, clipped = (ratio < lo ? lo : (ratio > hi ? hi : ratio)) * adv;
    const bool takes_plain = plain <= clipped;
    float pg = takes_plain ? -plain : -clipped;
    p.dlogp = takes_plain && free_d ? -plain : 0.f;
    if (a.dual_clip > 0.f && adv < 0.f && pg > -a.dual_clip * adv) pg = -a.dual_clip * adv, p.dlogp = 0.f;
    if (logp != logp) pg = float(logp);  // (a ratio of 1 does not see it)
    if (pg != pg) p.dlogp = pg;          // (no clip binds where the loss is NaN: an advantage or an old log-probability that is)
    p.kl = 0.f;
    if (a.ref_logp) {
        float k = float(double(w.ref_logp) - logp);
        const bool free_k = !(k <= -20.f || k >= 20.f);
        k = k < -20.f ? -20.f : (k > 20.f ? 20.f : k);
        p.kl = kl_of(k);
        pg = fmaf(a.kl_coef, p.kl, pg);
        if (free_k) p.dlogp -= a.kl_coef * (p.kl + k);
    }
    p.loss = a.ent_coef != 0.f ? pg - a.ent_coef * entropy : pg;
    return p;
}

// A policy row's share of the loss (a row without a weight in it, s = 0, has none whatever its own loss is).
__device__ __forceinline__ double share_of(const RowOf& w, const PolicyRow& p) { return w.scale > 0.f ? double(w.scale) * double(p.loss) : 0.0; }

// What a row comes to, from its statistics: s relative to the reference e (far: to the maximum itself).
struct RowDone {
    double logp, shift;
    float m, s, ln_s, entropy, g, h;
    PolicyRow p;
};
template <int EPI, bool ENT>
__device__ __forceinline__ RowDone row_done(const LossArgs& a, const RowOf& w, const Scale& c, float x_token, float m, float e, float s, float q, bool far) {
    RowDone r;
    if (!(m >= -FLT_MAX && m <= FLT_MAX)) s = NAN;  // no distribution
    r.shift = far ? 0.0 : shift_of(m, e, w.inv_t);
    const double sum = far ? double(s) : mended(s, m, e, c, r.shift), ln_s = ln_of(sum);
    r.m = m, r.s = float(sum), r.ln_s = float(ln_s);
    r.logp = (double(x_token) - double(m)) * double(w.inv_t) - (ln_s + r.shift);
    if (r.logp > 0.0) r.logp = 0.0;  // (by the last bits of the sum)
    r.entropy = ENT ? float(ln_s - kLn2 * double(q / s)) : 0.f;  // (the terms' mean exponent is q / s)
    if (EPI == EPI_POLICY) r.p = policy_row(a, w, r.logp, r.entropy), r.g = w.scale > 0.f ? w.scale * r.p.dlogp : 0.f, r.h = -a.ent_coef * w.scale;
    return r;
}
// Writes what the call wants of a row.  One thread.
template <int EPI, bool ENT, bool TERM = true>
__device__ __forceinline__ void write_row(const LossArgs& a, int row, const RowOf& w, const RowDone& r) {
    const bool live = w.live;
    if (a.logp) a.logp[row] = live ? float(r.logp) : 0.f;
    if (a.stats) a.stats[2 * int64_t(row)] = live ? r.m : 0.f, a.stats[2 * int64_t(row) + 1] = live ? shifted(r.s, r.shift) : 0.f;
    if (ENT && a.entropy) a.entropy[row] = live ? r.entropy : 0.f;
    if (EPI == EPI_POLICY) {
        if (a.kl) a.kl[row] = live ? r.p.kl : 0.f;
        if (a.row_loss) a.row_loss[row] = live ? r.p.loss : 0.f;
        if (a.g_logp) a.g_logp[row] = live ? r.g : 0.f;
        if (a.g_entropy) a.g_entropy[row] = live ? r.h : 0.f;
        if (TERM) a.row_term[row] = live ? share_of(w, r.p) : 0.0;
    } else if (EPI == EPI_PREF) {
        a.row_term[row] = live ? double(w.weight) * (r.logp - (a.ref_logp ? double(w.ref_logp) : 0.0)) : 0.0;
        a.row_scale[row] = live ? w.weight : 0.f;
        a.g_logp[row] = 0.f;  // (the rows of a pair get theirs from pairs_kernel)
    }
}

__device__ double block_sum(double v, double* sh) {  // the same value in every thread
    v = warp_sum(v);
    __syncthreads();
    if (lane_id() == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = lane_id() < int(blockDim.x >> 5) ? sh[lane_id()] : 0.0;
    return warp_sum(t);
}

// A kernel that may start before the one ahead of it in the stream has ended waits here for that one's results (no wait where it
// was launched the ordinary way).
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The CTA that comes last adds up the terms, in their order.  (Called by `callers` CTAs in all, each after its own terms are written.)
__device__ void last_sum(uint32_t* ticket, unsigned callers, const double* terms, int count, double scale, float* loss) {
    __shared__ bool last;
    __shared__ double sh_d[32];
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(ticket, 1u) + 1u == callers;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double t = 0.0;
    const int stride = int(blockDim.x);
    for (int r = threadIdx.x; r < count; r += 8 * stride) {  // (eight loads at a time: one CTA, and nobody to hide its waits)
        double v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = int64_t(r) + k * stride < count ? __ldcg(terms + r + k * stride) : 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += v[k];
    }
    t = block_sum(t, sh_d);
    if (threadIdx.x == 0) *loss = float(t * scale);
}

__device__ __forceinline__ void copy_async16(void* smem, const void* g) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(g) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() {  // waits for this thread's copies but its last N groups
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 16 logits of one thread, in V vectors `stride` apart
template <typename T, bool ENT>
__device__ __forceinline__ void add_block(Soft& s, const uint4* v, int stride, const Scale& c) {
    constexpr int E = 16 / sizeof(T), V = 16 / E;
    float x[16];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        float e[E];
        unpack<T>(v[k * stride], e);
#pragma unroll
        for (int j = 0; j < E; ++j) x[k * E + j] = e[j];
    }
    add_many<ENT, 16>(s, x, c);
}
template <typename T, bool ENT>
__device__ __forceinline__ void add_vec(Soft& s, uint4 v, const Scale& c) {
    float e[16 / sizeof(T)];
    unpack<T>(v, e);
    add_many<ENT, 16 / sizeof(T)>(s, e, c);
}
// a far row's thread sums (see is_far); m: the row's maximum
template <typename T, bool ENT, int NT>
__device__ __noinline__ Soft far_sums(const uint4* v, int cnt, bool have_edge, float x_edge, float m, float hi, float lo) {
    constexpr int E = 16 / sizeof(T);
    Soft a{m, 0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x % NT; i < cnt; i += NT) {
        float x[E];
        unpack<T>(v[i], x);
        for (int j = 0; j < E; ++j) {
            const float t = far_exponent(x[j], m, hi, lo), w = ex2_approx(t);
            a.s += w;
            if (ENT) a.q = fmaf(w, fmaxf(t, -1000.f), a.q);
        }
    }
    if (have_edge) {
        const float t = far_exponent(x_edge, m, hi, lo), w = ex2_approx(t);
        a.s += w;
        if (ENT) a.q = fmaf(w, fmaxf(t, -1000.f), a.q);
    }
    return a;
}

// vectors that a thread of the forward kernel has under way: kFwdRing steps of 16 logits each
template <typename T>
constexpr int kFwdRing = sizeof(T) == 4 ? 3 : 6;

// Where a CTA's slice of a row lies: `per` 16-byte vectors of the row's body; the scalars before the first and behind the last boundary
// belong to rank 0, one per thread.
template <typename T>
struct Slice {
    const T* x;       // the row
    int head, nv, v0, cnt;
    int edge;         // this thread's scalar, -1 without one
    __device__ __forceinline__ Slice(const LossArgs& a, int row, int rank, int per) {
        constexpr int E = 16 / sizeof(T);
        x = static_cast<const T*>(a.x) + int64_t(row) * a.ld;
        head = head_of(x, a.n), nv = (a.n - head) / E;
        v0 = min(rank * per, nv), cnt = min(per, nv - v0);
        const int i = int(threadIdx.x);
        edge = rank == 0 && i < a.n - nv * E ? (i < head ? i : i + nv * E) : -1;  // (fewer than 2 E scalars, one per thread)
    }
    __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(x + head) + v0; }
};

// The cluster's statistics of a row from its threads' sums; valid in warp 0 of every CTA.  data: the CTA's vectors, read again for a
// far row.
template <typename T, bool ENT>
__device__ __forceinline__ Soft row_sum(Soft s, const Scale& c, ReduceShared& sh, int ctas, const uint4* data, int cnt, bool have_edge, float x_edge,
                                        bool& far) {
    s = reduce<ENT>(s, c, sh, ctas, 0);
    far = threadIdx.x < 32 && is_far(s.m, c);
    if (__syncthreads_or(far)) {  // (every CTA of the cluster has the same statistics)
        if (threadIdx.x == 0) sh.m[0] = s.m;
        __syncthreads();
        const float m = sh.m[0];
        __syncthreads();
        s = reduce_far<ENT>(far_sums<T, ENT, kRowThreads>(data, cnt, have_edge, x_edge, m, c.hi, c.lo), m, sh, ctas);
        far = true;
    }
    return s;
}

// Statistics: one cluster per row.  A thread reads what it copied into shared memory itself, so that the copies need no barrier.
template <typename T, int EPI, bool ENT>
__global__ void __launch_bounds__(kRowThreads, 4) forward_kernel(const __grid_constant__ LossArgs a, int per) {
    constexpr int E = 16 / sizeof(T), NT = kRowThreads, V = 16 / E, D = kFwdRing<T>;
    extern __shared__ __align__(16) uint4 ring[];
    __shared__ ReduceShared sh;
    const int ctas = int(cluster_size()), rank = int(cluster_rank()), tid = threadIdx.x;
    const int row = int(blockIdx.x / unsigned(ctas));
    RowOf w = row_of<EPI>(a, row, false);
    if (w.live) {
        const Slice<T> at(a, row, rank, per);
        const uint4* v = at.body();
        const int cnt = at.cnt;
        const Scale c = scale_of(w.inv_t);
        Soft s = soft_empty(c);
#pragma unroll 1
        for (int k = 0; k < D - 1; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int i = (k * V + j) * NT + tid;
                if (i < cnt) copy_async16(ring + i, v + i);
            }
            copies_commit();
        }
        const float x_token = tid == 0 ? load_one(at.x + w.token) : 0.f;
        float x_edge = 0.f;
        if (at.edge >= 0) {
            x_edge = load_one(at.x + at.edge);
            const float e[1] = {x_edge};
            add_many<ENT, 1>(s, e, c);
        }
        int slot = 0;  // of the step at hand; the one before it is where the next copies go
#pragma unroll 1
        for (int i = tid; i < cnt; i += V * NT) {
            const int to = slot == 0 ? D - 1 : slot - 1;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int k = i + ((D - 1) * V + j) * NT;
                if (k < cnt) copy_async16(ring + (to * V + j) * NT + tid, v + k);
            }
            copies_commit();
            copies_but<D - 1>();
            const uint4* b = ring + slot * V * NT + tid;
            if (i + (V - 1) * NT < cnt) {
                add_block<T, ENT>(s, b, NT, c);
            } else {
                for (int j = 0; i + j * NT < cnt; ++j) add_vec<T, ENT>(s, b[j * NT], c);
            }
            slot = slot + 1 == D ? 0 : slot + 1;
        }
        copies_but<0>();
        bool far;
        s = row_sum<T, ENT>(s, c, sh, ctas, v, cnt, at.edge >= 0, x_edge, far);
        if (tid == 0 && rank == 0) {
            grid_dependency_wait();  // row_scale_kernel's results
            if (EPI == EPI_POLICY) w.scale = a.row_scale[row];
            write_row<EPI, ENT>(a, row, w, row_done<EPI, ENT>(a, w, c, x_token, s.m, s.e, s.s, s.q, far));
        }
    } else if (tid == 0 && rank == 0) {
        grid_dependency_wait();
        write_row<EPI, ENT>(a, row, w, RowDone{});
    }
    if (EPI == EPI_POLICY && rank == 0) last_sum(a.ticket, unsigned(a.rows), a.row_term, a.rows, 1.0, a.loss);
}

constexpr int kFusedThreads = 256, kFusedCtas = 5, kRowWarps = kFusedThreads / 32;

// A warp's partial statistics of a row, on their way to every CTA of the cluster; x: the token's logit from the warp that has it, 0 from
// the others (nobody reads it from memory: dx may be x, and another CTA may have written its part of the row by then).
struct Part {
    float m, s, q, x;
};
// stores to shared memory of CTA `cta` and counts the bytes on its barrier
__device__ __forceinline__ void send(Part* to, uint64_t* bar, int cta, const Part& p) {
    asm volatile(
        "{\n .reg .b32 d, b;\n mapa.shared::cluster.u32 d, %0, %2;\n mapa.shared::cluster.u32 b, %1, %2;\n"
        " st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [d], {%3, %4, %5, %6}, [b];\n}\n" ::"r"(smem_u32(to)),
        "r"(smem_u32(bar)), "r"(cta), "r"(__float_as_uint(p.m)), "r"(__float_as_uint(p.s)), "r"(__float_as_uint(p.q)), "r"(__float_as_uint(p.x))
        : "memory");
}
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Each warp's sums to every CTA of the cluster (its lane i tells CTA i).
template <bool ENT>
__device__ __forceinline__ void tell(Soft a, float x_token, const Scale& c, Part* mine, uint64_t* bar, int ctas) {
    a.s -= a.k, a.k = 0.f;
    const float m = warp_max_f(a.m);
    raise<ENT>(a, m, c);
    a.s = warp_sum_f(a.s);
    if (ENT) a.q = warp_sum_f(a.q);
    if (lane_id() < ctas) send(mine, bar, lane_id(), Part{m, a.s, a.q, x_token});
}
// The row's statistics from n warps' (one warp).  false: they did not come in their time.
template <bool ENT>
__device__ __forceinline__ bool hear(const Scale& c, const Part* parts, uint64_t* bar, uint32_t parity, int n, uint32_t limit, Soft& s, float& x_token) {
    if (lane_id() == 0) mbar_expect_tx(bar, uint32_t(n * sizeof(Part)));
    if (!__all_sync(0xffffffffu, mbar_wait(bar, parity, limit))) return false;
    float m = -INFINITY;
    for (int i = lane_id(); i < n; i += 32) m = fmaxf(m, parts[i].m);
    m = warp_max_f(m);
    s = Soft{m, ref_of(m, c), 0.f, 0.f, 0.f};
    float x = 0.f;
    for (int i = lane_id(); i < n; i += 32) {
        const Part p = parts[i];
        Soft t{p.m, ref_of(p.m, c), p.s, 0.f, p.q};
        raise<ENT>(t, m, c);
        s.s += t.s, x += p.x;
        if (ENT) s.q += t.q;
    }
    x_token = warp_sum_f(x);
    s.s = warp_sum_f(s.s);
    if (ENT) s.q = warp_sum_f(s.q);
    return true;
}

namespace fused {
// What a CTA knows of its rows so far, in one register (there are 48), the same in every thread: which row of the two this is; not the first
// row; exchanges so far, modulo 4; one exchange at least; second exchanges, modulo 2; a wait ran out
enum : uint32_t { ODD = 1, LATER = 2, LIVE = 4, LIVES = 12, SEEN = 16, FAR = 32, GONE = 64 };
}  // namespace fused

// A row from its statistics (one thread): what its gradient is made of, and what the call wants of it.  The CTA waits for it, so what it needs
// comes first.
template <bool ENT>
__device__ __forceinline__ void finish_row(const LossArgs& a, const RowOf& w, int row, int rank, bool first, const Scale& c, float x_token, const Soft& s, bool far,
                                           GradRow& q, bool& zero) {
    RowOf wr = w;
    if (first) {
        grid_dependency_wait();  // row_scale_kernel's results
        wr.scale = a.row_scale[row];
    }
    const RowDone d = row_done<EPI_POLICY, ENT>(a, wr, c, x_token, s.m, s.e, s.s, s.q, far);
    zero = d.g == 0.f && d.h == 0.f;
    q = grad_row(d.m, far, d.s, d.ln_s, c, wr.inv_t, wr.token, d.g, d.h, d.entropy);
    if (rank == 0) write_row<EPI_POLICY, ENT>(a, row, wr, d);
}
// A far row, whose sums are made again and exchanged once more, or a row of a CTA that is GONE.  The whole CTA, behind a barrier: a wait
// that ran out says nothing about where the CTA's other warps are.
template <typename T, bool ENT>
__device__ __noinline__ uint32_t rare_row(const LossArgs& a, const RowOf& w, int row, int rank, int ctas, uint32_t st, Scale c, float x_token, const uint4* slice,
                                          int cnt, bool have_edge, float x_edge, Part* parts, uint64_t* bar, const float& row_m, GradRow& q, bool& zero) {
    using namespace fused;
    const bool far = !(st & GONE);
    const int n_parts = ctas * kRowWarps;
    Soft s{0.f, ref_of(0.f, c), NAN, 0.f, NAN};
    if (far) {  // (every CTA of the cluster has the same statistics)
        const float m = row_m;
        const Scale one{1.f, 0.f, FLT_MAX};
        s = far_sums<T, ENT, kFusedThreads>(slice, cnt, have_edge, x_edge, m, c.hi, c.lo);
        s.m = 0.f, s.e = ref_of(0.f, one);  // (references alike: nothing is scaled on the way)
        tell<ENT>(s, 0.f, one, parts + 2 * n_parts + rank * kRowWarps + int(threadIdx.x >> 5), bar + 2, ctas);
        bool out = false;
        if (threadIdx.x < 32) {
            float none;
            out = !hear<ENT>(one, parts + 2 * n_parts, bar + 2, st & FAR ? 1 : 0, n_parts, a.wait_limit, s, none);
            s.m = m;
        }
        st ^= FAR;
        if (__syncthreads_or(out)) st |= GONE;
    }
    if (threadIdx.x == 0) {
        if (st & GONE) {
            grid_dependency_wait();  // (row_scale_kernel clears the word)
            atomicExch(a.ticket + 1, 1u);
            s = Soft{0.f, ref_of(0.f, c), NAN, 0.f, NAN};
        }
        finish_row<ENT>(a, w, row, rank, !(st & LATER), c, x_token, s, !(st & GONE), q, zero);
    }
    __syncthreads();
    return st;
}

// The policy loss with its gradient.  The clusters stay and take rows in turn, each CTA holding its slice of a row in shared memory
// from the read to the gradient: one read and one write of global memory.  As soon as a thread has written a vector's
// gradient it starts the copy of the same vector of the cluster's next row into the same place, so that the memory is
// busy while the statistics of that row wait for it; several CTAs per SM fill each other's waits (the exchange of the statistics, the row's
// scalars).  The statistics travel by stores that count on the receiver's mbarrier: a cluster barrier would hold every row until the
// gradient's stores of the row before it are acknowledged.
// Should a CTA's wait run out (it has a limit; nothing makes it run out but a store that is lost), the CTA says so in the workspace and is
// GONE: this row and all its later ones are NaN, without another exchange, since the barriers' phases no longer
// match.  The cluster's other CTAs then miss its statistics and go the same way.
// What bounds it is the clusters' lockstep: every row waits for the slowest of its CTAs (1480 x 151936 bf16: DRAM at 55 % of the copy rate, the special
// function units at 56 %, warps at the barrier a third of their time).  Measured beside it on 4096 x 151936 bf16, a third of the rows masked (501 us with
// two launches and two reads, 500 to 505 here): one CTA an SM with a ring of slices and a warp of its own for the scalars, 770; tasks of
// statistics and of gradients drawn from one counter, the second read from L2, 520 to 600; 384 or 512 threads, 534 and 554.
template <typename T, bool ENT>
__global__ void __launch_bounds__(kFusedThreads, kFusedCtas) fused_kernel(const __grid_constant__ LossArgs a, int per) {
    constexpr int EPI = EPI_POLICY;
    constexpr int E = 16 / sizeof(T), NT = kFusedThreads, V = 16 / E;
    extern __shared__ __align__(16) uint4 slice[];  // `per` vectors, then three sets of partial statistics (rows in turn; far rows)
    __shared__ GradRow s_q;
    __shared__ RowOf s_row[2];
    __shared__ uint64_t s_bar[3];
    __shared__ float s_m;
    __shared__ bool s_zero, s_far;
    const int ctas = int(cluster_size()), rank = int(cluster_rank()), tid = threadIdx.x;
    const int clusters = int(gridDim.x / unsigned(ctas));
    const int n_parts = ctas * kRowWarps, my_part = rank * kRowWarps + (tid >> 5);
    Part* const parts = reinterpret_cast<Part*>(slice + per);
    int row = int(blockIdx.x / unsigned(ctas));
    using namespace fused;
    uint32_t st = 0;
    if (tid < 32) {
        const RowOf w = row_of<EPI>(a, row, false);
        if (tid == 0) {
            s_row[0] = w;
            for (int i = 0; i < 3; ++i) mbar_init(&s_bar[i], 1);
            mbar_fence_init();
        }
    }
    __syncthreads();
    if (s_row[0].live) {
        const Slice<T> at(a, row, rank, per);
        const uint4* v = at.body();
#pragma unroll 4
        for (int i = tid; i < at.cnt; i += NT) copy_async16(slice + i, v + i);
        copies_commit();
    }
    cluster_barrier();  // every CTA's barriers are ready
#pragma unroll 1
    for (; row < a.rows; st = (st ^ ODD) | LATER, row += clusters) {
        const RowOf& w = s_row[st & ODD];
        const bool more = a.rows - row > clusters;
        if (more && tid >= NT - 32) {  // the next row's scalars; the wait is over at once but for the first row
            grid_dependency_wait();
            const RowOf r = row_of<EPI>(a, row + clusters, true);
            if (tid == NT - 32) s_row[(st ^ ODD) & ODD] = r;
        }
        const Slice<T> at(a, row, rank, per);
        const int cnt = at.cnt;
        float x_edge = 0.f;
        bool zero = true;
        if (w.live) {
            const Scale c = scale_of(w.inv_t);
            Soft s = soft_empty(c);
            if (at.edge >= 0) {
                x_edge = load_one(at.x + at.edge);
                const float e[1] = {x_edge};
                add_many<ENT, 1>(s, e, c);
            }
            copies_but<0>();
            int i = tid;
#pragma unroll 1
            for (; i + (V - 1) * NT < cnt; i += V * NT) add_block<T, ENT>(s, slice + i, NT, c);
#pragma unroll 1
            for (; i < cnt; i += NT) add_vec<T, ENT>(s, slice[i], c);
            // the token's logit goes along: one lane of the cluster has it
            const int tok = w.token - at.head - at.v0 * E;
            float x_token = at.edge >= 0 && w.token == at.edge ? x_edge : 0.f;
            if (tok >= 0 && tok < cnt * E && (tok / E) % NT == tid) x_token = load_one(reinterpret_cast<const T*>(slice) + tok);
            x_token = warp_sum_f(x_token);
            const int set = st & LIVE ? 1 : 0;
            const bool lose = a.lose_part && !(st & SEEN) && int(blockIdx.x) == ctas - 1 && tid < 32;
            if (!(st & GONE) && !lose) tell<ENT>(s, x_token, c, parts + set * n_parts + my_part, &s_bar[set], ctas);
            bool out = false;
            if (tid < 32 && !(st & GONE)) {
                out = !hear<ENT>(c, parts + set * n_parts, &s_bar[set], st & (2 * LIVE) ? 1 : 0, n_parts, a.wait_limit, s, x_token);
                if (tid == 0 && !out) {
                    s_far = is_far(s.m, c), s_m = s.m;
                    if (!is_far(s.m, c)) finish_row<ENT>(a, w, row, rank, !(st & LATER), c, x_token, s, false, s_q, s_zero);
                }
            }
            st = (st & ~LIVES) | ((st + LIVE) & LIVES) | SEEN;
            if (__syncthreads_or(out)) st |= GONE;
            if ((st & GONE) || s_far)
                st = rare_row<T, ENT>(a, w, row, rank, ctas, st, c, x_token, slice, cnt, at.edge >= 0, x_edge, parts, s_bar, s_m, s_q, s_zero);
            zero = s_zero;
        } else {
            if (tid == 0) {
                if (!(st & LATER)) grid_dependency_wait();
                if (rank == 0) write_row<EPI, ENT>(a, row, w, RowDone{});
            }
            __syncthreads();
        }
        // (s_row of the next row, s_q and s_zero are in place; their next writes come after every thread has read them: s_row's behind the
        // next row's barrier but one, the others' behind all warps' `tell` of the next row, or behind its barrier if that is not heard)
        GradRow q{};
        if (!zero) q = s_q;
        T* dx = static_cast<T*>(a.dx) + int64_t(row) * a.ld_dx;
        if (at.edge >= 0) store_one(dx + at.edge, zero ? 0.f : grad_of<ENT>(q, x_edge) + (at.edge == q.token ? q.d : 0.f));
        const bool vec = ((reinterpret_cast<uintptr_t>(at.x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
        T* body = dx + at.head + int64_t(at.v0) * E;
        uint4* out = reinterpret_cast<uint4*>(body);
        // the token's own element is written again by the thread that wrote its vector
        const int t = zero ? -1 : q.token - at.head - at.v0 * E;
        const bool mine = t >= 0 && t < cnt * E && (t / E) % NT == tid;
        const float x_mine = mine ? load_one(reinterpret_cast<const T*>(slice) + t) : 0.f;
        const uint4* next = nullptr;
        int refill = 0;
        if (more && s_row[(st ^ ODD) & ODD].live) {
            const Slice<T> n(a, row + clusters, rank, per);
            next = n.body(), refill = n.cnt;
        }
        int i = tid;
        if (zero && vec) {
#pragma unroll 4
            for (; i < cnt; i += NT) __stcs(out + i, make_uint4(0, 0, 0, 0));
            i = tid;  // (nothing refilled yet)
        } else if (vec && !q.far) {
            const int both = min(cnt, refill);
#pragma unroll 2
            for (; i < both; i += NT) {
                const uint4 g = grad_vec<T, ENT>(q, slice[i]);
                __stcs(out + i, g);
                copy_async16(slice + i, next + i);
            }
            for (int j = i; j < cnt; j += NT) __stcs(out + j, grad_vec<T, ENT>(q, slice[j]));
        } else {
            for (; i < cnt; i += NT) {
#pragma unroll 1
                for (int j = 0; j < E; ++j)
                    store_one(body + int64_t(i) * E + j, zero ? 0.f : grad_of<ENT>(q, load_one(reinterpret_cast<const T*>(slice + i) + j)));
            }
            i = tid;
        }
        if (mine) store_one(body + t, grad_of<ENT>(q, x_mine) + q.d);
#pragma unroll 4
        for (; i < refill; i += NT) copy_async16(slice + i, next + i);
        copies_commit();
    }
    copies_but<0>();
    cluster_barrier();  // nobody leaves while another CTA has stores for it to send
    if (st & GONE)      // ... or, where it did not wait for them, while they are under way
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (rank == 0) last_sum(a.ticket, unsigned(clusters), a.row_term, a.rows, 1.0, a.loss);
}

// ---------------------------------------------------------------------------------------------------------------
// short rows: a warp each
// ---------------------------------------------------------------------------------------------------------------

// A row of up to 8 KB fits the registers of one warp: it is read once, its statistics need no shared memory and no barrier, and (GRAD) its
// gradient is written from the registers.  The kernels above spend 4 to 7 us of a CTA on a row however short it is: 8000 rows of
// 2000 bf16 logits, policy loss with gradient, took 72 us with fused_kernel and take 33 here.
constexpr int kSmallRowThreads = 256, kSmallVectors = 16;  // vectors a lane, at most

// writes the gradient of a row's vectors from `first` on that a warp has in registers (q of zeros: zeros)
template <typename T, bool ENT, int K>
__device__ __forceinline__ void small_grad(const GradRow& q, const T* x, T* dx, int head, int first, int nv, int edge, float x_edge, const uint4 (&b)[K]) {
    constexpr int E = 16 / sizeof(T);
    __syncwarp();  // (every lane has read what it wants of the row: dx may be x)
    const bool zero = q.a == 0.f && q.b == 0.f && q.d == 0.f;
    const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int t = zero ? -1 : q.token - head;  // the token's place among the vectors
    if (edge >= 0) store_one(dx + edge, zero ? 0.f : grad_of<ENT>(q, x_edge) + (edge == q.token ? q.d : 0.f));
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = first + k * 32 + lane_id();
        if (i >= nv) continue;
        float e[E];
        if (zero) {
#pragma unroll
            for (int j = 0; j < E; ++j) e[j] = 0.f;
        } else {
            unpack<T>(b[k], e);
            if (!q.far) grad_many<ENT, E>(q, e);
            else
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = grad_of<ENT>(q, e[j]);
            if (t >= 0 && t / E == i)
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] += t % E == j ? q.d : 0.f;
        }
        if (vec) {
            __stcs(reinterpret_cast<uint4*>(dx + head) + i, pack<T>(e));
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) store_one(dx + head + int64_t(i) * E + j, e[j]);
        }
    }
}
// the row's scalars from given statistics
__device__ __forceinline__ GradRow grad_row_of(const LossArgs& a, int row, int token, float g, float h, bool ent) {
    const float inv_t = a.inv_t_rows ? a.inv_t_rows[row] : a.inv_t;
    const float m = a.stats[2 * int64_t(row)], sum = a.stats[2 * int64_t(row) + 1];
    const Scale c = scale_of(inv_t);
    const bool far = is_far(m, c);
    const double y = far ? 0.0 : shift_of(m, ref_of(m, c), inv_t);
    return grad_row(m, far, shifted(sum, -y), float(ln_of(double(sum)) - y), c, inv_t, token, g, h, ent ? a.entropy[row] : 0.f);
}

template <typename T, int EPI, bool ENT, bool GRAD, int K>
__global__ void __launch_bounds__(kSmallRowThreads, K > 8 ? 2 : 3) small_rows_kernel(const __grid_constant__ LossArgs a) {
    constexpr int E = 16 / sizeof(T);
    const int lane = lane_id();
    if (EPI == EPI_POLICY) grid_dependency_wait();  // row_scale_kernel's results
    const int warps = int(gridDim.x) * (kSmallRowThreads / 32);
    double total = 0.0;  // policy loss: this warp's share (its rows are always the same, in the same order)
    int64_t row64 = int64_t(blockIdx.x) * (kSmallRowThreads / 32) + (threadIdx.x >> 5);
    uint32_t words = row64 < a.rows ? row_word<EPI>(a, int(row64), true) : 0u;
#pragma unroll 1
    for (; row64 < a.rows; row64 += warps) {
        const int row = int(row64);
        const RowOf w = row_from<EPI>(a, row, words);
        if (row64 + warps < a.rows) words = row_word<EPI>(a, int(row64 + warps), true);  // (here by the time it is wanted)
        const T* x = static_cast<const T*>(a.x) + row64 * a.ld;
        T* const dx = GRAD ? static_cast<T*>(a.dx) + row64 * a.ld_dx : nullptr;
        const int head = head_of(x, a.n), nv = (a.n - head) / E, beside = a.n - nv * E;
        const uint4* v = reinterpret_cast<const uint4*>(x + head);
        const int edge = lane < beside ? (lane < head ? lane : lane + nv * E) : -1;  // (fewer than 2 E of them)
        uint4 b[K];
        float x_edge = 0.f;
        GradRow q{};
        if (w.live) {
auto load = [&](int first) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (first + k * 32 < nv) b[k] = first + k * 32 + lane < nv ? v[first + k * 32 + lane] : make_uint4(0, 0, 0, 0);
            };
            load(0);
            const float x_token = load_one(x + w.token);
            const Scale c = scale_of(w.inv_t);
            Soft s = soft_empty(c);
            if (edge >= 0) {
                x_edge = load_one(x + edge);
                const float e[1] = {x_edge};
                add_many<ENT, 1>(s, e, c);
            }
#pragma unroll 1
            for (int first = 0;;) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (first + k * 32 + lane < nv) add_vec<T, ENT>(s, b[k], c);
                first += 32 * K;
                if (GRAD || first >= nv) break;  // (with GRAD the row is in the registers as a whole)
                load(first);
            }
            __syncwarp();
            s.s -= s.k, s.k = 0.f;
            const float m = warp_max_f(s.m);
            raise<ENT>(s, m, c);
            s.s = warp_sum_f(s.s);
            if (ENT) s.q = warp_sum_f(s.q);
            const bool far = is_far(m, c);
            if (far) {
                Soft t = far_sums<T, ENT, 32>(v, nv, edge >= 0, x_edge, m, c.hi, c.lo);
                s.s = warp_sum_f(t.s), s.q = warp_sum_f(t.q);
            }
            const RowDone d = row_done<EPI, ENT>(a, w, c, x_token, s.m, s.e, s.s, s.q, far);
            if (lane == 0) write_row<EPI, ENT, EPI != EPI_POLICY>(a, row, w, d);
            if (EPI == EPI_POLICY) total += share_of(w, d.p);
            if (GRAD && !(d.g == 0.f && d.h == 0.f)) q = grad_row(d.m, far, d.s, d.ln_s, c, w.inv_t, w.token, d.g, d.h, d.entropy);
        } else if (lane == 0) {
            write_row<EPI, ENT, EPI != EPI_POLICY>(a, row, w, RowDone{});
        }
        if (GRAD) {
            small_grad<T, ENT, K>(q, x, dx, head, 0, nv, edge, x_edge, b);
        }
    }
    if (EPI == EPI_POLICY) {
        __shared__ double s_total[kSmallRowThreads / 32];
        if (lane == 0) s_total[threadIdx.x >> 5] = total;
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int i = 0; i < kSmallRowThreads / 32; ++i) t += s_total[i];
            a.row_term[blockIdx.x] = t;  // (a term per CTA: there are fewer of them than rows)
        }
        last_sum(a.ticket, gridDim.x, a.row_term, int(gridDim.x), 1.0, a.loss);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// gradient: grid = (rows, chunks)
// ---------------------------------------------------------------------------------------------------------------

constexpr int kGradThreads = 256;

template <typename T, bool ENT>
__global__ void __launch_bounds__(kGradThreads, 6) grad_kernel(const __grid_constant__ LossArgs a, int chunk) {
    constexpr int E = 16 / sizeof(T), NT = kGradThreads;
    __shared__ GradRow s_q;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int64_t j0 = int64_t(blockIdx.y) * chunk;
    const int n = a.n - j0 < chunk ? int(a.n - j0) : chunk;
    const T* x = static_cast<const T*>(a.x) + int64_t(row) * a.ld + j0;
    T* dx = static_cast<T*>(a.dx) + int64_t(row) * a.ld_dx + j0;
    const int token = a.token[row];
    const float g = a.g_logp[row], h = ENT ? a.g_entropy[row] : 0.f;
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int head = same ? head_of(x, n) : n, nv = (n - head) / E;
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
    uint4* dv = reinterpret_cast<uint4*>(dx + head);
    if (unsigned(token) >= unsigned(a.n) || (g == 0.f && h == 0.f)) {  // not read
#pragma unroll 4
        for (int i = tid; i < nv; i += NT) __stcs(dv + i, make_uint4(0, 0, 0, 0));
        for (int i = tid; i < n - nv * E; i += NT) store_one(dx + (i < head ? i : i + nv * E), 0.f);
        return;
    }
    // the first vectors are under way while one thread makes the row's scalars
    int i = tid;
    uint4 b[4];
    if (i + 3 * NT < nv) {
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = v[i + k * NT];
    }
    if (tid == 0) s_q = grad_row_of(a, row, token, g, h, ENT);
    // the token's own logit, before anything is written (dx may be x)
    const int64_t t64 = int64_t(token) - j0;
    const int at = t64 >= 0 && t64 < n ? int(t64) : -1, t_vec = at - head;
    const bool mine = at >= head && t_vec < nv * E && (t_vec / E) % NT == tid;
    const float x_token = mine ? load_one(x + at) : 0.f;
    __syncthreads();
    const GradRow q = s_q;
    if (!q.far) {
#pragma unroll 1
        while (i + 3 * NT < nv) {
            uint4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = grad_vec<T, ENT>(q, b[k]);
            const int next = i + 4 * NT;
            if (next + 3 * NT < nv) {
#pragma unroll
                for (int k = 0; k < 4; ++k) b[k] = v[next + k * NT];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) __stcs(dv + i + k * NT, o[k]);
            i = next;
        }
#pragma unroll 1
        for (; i < nv; i += NT) __stcs(dv + i, grad_vec<T, ENT>(q, v[i]));
        if (mine) store_one(dx + at, grad_of<ENT>(q, x_token) + q.d);
    } else {  // one by one
        for (int k = tid; k < nv * E; k += NT) {
            const int j = head + k;
            store_one(dx + j, grad_of<ENT>(q, load_one(x + j)) + (j == at ? q.d : 0.f));
        }
    }
    for (int k = tid; k < n - nv * E; k += NT) {
        const int j = k < head ? k : k + nv * E;
        store_one(dx + j, grad_of<ENT>(q, load_one(x + j)) + (j == at ? q.d : 0.f));
    }
}

// Short rows (see small_rows_kernel): a warp each.  60000 rows of 2000 bf16 logits: grad_kernel 186 us, this one 88.
template <typename T, bool ENT, int K>
__global__ void __launch_bounds__(kSmallRowThreads, K > 8 ? 2 : 3) small_grad_kernel(const __grid_constant__ LossArgs a) {
    constexpr int E = 16 / sizeof(T);
    const int lane = lane_id();
    const int64_t warps = int64_t(gridDim.x) * (kSmallRowThreads / 32);
#pragma unroll 1
    for (int64_t row64 = int64_t(blockIdx.x) * (kSmallRowThreads / 32) + (threadIdx.x >> 5); row64 < a.rows; row64 += warps) {
        const int row = int(row64), token = a.token[row];
        const float g = a.g_logp[row], h = ENT ? a.g_entropy[row] : 0.f;
        const T* x = static_cast<const T*>(a.x) + row64 * a.ld;
        const int head = head_of(x, a.n), nv = (a.n - head) / E, beside = a.n - nv * E;
        const uint4* v = reinterpret_cast<const uint4*>(x + head);
        const int edge = lane < beside ? (lane < head ? lane : lane + nv * E) : -1;
        uint4 b[K];
        float x_edge = 0.f;
        GradRow q{};
        const bool zero = unsigned(token) >= unsigned(a.n) || (g == 0.f && h == 0.f);
        T* const dx = static_cast<T*>(a.dx) + row64 * a.ld_dx;
#pragma unroll 1
        for (int first = 0;;) {
            if (!zero) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (first + k * 32 < nv) b[k] = first + k * 32 + lane < nv ? v[first + k * 32 + lane] : make_uint4(0, 0, 0, 0);
                if (first == 0) {
                    if (edge >= 0) x_edge = load_one(x + edge);
                    q = grad_row_of(a, row, token, g, h, ENT);
                }
            }
            small_grad<T, ENT, K>(q, x, dx, head, first, nv, first == 0 ? edge : -1, x_edge, b);
            first += 32 * K;
            if (first >= nv) break;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// weights, pairs, sums: small kernels
// ---------------------------------------------------------------------------------------------------------------

constexpr int kSmallThreads = 1024;

__device__ __forceinline__ float live_weight(const LossArgs& a, int row) {
    const int token = a.token[row];
    const float w = a.weight ? a.weight[row] : 1.f;  // (both loads before the first is looked at)
    return unsigned(token) < unsigned(a.n) && w > 0.f ? w : 0.f;
}
// the rows of sequence s, inside the batch whatever seq_start says
__device__ __forceinline__ int2 rows_of(const LossArgs& a, int s) {
    const int b = min(max(a.seq_start[s], 0), a.rows);
    return make_int2(b, min(max(a.seq_start[s + 1], b), a.rows));
}

// row_scale[rows] of the policy loss.  One CTA.
__device__ void row_scales(const LossArgs& a, int mean, double* sh) {
    const int tid = threadIdx.x;
    if (mean != WHIRL_MEAN_SEQS) {
        double k = 1.0;
        if (mean == WHIRL_MEAN_TOKENS) {
            double t = 0.0;
#pragma unroll 8
            for (int r = tid; r < a.rows; r += kSmallThreads) t += live_weight(a, r);
            t = block_sum(t, sh);
            k = t > 0.0 ? 1.0 / t : 0.0;
        }
#pragma unroll 8
        for (int r = tid; r < a.rows; r += kSmallThreads) a.row_scale[r] = float(k * live_weight(a, r));
        return;
    }
    // a warp per sequence: its weight's sum, then (knowing how many sequences have one) its rows
    for (int r = tid; r < a.rows; r += kSmallThreads) a.row_scale[r] = 0.f;
    double have = 0.0;
    for (int s = tid >> 5; s < a.seqs; s += kSmallThreads / 32) {
        const int2 b = rows_of(a, s);
        double t = 0.0;
        for (int r = b.x + lane_id(); r < b.y; r += 32) t += live_weight(a, r);
        t = warp_sum(t);
        if (lane_id() == 0) a.seq_term[s] = t, have += t > 0.0;
    }
    have = block_sum(have, sh);  // (its barriers also order the zeros before the scales)
    for (int s = tid >> 5; s < a.seqs; s += kSmallThreads / 32) {
        const double t = a.seq_term[s];
        if (!(t > 0.0)) continue;
        const int2 b = rows_of(a, s);
        for (int r = b.x + lane_id(); r < b.y; r += 32) a.row_scale[r] = float(double(live_weight(a, r)) / t / have);
    }
}
__global__ void __launch_bounds__(kSmallThreads) row_scale_kernel(const __grid_constant__ LossArgs a, int mean) {
    __shared__ double sh[32];
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) a.ticket[0] = a.ticket[1] = 0;
    row_scales(a, mean, sh);
}

// Loss of a pair and its derivative by h.
__device__ double2 pair_loss_of(const PairArgs& p, double h) {
    double loss, dh;
    if (p.kind == WHIRL_PREF_SIGMOID) {
        const double ls = p.smoothing, e = exp(-fabs(h)), l = log1p(e);
        const double up = h >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e), down = h >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e);
        // -log sigmoid(h) = max(-h, 0) + log(1 + e^-|h|)
        loss = (ls == 1.0 ? 0.0 : (1.0 - ls) * ((h < 0.0 ? -h : 0.0) + l)) + (ls == 0.0 ? 0.0 : ls * ((h > 0.0 ? h : 0.0) + l));
        if (h != h) loss = h;
        dh = ls * up - (1.0 - ls) * down;
    } else if (p.kind == WHIRL_PREF_HINGE) {
        loss = h != h ? h : (h < 1.0 ? 1.0 - h : 0.0);
        dh = h != h ? h : (h < 1.0 ? -1.0 : 0.0);
    } else {
        const double t = (h - 0.5) / double(p.beta);
        loss = t * t, dh = 2.0 * t / double(p.beta);
    }
    return make_double2(loss, dh);
}
__device__ void write_pair(const LossArgs& a, const PairArgs& p, int i, double loss, double chosen, double rejected) {
    a.seq_term[i] = loss;
    if (p.pair_loss) p.pair_loss[i] = float(loss);
    if (p.reward) p.reward[2 * i] = float(double(p.beta) * chosen), p.reward[2 * i + 1] = float(double(p.beta) * rejected);
}
// The sequences' sums of pair i, its loss, and the factor of every row's weight in g_logp (chosen, rejected).  The whole CTA.
__device__ double2 pair_done(const LossArgs& a, const PairArgs& p, int i, int2 (&b)[2], double* sh) {
    const int first = int(threadIdx.x), stride = int(blockDim.x);
    double P[2], W[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        b[k] = rows_of(a, 2 * i + k);
        double t = 0.0, w = 0.0;
#pragma unroll 8
        for (int r = b[k].x + first; r < b[k].y; r += stride) t += __ldcg(a.row_term + r), w += double(__ldcg(a.row_scale + r));
        P[k] = block_sum(t, sh);
        W[k] = 1.0;
        if (p.average) {
            w = block_sum(w, sh);
            W[k] = w > 0.0 ? 1.0 / w : 0.0;
            P[k] = w > 0.0 ? P[k] / w : 0.0;
        }
    }
    const double2 l = pair_loss_of(p, double(p.beta) * (P[0] - P[1]) - double(p.margin));
    if (first == 0) write_pair(a, p, i, l.x, P[0], P[1]);
    const double coef = double(p.beta) * l.y / double(p.pairs);
    return make_double2(coef * W[0], -coef * W[1]);
}

// One CTA per pair: the sequences' sums, the pair's loss, and the rows' g_logp.
constexpr int kPairThreads = 256;
__global__ void __launch_bounds__(kPairThreads) pairs_kernel(const __grid_constant__ LossArgs a, const __grid_constant__ PairArgs p) {
    __shared__ double sh[32];
    int2 b[2];
    const double2 c = pair_done(a, p, blockIdx.x, b, sh);
    for (int k = 0; k < 2; ++k)
        for (int r = b[k].x + int(threadIdx.x); r < b[k].y; r += kPairThreads) {
            const float w = a.row_scale[r];  // 0: the row does not count, whatever the pair comes to (NaN, infinity)
            a.g_logp[r] = w > 0.f ? float((k ? c.y : c.x) * double(w)) : 0.f;
        }
    last_sum(a.ticket, gridDim.x, a.seq_term, p.pairs, 1.0 / p.pairs, a.loss);
}

// A launch by clusters of `ctas` CTAs: one cluster per row, or (persistent) as many as fit at once.
template <typename... P>
cudaError_t cluster_launch(void (*f)(LossArgs, P...), std::atomic<uint64_t>& ready, const LossArgs& a, int ctas, int threads, size_t smem, bool persistent,
                           bool follows, cudaStream_t st, P... rest) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {  // bit per device: the function's limits are raised
        e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMost);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(unsigned(threads)), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(ctas), at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    int clusters = a.rows;
    if (persistent) {
        int fit = 0;
        cfg.gridDim = dim3(unsigned(ctas));
        e = cudaOccupancyMaxActiveClusters(&fit, f, &cfg);
        if (e != cudaSuccess) return e;
        clusters = std::min(clusters, std::max(fit, 1));
    }
    cfg.gridDim = dim3(unsigned(clusters) * unsigned(ctas));
    cfg.numAttrs = follows ? 2 : 1;  // (the policy loss follows row_scale_kernel)
    e = cudaLaunchKernelEx(&cfg, f, a, rest...);
    count_launch(LAUNCH_LOSS);
    return e;
}

int vectors_of(int n, int dtype) { return int((int64_t(n) * (dtype == WHIRL_F32 ? 4 : 2) + 15) / 16); }

// A warp per row: where it holds the whole row in its registers; or, where a row is read and done with piece by piece, for rows of up to 32 KB
// (statistics) or 16 KB (gradient) of which there are enough to fill the GPU with warps.  20000 rows of 4200 bf16 logits: statistics by CTAs 120 us, by warps
// 62; gradient 97 and 76.  3000 rows of 16000: statistics 31 by warps and 33 by CTAs, gradient 48 and 36.
bool is_small(int n, int dtype) { return vectors_of(n, dtype) <= 32 * kSmallVectors; }
bool is_short(const LossArgs& a, int dtype, int vectors) { return is_small(a.n, dtype) || (a.rows >= 148 * 16 && vectors_of(a.n, dtype) <= vectors); }
template <typename T, int EPI, bool ENT, bool GRAD>
cudaError_t small_typed(const LossArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    const int64_t want = (int64_t(a.rows) + kSmallRowThreads / 32 - 1) / (kSmallRowThreads / 32);
    cfg.gridDim = dim3(unsigned(std::min<int64_t>(want, 148 * 8))), cfg.blockDim = dim3(kSmallRowThreads), cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = EPI == EPI_POLICY ? 1 : 0;  // (the policy loss follows row_scale_kernel)
    const bool half = vectors_of(a.n, sizeof(T) == 4 ? WHIRL_F32 : WHIRL_BF16) <= 32 * 8;  // rows of up to 4 KB: half the registers, half as many warps more
    const cudaError_t e = half ? cudaLaunchKernelEx(&cfg, small_rows_kernel<T, EPI, ENT, GRAD, 8>, a) : cudaLaunchKernelEx(&cfg, small_rows_kernel<T, EPI, ENT, GRAD, 16>, a);
    count_launch(LAUNCH_LOSS);
    return e;
}
template <int EPI, bool GRAD>
cudaError_t small_launch(const LossArgs& a, int dtype, bool ent, cudaStream_t st) {
    if (dtype == WHIRL_F32) return ent ? small_typed<float, EPI, true, GRAD>(a, st) : small_typed<float, EPI, false, GRAD>(a, st);
    return ent ? small_typed<uint16_t, EPI, true, GRAD>(a, st) : small_typed<uint16_t, EPI, false, GRAD>(a, st);
}

template <typename T, int EPI, bool ENT>
cudaError_t forward_typed(const LossArgs& a, int ctas, int per, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return cluster_launch(forward_kernel<T, EPI, ENT>, ready, a, ctas, kRowThreads, size_t(kFwdRing<T>) * 16 * sizeof(T) * kRowThreads, false, EPI == EPI_POLICY, st, per);
}
template <int EPI>
cudaError_t forward_launch(const LossArgs& a, int dtype, bool ent, cudaStream_t st) {
    if (is_short(a, dtype, 2048)) return small_launch<EPI, false>(a, dtype, ent, st);
    const int nv = vectors_of(a.n, dtype);
    // Enough CTAs to fill the GPU three times over, 2 steps of the ring each at least: 1024 rows of 262144 f32 logits take 159 us with two
    // CTAs a row, 164 with one, 182 with four.
    int ctas = 1;
    while (ctas < 16 && int64_t(a.rows) * ctas < 1776 && nv / (2 * ctas) >= 2 * kRowThreads) ctas *= 2;
    const int per = (nv + ctas - 1) / ctas;
    if (dtype == WHIRL_F32) return ent ? forward_typed<float, EPI, true>(a, ctas, per, st) : forward_typed<float, EPI, false>(a, ctas, per, st);
    return ent ? forward_typed<uint16_t, EPI, true>(a, ctas, per, st) : forward_typed<uint16_t, EPI, false>(a, ctas, per, st);
}

template <typename T, bool ENT>
cudaError_t fused_typed(const LossArgs& a, int ctas, int per, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return cluster_launch(fused_kernel<T, ENT>, ready, a, ctas, kFusedThreads, size_t(per) * 16 + 3 * size_t(ctas) * kRowWarps * sizeof(Part), true, true, st, per);
}

}  // namespace

cudaError_t logprobs_launch(const LossArgs& a, int dtype, cudaStream_t st) { return forward_launch<EPI_NONE>(a, dtype, a.entropy != nullptr, st); }

template <typename T, bool ENT>
static cudaError_t small_grad_typed(const LossArgs& a, cudaStream_t st) {
    const dim3 grid(unsigned(std::min<int64_t>((int64_t(a.rows) + kSmallRowThreads / 32 - 1) / (kSmallRowThreads / 32), 148 * 8)));
    const bool half = vectors_of(a.n, sizeof(T) == 4 ? WHIRL_F32 : WHIRL_BF16) <= 32 * 8;
    if (half) small_grad_kernel<T, ENT, 8><<<grid, kSmallRowThreads, 0, st>>>(a);
    else small_grad_kernel<T, ENT, 16><<<grid, kSmallRowThreads, 0, st>>>(a);
    count_launch(LAUNCH_LOSS);
    return cudaGetLastError();
}

cudaError_t logprobs_grad_launch(const LossArgs& a, int dtype, cudaStream_t st) {
    if (is_short(a, dtype, 1024)) {
        if (dtype == WHIRL_F32) return a.g_entropy ? small_grad_typed<float, true>(a, st) : small_grad_typed<float, false>(a, st);
        return a.g_entropy ? small_grad_typed<uint16_t, true>(a, st) : small_grad_typed<uint16_t, false>(a, st);
    }
    // (a chunk per CTA; at most 65535 of them per row)
    const int chunk = int(std::max<int64_t>(16384, (int64_t(a.n) + 65534) / 65535));
    const dim3 grid(unsigned(a.rows), unsigned((int64_t(a.n) + chunk - 1) / chunk)), block(kGradThreads);
    if (dtype == WHIRL_F32) {
        if (a.g_entropy) grad_kernel<float, true><<<grid, block, 0, st>>>(a, chunk);
        else grad_kernel<float, false><<<grid, block, 0, st>>>(a, chunk);
    } else {
        if (a.g_entropy) grad_kernel<uint16_t, true><<<grid, block, 0, st>>>(a, chunk);
        else grad_kernel<uint16_t, false><<<grid, block, 0, st>>>(a, chunk);
    }
    count_launch(LAUNCH_LOSS);
    return cudaGetLastError();
}

cudaError_t policy_launch(const LossArgs& a, int dtype, int mean, cudaStream_t st) {
    row_scale_kernel<<<1, kSmallThreads, 0, st>>>(a, mean);
    count_launch(LAUNCH_LOSS);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const bool ent = a.ent_coef != 0.f || a.entropy;
    const int nv = vectors_of(a.n, dtype);
    if (a.dx && is_small(a.n, dtype)) return small_launch<EPI_POLICY, true>(a, dtype, ent, st);
    // The smallest cluster whose slices leave room for three CTAs an SM (rows of 1 MB: 16 CTAs 489 us, 8 CTAs 636; 512 KB: 8 CTAs 256, 16 CTAs
    // 277, 4 CTAs 309; 300 KB: 8 CTAs 487, 4 CTAs 535, 16 CTAs 663), and a larger one where the rows would not fill the GPU.
    int ctas = 1;
    while (ctas < 16 && int64_t(nv + ctas - 1) / ctas * 16 > 70 * 1024) ctas *= 2;
    while (ctas < 16 && int64_t(a.rows) * ctas < 592 && nv / (2 * ctas) >= kFusedThreads) ctas *= 2;
    const int64_t per = (int64_t(nv) + ctas - 1) / ctas;
    if (a.dx && per * 16 <= kSharedMost - 8192) {
        if (dtype == WHIRL_F32) return ent ? fused_typed<float, true>(a, ctas, int(per), st) : fused_typed<float, false>(a, ctas, int(per), st);
        return ent ? fused_typed<uint16_t, true>(a, ctas, int(per), st) : fused_typed<uint16_t, false>(a, ctas, int(per), st);
    }
    e = forward_launch<EPI_POLICY>(a, dtype, ent, st);
    return e == cudaSuccess && a.dx ? logprobs_grad_launch(a, dtype, st) : e;
}

cudaError_t preference_launch(const LossArgs& a, const PairArgs& p, int dtype, cudaStream_t st) {
    cudaError_t e = cudaMemsetAsync(a.ticket, 0, 8, st);
    if (e == cudaSuccess && p.pairs == 0) e = cudaMemsetAsync(a.loss, 0, 4, st);  // (no pairs: the loss is 0)
    if (e == cudaSuccess && a.rows > 0) e = forward_launch<EPI_PREF>(a, dtype, false, st);
    if (e != cudaSuccess) return e;
    if (p.pairs > 0) {
        pairs_kernel<<<p.pairs, kPairThreads, 0, st>>>(a, p);
        count_launch(LAUNCH_LOSS);
        e = cudaGetLastError();
    }
    return e == cudaSuccess && a.dx && a.rows > 0 ? logprobs_grad_launch(a, dtype, st) : e;
}

}  // namespace wb
