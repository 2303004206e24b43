// Log-probabilities of given tokens, the clipped policy loss and the preference loss, with their gradients down to the
// logits (formulas: include/whirl_b200.h).
//
// Every row needs its softmax statistics before any of its gradient can be written.  The statistics are one online pass: a
// thread keeps the largest logit it has met, the sum of exp((x - that) * inv_t) and (for the entropy) the sum of the
// exponentials times their exponents, and brings all three to a new maximum when one comes along; partial results merge the
// same way.  The gradient is one elementwise pass over the row.
#include "../../include/whirl_b200.h"

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdlib>
#include <cstdio>

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

// c = inv_t log2 e in two floats, hi rounded down so that lo >= 0 (a logit of -inf keeps its sign in both products).  With one float
// the exponents of a whole row are off in the same direction, by up to 6e-8 of their size: a bias of some 3e-7 in every
// log-probability, which sums over a sequence do not average out.
// most: logits are clamped to +-most where a reference is made of them, so that most * c stays finite.
struct Scale {
    float hi, lo, most;
};
__device__ __forceinline__ Scale scale_of(float inv_t) {
    const double c = double(inv_t) * 1.4426950408889634;
    Scale r;
    r.hi = __double2float_rd(c);
    r.lo = fmaxf(float(c - double(r.hi)), 1e-37f);
    r.most = fminf(1e37f / r.hi, FLT_MAX);
    return r;
}
// the reference exponent of a maximum
__device__ __forceinline__ float ref_of(float m, const Scale& c) { return fminf(fmaxf(m, -c.most), c.most) * c.hi; }

// Partial statistics of a set of logits: m their maximum (-inf without one), e = ref_of(m), s - k = sum 2^(x c - e) (k: what
// Kahan's sum owes), q = sum of the same terms times their exponent.  The exponent is one fused multiply-add from the logit; that e is a
// rounded product shifts all terms of a row by the same factor, which row_sum() takes out again.
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
        const float t = fmaf(x[0], c.hi, fmaf(x[0], c.lo, -a.e));
        sum = ex2_approx(t);
        if (ENT) qs = sum * fmaxf(t, -1000.f);
    } else {
        const F2 ne = f2(-a.e, -a.e), hi = f2(c.hi, c.hi), lo = f2(c.lo, c.lo);
        F2 w[N / 2 > 0 ? N / 2 : 1], q = f2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const F2 v = f2(x[2 * i], x[2 * i + 1]);
            const float2 t = split(fma2(v, hi, fma2(v, lo, ne)));
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

// The statistics of all threads of the CTA, then of all CTAs of the cluster; the result is valid in warp 0 of every CTA.  Every
// thread's sum is brought to the common maximum once (a tree of pairwise merges would scale it several times over, and
// ex2.approx errs downwards, 5e-8 on average, each time).
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
    a.m = 0.f, a.e = 0.f;  // (references alike: nothing is scaled)
    a = reduce<ENT>(a, one, sh, ctas, 1);
    a.m = m;
    return a;
}

// A row whose maximum is so large that its reference was clamped, or so low (rows of the type's lowest value) that its terms
// vanished: exponents from the differences to the maximum, which is known by then.  Thread sums only.
__device__ __forceinline__ bool is_far(const Soft& a) { return a.m >= -FLT_MAX && a.m <= FLT_MAX && !(a.s > 0.f && a.s <= FLT_MAX); }

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

// The row's scalars are worked out by one thread while the CTA waits, once per row, in a kernel whose loops own the instruction cache: a
// few short polynomials in 64 bits instead of the library's log, exp and expm1 (measured on the policy loss, 4096 x 151936 bf16: SCALARS).

// log of a positive finite number: s = 2^k f with f in [sqrt 1/2, sqrt 2), log f = 2 atanh z, z = (f - 1) / (f + 1), |z| < 0.172; the
// terms left out are below 1e-13.  NaN for what has no logarithm.
__device__ __forceinline__ double ln_of(double s) {
    if (!(s > 0.0 && s <= 1.7e308)) return NAN;
    const int hi = __double2hiint(s), k = (hi - 0x3fe6a09e) >> 20;
    const double f = __hiloint2double(hi - (k << 20), __double2loint(s)), b = f + 1.0;
    double r = double(__frcp_rn(float(b)));
    r = r * (2.0 - b * r);
    const double z = (f - 1.0) * r, y = z * z;
    double t = 1.0 / 13.0;
    t = fma(t, y, 1.0 / 11.0), t = fma(t, y, 1.0 / 9.0), t = fma(t, y, 1.0 / 7.0), t = fma(t, y, 1.0 / 5.0), t = fma(t, y, 1.0 / 3.0);
    return fma(double(k), kLn2, 2.0 * z * fma(t, y, 1.0));
}
// exp of |d| <= 25: d = n ln 2 + f, Taylor's sum to f^11 (what is left out is below 1e-14).  NaN stays.
__device__ __forceinline__ double exp_of(double d) {
    const double n = rint(d * 1.4426950408889634);
    constexpr double hi = double(0.6931471805599453f), lo = kLn2 - hi;  // (n * hi is exact)
    const double f = fma(n, -lo, fma(n, -hi, d));
    double t = 1.0 / 39916800.0;
    t = fma(t, f, 1.0 / 3628800.0), t = fma(t, f, 1.0 / 362880.0), t = fma(t, f, 1.0 / 40320.0), t = fma(t, f, 1.0 / 5040.0);
    t = fma(t, f, 1.0 / 720.0), t = fma(t, f, 1.0 / 120.0), t = fma(t, f, 1.0 / 24.0), t = fma(t, f, 1.0 / 6.0);
    t = fma(t, f, 0.5), t = fma(t, f, 1.0), t = fma(t, f, 1.0);
    return d == d ? __hiloint2double(__double2hiint(t) + (int(n) << 20), __double2loint(t)) : d;
}
// exp k - k - 1 for |k| <= 25, without the cancellation around 0
__device__ __forceinline__ double kl_of(double k) {
    if (fabs(k) > 0.35) return exp_of(k) - 1.0 - k;
    double t = 1.0 / 39916800.0;
    t = fma(t, k, 1.0 / 3628800.0), t = fma(t, k, 1.0 / 362880.0), t = fma(t, k, 1.0 / 40320.0), t = fma(t, k, 1.0 / 5040.0);
    t = fma(t, k, 1.0 / 720.0), t = fma(t, k, 1.0 / 120.0), t = fma(t, k, 1.0 / 24.0), t = fma(t, k, 1.0 / 6.0);
    return k * k * fma(t, k, 0.5);
}

// 2^(e - m c): what the rounded reference e of a row with maximum m puts into its sum.  Doubles: m c has to be exact to the last bits
// of e.
__device__ __forceinline__ double shift_of(double m, double e, double c) {
    const double y = kLn2 * (e - m * c);
    return fabs(y) < 1e-3 ? 1.0 + y * (1.0 + y * (0.5 + y * (1.0 / 6.0))) : exp_of(y < 25.0 ? y : 25.0);  // (|m c| <= 1e37: e is within 1e30 of it)
}

// The row's gradient: dx_j = w_j * (a + b * t_j), + d on the token, with t_j = x_j c - e (far: (x_j - e) c) and w_j = 2^t_j, whose sum
// over the row is s:
//   -inv_t g p_j - inv_t h p_j (log p_j + H),  p_j = w_j / s,  log p_j = ln 2 t_j - log s
//   => a = -(inv_t / s) (g + h (H - log s)),  b = -(inv_t / s) h ln 2
struct GradRow {
    float e, c, a, b, d;
    int token;
    bool far;
};
// sum: over exp((x - m) inv_t), m the row's maximum
__device__ __forceinline__ GradRow grad_row(float m, double sum, float inv_t, int token, double g, double h, double entropy) {
    GradRow q;
    q.c = inv_t * kLog2e, q.token = token;
    const float most = fminf(1e37f / q.c, FLT_MAX);
    q.far = !(m >= -most && m <= most);
    q.e = q.far ? m : m * q.c;
    const double s = q.far ? sum : sum / shift_of(m, q.e, q.c), k = double(inv_t) / s;
    q.a = float(-k * (g + (h == 0.0 ? 0.0 : h * (entropy - ln_of(s)))));
    q.b = float(-k * h * kLn2);
    q.d = float(double(inv_t) * g);
    return q;
}
template <bool ENT>
__device__ __forceinline__ float grad_of(const GradRow& q, float x) {
    const float t = q.far ? (x - q.e) * q.c : fmaf(x, q.c, -q.e), w = ex2_approx(t);
    return ENT ? w * fmaf(q.b, fmaxf(t, -1000.f), q.a) : w * q.a;
}
template <bool ENT, int N>
__device__ __forceinline__ void grad_many(const GradRow& q, float (&x)[N]) {  // (not for a far row)
    const F2 ne = f2(-q.e, -q.e), c = f2(q.c, q.c), a = f2(q.a, q.a), b = f2(q.b, q.b);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 t = split(fma2(f2(x[i], x[i + 1]), c, ne));
        const F2 w = f2(ex2_approx(t.x), ex2_approx(t.y));
        const float2 v = split(ENT ? mul2(w, fma2(b, f2(fmaxf(t.x, -1000.f), fmaxf(t.y, -1000.f)), a)) : mul2(w, a));
        x[i] = v.x, x[i + 1] = v.y;
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
constexpr int kSliceMost = 200 * 1024;  // bytes of a row's slice that a CTA can hold

// A row as a user's call describes it, and whether it counts.
struct RowOf {
    int token;
    float inv_t, weight;
    float adv, old_logp, ref_logp;  // (policy loss; the preference loss has ref_logp)
    float scale;                    // row_scale, where it was known when the row was read
    bool live;
};
// Read by a warp, one word per lane, so that a row costs one trip to memory; every lane gets the whole.
template <int EPI>
__device__ __forceinline__ RowOf row_of(const LossArgs& a, int row, bool with_scale) {
    const int lane = lane_id();
    const void* p = nullptr;
    if (lane == 0) p = a.token + row;
    else if (lane == 1 && a.inv_t_rows) p = a.inv_t_rows + row;
    else if (lane == 2 && a.weight) p = a.weight + row;
    else if (lane == 3 && EPI == EPI_POLICY) p = a.adv + row;
    else if (lane == 4 && EPI == EPI_POLICY && a.old_logp) p = a.old_logp + row;
    else if (lane == 5 && EPI != EPI_NONE && a.ref_logp) p = a.ref_logp + row;
    else if (lane == 6 && EPI == EPI_POLICY && with_scale) p = a.row_scale + row;
    else if (lane == 7 && a.seq_start) p = a.seq_start;
    else if (lane == 8 && a.seq_start) p = a.seq_start + a.seqs;
    const uint32_t got = p ? *static_cast<const uint32_t*>(p) : 0u;
    auto word = [&](int l) { return __shfl_sync(0xffffffffu, got, l); };
    auto real = [&](int l) { return __uint_as_float(word(l)); };
    RowOf r;
    r.token = int(word(0));
    const float it = real(1), wt = real(2);
    r.inv_t = a.inv_t_rows ? it : a.inv_t, r.weight = a.weight ? wt : 1.f;
    r.adv = real(3), r.old_logp = real(4), r.ref_logp = real(5), r.scale = real(6);
    const int first = int(word(7)), end = int(word(8));
    r.live = unsigned(r.token) < unsigned(a.n) && r.weight > 0.f && (!a.seq_start || (row >= first && row < end));
    return r;
}

// The policy loss of one row (all in 64 bits: differences of log-probabilities).
struct PolicyRow {
    double loss, kl, dlogp;
};
__device__ PolicyRow policy_row(const LossArgs& a, const RowOf& w, double logp, double entropy) {
    PolicyRow p;
    const double adv = w.adv;
    double ratio = 1.0, pg, dpg;
    bool free_d = true;
    if (a.old_logp) {
        double d = logp - double(w.old_logp);
        free_d = !(d <= -20.0 || d >= 20.0);
        d = d < -20.0 ? -20.0 : (d > 20.0 ? 20.0 : d);
        ratio = exp_of(d);
    }
    const double lo = 1.0 - double(a.clip_low), hi = 1.0 + double(a.clip_high);
    const double plain = ratio * adv, clipped = (ratio < lo ? lo : (ratio > hi ? hi : ratio)) * adv;
    const bool takes_plain = plain <= clipped;
    pg = takes_plain ? -plain : -clipped;
    dpg = takes_plain && free_d ? -plain : 0.0;
    if (a.dual_clip > 0.f && adv < 0.0 && pg > -double(a.dual_clip) * adv) pg = -double(a.dual_clip) * adv, dpg = 0.0;
    p.kl = 0.0;
    if (a.ref_logp) {
        double k = double(w.ref_logp) - logp;
        const bool free_k = !(k <= -20.0 || k >= 20.0);
        k = k < -20.0 ? -20.0 : (k > 20.0 ? 20.0 : k);
        p.kl = kl_of(k);
        pg += double(a.kl_coef) * p.kl;
        if (free_k) dpg -= double(a.kl_coef) * (p.kl + k);
    }
    p.loss = pg - (a.ent_coef != 0.f ? double(a.ent_coef) * entropy : 0.0);
    p.dlogp = dpg;
    return p;
}

// What a row comes to; with `write`, what the call wants of it is written.  One thread.  s: the row's statistics, of which s.s may be
// relative to a rounded reference (far: to the maximum itself).
struct RowDone {
    double sum, entropy, g, h;
};
template <int EPI, bool ENT>
__device__ __forceinline__ RowDone finish_row(const LossArgs& a, int row, bool write, const RowOf& w, float x_token, float m, float e, float s, float q,
                                           bool far) {
    RowDone done{};
    double logp = 0.0, entropy = 0.0, sum = 0.0;
    if (w.live) {
        const double c = double(w.inv_t) * 1.4426950408889634;
        // a row without a finite maximum has no distribution
        sum = (m >= -FLT_MAX && m <= FLT_MAX) ? (far ? double(s) : double(s) * shift_of(m, e, c)) : double(NAN);
        const double ls = ln_of(sum);
        logp = (double(x_token) - double(m)) * double(w.inv_t) - ls;
        // the terms' mean exponent is q / s from the reference, and e - m c more from the maximum
        if (ENT) entropy = ls - kLn2 * (double(q) / double(s) + (far ? 0.0 : double(e) - double(m) * c));
    } else {
        m = 0.f;
    }
    done.sum = sum, done.entropy = entropy;
    if (EPI != EPI_POLICY && !write) return done;
    if (write && a.logp) a.logp[row] = float(logp);
    if (write && a.stats) a.stats[2 * int64_t(row)] = m, a.stats[2 * int64_t(row) + 1] = float(sum);
    if (write && ENT && a.entropy) a.entropy[row] = float(entropy);
    if (EPI == EPI_POLICY) {
        PolicyRow p{};
        float scale = 0.f;
        if (w.live) scale = w.scale, p = policy_row(a, w, logp, entropy);
        done.g = float(double(scale) * p.dlogp), done.h = w.live ? -a.ent_coef * scale : 0.f;
        if (write) {
            if (a.kl) a.kl[row] = float(p.kl);
            if (a.row_loss) a.row_loss[row] = float(p.loss);
            if (a.g_logp) a.g_logp[row] = float(done.g);
            if (a.g_entropy) a.g_entropy[row] = float(done.h);
            a.row_term[row] = w.live ? double(scale) * p.loss : 0.0;
        }
    } else if (EPI == EPI_PREF) {
        a.row_term[row] = w.live ? double(w.weight) * (logp - (a.ref_logp ? double(w.ref_logp) : 0.0)) : 0.0;
        a.row_scale[row] = w.live ? w.weight : 0.f;
        a.g_logp[row] = 0.f;  // (the rows of a pair get theirs from pairs_kernel)
    }
    return done;
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

// The CTA that comes last adds up the rows' terms, in their order.  (Called by `callers` CTAs in all, each after its thread 0 has written
// the terms of its rows.)
__device__ void last_sum(const LossArgs& a, unsigned callers) {
    __shared__ bool last;
    __shared__ double sh_d[32];
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(a.ticket, 1u) + 1u == callers;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double t = 0.0;
    for (int r = threadIdx.x; r < a.rows; r += blockDim.x) t += __ldcg(a.row_term + r);
    t = block_sum(t, sh_d);
    if (threadIdx.x == 0) *a.loss = float(t);
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
template <typename T, bool ENT>
__device__ __noinline__ Soft far_sums(const uint4* v, int cnt, bool have_edge, float x_edge, float m, float c) {
    constexpr int E = 16 / sizeof(T);
    Soft a{m, 0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x; i < cnt; i += blockDim.x) {
        float x[E];
        unpack<T>(v[i], x);
        for (int j = 0; j < E; ++j) {
            const float t = (x[j] - m) * c, w = ex2_approx(t);
            a.s += w;
            if (ENT) a.q = fmaf(w, fmaxf(t, -1000.f), a.q);
        }
    }
    if (have_edge) {
        const float t = (x_edge - m) * c, w = ex2_approx(t);
        a.s += w;
        if (ENT) a.q = fmaf(w, fmaxf(t, -1000.f), a.q);
    }
    return a;
}

// vectors that a thread of the forward kernel has under way: kFwdRing steps of 16 logits each
template <typename T>
constexpr int kFwdRing = sizeof(T) == 4 ? 4 : 8;

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
    far = threadIdx.x < 32 && is_far(s);
    if (__syncthreads_or(far)) {  // (every CTA of the cluster has the same statistics)
        if (threadIdx.x == 0) sh.m[0] = s.m;
        __syncthreads();
        const float m = sh.m[0];
        __syncthreads();
        s = reduce_far<ENT>(far_sums<T, ENT>(data, cnt, have_edge, x_edge, m, c.hi), m, sh, ctas);
        far = true;
    }
    return s;
}

// Statistics: one cluster per row.  A thread reads what it copied into shared memory itself, so that the copies need no barrier.
template <typename T, int EPI, bool ENT>
__global__ void __launch_bounds__(kRowThreads, 3) forward_kernel(const __grid_constant__ LossArgs a, int per) {
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
            finish_row<EPI, ENT>(a, row, true, w, x_token, s.m, s.e, s.s, s.q, far);
        }
    } else if (tid == 0 && rank == 0) {
        grid_dependency_wait();
        finish_row<EPI, ENT>(a, row, true, w, 0.f, 0.f, 0.f, 0.f, 0.f, false);
    }
    if (EPI == EPI_POLICY && rank == 0) last_sum(a, unsigned(a.rows));
}

// A warp's partial statistics, on their way to every CTA of the cluster
template <bool ENT>
struct Part;
template <>
struct Part<false> {
    float m, s;
};
template <>
struct Part<true> {
    float m, s, q, pad;
};
// stores to shared memory of CTA `cta` and counts the bytes on its barrier
__device__ __forceinline__ void send(Part<false>* to, uint64_t* bar, int cta, float m, float s, float) {
    asm volatile(
        "{\n .reg .b32 d, b;\n mapa.shared::cluster.u32 d, %0, %2;\n mapa.shared::cluster.u32 b, %1, %2;\n"
        " st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [d], {%3, %4}, [b];\n}\n" ::"r"(smem_u32(to)),
        "r"(smem_u32(bar)), "r"(cta), "r"(__float_as_uint(m)), "r"(__float_as_uint(s))
        : "memory");
}
__device__ __forceinline__ void send(Part<true>* to, uint64_t* bar, int cta, float m, float s, float q) {
    asm volatile(
        "{\n .reg .b32 d, b;\n mapa.shared::cluster.u32 d, %0, %2;\n mapa.shared::cluster.u32 b, %1, %2;\n"
        " st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [d], {%3, %4, %5, %5}, [b];\n}\n" ::"r"(smem_u32(to)),
        "r"(smem_u32(bar)), "r"(cta), "r"(__float_as_uint(m)), "r"(__float_as_uint(s)), "r"(__float_as_uint(q))
        : "memory");
}
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

constexpr int kRowWarps = kRowThreads / 32;

// Each warp's sums to every CTA of the cluster (its lane i tells CTA i).
template <bool ENT>
__device__ __forceinline__ void tell(Soft a, const Scale& c, Part<ENT>* parts, uint64_t* bar, int ctas, int rank) {
    a.s -= a.k, a.k = 0.f;
    const float m = warp_max_f(a.m);
    raise<ENT>(a, m, c);
    a.s = warp_sum_f(a.s);
    if (ENT) a.q = warp_sum_f(a.q);
    if (lane_id() < ctas) send(parts + rank * kRowWarps + (threadIdx.x >> 5), bar, lane_id(), m, a.s, a.q);
}
// The row's statistics from all warps' (one warp).  A barrier that does not complete in its time gives a row of NaN.
template <bool ENT>
__device__ __forceinline__ Soft hear(const Scale& c, const Part<ENT>* parts, uint64_t* bar, uint32_t parity, int ctas, uint32_t& limit) {
    const int n = ctas * kRowWarps;
    if (lane_id() == 0) mbar_expect_tx(bar, uint32_t(n * sizeof(Part<ENT>)));
    const bool came = __all_sync(0xffffffffu, mbar_wait(bar, parity, limit));
    if (!came) limit = 1;  // (and the rows after it do not wait that long again)
    float m = -INFINITY;
    for (int i = lane_id(); i < n; i += 32) m = fmaxf(m, parts[i].m);
    m = warp_max_f(m);
    Soft s{m, ref_of(m, c), 0.f, 0.f, 0.f};
    for (int i = lane_id(); i < n; i += 32) {
        Soft p{parts[i].m, ref_of(parts[i].m, c), parts[i].s, 0.f, 0.f};
        if constexpr (ENT) p.q = parts[i].q;
        raise<ENT>(p, m, c);
        s.s += p.s;
        if (ENT) s.q += p.q;
    }
    s.s = warp_sum_f(s.s);
    if (ENT) s.q = warp_sum_f(s.q);
    if (!came) s.s = NAN;
    return s;
}

// The policy loss with its gradient.  The clusters stay and take rows in turn, each CTA holding its slice of a row in shared memory
// from the read to the gradient: one read and one write of global memory.  As soon as a thread has written a vector's
// gradient it starts the copy of the same vector of the cluster's next row into the same place, so that the memory is
// busy while the statistics of that row wait for it; several CTAs per SM fill each other's waits (the exchange of the statistics, the row's
// scalars).  The statistics travel by stores that count on the receiver's mbarrier: a cluster barrier would hold every row until the
// gradient's stores of the row before it are acknowledged.
template <typename T, int EPI, bool ENT>
__global__ void __launch_bounds__(kRowThreads, 5) fused_kernel(const __grid_constant__ LossArgs a, int per) {
    constexpr int E = 16 / sizeof(T), NT = kRowThreads, V = 16 / E;
    extern __shared__ __align__(16) uint4 slice[];  // `per` vectors, then three sets of partial statistics (rows in turn; far rows)
    __shared__ GradRow s_q;
    __shared__ RowOf s_row[2];
    __shared__ uint64_t s_bar[3];
    __shared__ float s_m;
    __shared__ bool s_zero, s_far;
    const int ctas = int(cluster_size()), rank = int(cluster_rank()), tid = threadIdx.x;
    const int clusters = int(gridDim.x / unsigned(ctas));
    Part<ENT>* const parts = reinterpret_cast<Part<ENT>*>(slice + per);
    int row = int(blockIdx.x / unsigned(ctas)), lives = 0, fars = 0;
    uint32_t limit = kWaitLimit;
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
    for (int k = 0; row < a.rows; ++k, row += clusters) {
        const RowOf& w = s_row[k & 1];
        const bool more = a.rows - row > clusters;
        if (more && tid >= NT - 32) {  // the next row's scalars; the wait is over at once but for the first row
            grid_dependency_wait();
            const RowOf r = row_of<EPI>(a, row + clusters, true);
            if (tid == NT - 32) s_row[(k + 1) & 1] = r;
        }
        const Slice<T> at(a, row, rank, per);
        const int cnt = at.cnt;
        float x_edge = 0.f;
        bool zero = true;
        if (w.live) {
            const Scale c = scale_of(w.inv_t);
            Soft s = soft_empty(c);
            const float x_token = tid == 0 ? load_one(at.x + w.token) : 0.f;
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
            const int set = lives & 1;
            tell<ENT>(s, c, parts + set * ctas * kRowWarps, &s_bar[set], ctas, rank);
            auto finish = [&](const Soft& r, bool far) {  // one thread
                RowOf wr = w;
                if (k == 0) {
                    grid_dependency_wait();  // row_scale_kernel's results
                    if (EPI == EPI_POLICY) wr.scale = a.row_scale[row];
                }
                const RowDone d = finish_row<EPI, ENT>(a, row, rank == 0, wr, x_token, r.m, r.e, r.s, r.q, far);
                s_zero = d.g == 0.0 && d.h == 0.0;
                s_q = grad_row(r.m, d.sum, wr.inv_t, wr.token, d.g, d.h, d.entropy);
            };
            if (tid < 32) {
                s = hear<ENT>(c, parts + set * ctas * kRowWarps, &s_bar[set], uint32_t(lives >> 1) & 1, ctas, limit);
                if (tid == 0) {
                    s_far = is_far(s), s_m = s.m;
                    if (!is_far(s)) finish(s, false);
                }
            }
            ++lives;
            __syncthreads();
            if (s_far) {  // (every CTA of the cluster has the same statistics)
                const float m = s_m;
                const Scale one{1.f, 0.f, FLT_MAX};
                s = far_sums<T, ENT>(slice, cnt, at.edge >= 0, x_edge, m, c.hi);
                s.m = 0.f, s.e = 0.f;  // (references alike: nothing is scaled on the way)
                tell<ENT>(s, one, parts + 2 * ctas * kRowWarps, &s_bar[2], ctas, rank);
                if (tid < 32) {
                    s = hear<ENT>(one, parts + 2 * ctas * kRowWarps, &s_bar[2], uint32_t(fars) & 1, ctas, limit);
                    s.m = m;
                    if (tid == 0) finish(s, true);
                }
                ++fars;
                __syncthreads();
            }
            zero = s_zero;
        } else {
            if (tid == 0) {
                if (k == 0) grid_dependency_wait();
                if (rank == 0) finish_row<EPI, ENT>(a, row, true, w, 0.f, 0.f, 0.f, 0.f, 0.f, false);
            }
            __syncthreads();
        }
        // (s_row of the next row, s_q and s_zero are in place; their next writes come after every thread has read them: s_row's behind the
        // next row's barrier but one, the others' behind all warps' `tell` of the next row)
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
        if (more && s_row[(k + 1) & 1].live) {
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
    cluster_barrier();  // nobody leaves while another CTA's stores are under way to it
    if (EPI == EPI_POLICY && rank == 0) last_sum(a, unsigned(clusters));
}

// ---------------------------------------------------------------------------------------------------------------
// gradient: grid = (rows, chunks)
// ---------------------------------------------------------------------------------------------------------------

constexpr int kGradThreads = 256;

template <typename T, bool ENT>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const __grid_constant__ LossArgs a, int chunk) {
    constexpr int E = 16 / sizeof(T), NT = kGradThreads;
    __shared__ GradRow s_q;
    __shared__ bool s_zero;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int64_t j0 = int64_t(blockIdx.y) * chunk;
    const int n = a.n - j0 < chunk ? int(a.n - j0) : chunk;
    const T* x = static_cast<const T*>(a.x) + int64_t(row) * a.ld + j0;
    T* dx = static_cast<T*>(a.dx) + int64_t(row) * a.ld_dx + j0;
    if (tid == 0) {
        const int token = a.token[row];
        const float g = a.g_logp[row], h = ENT ? a.g_entropy[row] : 0.f;
        s_zero = unsigned(token) >= unsigned(a.n) || (g == 0.f && h == 0.f);
        if (!s_zero) {
            const float inv_t = a.inv_t_rows ? a.inv_t_rows[row] : a.inv_t;
            const float m = a.stats[2 * int64_t(row)], sum = a.stats[2 * int64_t(row) + 1];
            s_q = grad_row(m, sum, inv_t, token, g, h, ENT ? a.entropy[row] : 0.f);
        }
    }
    __syncthreads();
    const bool zero = s_zero;
    GradRow q{};
    if (!zero) q = s_q;
    const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0 && !q.far;
    const int head = vec ? head_of(x, n) : n, nv = (n - head) / E;
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
    uint4* dv = reinterpret_cast<uint4*>(dx + head);
    const int64_t t64 = zero ? -1 : int64_t(q.token) - j0;
    const int at = t64 >= 0 && t64 < n ? int(t64) : -1;
    // the token's own logit, before anything is written (dx may be x)
    const int t_vec = at - head;
    const bool mine = at >= head && t_vec < nv * E && (t_vec / E) % NT == tid;
    const float x_token = mine ? load_one(x + at) : 0.f;
    if (zero) {
#pragma unroll 4
        for (int i = tid; i < nv; i += NT) __stcs(dv + i, make_uint4(0, 0, 0, 0));
    } else {
        int i = tid;
#pragma unroll 1
        for (; i + 3 * NT < nv; i += 4 * NT) {
            const uint4 b[4] = {v[i], v[i + NT], v[i + 2 * NT], v[i + 3 * NT]};
#pragma unroll
            for (int k = 0; k < 4; ++k) __stcs(dv + i + k * NT, grad_vec<T, ENT>(q, b[k]));
        }
#pragma unroll 1
        for (; i < nv; i += NT) __stcs(dv + i, grad_vec<T, ENT>(q, v[i]));
    }
    if (mine) store_one(dx + at, grad_of<ENT>(q, x_token) + q.d);
    for (int i = tid; i < head + (n - head - nv * E); i += NT) {
        const int j = i < head ? i : i + nv * E;
        store_one(dx + j, zero ? 0.f : grad_of<ENT>(q, load_one(x + j)) + (j == at ? q.d : 0.f));
    }
}

// ---------------------------------------------------------------------------------------------------------------
// weights, pairs, sums: small kernels
// ---------------------------------------------------------------------------------------------------------------

constexpr int kSmallThreads = 1024;

__device__ __forceinline__ float live_weight(const LossArgs& a, int row) {
    if (unsigned(a.token[row]) >= unsigned(a.n)) return 0.f;
    if (!a.weight) return 1.f;
    const float w = a.weight[row];
    return w > 0.f ? w : 0.f;
}
// the rows of sequence s, inside the batch whatever seq_start says
__device__ __forceinline__ int2 rows_of(const LossArgs& a, int s) {
    const int b = min(max(a.seq_start[s], 0), a.rows);
    return make_int2(b, min(max(a.seq_start[s + 1], b), a.rows));
}

// row_scale[rows] of the policy loss.  One CTA.
__global__ void __launch_bounds__(kSmallThreads) row_scale_kernel(LossArgs a, int mean) {
    __shared__ double sh[32];
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) *a.ticket = 0;
    if (mean != WHIRL_MEAN_SEQS) {
        double k = 1.0;
        if (mean == WHIRL_MEAN_TOKENS) {
            double t = 0.0;
            for (int r = tid; r < a.rows; r += kSmallThreads) t += live_weight(a, r);
            t = block_sum(t, sh);
            k = t > 0.0 ? 1.0 / t : 0.0;
        }
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

// loss[0] = scale * sum of terms[count], in a fixed order.  One CTA.
__global__ void __launch_bounds__(kSmallThreads) sum_kernel(const double* terms, int count, double scale, float* loss) {
    __shared__ double sh[32];
    double t = 0.0;
    for (int i = threadIdx.x; i < count; i += kSmallThreads) t += terms[i];
    t = block_sum(t, sh);
    if (threadIdx.x == 0) *loss = float(t * scale);
}

// One CTA per pair: the sequences' sums, the pair's loss, and the rows' g_logp.
constexpr int kPairThreads = 128;
__global__ void __launch_bounds__(kPairThreads) pairs_kernel(LossArgs a, PairArgs p) {
    __shared__ double sh[32];
    const int i = blockIdx.x, tid = threadIdx.x;
    int2 b[2];
    double P[2], W[2];
    for (int k = 0; k < 2; ++k) {
        b[k] = rows_of(a, 2 * i + k);
        double t = 0.0, w = 0.0;
        for (int r = b[k].x + tid; r < b[k].y; r += kPairThreads) t += a.row_term[r], w += double(a.row_scale[r]);
        P[k] = block_sum(t, sh);
        W[k] = 1.0;
        if (p.average) {
            w = block_sum(w, sh);
            W[k] = w > 0.0 ? 1.0 / w : 0.0;
            P[k] = w > 0.0 ? P[k] / w : 0.0;
        }
    }
    const double beta = p.beta, h = beta * (P[0] - P[1]) - double(p.margin);
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
        dh = h < 1.0 ? -1.0 : 0.0;
    } else {
        const double t = (h - 0.5) / beta;
        loss = t * t, dh = 2.0 * t / beta;
    }
    const double coef = beta * dh / double(p.pairs);
    for (int k = 0; k < 2; ++k)
        for (int r = b[k].x + tid; r < b[k].y; r += kPairThreads) a.g_logp[r] = float((k ? -coef : coef) * W[k] * double(a.row_scale[r]));
    if (tid == 0) {
        a.seq_term[i] = loss;
        if (p.pair_loss) p.pair_loss[i] = float(loss);
        if (p.reward) p.reward[2 * i] = float(beta * P[0]), p.reward[2 * i + 1] = float(beta * P[1]);
    }
}

// A launch of forward_kernel / fused_kernel: `ctas` CTAs in a cluster, `per` vectors of a row each, at most `clusters` clusters.
template <typename F>
cudaError_t cluster_launch(F f, std::atomic<uint64_t>& ready, const LossArgs& a, int ctas, int per, size_t smem, bool persistent, bool follows, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {  // bit per device: the function's limits are raised
        e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceMost);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kRowThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
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
        if (getenv("WB_V")) fprintf(stderr, "fit %d ctas %d smem %zu\n", fit, ctas, smem);
    }
    cfg.gridDim = dim3(unsigned(clusters) * unsigned(ctas));
    cfg.numAttrs = follows ? 2 : 1;  // (the policy loss follows row_scale_kernel)
    e = cudaLaunchKernelEx(&cfg, f, a, per);
    count_launch(LAUNCH_LOSS);
    return e;
}

int vectors_of(int n, int dtype) { return int((int64_t(n) * (dtype == WHIRL_F32 ? 4 : 2) + 15) / 16); }

template <typename T, int EPI, bool ENT>
cudaError_t forward_typed(const LossArgs& a, int ctas, int per, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return cluster_launch(forward_kernel<T, EPI, ENT>, ready, a, ctas, per, size_t(kFwdRing<T>) * 16 * sizeof(T) * kRowThreads, false, EPI == EPI_POLICY, st);
}
template <int EPI>
cudaError_t forward_launch(const LossArgs& a, int dtype, bool ent, cudaStream_t st) {
    const int nv = vectors_of(a.n, dtype);
    int ctas = 1;
    while (ctas < 16 && int64_t(a.rows) * ctas < 1776 && nv / (2 * ctas) >= 2 * kRowThreads) ctas *= 2;
    if (const char* v = getenv("WB_CF")) ctas = atoi(v);
    const int per = (nv + ctas - 1) / ctas;
    if (dtype == WHIRL_F32) return ent ? forward_typed<float, EPI, true>(a, ctas, per, st) : forward_typed<float, EPI, false>(a, ctas, per, st);
    return ent ? forward_typed<uint16_t, EPI, true>(a, ctas, per, st) : forward_typed<uint16_t, EPI, false>(a, ctas, per, st);
}

template <typename T, bool ENT>
cudaError_t fused_typed(const LossArgs& a, int ctas, int per, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return cluster_launch(fused_kernel<T, EPI_POLICY, ENT>, ready, a, ctas, per, size_t(per) * 16 + 3 * size_t(ctas) * kRowWarps * sizeof(Part<ENT>), true, true, st);
}

}  // namespace

cudaError_t logprobs_launch(const LossArgs& a, int dtype, cudaStream_t st) { return forward_launch<EPI_NONE>(a, dtype, a.entropy != nullptr, st); }

cudaError_t logprobs_grad_launch(const LossArgs& a, int dtype, cudaStream_t st) {
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
    int ctas = 1, most = 44 * 1024;
    if (const char* v = getenv("WB_SL")) most = atoi(v) * 1024;
    while (ctas < 16 && int64_t(nv + ctas - 1) / ctas * 16 > most) ctas *= 2;
    while (ctas < 16 && int64_t(a.rows) * ctas < 592 && nv / (2 * ctas) >= kRowThreads) ctas *= 2;
    if (const char* v = getenv("WB_CG")) ctas = atoi(v);
    const int64_t per = (int64_t(nv) + ctas - 1) / ctas;
    if (a.dx && per * 16 <= kSliceMost) {
        if (dtype == WHIRL_F32) return ent ? fused_typed<float, true>(a, ctas, int(per), st) : fused_typed<float, false>(a, ctas, int(per), st);
        return ent ? fused_typed<uint16_t, true>(a, ctas, int(per), st) : fused_typed<uint16_t, false>(a, ctas, int(per), st);
    }
    e = forward_launch<EPI_POLICY>(a, dtype, ent, st);
    return e == cudaSuccess && a.dx ? logprobs_grad_launch(a, dtype, st) : e;
}

cudaError_t preference_launch(const LossArgs& a, const PairArgs& p, int dtype, float* loss, cudaStream_t st) {
    if (a.rows > 0) {
        const cudaError_t e = forward_launch<EPI_PREF>(a, dtype, false, st);
        if (e != cudaSuccess) return e;
    }
    if (p.pairs > 0) {
        pairs_kernel<<<p.pairs, kPairThreads, 0, st>>>(a, p);
        count_launch(LAUNCH_LOSS);
    }
    if (a.dx && a.rows > 0) {
        const cudaError_t e = logprobs_grad_launch(a, dtype, st);
        if (e != cudaSuccess) return e;
    }
    sum_kernel<<<1, kSmallThreads, 0, st>>>(a.seq_term, p.pairs, p.pairs > 0 ? 1.0 / p.pairs : 0.0, loss);
    count_launch(LAUNCH_LOSS);
    return cudaGetLastError();
}

}  // namespace wb
