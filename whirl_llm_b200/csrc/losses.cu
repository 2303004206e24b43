// Log-probabilities of given tokens, the clipped policy loss and the preference loss, with their gradients down to the
// logits (formulas: include/whirl_b200.h).
//
// Every row needs its softmax statistics before any of its gradient can be written.  The statistics are one online pass: a
// thread keeps the largest logit it has met, the sum of exp((x - that) * inv_t) and (for the entropy) the sum of the
// exponentials times their exponents, and brings all three to a new maximum when one comes along; partial results merge the
// same way.  The gradient is one elementwise pass over the row.
#include "../../include/whirl_b200.h"

#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "kernels.h"

namespace wb {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// softmax statistics
// ---------------------------------------------------------------------------------------------------------------

// Partial statistics of a set of logits: m their maximum (-inf without one), s = sum 2^((x - r) c), q = sum of the same terms
// times their exponent (x - r) c, with the reference r = max(m, -FLT_MAX) and c = inv_t log2 e.  (The exponent is formed from
// the difference, not as x c - r c: rows of the type's lowest values stay exact, and so does the term of the maximum.)
struct Soft {
    float m = -INFINITY, s = 0.f, q = 0.f;
};
__device__ __forceinline__ float ref_of(float m) { return fmaxf(m, -FLT_MAX); }

template <bool ENT>
__device__ __forceinline__ void raise(Soft& a, float m, float c) {  // moves a's reference to that of m >= a.m
    const float t = (ref_of(a.m) - ref_of(m)) * c, f = ex2_approx(t);
    if (ENT) a.q = a.s == 0.f ? 0.f : f * fmaf(fmaxf(t, -1000.f), a.s, a.q);
    a.s = a.s == 0.f ? 0.f : a.s * f;
    a.m = m;
}
template <bool ENT>
__device__ __forceinline__ void merge(Soft& a, Soft b, float c) {
    const float m = fmaxf(a.m, b.m);
    raise<ENT>(a, m, c);
    raise<ENT>(b, m, c);
    a.s += b.s;
    if (ENT) a.q += b.q;
}
template <bool ENT>
__device__ __forceinline__ void add(Soft& a, float x, float r, float c) {
    const float t = (x - r) * c, w = ex2_approx(t);
    a.s += w;
    if (ENT) a.q = fmaf(w, fmaxf(t, -1000.f), a.q);  // (0 * -inf is not what a forbidden token adds)
}
template <bool ENT, int N>
__device__ __forceinline__ void add_many(Soft& a, const float (&x)[N], float c) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > a.m) raise<ENT>(a, m, c);
    const float r = ref_of(a.m);
#pragma unroll
    for (int i = 0; i < N; ++i) add<ENT>(a, x[i], r, c);
}

template <bool ENT>
__device__ Soft block_merge(Soft a, float c, Soft* sh) {  // the result is valid in every thread of warp 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Soft b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o), b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        if (ENT) b.q = __shfl_xor_sync(0xffffffffu, a.q, o);
        merge<ENT>(a, b, c);
    }
    const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if (lane_id() == 0) sh[w] = a;
    __syncthreads();
    if (w == 0) {
        a = lane_id() < nw ? sh[lane_id()] : Soft{};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Soft b;
            b.m = __shfl_xor_sync(0xffffffffu, a.m, o), b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
            if (ENT) b.q = __shfl_xor_sync(0xffffffffu, a.q, o);
            merge<ENT>(a, b, c);
        }
    }
    return a;
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

// The row's gradient: dx_j = w_j * (a + b * t_j), + d on the token, with t_j = (x_j - r) c and w_j = 2^t_j.
//   -inv_t g p_j - inv_t h p_j (log p_j + H),  p_j = w_j / sum,  log p_j = ln 2 t_j - log sum
//   => a = -(inv_t / sum) (g + h (H - log sum)),  b = -(inv_t / sum) h ln 2
struct GradRow {
    float r, c, a, b, d;
    int token;
};
__device__ __forceinline__ GradRow grad_row(float m, double sum, double inv_t, int token, double g, double h, double entropy) {
    const double k = inv_t / sum;
    GradRow q;
    q.r = ref_of(m), q.c = float(inv_t) * kLog2e, q.token = token;
    q.a = float(-k * (g + (h == 0.0 ? 0.0 : h * (entropy - log(sum)))));
    q.b = float(-k * h * 0.6931471805599453);
    q.d = float(inv_t * g);
    return q;
}
template <bool ENT>
__device__ __forceinline__ float grad_of(const GradRow& q, float x) {
    const float t = (x - q.r) * q.c, w = ex2_approx(t);
    return ENT ? w * fmaf(q.b, fmaxf(t, -1000.f), q.a) : w * q.a;
}

// ---------------------------------------------------------------------------------------------------------------
// forward: one CTA per row
// ---------------------------------------------------------------------------------------------------------------

constexpr int kFwdThreads = 512;

// the row as a user's call describes it, and whether it counts
struct RowOf {
    int token;
    float inv_t;
    bool live;
};
__device__ __forceinline__ RowOf row_of(const LossArgs& a, int row) {
    RowOf r;
    r.token = a.token[row];
    r.inv_t = a.inv_t_rows ? a.inv_t_rows[row] : a.inv_t;
    r.live = unsigned(r.token) < unsigned(a.n);
    if (a.weight) r.live = r.live && a.weight[row] > 0.f;
    if (a.seq_start) r.live = r.live && row >= a.seq_start[0] && row < a.seq_start[a.seqs];
    return r;
}

// The policy loss of one row (all in 64 bits: differences of log-probabilities).
struct PolicyRow {
    double loss, kl, dlogp;
};
__device__ PolicyRow policy_row(const LossArgs& a, int row, double logp, double entropy) {
    PolicyRow p;
    const double adv = a.adv[row];
    double ratio = 1.0, pg, dpg;
    bool free_d = true;
    if (a.old_logp) {
        double d = logp - double(a.old_logp[row]);
        free_d = !(d <= -20.0 || d >= 20.0);
        d = d < -20.0 ? -20.0 : (d > 20.0 ? 20.0 : d);
        ratio = exp(d);
    }
    const double lo = 1.0 - double(a.clip_low), hi = 1.0 + double(a.clip_high);
    const double plain = ratio * adv, clipped = (ratio < lo ? lo : (ratio > hi ? hi : ratio)) * adv;
    const bool takes_plain = plain <= clipped;
    pg = takes_plain ? -plain : -clipped;
    dpg = takes_plain && free_d ? -plain : 0.0;
    if (a.dual_clip > 0.f && adv < 0.0 && pg > -double(a.dual_clip) * adv) pg = -double(a.dual_clip) * adv, dpg = 0.0;
    p.kl = 0.0;
    if (a.ref_logp) {
        double k = double(a.ref_logp[row]) - logp;
        const bool free_k = !(k <= -20.0 || k >= 20.0);
        k = k < -20.0 ? -20.0 : (k > 20.0 ? 20.0 : k);
        const double e = expm1(k);
        p.kl = e - k;
        pg += double(a.kl_coef) * p.kl;
        if (free_k) dpg -= double(a.kl_coef) * e;
    }
    p.loss = pg - (a.ent_coef != 0.f ? double(a.ent_coef) * entropy : 0.0);
    p.dlogp = dpg;
    return p;
}

// Writes what a call wants of one row.  One thread.
template <int EPI, bool ENT>
__device__ void finish_row(const LossArgs& a, int row, bool live, int token, float inv_t, float x_token, const Soft& s) {
    double logp = 0.0, entropy = 0.0, sum = 0.0;
    float m = 0.f;
    if (live) {
        m = s.m;
        // a row without a finite maximum has no distribution
        sum = (m >= -FLT_MAX && m <= FLT_MAX) ? double(s.s) : double(NAN);
        const double ls = log(sum);
        logp = (double(x_token) - double(m)) * double(inv_t) - ls;
        if (ENT) entropy = ls - 0.6931471805599453 * double(s.q) / sum;
    }
    if (a.logp) a.logp[row] = float(logp);
    if (a.stats) a.stats[2 * int64_t(row)] = m, a.stats[2 * int64_t(row) + 1] = float(sum);
    if (ENT && a.entropy) a.entropy[row] = float(entropy);
    if (EPI == EPI_POLICY) {
        PolicyRow p{};
        float scale = 0.f;
        if (live) scale = a.row_scale[row], p = policy_row(a, row, logp, entropy);
        if (a.kl) a.kl[row] = float(p.kl);
        a.row_loss[row] = float(p.loss);
        a.g_logp[row] = float(double(scale) * p.dlogp);
        if (a.g_entropy) a.g_entropy[row] = live ? -a.ent_coef * scale : 0.f;
        a.row_term[row] = live ? double(scale) * p.loss : 0.0;
    } else if (EPI == EPI_PREF) {
        const float w = !live ? 0.f : (a.weight ? a.weight[row] : 1.f);
        a.row_term[row] = live ? double(w) * (logp - (a.ref_logp ? double(a.ref_logp[row]) : 0.0)) : 0.0;
        a.row_scale[row] = w;
        a.g_logp[row] = 0.f;  // (the rows of a pair get theirs from pairs_kernel)
    }
}

template <typename T, int EPI, bool ENT>
__global__ void __launch_bounds__(kFwdThreads) forward_kernel(LossArgs a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ Soft sh[32];
    const int row = blockIdx.x, tid = threadIdx.x;
    const RowOf w = row_of(a, row);
    if (!w.live) {
        if (tid == 0) finish_row<EPI, ENT>(a, row, false, w.token, w.inv_t, 0.f, Soft{});
        return;
    }
    const float c = w.inv_t * kLog2e;
    const T* x = static_cast<const T*>(a.x) + int64_t(row) * a.ld;
    const int head = head_of(x, a.n), nv = (a.n - head) / E;
    Soft s;
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
#pragma unroll 4
    for (int i = tid; i < nv; i += kFwdThreads) {
        float e[E];
        unpack<T>(v[i], e);
        add_many<ENT>(s, e, c);
    }
    for (int i = tid; i < head + (a.n - head - nv * E); i += kFwdThreads) {
        const float e[1] = {load_one(x + (i < head ? i : i + nv * E))};
        add_many<ENT>(s, e, c);
    }
    s = block_merge<ENT>(s, c, sh);
    if (tid == 0) finish_row<EPI, ENT>(a, row, true, w.token, w.inv_t, load_one(x + w.token), s);
}

// ---------------------------------------------------------------------------------------------------------------
// gradient: grid = (rows, chunks)
// ---------------------------------------------------------------------------------------------------------------

constexpr int kGradThreads = 256;

template <typename T, bool ENT>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(LossArgs a, int chunk) {
    constexpr int E = 16 / sizeof(T);
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
    const int at = zero ? -1 : int(int64_t(q.token) - j0 < 0 || int64_t(q.token) - j0 >= n ? -1 : int64_t(q.token) - j0);
    const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int head = vec ? head_of(x, n) : n, nv = (n - head) / E;
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
    uint4* dv = reinterpret_cast<uint4*>(dx + head);
#pragma unroll 4
    for (int i = tid; i < nv; i += kGradThreads) {
        float e[E];
        if (zero) {
            dv[i] = make_uint4(0, 0, 0, 0);
        } else {
            unpack<T>(v[i], e);
#pragma unroll
            for (int k = 0; k < E; ++k) e[k] = grad_of<ENT>(q, e[k]);
            const int o = at - head - i * E;
#pragma unroll
            for (int k = 0; k < E; ++k) e[k] = o == k ? e[k] + q.d : e[k];
            dv[i] = pack<T>(e);
        }
    }
    for (int i = tid; i < head + (n - head - nv * E); i += kGradThreads) {
        const int j = i < head ? i : i + nv * E;
        float e = 0.f;
        if (!zero) {
            e = grad_of<ENT>(q, load_one(x + j));
            if (j == at) e += q.d;
        }
        store_one(dx + j, e);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// weights, pairs, sums: small kernels
// ---------------------------------------------------------------------------------------------------------------

constexpr int kSmallThreads = 1024;

__device__ double block_sum(double v, double* sh) {  // the same value in every thread
    v = warp_sum(v);
    __syncthreads();
    if (lane_id() == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = lane_id() < int(blockDim.x >> 5) ? sh[lane_id()] : 0.0;
    return warp_sum(t);
}

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

template <int EPI>
cudaError_t forward_launch(const LossArgs& a, int dtype, bool ent, cudaStream_t st) {
    const dim3 grid(unsigned(a.rows)), block(kFwdThreads);
    if (dtype == WHIRL_F32) {
        if (ent) forward_kernel<float, EPI, true><<<grid, block, 0, st>>>(a);
        else forward_kernel<float, EPI, false><<<grid, block, 0, st>>>(a);
    } else {
        if (ent) forward_kernel<uint16_t, EPI, true><<<grid, block, 0, st>>>(a);
        else forward_kernel<uint16_t, EPI, false><<<grid, block, 0, st>>>(a);
    }
    count_launch(LAUNCH_LOSS);
    return cudaGetLastError();
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

cudaError_t policy_launch(const LossArgs& a, int dtype, int mean, float* loss, cudaStream_t st) {
    row_scale_kernel<<<1, kSmallThreads, 0, st>>>(a, mean);
    count_launch(LAUNCH_LOSS);
    cudaError_t e = forward_launch<EPI_POLICY>(a, dtype, a.ent_coef != 0.f || a.entropy, st);
    if (e != cudaSuccess) return e;
    if (a.dx) {
        e = logprobs_grad_launch(a, dtype, st);
        if (e != cudaSuccess) return e;
    }
    sum_kernel<<<1, kSmallThreads, 0, st>>>(a.row_term, a.rows, 1.0, loss);
    count_launch(LAUNCH_LOSS);
    return cudaGetLastError();
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
