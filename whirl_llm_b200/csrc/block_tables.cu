// Cache block tables and slot maps from the sequences' lengths (rules: include/whirl_b200.h).
//
// Everything a sequence gets depends on prefix sums over the sequences before it: rows asked for, blocks given back, blocks
// needed, rows granted.  plan_kernel (one CTA) forms them; fill_kernel (the whole GPU) then works out every row and every block
// that changes hands from the plan alone.  A block that a sequence gives back in this step and another takes is read from the
// giver's table, not from the stack, so nothing in fill_kernel waits for anything else in it:
//   reads  free_ids below the old count, table entries below a sequence's old owned (a giver's behind its target among them)
//   writes free_ids from the old count on, table entries from a taker's old owned on (a taker is never a giver)
// Bound by latency: 16 sequences with 9 rows each take 8 us of the GPU (launches 2, plan 3, fill 3), 256 sequences with 524288 rows 12 us (8.4 MB of
// maps, 1.3 us at the copy rate), 1024 sequences of which a quarter swaps some 400 blocks each 14 us; the call through the Python binding takes 24.
#include "../../include/whirl_b200.h"

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace wb {

namespace {

struct Head {     // of the plan
    int count;    // free blocks before the step
    int rows;     // rows granted
    int64_t have; // blocks at hand: count + given back
};
// per sequence: old owned, target (old owned again where nothing changes hands), blocks given back and blocks taken before it
struct Plan {
    Head* head;
    int32_t *owned, *target;
    int32_t *back, *taken;  // (blocks that exist: both fit 32 bits; of a sequence that is refused, taken is not read)
};
__host__ __device__ Plan plan_of(void* ws, int seqs) {
    Plan p;
    uint8_t* b = static_cast<uint8_t*>(ws);
    const size_t n = (size_t(seqs) * 4 + 255) / 256 * 256;
    p.head = reinterpret_cast<Head*>(b);
    p.owned = reinterpret_cast<int32_t*>(b + 256), p.target = reinterpret_cast<int32_t*>(b + 256 + n);
    p.back = reinterpret_cast<int32_t*>(b + 256 + 2 * n), p.taken = reinterpret_cast<int32_t*>(b + 256 + 3 * n);
    return p;
}

constexpr int kPlanThreads = 1024;

// N running sums over the CTA at once: v becomes the inclusive prefix sums, total the sums.  sh: 32 words each, free again behind the
// call's last barrier
template <int N>
__device__ __forceinline__ void block_scan(int64_t (&v)[N], int64_t (&total)[N], int64_t (*sh)[32]) {
    const int w = threadIdx.x >> 5, lane = lane_id();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t t = __shfl_up_sync(0xffffffffu, v[k], o);
            if (lane >= o) v[k] += t;
        }
    if (lane == 31)
#pragma unroll
        for (int k = 0; k < N; ++k) sh[k][w] = v[k];
    __syncthreads();
    // every warp adds up the warps before it itself: one barrier less than a second scan by one of them
    int64_t t[N];
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] = sh[k][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t u = __shfl_up_sync(0xffffffffu, t[k], o);
            if (lane >= o) t[k] += u;
        }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int64_t before = __shfl_sync(0xffffffffu, t[k], (w - 1) & 31);
        total[k] = __shfl_sync(0xffffffffu, t[k], 31);
        if (w) v[k] += before;
    }
    __syncthreads();
}

struct Wish {  // what a sequence asks for
    int64_t add, target;
    int own;
    bool valid;
};
__device__ __forceinline__ Wish wish_of(const int32_t* length, const int32_t* n_new, const whirl_block_tables& t, int s) {
    Wish w{0, 0, 0, false};
    if (s < t.seqs) {
        const int64_t len = length[s], add = n_new[s];
        const int own = t.owned[s];
        const int64_t sum = len + add;
        w.own = min(max(own, 0), t.max_blocks);
        w.valid = len >= 0 && add >= 0 && sum <= INT32_MAX;
        if (w.valid) w.target = (uint32_t(sum) + uint32_t(t.block_size) - 1) / uint32_t(t.block_size);
        w.valid = w.valid && w.target <= t.max_blocks;
        w.add = w.valid ? add : 0;
    }
    return w;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* length, const int32_t* n_new, whirl_block_tables t, whirl_step_rows r,
                                                           void* ws) {
    __shared__ int64_t sh[3][32];
    asm volatile("griddepcontrol.launch_dependents;");
    const Plan p = plan_of(ws, t.seqs);
    const int tid = threadIdx.x;
    const int count = min(max(*t.free_count, 0), t.num_blocks);
    // As if everybody were granted: rows, blocks given back and blocks needed in one pass.  Where the sums stay inside max_rows and the
    // blocks at hand, that is the answer.
    int64_t rows = 0, back = 0, needs = 0;
    for (int base = 0; base < t.seqs; base += kPlanThreads) {
        const int s = base + tid;
        const Wish w = wish_of(length, n_new, t, s);
        const int64_t give = w.valid && w.own > w.target ? w.own - w.target : 0, need = w.valid && w.target > w.own ? w.target - w.own : 0;
        int64_t v[3] = {w.add, give, need}, total[3];
        block_scan(v, total, sh);
        if (s < t.seqs) {
            r.status[s] = w.valid ? WHIRL_SEQ_OK : WHIRL_SEQ_INVALID;
            p.owned[s] = w.own, p.target[s] = w.valid ? int(w.target) : w.own;
            p.back[s] = int(min(back + v[1] - give, int64_t(INT32_MAX))), p.taken[s] = int(min(needs + v[2] - need, int64_t(INT32_MAX)));
            r.row0[s] = int(min(rows + v[0] - w.add, int64_t(INT32_MAX)));
        }
        rows += total[0], back += total[1], needs += total[2];
    }
    int64_t have = count + back, used = needs;
    if (rows <= r.max_rows && needs <= have) {
        for (int s = tid; s < t.seqs; s += kPlanThreads) t.owned[s] = p.target[s];  // (each thread reads what it wrote itself)
    } else {
        // rows asked for -> who fits -> blocks given back
        int64_t asked = 0;
        back = 0;
        for (int base = 0; base < t.seqs; base += kPlanThreads) {
            const int s = base + tid;
            const Wish w = wish_of(length, n_new, t, s);
            int64_t v[1] = {w.add}, total[1];
            block_scan(v, total, sh);
            const bool fits = w.valid && (w.add == 0 || asked + v[0] <= r.max_rows);
            asked += total[0];
            const int64_t give = fits && w.own > w.target ? w.own - w.target : 0;
            v[0] = give;
            block_scan(v, total, sh);
            if (s < t.seqs) {
                if (!fits) p.target[s] = w.own;
                if (!fits && w.valid) r.status[s] = WHIRL_SEQ_REFUSED;
                p.back[s] = int(min(back + v[0] - give, int64_t(INT32_MAX)));
            }
            back += total[0];
        }
        // blocks needed -> who gets them -> rows
        have = count + back;
        needs = rows = used = 0;
        for (int base = 0; base < t.seqs; base += kPlanThreads) {
            const int s = base + tid;
            const bool in = s < t.seqs;
            const int own = in ? p.owned[s] : 0, target = in ? p.target[s] : 0;
            const int64_t need = target > own ? target - own : 0;
            int64_t v[1] = {need}, total[1];
            block_scan(v, total, sh);
            const bool ok = in && r.status[s] == WHIRL_SEQ_OK && (need == 0 || needs + v[0] <= have);
            if (in) p.taken[s] = int(min(needs + v[0] - need, int64_t(INT32_MAX)));
            needs += total[0];
            const int64_t add = ok ? n_new[s] : 0;
            int64_t u[2] = {add, ok ? need : 0}, sum[2];
            block_scan(u, sum, sh);
            if (in) {
                r.row0[s] = int(rows + u[0] - add);
                if (ok) t.owned[s] = target;
                else if (need) p.target[s] = own, r.status[s] = WHIRL_SEQ_REFUSED;
            }
            rows += sum[0], used += sum[1];
        }
    }
    if (tid == 0) {
        r.row0[t.seqs] = int(rows);
        *t.free_count = int(min(have - used, int64_t(t.num_blocks)));
        p.head->count = count, p.head->rows = int(rows), p.head->have = have;
    }
}

// the last s in [0, n) with v[s] <= at (v not decreasing, v[0] <= at)
__device__ __forceinline__ int last_upto(const int32_t* v, int n, int at) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Block k (counted over the step) that is taken from the stack.  giver: the last one met, tried first (neighbouring blocks come from the
// same one; a search is ten dependent loads).
__device__ __forceinline__ int block_taken(const whirl_block_tables& t, const Plan& p, int count, int64_t have, int k, int& giver) {
    const int64_t at = have - 1 - k;
    if (at < count) return at >= 0 ? t.free_ids[at] : -1;
    const int g = int(at - count);
    if (giver < 0 || g < p.back[giver] || g >= p.back[giver] + (p.owned[giver] - p.target[giver])) giver = last_upto(p.back, t.seqs, g);
    return t.table[int64_t(giver) * t.max_blocks + p.target[giver] + (g - p.back[giver])];
}

constexpr int kFillThreads = 256;

// group: threads per sequence, a power of two from 32 on
__global__ void __launch_bounds__(kFillThreads) fill_kernel(const int32_t* length, whirl_block_tables t, whirl_step_rows r, void* ws, int group) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // plan_kernel's results (the launch overlaps it)
    const Plan p = plan_of(ws, t.seqs);
    const int count = p.head->count, rows = p.head->rows;
    const int64_t have = p.head->have;
    const int64_t tid = int64_t(blockIdx.x) * kFillThreads + threadIdx.x, threads = int64_t(gridDim.x) * kFillThreads;
    // four rows a thread: one search, and 16-byte stores where the arrays allow them
    const bool wide = ((reinterpret_cast<uintptr_t>(r.slot) | reinterpret_cast<uintptr_t>(r.position) | reinterpret_cast<uintptr_t>(r.seq)) & 15) == 0;
    for (int64_t i0 = tid * 4; i0 < r.max_rows; i0 += threads * 4) {
        int64_t slot[4];
        int pos[4], seq[4], s = -1, b = -1, id = 0, giver = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = i0 + k;
            slot[k] = -1, pos[k] = 0, seq[k] = -1;
            if (i < rows) {
                int now = s < 0 ? last_upto(r.row0, t.seqs, int(i)) : s;
                while (r.row0[now + 1] <= i) ++now;  // (row0[seqs] = rows > i)
                pos[k] = length[now] + int(i) - r.row0[now];
                const int at = pos[k] / t.block_size;
                if (now != s || at != b) {
                    const int own = p.owned[now];
                    id = at < own ? t.table[int64_t(now) * t.max_blocks + at] : block_taken(t, p, count, have, p.taken[now] + at - own, giver);
                }
                s = now, b = at;
                slot[k] = int64_t(id) * t.block_size + pos[k] % t.block_size, seq[k] = now;
            }
        }
        if (wide && i0 + 4 <= r.max_rows) {
            reinterpret_cast<longlong2*>(r.slot + i0)[0] = make_longlong2(slot[0], slot[1]);
            reinterpret_cast<longlong2*>(r.slot + i0)[1] = make_longlong2(slot[2], slot[3]);
            if (r.position) *reinterpret_cast<int4*>(r.position + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            if (r.seq) *reinterpret_cast<int4*>(r.seq + i0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i0 + k >= r.max_rows) break;
                r.slot[i0 + k] = slot[k];
                if (r.position) r.position[i0 + k] = pos[k];
                if (r.seq) r.seq[i0 + k] = seq[k];
            }
        }
    }
    // what changes hands
    const int lane = int(tid & (group - 1));
    for (int64_t s = tid / group; s < t.seqs; s += threads / group) {
        const int own = p.owned[s], target = p.target[s];
        int32_t* row = t.table + s * t.max_blocks;
        for (int j = target + lane; j < own; j += group) {
            const int64_t to = int64_t(count) + p.back[s] + (j - target);
            if (to < t.num_blocks) t.free_ids[to] = row[j];
        }
        int giver = -1;
        for (int j = own + lane; j < target; j += group) row[j] = block_taken(t, p, count, have, p.taken[s] + (j - own), giver);
    }
}

}  // namespace

size_t block_tables_ws_bytes(int seqs) { return 256 + 4 * ((size_t(seqs) * 4 + 255) / 256 * 256); }

cudaError_t block_tables_launch(const int32_t* length, const int32_t* n_new, const whirl_block_tables& t, const whirl_step_rows& r, void* ws,
                                int sm_count, cudaStream_t st) {
    plan_kernel<<<1, kPlanThreads, 0, st>>>(length, n_new, t, r, ws);
    count_launch(LAUNCH_BLOCKS);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // four rows a thread; a quarter of a CTA per sequence where there are CTAs enough, so that long lists of blocks move side by side
    const int64_t want = std::max((int64_t(r.max_rows) + 4 * kFillThreads - 1) / (4 * kFillThreads), (int64_t(t.seqs) * 64 + kFillThreads - 1) / kFillThreads);
    if (want == 0) return cudaSuccess;
    const int64_t ctas = std::min<int64_t>(want, int64_t(sm_count) * 8);
    int group = 32;
    while (group < kFillThreads && int64_t(t.seqs) * group * 2 <= ctas * kFillThreads) group *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas)), cfg.blockDim = dim3(kFillThreads), cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, fill_kernel, length, t, r, ws, group);
    count_launch(LAUNCH_BLOCKS);
    return e;
}

}  // namespace wb
