// Cache block tables and slot maps from the sequences' lengths (rules: include/whirl_b200.h).
//
// Everything a sequence gets depends on prefix sums over the sequences before it: rows asked for, blocks given back, blocks
// needed, rows granted.  plan_kernel (one CTA) forms them; fill_kernel (the whole GPU) then works out every row and every block
// that changes hands from the plan alone.  A block that a sequence gives back in this step and another takes is read from the
// giver's table, not from the stack, so nothing in fill_kernel waits for anything else in it:
//   reads  free_ids below the old count, table entries below a sequence's old owned (a giver's behind its target among them)
//   writes free_ids from the old count on, table entries from a taker's old owned on (a taker is never a giver)
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

__device__ __forceinline__ int64_t warp_scan_incl64(int64_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane_id() >= o) v += t;
    }
    return v;
}
// inclusive prefix sum over the CTA; total = the sum.  sh: 33 words, free again after the call's last barrier
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sh, int64_t& total) {
    const int w = threadIdx.x >> 5;
    v = warp_scan_incl64(v);
    if (lane_id() == 31) sh[w] = v;
    __syncthreads();
    if (w == 0) {
        const int64_t t = warp_scan_incl64(sh[lane_id()]);
        sh[lane_id()] = t;
    }
    __syncthreads();
    const int64_t before = w ? sh[w - 1] : 0;
    total = sh[kPlanThreads / 32 - 1];
    __syncthreads();
    return before + v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* length, const int32_t* n_new, whirl_block_tables t, whirl_step_rows r,
                                                           void* ws) {
    __shared__ int64_t sh[33];
    const Plan p = plan_of(ws, t.seqs);
    const int tid = threadIdx.x;
    const int count = min(max(*t.free_count, 0), t.num_blocks);
    int64_t total;
    // rows asked for -> who fits -> blocks given back
    int64_t asked = 0, back = 0;
    for (int base = 0; base < t.seqs; base += kPlanThreads) {
        const int s = base + tid;
        const bool in = s < t.seqs;
        const int64_t len = in ? length[s] : 0, add = in ? n_new[s] : 0;
        const int64_t target = (len + add + t.block_size - 1) / t.block_size;
        const bool valid = in && len >= 0 && add >= 0 && len + add <= INT32_MAX && target <= t.max_blocks;
        const int64_t rows = asked + block_scan(valid ? add : 0, sh, total);
        asked += total;
        const bool fits = valid && (add == 0 || rows <= r.max_rows);
        const int own = in ? min(max(t.owned[s], 0), t.max_blocks) : 0;
        const int64_t give = fits && own > target ? own - target : 0;
        const int64_t upto = back + block_scan(give, sh, total);
        back += total;
        if (in) {
            r.status[s] = fits ? WHIRL_SEQ_OK : (valid ? WHIRL_SEQ_REFUSED : WHIRL_SEQ_INVALID);
            p.owned[s] = own, p.target[s] = fits ? int(target) : own, p.back[s] = int(min(upto - give, int64_t(INT32_MAX)));
        }
    }
    // blocks needed -> who gets them -> rows  (each thread reads back what it wrote itself)
    const int64_t have = count + back;
    int64_t needs = 0, row = 0, used = 0;
    for (int base = 0; base < t.seqs; base += kPlanThreads) {
        const int s = base + tid;
        const bool in = s < t.seqs;
        const int own = in ? p.owned[s] : 0, target = in ? p.target[s] : 0;
        const int64_t need = target > own ? target - own : 0;
        const int64_t upto = needs + block_scan(need, sh, total);
        needs += total;
        const bool ok = in && r.status[s] == WHIRL_SEQ_OK && (need == 0 || upto <= have);
        const int64_t add = ok ? n_new[s] : 0;
        const int64_t end = row + block_scan(add, sh, total);
        row += total;
        block_scan(ok ? need : 0, sh, total);
        used += total;
        if (in) {
            p.taken[s] = int(min(upto - need, int64_t(INT32_MAX)));
            r.row0[s] = int(end - add);
            if (ok) t.owned[s] = target;
            else if (need) p.target[s] = own, r.status[s] = WHIRL_SEQ_REFUSED;
        }
    }
    if (tid == 0) {
        r.row0[t.seqs] = int(row);
        *t.free_count = int(min(have - used, int64_t(t.num_blocks)));
        p.head->count = count, p.head->rows = int(row), p.head->have = have;
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

// block k (counted over the step) that is taken from the stack
__device__ __forceinline__ int block_taken(const whirl_block_tables& t, const Plan& p, int count, int64_t have, int k) {
    const int64_t at = have - 1 - k;
    if (at < count) return at >= 0 ? t.free_ids[at] : -1;
    const int g = int(at - count), s = last_upto(p.back, t.seqs, g);  // the giver: the last sequence before whom at most g were given
    return t.table[int64_t(s) * t.max_blocks + p.target[s] + (g - p.back[s])];
}

constexpr int kFillThreads = 256;

__global__ void __launch_bounds__(kFillThreads) fill_kernel(const int32_t* length, whirl_block_tables t, whirl_step_rows r, void* ws) {
    const Plan p = plan_of(ws, t.seqs);
    const int count = p.head->count, rows = p.head->rows;
    const int64_t have = p.head->have;
    const int64_t tid = int64_t(blockIdx.x) * kFillThreads + threadIdx.x, threads = int64_t(gridDim.x) * kFillThreads;
    for (int64_t i = tid; i < r.max_rows; i += threads) {
        int64_t slot = -1;
        int pos = 0, s = -1;
        if (i < rows) {
            s = last_upto(r.row0, t.seqs, int(i));
            pos = length[s] + int(i) - r.row0[s];
            const int b = pos / t.block_size, own = p.owned[s];
            const int id = b < own ? t.table[int64_t(s) * t.max_blocks + b] : block_taken(t, p, count, have, p.taken[s] + b - own);
            slot = int64_t(id) * t.block_size + pos % t.block_size;
        }
        r.slot[i] = slot;
        if (r.position) r.position[i] = pos;
        if (r.seq) r.seq[i] = s;
    }
    // a warp per sequence: what changes hands
    for (int64_t s = tid >> 5; s < t.seqs; s += threads >> 5) {
        const int own = p.owned[s], target = p.target[s];
        int32_t* row = t.table + s * t.max_blocks;
        for (int j = target + lane_id(); j < own; j += 32) {
            const int64_t to = int64_t(count) + p.back[s] + (j - target);
            if (to < t.num_blocks) t.free_ids[to] = row[j];
        }
        for (int j = own + lane_id(); j < target; j += 32) row[j] = block_taken(t, p, count, have, p.taken[s] + (j - own));
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
    const int64_t want = std::max((int64_t(r.max_rows) + kFillThreads - 1) / kFillThreads, (int64_t(t.seqs) * 32 + kFillThreads - 1) / kFillThreads);
    if (want == 0) return cudaSuccess;
    fill_kernel<<<unsigned(std::min<int64_t>(want, int64_t(sm_count) * 8)), kFillThreads, 0, st>>>(length, t, r, ws);
    count_launch(LAUNCH_BLOCKS);
    return cudaGetLastError();
}

}  // namespace wb
