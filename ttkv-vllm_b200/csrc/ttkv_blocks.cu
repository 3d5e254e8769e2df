// Block tables and slot maps built on the device from request lengths (ttkv_plan_step) and the
// return of finished requests' blocks (ttkv_release_blocks).
//
// Mathematics: need_r = ceil(seq_r / bs) - ceil((seq_r - new_r) / bs); an inclusive prefix sum over
// the requests gives each one its range of the free list, and a token at position p of request r
// lies in slot table[r][p / bs] * bs + p % bs. All integers.
//
// Bound: launch and load latency (a step moves a few KB to a few hundred KB). So one launch, one
// cluster of 8 CTAs: every CTA repeats the prefix sum over all requests (a few hundred loads) rather
// than waiting for another CTA's, keeps each request's start in shared memory, and fills its share
// of the tokens and of the table rows. The cluster's barrier orders every CTA's read of the count
// before the write of the new one, which may be the same word.
#include <cooperative_groups.h>

#include "ttkv_common.cuh"

namespace ttkv {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanCtas = 8;        // the largest portable cluster
constexpr int kPlanThreads = 512;

struct PlanParams {
    int32_t* table;
    int64_t bt_stride;
    int32_t bt_cols;
    const int32_t* lens;            // seq_lens of a plan, lens of a release
    const int32_t* qsl;
    int32_t n_reqs;
    int32_t* free_blocks;
    int32_t capacity;
    const int32_t* count;
    int32_t* count_out;
    int32_t bs;
    int64_t* slots;
    int64_t* positions;
    int32_t n_tokens;
    int32_t* status;
};

__device__ __forceinline__ int blocks_of(int tokens, int bs) {
    return tokens > 0 ? int((unsigned(tokens) + unsigned(bs) - 1u) / unsigned(bs)) : 0;
}

// Inclusive scan of v over the CTA's threads; `total` = the CTA's sum. wsum: 32 words of shared memory.
__device__ __forceinline__ long long scan_inclusive(long long v, long long* wsum, long long& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) wsum[w] = v;
    __syncthreads();
    long long before = 0, all = 0;
    #pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i) {
        const long long s = wsum[i];
        before += i < w ? s : 0;
        all += s;
    }
    __syncthreads();
    total = all;
    return v + before;
}

// base[r]: request r's first entry of its range of the free list, counted from the list's end (plan)
// or from its old end (release); -1: refused. Returns the blocks taken or returned in all.
template <bool RELEASE>
__device__ int assign_ranges(const PlanParams& P, int avail, int32_t* base, long long* wsum, int32_t* taken) {
    const int tid = threadIdx.x;
    const bool first = blockIdx.x == 0;
    long long carry = 0;
    if (tid == 0) *taken = 0;
    __syncthreads();
    for (int r0 = 0; r0 < P.n_reqs; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int need = 0;
        bool ok = r < P.n_reqs;
        if (ok) {
            const int seq = P.lens[r];
            if (RELEASE) {
                need = blocks_of(seq, P.bs);
            } else {
                const int a = P.qsl[r], b = P.qsl[r + 1];
                if (a < 0 || b < a || b > P.n_tokens || seq < b - a) {
                    ok = false;
                    if (first) report(P.status, TTKV_STATUS_QUERY);
                } else {
                    need = blocks_of(seq, P.bs) - blocks_of(seq - (b - a), P.bs);
                }
            }
            if (ok && blocks_of(seq, P.bs) > P.bt_cols) {
                ok = false;
                need = 0;
                if (first) report(P.status, TTKV_STATUS_ROW_SHORT);
            }
        }
        long long total;
        const long long end = carry + scan_inclusive(need, wsum, total);
        if (ok && need > 0 && end > avail) {                 // and so for every later request with a need
            ok = false;
            if (first) report(P.status, RELEASE ? TTKV_STATUS_POOL_FULL : TTKV_STATUS_POOL_EMPTY);
        }
        if (r < P.n_reqs) base[r] = ok ? int32_t(min(end - need, (long long)avail)) : -1;
        if (ok && need > 0) atomicMax(taken, int32_t(end));
        carry += total;
    }
    __syncthreads();
    return *taken;
}

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) plan_step_kernel(const PlanParams P) {
    extern __shared__ int32_t plan_smem[];
    __shared__ long long wsum[32];
    __shared__ int32_t taken;
    int32_t* base = plan_smem;                       // [n_reqs]
    int32_t* start = plan_smem + P.n_reqs;           // [n_reqs + 1] query_start_loc
    const int tid = threadIdx.x, rank = blockIdx.x;
    const int count = min(max(*P.count, 0), P.capacity);
    for (int r = tid; r <= P.n_reqs; r += kPlanThreads) start[r] = P.qsl[r];
    const int used = assign_ranges<false>(P, count, base, wsum, &taken);

    // the table rows: a warp per request
    const int lane = tid & 31;
    for (int r = rank * (kPlanThreads / 32) + (tid >> 5); r < P.n_reqs; r += kPlanCtas * (kPlanThreads / 32)) {
        const int seq = P.lens[r], ql = start[r + 1] - start[r];
        int32_t* row = P.table + int64_t(r) * P.bt_stride;
        const int held = blocks_of(seq - max(ql, 0), P.bs);
        if (base[r] < 0) {
            if (lane == 0 && held < P.bt_cols) row[held] = -1;
            continue;
        }
        const int want = blocks_of(seq, P.bs);
        for (int i = held + lane; i < want; i += 32) row[i] = P.free_blocks[count - 1 - (base[r] + i - held)];
    }

    // the tokens: request by a binary search of the starts
    for (int t = rank * kPlanThreads + tid; t < P.n_tokens; t += kPlanCtas * kPlanThreads) {
        int lo = 0, hi = P.n_reqs;                   // the last r with start[r] <= t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (start[mid + 1] <= t) lo = mid + 1; else hi = mid;
        }
        int64_t slot = -1;
        int pos = 0;
        if (lo < P.n_reqs && t >= start[lo] && base[lo] >= 0) {
            const int seq = P.lens[lo], ql = start[lo + 1] - start[lo];
            pos = seq - ql + (t - start[lo]);
            const int held = blocks_of(seq - ql, P.bs), bi = int(unsigned(pos) / unsigned(P.bs));
            const int blk = bi < held ? P.table[int64_t(lo) * P.bt_stride + bi]
                                      : P.free_blocks[count - 1 - (base[lo] + bi - held)];
            if (blk >= 0) slot = int64_t(blk) * P.bs + (pos - bi * P.bs);
        }
        P.slots[t] = slot;
        if (P.positions) P.positions[t] = pos;
    }
    cg::this_cluster().sync();                       // every CTA has read the count
    if (rank == 0 && tid == 0) *P.count_out = count - used;
}

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) release_blocks_kernel(const PlanParams P) {
    extern __shared__ int32_t plan_smem[];
    __shared__ long long wsum[32];
    __shared__ int32_t taken;
    int32_t* base = plan_smem;
    const int tid = threadIdx.x, rank = blockIdx.x, lane = tid & 31;
    const int count = min(max(*P.count, 0), P.capacity);
    const int used = assign_ranges<true>(P, P.capacity - count, base, wsum, &taken);
    for (int r = rank * (kPlanThreads / 32) + (tid >> 5); r < P.n_reqs; r += kPlanCtas * (kPlanThreads / 32)) {
        if (base[r] < 0) continue;
        const int n = blocks_of(P.lens[r], P.bs);
        const int32_t* row = P.table + int64_t(r) * P.bt_stride;
        bool bad = false;
        for (int i = lane; i < n; i += 32) {
            const int32_t id = row[i];
            bad |= id < 0;
            P.free_blocks[count + base[r] + i] = id;
        }
        if (bad) report(P.status, TTKV_STATUS_BLOCK_RANGE);
    }
    cg::this_cluster().sync();
    if (rank == 0 && tid == 0) *P.count_out = count + used;
}

int check_plan(const PlanParams& P) {
    if (!P.count || !P.count_out || (P.n_reqs > 0 && !P.lens) || (P.n_reqs > 0 && P.bt_cols > 0 && !P.table) ||
        (P.capacity > 0 && !P.free_blocks))
        return fail(TTKV_ERR_ARG, "plan: null pointer");
    if (P.n_reqs < 0 || P.bt_cols < 0 || P.capacity < 0 || P.n_tokens < 0)
        return fail(TTKV_ERR_ARG, "plan: a negative size");
    if (P.bs < 1) return fail(TTKV_ERR_ARG, "plan: block size %d", P.bs);
    if (P.n_reqs > 1 && P.bt_stride < P.bt_cols) return fail(TTKV_ERR_ARG, "plan: block-table rows overlap");
    if (P.n_reqs > TTKV_PLAN_MAX_REQS)
        return fail(TTKV_ERR_UNSUPPORTED, "plan: %d requests > %d", P.n_reqs, TTKV_PLAN_MAX_REQS);
    return TTKV_OK;
}

template <typename K>
int launch_plan(K kernel, const PlanParams& P, size_t smem, const char* what, void* stream) {
    if (int e = raise_smem_limit(reinterpret_cast<const void*>(kernel), what)) return e;
    kernel<<<kPlanCtas, kPlanThreads, smem, static_cast<cudaStream_t>(stream)>>>(P);
    return check_launch(what);
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" int ttkv_plan_step(int32_t* block_table, int64_t bt_stride, int32_t bt_cols, const int32_t* seq_lens,
                              const int32_t* query_start_loc, int32_t n_reqs, const int32_t* free_blocks,
                              int32_t capacity, const int32_t* free_count, int32_t* free_count_out,
                              int32_t block_size, int64_t* slots, int64_t* positions, int32_t n_tokens,
                              int32_t* status, void* stream) {
    PlanParams P{block_table, bt_stride, bt_cols, seq_lens, query_start_loc, n_reqs,
                 const_cast<int32_t*>(free_blocks), capacity, free_count, free_count_out, block_size,
                 slots, positions, n_tokens, status};
    if (int e = check_plan(P)) return e;
    if (!query_start_loc || (n_tokens > 0 && !slots)) return fail(TTKV_ERR_ARG, "plan: null pointer");
    return launch_plan(plan_step_kernel, P, (2 * size_t(n_reqs) + 1) * sizeof(int32_t), "plan_step_kernel", stream);
}

extern "C" int ttkv_release_blocks(const int32_t* block_table, int64_t bt_stride, int32_t bt_cols,
                                   const int32_t* lens, int32_t n_reqs, int32_t* free_blocks, int32_t capacity,
                                   const int32_t* free_count, int32_t* free_count_out, int32_t block_size,
                                   int32_t* status, void* stream) {
    PlanParams P{const_cast<int32_t*>(block_table), bt_stride, bt_cols, lens, nullptr, n_reqs, free_blocks,
                 capacity, free_count, free_count_out, block_size, nullptr, nullptr, 0, status};
    if (int e = check_plan(P)) return e;
    return launch_plan(release_blocks_kernel, P, (size_t(n_reqs) + 1) * sizeof(int32_t), "release_blocks_kernel", stream);
}
