// Block tables and slot maps built on the device from request lengths (ttkv_plan_step) and the
// return of finished requests' blocks (ttkv_release_blocks).
//
// Mathematics: need_r = ceil(seq_r / bs) - ceil((seq_r - new_r) / bs); an inclusive prefix sum over
// the requests gives each one its range of the free list, and a token at position p of request r
// lies in slot table[r][p / bs] * bs + p % bs. All integers.
//
// Bound: launch and load latency (a step moves a few KB to a few hundred KB). So one launch, one
// cluster of CTAs: every CTA repeats the prefix sum over all requests (a few hundred loads) rather than
// waiting for another CTA's, keeps each request's lengths and its end in the free list in shared
// memory, and then takes its share of the blocks that change hands and of the tokens, each found by a
// binary search, so that a step has two rounds of loads whatever its mix of lengths. One decode token
// for each of 8, 1024, 4096 and 16384 requests takes 8.3, 12.3, 22.5 and 64 us from an idle GPU (8.6,
// 13.3, 32.8 and 111 with one CTA), 16384 tokens of 64 requests 12.3 (45 with one). A release writes
// the ids as it reads them, behind the list's end, and starts over without a request's where one is
// negative or the room was too little: looking at all of them first would be a third round of loads. The cluster's barrier orders
// every CTA's read of the count before the write of the new one, which may be the same word.
#include <cooperative_groups.h>

#include <utility>

#include "ttkv_async.cuh"
#include "ttkv_common.cuh"

namespace ttkv {
namespace {

namespace cg = cooperative_groups;

constexpr int kPlanCtas = 8;        // the largest portable cluster
constexpr int kPlanThreads = 512;

using PlanParams = ttkv_plan_args_t;

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

// A request in shared memory: its tokens, its start (plan) and the end of its range of the free list,
// counted from the list's end (plan) or from its old end (release). A refused request's range is empty
// and its length is kept as ~seq.
struct PlanSmem {
    int32_t* len;
    int32_t* end;
    int32_t* start;                                  // [n_reqs + 1]
};

// Release: the length of a request whose row holds a negative id.
constexpr int32_t kBadRow = INT32_MIN;

// Fills len and end; returns the blocks taken or returned in all, and whether the room was too little.
// again (release): requests whose length is kBadRow are left out.
template <bool RELEASE>
__device__ int assign_ranges(const PlanParams& P, int avail, const PlanSmem& M, long long* wsum, int32_t* taken, bool& lacking,
                             bool again = false) {
    const int tid = threadIdx.x;
    const bool first = blockIdx.x == 0;
    long long carry = 0;
    if (tid == 0) *taken = 0;
    __syncthreads();
    for (int r0 = 0; r0 < P.n_reqs; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int need = 0, seq = 0;
        bool ok = r < P.n_reqs;
        if (ok) {
            seq = P.lens[r];
            if (RELEASE) {
                ok = !again || M.len[r] != kBadRow;
                need = ok ? blocks_of(seq, P.block_size) : 0;
            } else {
                const int a = P.query_start_loc[r], b = P.query_start_loc[r + 1];
                M.start[r] = a;
                if (r == P.n_reqs - 1) M.start[P.n_reqs] = b;
                if (a < 0 || b < a || b > P.n_tokens || seq < b - a) {
                    ok = false;
                    if (first) report(P.status, TTKV_STATUS_QUERY);
                } else {
                    need = blocks_of(seq, P.block_size) - blocks_of(seq - (b - a), P.block_size);
                }
            }
            if (ok && blocks_of(seq, P.block_size) > P.bt_cols) {
                ok = false;
                need = 0;
                if (first) report(P.status, TTKV_STATUS_ROW_SHORT);
            }
        }
        long long total;
        const long long end = carry + scan_inclusive(need, wsum, total);
        if (ok && need > 0 && end > avail) ok = false;      // and so for every later request with a need
        if (ok && need > 0) atomicMax(taken, int32_t(end));
        if (r < P.n_reqs) {
            M.len[r] = ok ? seq : ~max(seq, 0);
            M.end[r] = ok || end <= avail ? int32_t(min(end, (long long)avail)) : -1;
        }
        carry += total;
    }
    lacking = carry > avail;
    __syncthreads();
    // from the first refusal for want of room on, every end is the last one granted
    const int used = *taken;
    for (int r = tid; r < P.n_reqs; r += kPlanThreads)
        if (M.end[r] < 0 || M.end[r] > used) M.end[r] = used;
    if (!RELEASE && P.n_reqs == 0 && tid == 0) M.start[0] = 0;
    __syncthreads();
    return used;
}

// The first request whose value in `ends` is above e (n_reqs: none).
__device__ __forceinline__ int find(const int32_t* ends, int n_reqs, int e) {
    int lo = 0, hi = n_reqs;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] <= e) lo = mid + 1; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_step_kernel(const PlanParams P) {
    extern __shared__ int32_t plan_smem[];
    __shared__ long long wsum[32];
    __shared__ int32_t taken;
    const PlanSmem M{plan_smem, plan_smem + P.n_reqs, plan_smem + 2 * P.n_reqs};
    const int at = blockIdx.x * kPlanThreads + threadIdx.x, step = gridDim.x * kPlanThreads;
    pdl_wait();
    pdl_trigger();
    const int count = min(max(*P.free_count, 0), P.capacity);
    bool lacking;
    const int used = assign_ranges<false>(P, count, M, wsum, &taken, lacking);
    if (lacking && at == 0) report(P.status, TTKV_STATUS_POOL_EMPTY);

    // a refused request's row: no block behind those that it holds, as far as it would have reached, so that
    // a later step that takes them for its own does not meet what another request left there
    for (int r = at; r < P.n_reqs; r += step) {
        if (M.len[r] >= 0) continue;
        const int seq = ~M.len[r], fresh = max(M.start[r + 1] - M.start[r], 0), held = blocks_of(seq - fresh, P.block_size);
        const int end = fresh > seq ? 1 : min(max(blocks_of(seq, P.block_size), held + 1), P.bt_cols);
        for (int i = held; i < min(end, P.bt_cols); ++i) P.block_table[int64_t(r) * P.bt_stride + i] = -1;
    }
    // the blocks taken, into their rows
    for (unsigned i = at; i < unsigned(used); i += step) {
        const int e = int(i);
        const int r = find(M.end, P.n_reqs, e), first = r ? M.end[r - 1] : 0;
        const int held = blocks_of(M.len[r] - (M.start[r + 1] - M.start[r]), P.block_size);
        const int32_t id = P.free_blocks[count - 1 - e];
        if (id < 0) report(P.status, TTKV_STATUS_BLOCK_RANGE);
        P.block_table[int64_t(r) * P.bt_stride + held + (e - first)] = id;
    }
    // the tokens
    for (unsigned i = at; i < unsigned(P.n_tokens); i += step) {
        const int t = int(i);
        const int r = find(M.start + 1, P.n_reqs, t);
        int64_t slot = -1;
        int pos = 0;
        if (r < P.n_reqs && t >= M.start[r] && M.len[r] >= 0) {
            const int ql = M.start[r + 1] - M.start[r], first = r ? M.end[r - 1] : 0;
            pos = M.len[r] - ql + (t - M.start[r]);
            const int held = blocks_of(M.len[r] - ql, P.block_size), bi = int(unsigned(pos) / unsigned(P.block_size));
            const int blk = bi < held ? P.block_table[int64_t(r) * P.bt_stride + bi] : P.free_blocks[count - 1 - (first + bi - held)];
            if (blk >= 0) slot = int64_t(blk) * P.block_size + (pos - bi * P.block_size);
        }
        P.slots[t] = slot;
        if (P.positions) P.positions[t] = pos;
    }
    cg::this_cluster().sync();                       // every CTA has read the count
    if (at == 0) *P.free_count_out = count - used;
}

// The granted requests' ids onto the list's end, this thread's share of them; whether one is negative.
__device__ bool push_ids(const PlanParams& P, const PlanSmem& M, int count, int used, int at, int step) {
    bool bad = false;
    #pragma unroll 4
    for (unsigned i = at; i < unsigned(used); i += step) {
        const int e = int(i);
        const int r = find(M.end, P.n_reqs, e);
        const int32_t id = P.block_table[int64_t(r) * P.bt_stride + (e - (r ? M.end[r - 1] : 0))];
        bad |= id < 0;
        P.free_blocks[count + e] = id;
    }
    return bad;
}

__global__ void __launch_bounds__(kPlanThreads) release_blocks_kernel(const PlanParams P) {
    extern __shared__ int32_t plan_smem[];
    __shared__ long long wsum[32];
    __shared__ int32_t taken;
    __shared__ int bad_row;                          // some CTA of the cluster met a negative id
    const PlanSmem M{plan_smem, plan_smem + P.n_reqs, nullptr};
    const int at = blockIdx.x * kPlanThreads + threadIdx.x, step = gridDim.x * kPlanThreads;
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) bad_row = 0;
    auto begun = cluster.barrier_arrive();
    pdl_wait();
    pdl_trigger();
    const int count = min(max(*P.free_count, 0), P.capacity), avail = P.capacity - count;
    bool lacking;
    int used = assign_ranges<true>(P, avail, M, wsum, &taken, lacking);
    cluster.barrier_wait(std::move(begun));          // every CTA's bad_row may be written
    if (push_ids(P, M, count, used, at, step))
        for (int c = 0; c < kPlanCtas; ++c) *cluster.map_shared_rank(&bad_row, c) = 1;
    cluster.sync();
    if (bad_row || lacking) {                        // (the same in every CTA) once more without the rows that hold one
        const int lane = threadIdx.x & 31;
        for (int r = threadIdx.x >> 5; r < P.n_reqs; r += kPlanThreads / 32) {
            const int nb = blocks_of(P.lens[r], P.block_size);
            bool bad = false;
            if (nb <= P.bt_cols)
                for (int k = lane; k < nb; k += 32) bad |= P.block_table[int64_t(r) * P.bt_stride + k] < 0;
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) M.len[r] = bad ? kBadRow : 0;
            if (bad && lane == 0 && blockIdx.x == 0) report(P.status, TTKV_STATUS_BLOCK_RANGE);
        }
        __syncthreads();
        used = assign_ranges<true>(P, avail, M, wsum, &taken, lacking, true);
        push_ids(P, M, count, used, at, step);
    }
    if (at == 0) {
        if (lacking) report(P.status, TTKV_STATUS_POOL_FULL);
        *P.free_count_out = count + used;
    }
}

int check_plan(const ttkv_plan_args_t* p) {
    if (!p) return fail(TTKV_ERR_ARG, "plan: null arguments");
    const ttkv_plan_args_t& P = *p;
    if (!P.free_count || !P.free_count_out || (P.n_reqs > 0 && !P.lens) ||
        (P.n_reqs > 0 && P.bt_cols > 0 && !P.block_table) || (P.capacity > 0 && !P.free_blocks))
        return fail(TTKV_ERR_ARG, "plan: null pointer");
    if (P.n_reqs < 0 || P.bt_cols < 0 || P.capacity < 0 || P.n_tokens < 0) return fail(TTKV_ERR_ARG, "plan: a negative size");
    if (P.block_size < 1) return fail(TTKV_ERR_ARG, "plan: block size %d", P.block_size);
    if (P.n_reqs > 1 && P.bt_stride < P.bt_cols) return fail(TTKV_ERR_ARG, "plan: block-table rows overlap");
    if (P.n_reqs > TTKV_PLAN_MAX_REQS)
        return fail(TTKV_ERR_UNSUPPORTED, "plan: %d requests > %d", P.n_reqs, TTKV_PLAN_MAX_REQS);
    return TTKV_OK;
}

template <typename K>
int launch_plan(K kernel, const PlanParams& P, size_t smem, const char* what) {
    if (int e = raise_smem_limit(reinterpret_cast<const void*>(kernel), what)) return e;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kPlanCtas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kPlanCtas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(P.stream);
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(TTKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    }
    return TTKV_OK;
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" int ttkv_plan_step(const ttkv_plan_args_t* args) {
    if (int e = check_plan(args)) return e;
    if (!args->query_start_loc || (args->n_tokens > 0 && !args->slots)) return fail(TTKV_ERR_ARG, "plan: null pointer");
    return launch_plan(plan_step_kernel, *args, (3 * size_t(args->n_reqs) + 1) * sizeof(int32_t), "plan_step_kernel");
}

extern "C" int ttkv_release_blocks(const ttkv_plan_args_t* args) {
    if (int e = check_plan(args)) return e;
    return launch_plan(release_blocks_kernel, *args, (2 * size_t(args->n_reqs) + 1) * sizeof(int32_t), "release_blocks_kernel");
}
