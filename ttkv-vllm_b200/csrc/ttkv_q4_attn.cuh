// Attention over the 4-bit paged cache: what its two kernels share. q4_stream_kernel (ttkv_q4_stream.cu)
// takes one or a few queries per request, q4_chunk_kernel (ttkv_q4_chunk.cu) chunks of them.
#pragma once

#include <algorithm>

#include "ttkv_async.cuh"
#include "ttkv_q4.cuh"

namespace ttkv {
namespace q4 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCtas = 148;               // one CTA per SM of a B200; workspaces are sized for it
constexpr int kMaxSeq = 0x7fffff00;         // a tile behind the last token still has a 32-bit position

struct AttnParams {
    const uint8_t* cache;
    int64_t n_blocks;
    int32_t H, G, block_size, bs_shift;     // log2 of the block size, -1 where it is no power of two
    const int32_t* block_table;
    int64_t bt_stride;
    int32_t bt_cols;
    const int32_t* seq_lens;
    const int32_t* q_start;                 // null: one query per request
    const int32_t* q_len;
    int32_t n_reqs, n_rows, max_q, max_seq; // the last two bound q_len and seq_lens
    const void* q;
    int32_t dtype, q_vec, out_vec;
    int64_t q_stride;
    float scale;
    void* out;
    int64_t out_stride;
    int32_t n_ctas;
    float* part_ml;                         // [n_ctas][2][rows of a block][2]
    float* part_o;                          // [n_ctas][2][rows of a block][D]
    float* first;                           // [n_ctas][warps] parts of the warps' first segments (streaming kernel)
    int32_t* rec;                           // [n_ctas][8] what each CTA leaves to the merge (chunk kernel)
    int32_t* status;
};

// ------------------------------------------------------------------ the batch
// A request's tokens, queries (none where it is refused) and first query row.
struct Req {
    int seq, ql, q0;
};

__device__ __forceinline__ Req request(const AttnParams& P, int r, bool tell) {
    Req a;
    a.seq = max(P.seq_lens[r], 0);
    a.ql = P.q_len ? P.q_len[r] : 1;
    a.q0 = P.q_start ? P.q_start[r] : r;
    int code = 0;
    if (P.q_len && a.ql > 0 &&
        (a.ql > a.seq || a.ql > P.max_q || a.q0 < 0 || int64_t(a.q0) + a.ql > P.n_rows)) code = TTKV_STATUS_QUERY;
    else if (a.seq > P.max_seq && a.ql > 0) code = TTKV_STATUS_SEQ_BOUND;
    else if (a.seq > int64_t(P.bt_cols) * P.block_size && a.ql > 0) code = TTKV_STATUS_ROW_SHORT;
    if (code && tell) report(P.status, code);
    if (code || a.ql < 0) a.ql = 0;
    return a;
}

__device__ __forceinline__ int row_blocks(const Req& a, int G, int rows) { return int((unsigned(a.ql) * unsigned(G) + rows - 1) / rows); }

// The list of T units shared out to n CTAs: CTA c owns [c S, (c + 1) S), S = ceil(T / n), cut at T.
__device__ __forceinline__ int share_size(int T, int n) { return (T + n - 1) / n; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// ------------------------------------------------------------------ partial results
// Weighted sum of partials (max m_i, sum l_i, rows o_i relative to m_i): relative to M = max m_i.
__device__ __forceinline__ float part_weight(float m, float M) { return M == -INFINITY ? 1.f : ex2(m - M); }

// Four output values from element i of the output.
__device__ __forceinline__ void store4(const AttnParams& P, int64_t i, float4 x) {
    if (P.out_vec) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + i) =
            make_uint2(pack2(x.x, x.y, P.dtype), pack2(x.z, x.w, P.dtype));
    } else {
        store_elt(P.out, P.dtype, i, x.x);
        store_elt(P.out, P.dtype, i + 1, x.y);
        store_elt(P.out, P.dtype, i + 2, x.z);
        store_elt(P.out, P.dtype, i + 3, x.w);
    }
}

// Four output values o / l from lane index `lane` (a multiple of 4) of row (query j, head g of h).
__device__ __forceinline__ void store_out(const AttnParams& P, const Req& rq, int h, int row, int D, int lane, float4 o,
                                          float l) {
    const int j = row / P.G, g = row - j * P.G;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t i = int64_t(rq.q0 + j) * P.out_stride + int64_t(h * P.G + g) * D + lane;
    store4(P, i, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------ host
inline int sm_count(int* n) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return fail(TTKV_ERR_CUDA, "no CUDA device");
    }
    return TTKV_OK;
}

// ttkv_q4_chunk.cu
size_t chunk_workspace_bytes(int d);
int run_chunk(const ttkv_q4_cache_t* c, AttnParams P, void* ws, size_t ws_bytes, cudaStream_t st);

}  // namespace q4
}  // namespace ttkv
