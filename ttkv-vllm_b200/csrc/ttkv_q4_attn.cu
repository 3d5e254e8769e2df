// Attention over the 4-bit paged cache: one query token per request (ttkv_q4_decode) or a chunk of
// them (ttkv_q4_prefill).
//
//   o = sum_t p_t V_t / sum_t p_t,   p_t = exp(scale q . K_t),   K_t = m_t + s_t c_t (V alike)
//
// q4_stream_kernel reads every stored byte once per block of 8 NT (query, head) rows and is bound by
// memory. The codes c are never turned into values: they are exact operands of the tensor cores,
// and scales and minima act on the products,
//
//   q . K_t = s_t (q . c_t) + m_t sum(q)
//   o       = sum_t (p_t s_t) (c_t - 7.5) + sum_t p_t (m_t + 7.5 s_t).
//
// A code in the low bits of an fp16 is the subnormal c 2^-24, so one mask makes two operands of a
// word (the next nibble's come out as c 2^-20: q is stored with the factor, o divided by it); eight
// values cost five instructions. p_t s_t is rounded to fp16, an operand of the matrix product, after
// scaling by a power of two that keeps the largest near 2^14. It multiplies c - 7.5 (the second sum
// takes the rounded weight's share of 7.5, and is fp32), so the rounding error is that of weights on
// centred values: 2^-12 of each term at most.
#include <algorithm>

#include "ttkv_async.cuh"
#include "ttkv_q4.cuh"

namespace ttkv {
namespace {

using namespace q4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;                   // warps of a streaming CTA, each on its own run of tokens
constexpr int kUnit = 64;                   // tokens of a unit of work: one softmax step of a warp

struct AttnParams {
    const uint8_t* cache;
    int64_t n_blocks;
    int32_t H, G, block_size;
    const int32_t* block_table;
    int64_t bt_stride;
    int32_t bt_cols;
    const int32_t* seq_lens;
    const int32_t* q_start;                 // null: one query per request
    const int32_t* q_len;
    int32_t n_reqs, n_rows, max_q, max_seq;
    const void* q;
    int32_t dtype, q_vec, out_vec;
    int64_t q_stride;
    float scale;
    void* out;
    int64_t out_stride;
    int32_t n_ctas;
    int64_t* prefix;                        // [n_reqs + 1] units before each request (workspace)
    float* part_ml;                         // [n_ctas][2][rows][2]
    float* part_o;                          // [n_ctas][2][rows][D]
    int32_t* status;
};

// ------------------------------------------------------------------ the batch
// A request's tokens, queries and rows (query, head of the group), or n = 0 where it is refused.
struct Req {
    int seq, ql, q0;
    bool refused;
};

__device__ __forceinline__ Req request(const AttnParams& P, int r, bool tell) {
    Req a;
    a.seq = max(P.seq_lens[r], 0);
    a.ql = P.q_len ? P.q_len[r] : 1;
    a.q0 = P.q_start ? P.q_start[r] : r;
    a.refused = false;
    int code = 0;
    if (P.q_len && a.ql > 0 &&
        (a.ql > a.seq || a.ql > P.max_q || a.q0 < 0 || int64_t(a.q0) + a.ql > P.n_rows)) code = TTKV_STATUS_QUERY;
    else if (P.max_seq > 0 && a.seq > P.max_seq && a.ql > 0) code = TTKV_STATUS_SEQ_BOUND;
    else if ((int64_t(a.seq) + P.block_size - 1) / P.block_size > P.bt_cols && a.ql > 0) code = TTKV_STATUS_ROW_SHORT;
    if (code) {
        a.refused = true;
        if (tell) report(P.status, code);
    }
    if (a.refused || a.ql < 0) a.ql = 0;
    return a;
}

__device__ __forceinline__ int row_blocks(const Req& a, int G, int rows) { return int((int64_t(a.ql) * G + rows - 1) / rows); }
__device__ __forceinline__ int units_of(const Req& a) { return a.ql > 0 ? (a.seq + kUnit - 1) / kUnit : 0; }

// The CTA that owns unit u of T shared out to n CTAs, CTA c owning [c T / n, (c + 1) T / n).
__device__ __forceinline__ int64_t share_begin(int64_t c, int64_t T, int64_t n) { return c * T / n; }
__device__ __forceinline__ int64_t owner_of(int64_t u, int64_t T, int64_t n) { return ((u + 1) * n - 1) / T; }

// ------------------------------------------------------------------ warp-level products
// D += A (16 x 16, row) . B (16 x 8, column), fp16 operands and fp32 sums.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

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

// ------------------------------------------------------------------ one warp's rows
// Fragment places of lane (b = lane / 4, a = lane % 4): stored tokens b and b + 8 of a panel as rows
// of S^T, rows 2 a and 2 a + 1 of each block of 8 (query, head) rows as its columns; output lanes
// 32 j + 4 b + (0..3) as rows of O^T.
template <int D, int GRP, int NT>
struct WarpRows {
    static constexpr int NW = D / 32, NG = D / GRP, WPG = GRP / 32, ROWS = 8 * NT;
    uint32_t qf[NT][2 * NW][2];         // q 2^e as B fragments, lanes 8 a + (0..7) of each 32
    float q1[NT][2][NG], qm[NT][2];     // sums of q 2^e over each group; 2^-e scale log2(e)
    int lim[NT][2], min_lim;            // tokens each row sees; the fewest any row of the block does
    float m[NT][2], l[NT][2];           // running max (base 2) and this lane's share of the sum
    float o[2 * NW][NT][4];             // (p s 2^vn) . c
    float dsum[NT][2][NG];              // this lane's share of 2^vn p (m + 7.5 s) - 7.5 (p s 2^vn)
    float vn;                           // 2^vn, the scaling of the weights

    __device__ __forceinline__ void start(const AttnParams& P, const Req& rq, int h, int rb, int lane) {
        const int b = lane >> 2, a = lane & 3;
        const int n_rows = rq.ql * P.G;
        min_lim = 0x7fffffff;
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // row b's fragment, and its sums and factor to the lanes that hold its columns
            const int row = rb * ROWS + 8 * nt + b;
            const bool live = row < n_rows;
            const int j = live ? row / P.G : 0, g = live ? row - j * P.G : 0;
            const int64_t src = int64_t(rq.q0 + j) * P.q_stride + int64_t(h * P.G + g) * D + 8 * a;
            float x[NW][8], big = 0.f;
            #pragma unroll
            for (int w = 0; w < NW; ++w) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) x[w][i] = 0.f;
                if (live) load8(P.q, P.dtype, src + 32 * w, P.q_vec, x[w]);
                #pragma unroll
                for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[w][i]));
            }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // e brings the row's largest |q| into [1, 2): fp16 then holds every element to 2^-20 of it
            const int e = big > 0.f && big < INFINITY ? 127 - int(__float_as_uint(big) >> 23) : 0;
            const float up = __uint_as_float(uint32_t(min(127 + e, 254)) << 23);
            float sum[NG];
            #pragma unroll
            for (int k = 0; k < NG; ++k) sum[k] = 0.f;
            #pragma unroll
            for (int w = 0; w < NW; ++w) {
                #pragma unroll
                for (int i = 0; i < 8; ++i) { x[w][i] *= up; sum[w / WPG] += x[w][i]; }
                // nibbles 0, 2, 4, 6 of a word are multiplied as c 2^-24, nibbles 1, 3, 5, 7 as c 2^-20
                qf[nt][2 * w][0] = half2_bits(x[w][0], x[w][4]);
                qf[nt][2 * w][1] = half2_bits(x[w][1] * 0.0625f, x[w][5] * 0.0625f);
                qf[nt][2 * w + 1][0] = half2_bits(x[w][2], x[w][6]);
                qf[nt][2 * w + 1][1] = half2_bits(x[w][3] * 0.0625f, x[w][7] * 0.0625f);
            }
            const float fac = P.scale * kLog2e * __uint_as_float(uint32_t(max(127 - e, 1)) << 23);
            const int seen = live ? rq.seq - rq.ql + j + 1 : 0;
            if (live) min_lim = min(min_lim, seen);
            #pragma unroll
            for (int k = 0; k < NG; ++k) {
                sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
                sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
            }
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int from = (2 * a + c) * 4;
                #pragma unroll
                for (int k = 0; k < NG; ++k) {
                    q1[nt][c][k] = __shfl_sync(0xffffffffu, sum[k], from);
                    dsum[nt][c][k] = 0.f;
                }
                qm[nt][c] = __shfl_sync(0xffffffffu, fac, from);
                lim[nt][c] = __shfl_sync(0xffffffffu, seen, from);
                m[nt][c] = -INFINITY;
                l[nt][c] = 0.f;
            }
            #pragma unroll
            for (int i = 0; i < 2 * NW; ++i)
                #pragma unroll
                for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
        }
        #pragma unroll
        for (int k = 4; k < 32; k <<= 1) min_lim = min(min_lim, __shfl_xor_sync(0xffffffffu, min_lim, k));
        vn = 274877906944.f;                                     // 2^38: the least scale in [2^14, 2^15)
    }

    // Tokens [t0, t0 + 64), panel p of them at pan[p] (null: none, or a block id outside the cache).
    template <bool MASK>
    __device__ __forceinline__ void step_masked(const uint8_t* const (&pan)[4], int t0, int seq, int lane) {
        const int b = lane >> 2, a = lane & 3;
        float s[4][NT][4];
        float tmax[NT][2], vmax = 0.f;
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) tmax[nt][0] = tmax[nt][1] = -INFINITY;
        #pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int ta = t0 + 16 * p + b;                       // this lane's tokens: ta and ta + 8
            if (MASK && t0 + 16 * p >= seq) {                     // no token of this panel (warp-uniform)
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) s[p][nt][i] = -INFINITY;
                continue;
            }
            uint32_t lo[NW], hi[NW], sm[2][NG];
            load_words(pan[p] + b * (D / 2) + a * (D / 8), lo);
            load_words(pan[p] + (b + 8) * (D / 2) + a * (D / 8), hi);
            load_words(pan[p] + k_meta_offset(D) + b * NG * 4, sm[0]);
            load_words(pan[p] + k_meta_offset(D) + (b + 8) * NG * 4, sm[1]);
            float acc[NG][NT][4];
            #pragma unroll
            for (int g = 0; g < NG; ++g)
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) acc[g][nt][i] = 0.f;
            #pragma unroll
            for (int w = 0; w < NW; ++w) {
                const uint32_t l8 = lo[w] >> 8, h8 = hi[w] >> 8;
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816(acc[w / WPG][nt], lo[w] & 0x000f000fu, hi[w] & 0x000f000fu, lo[w] & 0x00f000f0u,
                             hi[w] & 0x00f000f0u, qf[nt][2 * w][0], qf[nt][2 * w][1]);
                    mma16816(acc[w / WPG][nt], l8 & 0x000f000fu, h8 & 0x000f000fu, l8 & 0x00f000f0u, h8 & 0x00f000f0u,
                             qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
                }
            }
            float2 f[2][NG];
            #pragma unroll
            for (int i = 0; i < 2; ++i)
                #pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f[i][g] = __half22float2(*reinterpret_cast<const __half2*>(&sm[i][g]));
                    f[i][g].x *= 16777216.f;                      // 2^24 of the codes
                }
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = i & 1;
                    float x = 0.f;
                    #pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float u = fmaf(f[i >> 1][g].x, acc[g][nt][i], f[i >> 1][g].y * q1[nt][c][g]);
                        x = g ? x + u : u;
                    }
                    x *= qm[nt][c];
                    if (MASK && ta + 8 * (i >> 1) >= lim[nt][c]) x = -INFINITY;
                    s[p][nt][i] = x;
                    tmax[nt][c] = fmaxf(tmax[nt][c], x);
                }
        }
        // the V scales of this lane's tokens (each token's lanes hold the same): their largest keeps
        // the fp16 weights in range
        uint32_t vm[4][2][NG];
        #pragma unroll
        for (int p = 0; p < 4; ++p) {
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool live = !MASK || t0 + 16 * p + b + 8 * i < seq;
                if (live) load_words(pan[p] + v_meta_offset(D, GRP) + (b + 8 * i) * NG * 4, vm[p][i]);
                #pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (!live) vm[p][i][g] = 0u;
                    vmax = fmaxf(vmax, __half2float(__ushort_as_half(uint16_t(vm[p][i][g] & 0xffffu))));
                }
            }
        }
        #pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
            vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, k));
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                tmax[nt][0] = fmaxf(tmax[nt][0], __shfl_xor_sync(0xffffffffu, tmax[nt][0], k));
                tmax[nt][1] = fmaxf(tmax[nt][1], __shfl_xor_sync(0xffffffffu, tmax[nt][1], k));
            }
        }
        // 2^vn with vmax 2^vn in [2^14, 2^15); it only falls, and what is summed falls with it
        float vfall = 1.f;
        {
            const float want = vmax > 0.f ? __uint_as_float(uint32_t(268 - int(__float_as_uint(vmax) >> 23)) << 23) : vn;
            if (want < vn) { vfall = want / vn; vn = want; }
        }
        bool moved = vfall != 1.f;
        float corr[NT][2];
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float mn = fmaxf(m[nt][c], tmax[nt][c]);
                corr[nt][c] = m[nt][c] == -INFINITY ? 1.f : ex2(m[nt][c] - mn);
                moved |= corr[nt][c] != 1.f;
                m[nt][c] = mn;
                l[nt][c] *= corr[nt][c];
                corr[nt][c] *= vfall;
                #pragma unroll
                for (int g = 0; g < NG; ++g) dsum[nt][c][g] *= corr[nt][c];
            }
        if (__any_sync(0xffffffffu, moved)) {
            #pragma unroll
            for (int i = 0; i < 2 * NW; ++i)
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) o[i][nt][k] *= corr[nt][k & 1];
        }
        #pragma unroll
        for (int p = 0; p < 4; ++p) {
            if (MASK && t0 + 16 * p >= seq) continue;
            float pr[NT][4];
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float mm = MASK && m[nt][i & 1] == -INFINITY ? 0.f : m[nt][i & 1];
                    pr[nt][i] = ex2(s[p][nt][i] - mm);
                    l[nt][i & 1] += pr[nt][i];
                }
            uint32_t pf[NG][NT][2];
            #pragma unroll
            for (int g = 0; g < NG; ++g)
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&vm[p][i][g]));
                    const float sv = sm.x * vn, mid = fmaf(7.5f, sv, sm.y * vn);
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float p0 = pr[nt][2 * i], p1 = pr[nt][2 * i + 1];
                        float w0 = p0 * sv, w1 = p1 * sv, d0 = p0 * mid, d1 = p1 * mid;
                        if (MASK) {                              // a weight of 0 on a NaN counts as none
                            const int t = t0 + 16 * p + b + 8 * i;
                            if (t >= lim[nt][0]) w0 = d0 = 0.f;
                            if (t >= lim[nt][1]) w1 = d1 = 0.f;
                        }
                        const __half2 wh = __floats2half2_rn(w0, w1);
                        const float2 wf = __half22float2(wh);
                        dsum[nt][0][g] += fmaf(-7.5f, wf.x, d0);
                        dsum[nt][1][g] += fmaf(-7.5f, wf.y, d1);
                        pf[g][nt][i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&wh));
                    }
                }
            uint32_t lo[NW], hi[NW];                             // tokens 2 a, 2 a + 1 and those + 8
            load_words(pan[p] + 8 * D + a * D + b * (D / 8), lo);
            load_words(pan[p] + 8 * D + (a + 4) * D + b * (D / 8), hi);
            #pragma unroll
            for (int w = 0; w < NW; ++w) {
                const uint32_t l8 = lo[w] >> 8, h8 = hi[w] >> 8;
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t b0 = pf[w / WPG][nt][0], b1 = pf[w / WPG][nt][1];
                    mma16816(o[2 * w][nt], lo[w] & 0x000f000fu, lo[w] & 0x00f000f0u, hi[w] & 0x000f000fu,
                             hi[w] & 0x00f000f0u, b0, b1);
                    mma16816(o[2 * w + 1][nt], l8 & 0x000f000fu, l8 & 0x00f000f0u, h8 & 0x000f000fu, h8 & 0x00f000f0u,
                             b0, b1);
                }
            }
        }
    }

    // Sums over the lanes that share columns; o becomes sum p V relative to m, l the whole sum.
    __device__ __forceinline__ void finish() {
        const float back = 1.f / vn;
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                #pragma unroll
                for (int k = 4; k < 32; k <<= 1) {
                    l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], k);
                    #pragma unroll
                    for (int g = 0; g < NG; ++g) dsum[nt][c][g] += __shfl_xor_sync(0xffffffffu, dsum[nt][c][g], k);
                }
            }
        #pragma unroll
        for (int i = 0; i < 2 * NW; ++i)
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int k = 0; k < 4; ++k)                       // rows + 8 of a fragment came in as c 2^-20
                    o[i][nt][k] = fmaf(o[i][nt][k], k < 2 ? 16777216.f : 1048576.f, dsum[nt][k & 1][i / 2 / WPG]) * back;
    }
};

// ------------------------------------------------------------------ partial results
// Weighted sum of partials (max m_i, sum l_i, rows o_i relative to m_i): relative to M = max m_i.
__device__ __forceinline__ float part_weight(float m, float M) { return M == -INFINITY ? 1.f : ex2(m - M); }

// Four output values o / l from lane index `lane` (a multiple of 4) of row (query j, head g of h).
__device__ __forceinline__ void store_out(const AttnParams& P, const Req& rq, int h, int row, int D, int lane, float4 o,
                                          float l) {
    const int j = row / P.G, g = row - j * P.G;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t i = int64_t(rq.q0 + j) * P.out_stride + int64_t(h * P.G + g) * D + lane;
    const float x[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    if (P.out_vec) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + i) =
            make_uint2(pack2(x[0], x[1], P.dtype), pack2(x[2], x[3], P.dtype));
    } else {
        #pragma unroll
        for (int k = 0; k < 4; ++k) store_elt(P.out, P.dtype, i + k, x[k]);
    }
}

// ------------------------------------------------------------------ the streaming kernel
// The work is the list of (request, KV head, row block, 64-token unit), shared out evenly: CTA c of
// n owns [c T / n, (c + 1) T / n), each of its warps an eighth of that. A warp's run crosses from one
// (request, head, row block) to the next; what a run holds of one is a segment. A segment that is
// whole writes its output; the others meet in shared memory at the end of the CTA, and what is still
// a part then goes to the workspace for q4_merge_kernel (at most the CTA's first and its last).
template <int D, int GRP, int NT>
__global__ void __launch_bounds__(32 * kWarps) q4_stream_kernel(const AttnParams P) {
    using Rows = WarpRows<D, GRP, NT>;
    constexpr int ROWS = 8 * NT, SLOTS = 2 * kWarps;
    extern __shared__ __align__(16) unsigned char smem[];
    float* po = reinterpret_cast<float*>(smem);                                       // [SLOTS][ROWS][D]
    float* pml = po + SLOTS * ROWS * D;                                               // [SLOTS][ROWS][2]
    uint8_t* nan_panel = reinterpret_cast<uint8_t*>(pml + SLOTS * ROWS * 2);          // codes 0, scales NaN
    __shared__ long long pre[32 * kWarps + 1], wsum[kWarps];
    __shared__ long long pid[SLOTS];                     // first unit of the slot's (request, head, row block), -1: none
    __shared__ int pr[SLOTS], ph[SLOTS], prb[SLOTS];

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    const bool tell = blockIdx.x == 0;

    // ---- units of the requests before each thread's share of them
    const int per = (P.n_reqs + 32 * kWarps - 1) / (32 * kWarps);
    const int rlo = min(tid * per, P.n_reqs), rhi = min(rlo + per, P.n_reqs);
    long long mine = 0;
    for (int r = rlo; r < rhi; ++r) {
        const Req a = request(P, r, tell);
        mine += (long long)P.H * row_blocks(a, P.G, ROWS) * units_of(a);
    }
    long long inc = mine;
    #pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, k);
        if (lane >= k) inc += y;
    }
    if (lane == 31) wsum[w] = inc;
    if (tid < SLOTS) pid[tid] = -1;
    for (int i = tid; i < panel_bytes(D, GRP) / 4; i += 32 * kWarps)
        reinterpret_cast<uint32_t*>(nan_panel)[i] = i < 16 * D / 4 ? 0u : 0x00007e00u;
    __syncthreads();
    for (int i = 0; i < w; ++i) inc += wsum[i];
    pre[tid] = inc - mine;
    if (tid == 32 * kWarps - 1) pre[tid + 1] = inc;
    __syncthreads();
    const long long T = pre[32 * kWarps];
    if (tell) {
        long long u = inc - mine;
        for (int r = rlo; r < rhi; ++r) {
            P.prefix[r] = u;
            const Req a = request(P, r, false);
            u += (long long)P.H * row_blocks(a, P.G, ROWS) * units_of(a);
        }
        if (tid == 0) P.prefix[P.n_reqs] = T;
    }
    const long long ca = share_begin(blockIdx.x, T, P.n_ctas), cb = share_begin(blockIdx.x + 1, T, P.n_ctas);
    if (ca == cb) return;

    // ---- this warp's run
    long long u = ca + w * (cb - ca) / kWarps;
    const long long ue = ca + (w + 1) * (cb - ca) / kWarps;
    if (u < ue) {
        int lo = 0, hi = 32 * kWarps - 1;                // the last chunk of requests that begins at or before u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= u) lo = mid; else hi = mid - 1;
        }
        int r = lo * per;
        long long off = u - pre[lo];
        bool first = true;
        while (u < ue) {
            const Req rq = request(P, r, false);
            const int U = units_of(rq), nrb = row_blocks(rq, P.G, ROWS);
            if (off >= (long long)P.H * nrb * U) { off -= (long long)P.H * nrb * U; ++r; continue; }
            const int pair = int(off / U), ui = int(off - (long long)pair * U);
            const int h = pair / nrb, rb = pair - h * nrb;
            const int n_here = int(min((long long)(U - ui), ue - u));
            Rows R;
            R.start(P, rq, h, rb, lane);
            const int32_t* brow = P.block_table + int64_t(r) * P.bt_stride;
            for (int i = 0; i < n_here; ++i) {
                const int t0 = (ui + i) * kUnit;
                const uint8_t* pan[4];
                #pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const int t = t0 + 16 * p;
                    pan[p] = nullptr;
                    if (t < rq.seq) {
                        const int bi = t / P.block_size, blk = brow[bi];
                        if (blk >= 0 && blk < P.n_blocks) {
                            pan[p] = P.cache + ((int64_t(blk) * P.H + h) * (P.block_size / kPanelTokens) +
                                                (t - bi * P.block_size) / kPanelTokens) * panel_bytes(D, GRP);
                        } else {
                            pan[p] = nan_panel;
                            if (lane == 0) report(P.status, TTKV_STATUS_BLOCK_RANGE);
                        }
                    }
                }
                if (t0 + kUnit <= R.min_lim) R.template step_masked<false>(pan, t0, rq.seq, lane);
                else R.template step_masked<true>(pan, t0, rq.seq, lane);
            }
            R.finish();
            const bool whole = ui == 0 && n_here == U;
            const int slot = 2 * w + (first ? 0 : 1);
            const int b = lane >> 2, a = lane & 3;
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int i = 8 * nt + 2 * a + c, row = rb * ROWS + i;
                    #pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        const float4 o = make_float4(R.o[2 * k][nt][c], R.o[2 * k][nt][2 + c], R.o[2 * k + 1][nt][c],
                                                     R.o[2 * k + 1][nt][2 + c]);
                        if (!whole) *reinterpret_cast<float4*>(po + (slot * ROWS + i) * D + 32 * k + 4 * b) = o;
                        else if (row < rq.ql * P.G) store_out(P, rq, h, row, D, 32 * k + 4 * b, o, R.l[nt][c]);
                    }
                    if (!whole && b == 0) {
                        pml[(slot * ROWS + i) * 2] = R.m[nt][c];
                        pml[(slot * ROWS + i) * 2 + 1] = R.l[nt][c];
                    }
                }
            if (!whole && lane == 0) {
                pid[slot] = u - ui;
                pr[slot] = r;
                ph[slot] = h;
                prb[slot] = rb;
            }
            first = false;
            u += n_here;
            off += n_here;
        }
    }
    __syncthreads();

    // ---- what the warps hold of the same (request, head, row block), joined
    for (int s0 = 0; s0 < SLOTS;) {
        const long long id = pid[s0];
        int s1 = s0 + 1;
        if (id < 0) { s0 = s1; continue; }
        int last = s0;
        for (; s1 < SLOTS && (pid[s1] < 0 || pid[s1] == id); ++s1)
            if (pid[s1] == id) last = s1;
        const Req rq = request(P, pr[s0], false);
        const int h = ph[s0], rb = prb[s0];
        const bool whole = id >= ca && id + units_of(rq) <= cb;
        const int64_t g0 = (int64_t(blockIdx.x) * 2 + (ca >= id ? 0 : 1)) * ROWS;
        for (int e = tid; e < ROWS * (D / 4); e += 32 * kWarps) {
            const int i = e / (D / 4), ln = 4 * (e - i * (D / 4));
            float M = -INFINITY;
            for (int s = s0; s <= last; ++s)
                if (pid[s] == id) M = fmaxf(M, pml[(s * ROWS + i) * 2]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
            for (int s = s0; s <= last; ++s) {
                if (pid[s] != id) continue;
                const float wt = part_weight(pml[(s * ROWS + i) * 2], M);
                const float4 x = *reinterpret_cast<const float4*>(po + (s * ROWS + i) * D + ln);
                l = fmaf(wt, pml[(s * ROWS + i) * 2 + 1], l);
                o.x = fmaf(wt, x.x, o.x); o.y = fmaf(wt, x.y, o.y); o.z = fmaf(wt, x.z, o.z); o.w = fmaf(wt, x.w, o.w);
            }
            if (whole) {
                if (rb * ROWS + i < rq.ql * P.G) store_out(P, rq, h, rb * ROWS + i, D, ln, o, l);
            } else {
                *reinterpret_cast<float4*>(P.part_o + (g0 + i) * D + ln) = o;
                if (ln == 0) {
                    P.part_ml[(g0 + i) * 2] = M;
                    P.part_ml[(g0 + i) * 2 + 1] = l;
                }
            }
        }
        s0 = s1;
    }
}

// ------------------------------------------------------------------ the merge
// One CTA per (request, KV head, row): the parts that the CTAs left of its (request, head, row block),
// found from the shares; also the zeros of an empty request. D / 4 threads take four lanes each of
// one part, the CTA's thread groups different parts.
constexpr int kMergeThreads = 256;

__global__ void __launch_bounds__(kMergeThreads) q4_merge_kernel(const AttnParams P, int D, int rows_block) {
    __shared__ float4 so[kMergeThreads];
    __shared__ float sm[kMergeThreads / 16], sl[kMergeThreads / 16], smax[kMergeThreads / 32];
    const int r = blockIdx.y, tid = threadIdx.x;
    const Req rq = request(P, r, false);
    const int per_head = P.max_q * P.G;
    const int h = blockIdx.x / per_head, row = blockIdx.x - h * per_head;
    if (rq.ql <= 0 || row >= rq.ql * P.G) return;
    const int lanes = D / 4, grp = tid / lanes, ngrp = kMergeThreads / lanes, ln = 4 * (tid - grp * lanes);
    const int U = units_of(rq);
    if (U == 0) {
        if (grp == 0) store_out(P, rq, h, row, D, ln, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
        return;
    }
    const int nrb = row_blocks(rq, P.G, rows_block), rb = row / rows_block, i = row - rb * rows_block;
    const int64_t T = P.prefix[P.n_reqs], n = P.n_ctas;
    const int64_t u0 = P.prefix[r] + (int64_t(h) * nrb + rb) * U;
    const int64_t c0 = owner_of(u0, T, n), c1 = owner_of(u0 + U - 1, T, n);
    if (c0 == c1) return;                                        // that CTA has written the output
    auto slot = [&](int64_t c) -> int64_t {
        const int64_t a = share_begin(c, T, n);
        if (a == share_begin(c + 1, T, n)) return -1;            // fewer units than CTAs: nothing there
        return (c * 2 + (a >= u0 ? 0 : 1)) * rows_block + i;
    };
    float M = -INFINITY;
    for (int64_t c = c0 + tid; c <= c1; c += kMergeThreads) {
        const int64_t s = slot(c);
        if (s >= 0) M = fmaxf(M, P.part_ml[2 * s]);
    }
    #pragma unroll
    for (int k = 1; k < 32; k <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
    if ((tid & 31) == 0) smax[tid >> 5] = M;
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < kMergeThreads / 32; ++k) M = fmaxf(M, smax[k]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    #pragma unroll 4
    for (int64_t c = c0 + grp; c <= c1; c += ngrp) {
        const int64_t s = slot(c);
        if (s < 0) continue;
        const float wt = part_weight(P.part_ml[2 * s], M);
        const float4 x = *reinterpret_cast<const float4*>(P.part_o + s * D + ln);
        l = fmaf(wt, P.part_ml[2 * s + 1], l);
        o.x = fmaf(wt, x.x, o.x); o.y = fmaf(wt, x.y, o.y); o.z = fmaf(wt, x.z, o.z); o.w = fmaf(wt, x.w, o.w);
    }
    so[tid] = o;
    if (ln == 0) sl[grp] = l;
    __syncthreads();
    if (grp) return;
    l = 0.f;
    for (int k = 0; k < ngrp; ++k) l += sl[k];
    for (int k = 1; k < ngrp; ++k) {
        const float4 x = so[k * lanes + tid];
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
    }
    store_out(P, rq, h, row, D, ln, o, l);
}

// ------------------------------------------------------------------ host
int sm_count(int* n) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return fail(TTKV_ERR_CUDA, "no CUDA device");
    }
    return TTKV_OK;
}

constexpr int kMaxStreamCtas = 2 * 148;          // the workspace is sized for it (a B200 has 148 SMs)

// Rows a streaming warp takes at once: 8 (query, head) rows a fragment, two fragments above that.
int stream_nt(int64_t rows) { return rows > 8 ? 2 : 1; }

size_t stream_workspace(int d, int n_reqs, int nt) {
    const size_t rows = size_t(kMaxStreamCtas) * 2 * 8 * nt;
    return ((size_t(n_reqs) + 1) * 8 + 15) / 16 * 16 + rows * (d + 2) * sizeof(float);
}

int check_attn(const ttkv_q4_cache_t* cache, const ttkv_q4_batch_t* batch, const void* q, int32_t q_dtype,
               int64_t q_stride, int32_t HQ, const void* out, int64_t out_stride) {
    if (int e = check_cache(cache)) return e;
    if (!batch || batch->n_reqs < 0 || batch->bt_cols < 0) return fail(TTKV_ERR_ARG, "4-bit read: batch");
    if (batch->n_reqs > 65535) return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: %d requests in one call", batch->n_reqs);
    if (batch->n_reqs > 0 && (!batch->seq_lens || !q || !out || (batch->bt_cols > 0 && !batch->block_table)))
        return fail(TTKV_ERR_ARG, "4-bit read: null pointer");
    if (HQ < cache->H || HQ % cache->H) return fail(TTKV_ERR_ARG, "HQ=%d is not a multiple of H=%d", HQ, cache->H);
    if (q_dtype != TTKV_F16 && q_dtype != TTKV_BF16)
        return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: queries and outputs are fp16 or bf16");
    if (q_stride < 0 || out_stride < 0) return fail(TTKV_ERR_ARG, "4-bit read: a negative stride");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 1)
        return fail(TTKV_ERR_ALIGN, "4-bit read: q or out at an odd address");
    return TTKV_OK;
}

template <int D, int GRP, int NT>
int launch_stream(AttnParams P, cudaStream_t st) {
    auto k = q4_stream_kernel<D, GRP, NT>;
    if (int e = raise_smem_limit(reinterpret_cast<const void*>(k), "q4_stream_kernel")) return e;
    const size_t smem = size_t(2 * kWarps) * 8 * NT * (D + 2) * sizeof(float) + panel_bytes(D, GRP);
    k<<<P.n_ctas, 32 * kWarps, smem, st>>>(P);
    if (int e = check_launch("q4_stream_kernel")) return e;
    q4_merge_kernel<<<dim3(unsigned(P.H * P.max_q * P.G), unsigned(P.n_reqs)), kMergeThreads, 0, st>>>(P, D, 8 * NT);
    return check_launch("q4_merge_kernel");
}

int run_stream(const ttkv_q4_cache_t* c, AttnParams P, void* ws, size_t ws_bytes, cudaStream_t st) {
    const int nt = stream_nt(int64_t(P.max_q) * P.G);
    if (!ws || ws_bytes < stream_workspace(c->d, P.n_reqs, nt))
        return fail(TTKV_ERR_WORKSPACE, "4-bit read: workspace of %zu bytes, %zu needed", ws_bytes,
                    stream_workspace(c->d, P.n_reqs, nt));
    if (reinterpret_cast<uintptr_t>(ws) & 15) return fail(TTKV_ERR_ALIGN, "4-bit read: workspace not 16-byte aligned");
    int sms = 0;
    if (int e = sm_count(&sms)) return e;
    P.n_ctas = std::min(sms, kMaxStreamCtas);
    const size_t rows = size_t(P.n_ctas) * 2 * 8 * nt;
    P.prefix = static_cast<int64_t*>(ws);
    P.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + ((size_t(P.n_reqs) + 1) * 8 + 15) / 16 * 16);
    P.part_ml = P.part_o + rows * c->d;
#define TTKV_Q4_STREAM(D, GRP)                                                                         if (c->d == D && c->group == GRP) return nt == 2 ? launch_stream<D, GRP, 2>(P, st) : launch_stream<D, GRP, 1>(P, st);
    TTKV_Q4_STREAM(64, 32) TTKV_Q4_STREAM(64, 64) TTKV_Q4_STREAM(128, 32) TTKV_Q4_STREAM(128, 64) TTKV_Q4_STREAM(128, 128)
#undef TTKV_Q4_STREAM
    return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: geometry");
}

AttnParams attn_params(const ttkv_q4_cache_t* c, const ttkv_q4_batch_t* b, const void* q, int32_t dtype,
                       int64_t q_stride, int32_t HQ, float scale, void* out, int64_t out_stride, int32_t* status) {
    AttnParams P{};
    P.cache = c->base; P.n_blocks = c->n_blocks; P.H = c->H; P.G = HQ / c->H; P.block_size = c->block_size;
    P.block_table = b->block_table; P.bt_stride = b->bt_stride; P.bt_cols = b->bt_cols; P.seq_lens = b->seq_lens;
    P.n_reqs = b->n_reqs; P.q = q; P.dtype = dtype; P.q_stride = q_stride; P.scale = scale;
    P.out = out; P.out_stride = out_stride; P.status = status;
    P.q_vec = rows_aligned(q, dtype, q_stride);
    P.out_vec = (reinterpret_cast<uintptr_t>(out) & 7) == 0 && (out_stride & 3) == 0;
    return P;
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" size_t ttkv_q4_decode_workspace_bytes(const ttkv_q4_cache_t* cache, int32_t n_reqs, int32_t HQ) {
    if (!cache || cache->H < 1 || HQ < cache->H || n_reqs < 0) return 0;
    return stream_workspace(cache->d, n_reqs, stream_nt(HQ / cache->H));
}

extern "C" int ttkv_q4_decode(const ttkv_q4_cache_t* cache, const ttkv_q4_batch_t* batch, const void* q,
                              int32_t q_dtype, int64_t q_stride, int32_t HQ, float scale, void* out,
                              int64_t out_stride, void* workspace, size_t workspace_bytes, int32_t* status,
                              void* stream) {
    if (int e = check_attn(cache, batch, q, q_dtype, q_stride, HQ, out, out_stride)) return e;
    if (batch->n_reqs == 0) return TTKV_OK;
    AttnParams P = attn_params(cache, batch, q, q_dtype, q_stride, HQ, scale, out, out_stride, status);
    P.n_rows = batch->n_reqs;
    P.max_q = 1;
    return run_stream(cache, P, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" size_t ttkv_q4_prefill_workspace_bytes(const ttkv_q4_cache_t* cache, int32_t n_reqs, int32_t HQ,
                                                  int32_t max_q_len, int32_t max_seq_len) {
    if (!cache || cache->H < 1 || HQ < cache->H || n_reqs < 0 || max_q_len < 0) return 0;
    return stream_workspace(cache->d, n_reqs, stream_nt(int64_t(max_q_len) * (HQ / cache->H)));
}

extern "C" int ttkv_q4_prefill(const ttkv_q4_cache_t* cache, const ttkv_q4_batch_t* batch, const int32_t* q_start,
                               const int32_t* q_len, const void* q, int32_t q_dtype, int64_t q_stride, int32_t n_rows,
                               int32_t HQ, float scale, void* out, int64_t out_stride, int32_t max_q_len,
                               int32_t max_seq_len, void* workspace, size_t workspace_bytes, int32_t* status,
                               void* stream) {
    if (int e = check_attn(cache, batch, q, q_dtype, q_stride, HQ, out, out_stride)) return e;
    if (max_q_len < 0 || max_seq_len < 0 || n_rows < 0) return fail(TTKV_ERR_ARG, "4-bit prefill: a negative size");
    if (batch->n_reqs > 0 && (!q_start || !q_len)) return fail(TTKV_ERR_ARG, "4-bit prefill: q_start or q_len missing");
    if (batch->n_reqs == 0 || n_rows == 0 || max_q_len == 0) return TTKV_OK;
    if (int64_t(max_q_len) * HQ > 0x7fffffff) return fail(TTKV_ERR_UNSUPPORTED, "4-bit prefill: %d queries of %d heads", max_q_len, HQ);
    AttnParams P = attn_params(cache, batch, q, q_dtype, q_stride, HQ, scale, out, out_stride, status);
    P.q_start = q_start; P.q_len = q_len; P.n_rows = n_rows; P.max_q = max_q_len; P.max_seq = std::max(max_seq_len, 1);
    return run_stream(cache, P, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
