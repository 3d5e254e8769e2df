// Chunks of queries over the 4-bit paged cache on the 5th-generation tensor cores.
//
//   S = Q K^T,  P = exp(scale S - m) masked,  O += P V,  out = O / sum P
//
// A chunk has many (query, head) rows per stored token, so products bound it, not memory: a CTA takes
// 256 rows of one KV head (two tiles of 128, the M of an MMA, whose products and softmaxes run in
// turn) over stored tiles of 128 tokens. Each stored tile is turned into fp16 operands once for both:
// K^ = m + s c and V^, rounded once to fp16 (the codes as exact operands with their scales applied to S
// and P would cost the softmax twice its instructions, and with groups below d a product each). V^ is off
// by 2^-11 of an element at most, as is each weight, which is what fp16 outputs are off by themselves.
// Rounded keys put 2^-11 of sum |q_i K_i| on a score at most, which grows with the keys and not with their
// spread: 5e-4 to 1e-3 of the output with a few large channels, up to 1.8e-3 where channels have offsets of
// three times their spread, against the 1.7e-3 that bf16 outputs are off by themselves and the 2.1e-4 of
// fp16. So for fp16 queries (FINE) a key is the sum of two fp16, its rounding and what that leaves, with a
// product each: 3.3e-4 in all, and 282 and 854 us for the 251 and 734 of the chunks below. (V as a sum of two
// as well gives 2.7e-4 and takes 20 to 25 percent more.) Scores, sums and O are fp32. P is fp16, of which the weights are
// held in the upper part: the largest of a segment's first half is 2^8 and none passes 2^15, so they keep
// 11 bits down to 2^-22 of it and vanish only below 2^-33 (2^-25 with a largest of 1, which lost half of what
// 16383 tokens weigh together, each 18 nats below the first).
// The running maximum moves only when a half's weights outgrow that (then O in tensor memory is rescaled).
//
// Roles: two softmax warpgroups (a thread owns a row, i.e. a lane of tensor memory), a warpgroup that
// dequantises K and one for V, two warps that issue the products, one per row tile, and a warp that
// fetches the stored panels, by bulk copies into a ring a tile and a half deep. Operands are
// double-buffered in shared memory in the 128-byte-swizzled K-major layout of the MMA. Scores are made
// 64 tokens at a time into two buffers in turn, so the next half's product runs under this half's
// softmax, whose P replaces the scores in place. The stored order of the codes needs no transposition:
// a K word is a 16-byte chunk of its token's row (the dims of a chunk in the order 0 4 1 5 2 6 3 7,
// which Q repeats), and four V words are chunks of eight tokens of four lanes. The roles' loops are
// kept short (rolled where the data lies in shared memory): together they have to stay in the SM's
// instruction cache, and unrolled they streamed 19 KB of code per tile through it.
//
// 256 queries of 24 heads over 7379 tokens of each of 8 requests take 251 us without the merge, 727
// TFLOP/s; 1024 to 2048 queries of 32 heads over 8192 to 16384 tokens of two requests 734, 827 TFLOP/s,
// half of a library matrix product's rate (bf16, under the profiler; 230 and 680 in a program). A stored tile takes about 4500 cycles, in 2050 of which the
// tensor cores compute; the exponentials take 2050 of their pipe, the operands 2700 of shared memory's
// (A of the scores is read again with each 64 tokens), and each role is busy for 3500 to 4000, slowed by
// the others' instructions. Without any one role's arithmetic it is 4 to 6 percent faster, without all 10.
// Scores a half ahead in a buffer of their own, with the maximum sought in every half, took 3 percent more
// time; rings of their own for K and V changed nothing; product warps of one running lane took 5 percent
// more, as what their instructions need was then moved lane by lane.
//
// The work list is (request, KV head, row block, stored tile up to the block's causal limit), shared
// out evenly to one CTA per SM as in the streaming kernel; the parts that a share's borders cut go
// through the workspace to q4_chunk_merge_kernel.
#include "ttkv_q4_attn.cuh"
#include "ttkv_umma.cuh"

namespace ttkv {
namespace {

using namespace q4;
using namespace umma;

constexpr int TN = 128;                      // stored tokens of a tile
constexpr int TM = 128;                      // rows of a tile
constexpr int CROWS = 2 * TM;                // rows of a block
constexpr int TH = TN / 2;                   // tokens of a half, the step of the softmax
constexpr int kChunkThreads = 20 * 32;       // softmax 8 warps, K 4, V 4, products 2, fetching 1 (and 1 idle)
// Registers a thread: at launch, and of each role after its own setting. A warpgroup waits in its
// setting until the others have given theirs up, so the shares must not exceed the launch's total.
constexpr int kRegsLaunch = 96, kRegsSoftmax = 128, kRegsOperands = 80, kRegsProducts = 64;
static_assert(2 * kRegsSoftmax + 2 * kRegsOperands + kRegsProducts <= 5 * kRegsLaunch, "register shares");
constexpr uint32_t kTmemCols = 512;          // S of row tile 0 and 1, O of each, at 128 columns
constexpr float kWeightMost = 32768.f;       // of a half's weights in all: each is a finite fp16
constexpr float kWeightBits = 8.f;           // the largest weight when the maximum has been looked for, as a power of two:
                                             // 64 such weights stay below that, so a flat row does not look again
static_assert(TH * 256 <= 32768, "a half of the largest weights");
constexpr int kFlags = 8;                    // tiles whose NaN values are remembered

// Row tiles' tensor memory: S of a half in buffer y (then P in its first 32 columns) and O.
__device__ __forceinline__ uint32_t s_col(int x, uint32_t y) { return 128u * x + 64u * y; }
__device__ __forceinline__ uint32_t o_col(int x) { return 256u + 128u * x; }

template <int D, int GRP, bool FINE>
struct ChunkSmem {
    // A stage of K: a tile, or a half of one with what its rounding left behind it
    static constexpr int Q = TM * D * 2, K = TN * D * 2, V = D * TN * 2;
    // Panels of the ring: a multiple of four, so that a place always holds panels of the same warps of K and V.
    // Each warp then sees every phase of its places; one that skipped some could take the phase before the
    // last for the one that it waits for, and read a place that is still being filled
    static constexpr int PANEL = panel_bytes(D, GRP), RING = std::min(16, 30 * 1024 / PANEL) / 4 * 4;
    static_assert(RING >= 8 && RING % 4 == 0, "places of the ring");
    static constexpr int off_q = 0, off_k = 2 * Q, off_v = off_k + 2 * K, off_ring = off_v + 2 * V;
    static constexpr int BYTES = off_ring + RING * PANEL + 1024;
    // 64 dims of 128 rows; of a stage's tokens; 64 tokens of D lanes
    static constexpr int QATOM = TM * 128, KATOM = (FINE ? TH : TN) * 128, VATOM = D * 128;
};

struct ChunkBars {
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2];        // operand stages
    uint64_t rfull[16], rempty[16];                           // panels of the ring
    // row tiles; of halves one for each buffer: a half is waited for before the one after the next is made,
    // so no phase is missed
    uint64_t qfull[2], sfull[2][2], pfull[2][2], pvdone[2][2];
    uint64_t noted[2];                                        // a segment's flags of NaN have all been read
};

// A CTA's (or a role's) place in the work list.
struct Segments {
    int u, ue;                               // the next unit and the end of the share
    int r, h, rb, ui, U, nrb;                // request, KV head, row block, tile of U
    Req rq;

    // Tiles that row block b reads: up to the limit of its last query.
    __device__ __forceinline__ static int tiles(const Req& a, int G, int b) {
        const int last = min((b * CROWS + CROWS - 1) / G, a.ql - 1);
        return (a.seq - a.ql + last + 1 + TN - 1) / TN;
    }
    __device__ __forceinline__ static int per_head(const Req& a, int G) {
        const int n = row_blocks(a, G, CROWS);
        int sum = 0;
        for (int b = 0; b < n; ++b) sum += tiles(a, G, b);
        return sum;
    }
    __device__ __forceinline__ void load(const AttnParams& P) {
        rq = request(P, r, false);
        nrb = row_blocks(rq, P.G, CROWS);
    }
    // To unit u, `off` units behind the first of request r (or of a later one).
    __device__ __forceinline__ void seek(const AttnParams& P, int off) {
        int ph;
        for (;; ++r) {
            load(P);
            ph = per_head(rq, P.G);
            if (off < ph * P.H) break;
            off -= ph * P.H;
        }
        h = off / ph;
        off -= h * ph;
        for (rb = 0;; ++rb) {
            U = tiles(rq, P.G, rb);
            if (off < U) break;
            off -= U;
        }
        ui = off;
    }
    __device__ __forceinline__ int here() const { return min(U - ui, ue - u); }   // tiles of this segment
    __device__ __forceinline__ void skip(const AttnParams& P, int n) {           // past n tiles of it
        u += n;
        ui += n;
        if (u >= ue || ui < U) return;
        ui = 0;
        if (++rb == nrb) {
            rb = 0;
            if (++h == P.H) {
                h = 0;
                do { ++r; load(P); } while (nrb == 0);
            }
        }
        U = tiles(rq, P.G, rb);
    }
};

__device__ __forceinline__ uint32_t h2u(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 u2h(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }

// Two codes of a word as exact fp16 integers: an fp16 1024 + c, less 1024. HI: the upper nibble of a
// byte, 1024 + 16 c.
template <bool HI>
__device__ __forceinline__ __half2 codes2(uint32_t w) {
    if (HI) return __hfma2(u2h((w & 0x00f000f0u) | 0x64006400u), u2h(0x2c002c00u), u2h(0xd400d400u));   // x / 16 - 64
    return __hsub2(u2h((w & 0x000f000fu) | 0x64006400u), u2h(0x64006400u));
}

// minimum + scale * code of two codes, exact to fp32, as the sum of an fp16 and of the fp16 of what that leaves.
__device__ __forceinline__ void split2(__half2 codes, float2 sm, uint32_t& hi, uint32_t& lo) {
    const float2 c = __half22float2(codes);
    const float2 x = make_float2(fmaf(c.x, sm.x, sm.y), fmaf(c.y, sm.x, sm.y));
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 r = __half22float2(h);
    hi = h2u(h);
    lo = half2_bits(x.x - r.x, x.y - r.y);
}

__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one;
}

// The panels of a stored tile, one each in lanes 0 to 7: index in the cache, or that there is none or
// that its block id is outside the cache.
constexpr int kNoPanel = -1, kBadPanel = -2;

__device__ __forceinline__ int panels_of(const AttnParams& P, int r, int h, int tile, int seq, int lane) {
    const int t = tile * TN + 16 * lane;
    if (lane >= 8 || t >= seq) return kNoPanel;
    const int bi = t / P.block_size;
    const int blk = P.block_table[int64_t(r) * P.bt_stride + bi];
    if (blk < 0 || blk >= P.n_blocks) return kBadPanel;
    // (an index of panels: the memory of a GPU holds fewer than 2^31)
    return int((int64_t(blk) * P.H + h) * (P.block_size / kPanelTokens)) + (t - bi * P.block_size) / kPanelTokens;
}

// Bounded wait for a barrier's phase (about 2 s). The clock is read once in many tries, and a warp with
// time to spare sleeps in between: polling takes issue slots from the warps that it waits for.
template <bool IDLE>
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        #pragma unroll 1
        for (int i = 0; i < 64; ++i) {
            if (IDLE) __nanosleep(64);
            if (mbar_try(bar, parity)) return true;
        }
        if (clock64() - t0 > kWaitCycles) return false;
    }
}

// Eight 16-bit elements to memory that is not 16-byte aligned.
__device__ __forceinline__ void store_chunk_unaligned(uint16_t* p, uint4 v) {
    #pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = i < 4 ? (i < 2 ? v.x : v.y) : (i < 6 ? v.z : v.w);
        p[i] = uint16_t(u >> (16 * (i & 1)));
    }
}

template <int D, int GRP, bool FINE>
__global__ void __launch_bounds__(kChunkThreads, 1) q4_chunk_kernel(const AttnParams P) {
    using S = ChunkSmem<D, GRP, FINE>;
    constexpr int NG = D / GRP, NW = D / 32, WPG = GRP / 32, PANEL = S::PANEL, RING = S::RING;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ ChunkBars B;
    __shared__ uint32_t tmem_base;
    int* pre = reinterpret_cast<int*>(smem + S::off_ring);   // [kChunkThreads + 1], until the roles begin
    __shared__ long long wsum[kChunkThreads / 32];
    __shared__ __align__(16) uint8_t vbad[kFlags][TN];                    // groups whose V is NaN, a bit each
    __shared__ int any_bad[kFlags];

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    const bool tell = blockIdx.x == 0;
    if (w == 16) tmem_alloc(&tmem_base, kTmemCols);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.kfull[i], 128);
            mbar_init(&B.kempty[i], 2);
            mbar_init(&B.vfull[i], 128);
            mbar_init(&B.vempty[i], 2);
            mbar_init(&B.qfull[i], 128);
            mbar_init(&B.noted[i], 128);
            for (int y = 0; y < 2; ++y) {
                mbar_init(&B.sfull[i][y], 1);
                mbar_init(&B.pfull[i][y], 128);
                mbar_init(&B.pvdone[i][y], 1);
            }
        }
    }
    if (tid < RING) {
        mbar_init(&B.rfull[tid], 1);
        mbar_init(&B.rempty[tid], 2);
    }
    for (int i = tid; i < kFlags * TN; i += kChunkThreads) (&vbad[0][0])[i] = 0;
    if (tid < kFlags) any_bad[tid] = 0;
    pdl_wait();

    // ---- units of the requests before each thread's share of them
    const int per = (P.n_reqs + kChunkThreads - 1) / kChunkThreads;
    const int rlo = min(tid * per, P.n_reqs), rhi = min(rlo + per, P.n_reqs);
    long long sum = 0;
    for (int r = rlo; r < rhi; ++r) {
        const Req a = request(P, r, tell);
        sum += (long long)P.H * Segments::per_head(a, P.G);
    }
    long long inc = sum;
    #pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, k);
        if (lane >= k) inc += y;
    }
    if (lane == 31) wsum[w] = inc;
    tc_before();
    __syncthreads();
    tc_after();
    for (int i = 0; i < w; ++i) inc += wsum[i];
    pre[tid] = int(inc - sum);
    if (tid == kChunkThreads - 1) {
        const bool vast = inc > 0x7fff0000;                   // 2^31 tiles: reported, and nothing done
        pre[kChunkThreads] = vast ? 0 : int(inc);
        if (vast && tell) report(P.status, TTKV_STATUS_SEQ_BOUND);
    }
    __syncthreads();
    const int T = pre[kChunkThreads], share = share_size(T, P.n_ctas);
    const int ca = min(int(blockIdx.x) * share, T), cb = min(ca + share, T);
    pdl_trigger();
    const uint32_t tmem = tmem_base;
    bool dead = false;                                        // a bounded wait ran out: no further waits
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !wait_phase<false>(bar, parity & 1u)) {
            dead = true;
            report(P.status, TTKV_STATUS_TIMEOUT);
        }
    };
    auto wait_idle = [&](uint64_t* bar, uint32_t parity) {    // by warps that are ahead of the others
        if (!dead && !wait_phase<true>(bar, parity & 1u)) {
            dead = true;
            report(P.status, TTKV_STATUS_TIMEOUT);
        }
    };
    Segments sg;
    sg.u = ca;
    sg.ue = cb;
    if (ca < cb) {
        int lo = 0, hi = kChunkThreads - 1;                   // the last chunk of requests that begins at or before ca
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= ca) lo = mid; else hi = mid - 1;
        }
        sg.r = lo * per;
        sg.seek(P, ca - pre[lo]);
    }
    fence_async_smem();                                       // `pre` gives way to the first panels
    __syncthreads();
    if (tid == 0) {                                           // for the merge: no row block begun here and cut, so far
        P.rec[8 * blockIdx.x] = -1;
    }

    if (w < 8) {                                              // (fewer tiles than CTAs: nothing to do in any role)
        // ============================================================== softmax: row tile x, row t
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kRegsSoftmax));
        const int x = w >> 2, t = tid & 127;
        const uint32_t lane_base = tmem + (uint32_t(32 * (w & 3)) << 16);
        unsigned char* qb = smem + S::off_q + x * S::Q;
        uint32_t n_s = 0, n_tile = 0;                         // halves of this row tile; stored tiles of the CTA
        for (; sg.u < sg.ue;) {
            const Req rq = sg.rq;
            const int n = sg.here(), begin = sg.ui, U = sg.U, h = sg.h, rb = sg.rb, r = sg.r, u0 = sg.u - sg.ui;
            const int n_rows = rq.ql * P.G, row = rb * CROWS + x * TM + t;
            sg.skip(P, n);
            if (rb * CROWS + x * TM >= n_rows) { n_tile += n; continue; }       // no rows in this tile
            const bool live = row < n_rows;
            const int j = live ? row / P.G : 0, g = live ? row - j * P.G : 0;
            const int lim = live ? rq.seq - rq.ql + j + 1 : 0;                  // sees stored tokens below it
            float qf = 0.f;
            {
                // the warp's 32 rows, D / 8 lanes to a row, a chunk of eight dims each
                constexpr int LPR = D / 8, RPI = 32 / LPR;    // lanes a row, rows at once
                const int c = lane % LPR;
                const int64_t src = live ? int64_t(rq.q0 + j) * P.q_stride + int64_t(h * P.G + g) * D : -1;
                auto place = [&](int i) -> uint4* {           // the chunk of row i RPI + lane / LPR of the warp
                    return reinterpret_cast<uint4*>(qb + (c >> 3) * S::QATOM + kmajor_off(t - lane + i * RPI + lane / LPR, c & 7));
                };
                // as it is, all loads in flight at once; then each chunk in place
                if (P.q_vec) {
                    uint4 raw[LPR];
                    #pragma unroll
                    for (int i = 0; i < LPR; ++i) {
                        const int64_t from = __shfl_sync(0xffffffffu, src, i * RPI + lane / LPR);
                        raw[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.q) + max(from, int64_t(0)) + 8 * c);
                    }
                    #pragma unroll
                    for (int i = 0; i < LPR; ++i) *place(i) = raw[i];
                } else {
                    #pragma unroll 1
                    for (int i = 0; i < LPR; ++i) {
                        const int64_t from = __shfl_sync(0xffffffffu, src, i * RPI + lane / LPR);
                        const uint16_t* p = static_cast<const uint16_t*>(P.q) + max(from, int64_t(0)) + 8 * c;
                        *place(i) = make_uint4(p[0] | (uint32_t(p[1]) << 16), p[2] | (uint32_t(p[3]) << 16),
                                               p[4] | (uint32_t(p[5]) << 16), p[6] | (uint32_t(p[7]) << 16));
                    }
                }
                #pragma unroll 1
                for (int i = 0; i < LPR; ++i) {
                    const uint4 raw = *place(i);
                    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
                    const bool none = __shfl_sync(0xffffffffu, src, i * RPI + lane / LPR) < 0;
                    float v[8], big = 0.f;
                    #pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        float2 f = P.dtype == TTKV_BF16
                            ? make_float2(__uint_as_float(u[z] << 16), __uint_as_float(u[z] & 0xffff0000u)) : __half22float2(u2h(u[z]));
                        if (none) f = make_float2(0.f, 0.f);
                        v[2 * z] = f.x;
                        v[2 * z + 1] = f.y;
                        big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                    #pragma unroll
                    for (int z = 1; z < LPR; z <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, z));
                    // e brings the row's largest |q| into [1, 2); a negative scale's sign goes to q
                    const int e = big > 0.f && big < INFINITY ? 127 - int(__float_as_uint(big) >> 23) : 0;
                    const float up = copysignf(__uint_as_float(uint32_t(min(127 + e, 254)) << 23), P.scale);
                    // dims 0 4 1 5 2 6 3 7, the order of a word's codes
                    *place(i) = make_uint4(half2_bits(v[0] * up, v[4] * up), half2_bits(v[1] * up, v[5] * up),
                                           half2_bits(v[2] * up, v[6] * up), half2_bits(v[3] * up, v[7] * up));
                    const int e_row = __shfl_sync(0xffffffffu, e, (lane % RPI) * LPR);
                    if (lane / RPI == i)                      // this lane's own row
                        // (not 0, which would make NaN of a masked score of -inf)
                        qf = fmaxf(fabsf(P.scale) * kLog2e * __uint_as_float(uint32_t(max(127 - e_row, 1)) << 23), 1e-38f);
                }
            }
            fence_async_smem();
            mbar_arrive(&B.qfull[x]);

            float m = -INFINITY, l = 0.f;                     // m: what scores are taken against, 8 below a maximum
            uint32_t bad = 0;                                 // groups of V that are NaN in a token that this row sees
            auto note_bad = [&](int i, uint32_t k) {          // tile i of the segment, k-th of the CTA: V consumed
                const uint32_t f = k & (kFlags - 1);
                if (*reinterpret_cast<volatile int*>(&any_bad[f]) == 0) return;
                for (int c = 0; c < TN; ++c)
                    if ((begin + i) * TN + c < lim) bad |= *reinterpret_cast<volatile uint8_t*>(&vbad[f][c]);
            };
            for (int i = 0; i < 2 * n; ++i, ++n_s) {          // halves
                const uint32_t sc = lane_base + s_col(x, n_s & 1);
                wait(&B.sfull[x][n_s & 1], n_s >> 1);                       // (and P . V of the half before the last has ended)
                tc_after();
                if (i > 0 && (i & 1) == 0) note_bad((i >> 1) - 1, n_tile + (i >> 1) - 1);
                const int seen = lim - (begin * TN + i * TH); // tokens of the half that the row sees
                const bool full = __all_sync(0xffffffffu, seen >= TH);
                // weights against the maximum so far, which may be exceeded as long as no fp16 weight overflows:
                // the half's sum tells. The maximum is looked for in the first half and, rarely, when it does
                uint32_t p[2][16];
                float sum;
                for (bool raise = i == 0;; raise = true) {
                    float s[2][32];
                    tmem_ld32(sc, s[0]);
                    tmem_ld32(sc + 32, s[1]);
                    tmem_wait_ld();
                    if (!full) {
                        #pragma unroll
                        for (int c = 0; c < 2; ++c)
                            #pragma unroll
                            for (int k = 0; k < 32; ++k) s[c][k] = 32 * c + k < seen ? s[c][k] : -INFINITY;
                    }
                    if (raise) {
                        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        #pragma unroll
                        for (int c = 0; c < 2; ++c)
                            #pragma unroll
                            for (int k = 0; k < 32; ++k) m4[k & 3] = fmaxf(m4[k & 3], s[c][k]);
                        const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * qf - kWeightBits;
                        float corr = 1.f;
                        if (mt > m) {                         // (m is -inf at first)
                            corr = m == -INFINITY ? 0.f : ex2(m - mt);
                            m = mt;
                            l *= corr;
                        }
                        if (i > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
                            wait(&B.pvdone[x][(n_s - 1) & 1], (n_s - 1) >> 1);    // O holds every half before this one
                            tc_after();
                            #pragma unroll 1
                            for (int c = 0; c < D / 16; ++c) {
                                float o[16];
                                tmem_ld16(lane_base + o_col(x) + 16 * c, o);
                                tmem_wait_ld();
                                uint32_t v[16];
                                #pragma unroll
                                for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(o[k] * corr);
                                tmem_st16u(lane_base + o_col(x) + 16 * c, v);
                            }
                        }
                    }
                    const float mm = m == -INFINITY ? 0.f : m;    // a row that sees nothing yet has weights of 0
                    float2 ls = make_float2(0.f, 0.f);
                    #pragma unroll
                    for (int c = 0; c < 2; ++c)
                        #pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float2 a = __ffma2_rn(make_float2(s[c][2 * k], s[c][2 * k + 1]), make_float2(qf, qf), make_float2(-mm, -mm));
                            const float2 e = make_float2(ex2(a.x), ex2(a.y));
                            ls = __fadd2_rn(ls, e);
                            p[c][k] = half2_bits(e.x, e.y);
                        }
                    sum = ls.x + ls.y;
                    if (raise || !__any_sync(0xffffffffu, sum > kWeightMost)) break;
                }
                l += sum;
                tmem_st16u(sc, p[0]);
                tmem_st16u(sc + 16, p[1]);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_before();
                mbar_arrive(&B.pfull[x][n_s & 1]);
            }
            n_tile += n;
            // ---- O / l, or the parts
            wait(&B.pvdone[x][(n_s - 1) & 1], (n_s - 1) >> 1);
            tc_after();
            note_bad(n - 1, n_tile - 1);
            mbar_arrive(&B.noted[x]);
            const bool whole = begin == 0 && n == U;
            // 32 output lanes at a time, through the warp's rows of Q (read by the last product) so that
            // neighbouring lanes of the warp write neighbouring bytes
            const int64_t pr = (int64_t(blockIdx.x) * 2 + (ca >= u0 ? 0 : 1)) * CROWS + x * TM + t;
            // (a row that has queries sees a token; its weights add up to 0 only where its scores are all -inf, of a
            // query with an infinity: 0 times 1 / 0 is the NaN that it should be)
            const float inv = whole ? 1.f / l : 1.f;
            const int64_t dst = !live ? -1 : whole ? int64_t(rq.q0 + j) * P.out_stride + int64_t(h * P.G + g) * D : pr * D;
            uint4* stage = reinterpret_cast<uint4*>(qb + (w & 3) * 4096);
            #pragma unroll 1
            for (int c = 0; c < NW; ++c) {
                float o[32];
                tmem_ld32(lane_base + o_col(x) + 32u * c, o); // column 32 c + 8 i + b holds lane 32 c + 4 b + i
                tmem_wait_ld();
                const float f = (bad >> (c / WPG)) & 1u ? __int_as_float(0x7fc00000) : inv;
                #pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= f;
                __syncwarp();
                if (!whole) {                                 // 128 bytes a row: 8 lanes, 4 rows at once
                    #pragma unroll
                    for (int b = 0; b < 8; ++b)
                        stage[8 * lane + (b ^ (lane & 7))] = make_uint4(__float_as_uint(o[b]), __float_as_uint(o[8 + b]),
                                                                        __float_as_uint(o[16 + b]), __float_as_uint(o[24 + b]));
                    __syncwarp();
                    #pragma unroll 2
                    for (int k = 0; k < 8; ++k) {
                        const int rl = 4 * k + (lane >> 3), b = lane & 7;
                        const int64_t to = __shfl_sync(0xffffffffu, dst, rl);
                        if (to >= 0) *reinterpret_cast<uint4*>(P.part_o + to + 32 * c + 4 * b) = stage[8 * rl + (b ^ (rl & 7))];
                    }
                } else {                                      // 64 bytes a row: 4 lanes, 8 rows at once
                    #pragma unroll
                    for (int b = 0; b < 8; b += 2)
                        stage[4 * lane + ((b >> 1) ^ ((lane >> 1) & 3))] =
                            make_uint4(pack2(o[b], o[8 + b], P.dtype), pack2(o[16 + b], o[24 + b], P.dtype),
                                       pack2(o[b + 1], o[9 + b], P.dtype), pack2(o[17 + b], o[25 + b], P.dtype));
                    __syncwarp();
                    #pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
                        const int rl = 8 * k + (lane >> 2), b = lane & 3;
                        const int64_t to = __shfl_sync(0xffffffffu, dst, rl);
                        if (to < 0) continue;
                        uint16_t* p = static_cast<uint16_t*>(P.out) + to + 32 * c + 8 * b;
                        const uint4 v = stage[4 * rl + (b ^ ((rl >> 1) & 3))];
                        if (P.out_vec == 2) *reinterpret_cast<uint4*>(p) = v;
                        else store_chunk_unaligned(p, v);
                    }
                }
            }
            if (live && !whole) *reinterpret_cast<float2*>(P.part_ml + 2 * pr) = make_float2(m, l);
            if (x == 0 && t == 0 && begin == 0 && n < U) {    // begun here and cut: this CTA's entry of the merge
                int32_t* rec = P.rec + 8 * blockIdx.x;
                rec[0] = r;
                rec[1] = h;
                rec[2] = rb;
                rec[3] = u0;
                rec[4] = U;
                rec[5] = share;
            }
        }
    } else if (w < 12) {
        // ============================================================== K of a tile as fp16 rows
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsOperands));
        // panels wk and wk + 4, eight tokens at a time: lane (b token of them, a chunk of its row), so that
        // eight lanes read 128 bytes of codes and write eight different chunks of the swizzled rows
        const int wk = w - 8, b = (lane >> 3) ^ ((lane & 4) ? 5 : 0), a = lane & 3;
        uint32_t n_tile = 0;
        while (sg.u < sg.ue) {
            const int n = sg.here(), first = sg.ui, seq = sg.rq.seq;
            sg.skip(P, n);
            for (int it = 0; it < n; ++it, ++n_tile) {
                if (!FINE) wait_idle(&B.kempty[n_tile & 1], (n_tile >> 1) + 1);
                #pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                    const int p = wk + 4 * (i >> 1), o = 8 * (i & 1) + b, row = 16 * p + o, st = FINE ? i >> 1 : n_tile & 1;
                    const uint32_t g = 8 * n_tile + p, slot = g % RING;
                    const unsigned char* pan = smem + S::off_ring + slot * PANEL;
                    unsigned char* kb = smem + S::off_k + st * S::K;
                    if (FINE && (i & 1) == 0) wait_idle(&B.kempty[st], n_tile + 1);
                    if ((i & 1) == 0) wait(&B.rfull[slot], g / RING);
                    uint32_t kw[NW], km[NG];
                    load_words(pan + o * (D / 2) + a * (D / 8), kw);
                    load_words(pan + k_meta_offset(D) + o * NG * 4, km);
                    const bool none = (first + it) * TN + row >= seq;          // behind the last token: zeros
                    #pragma unroll
                    for (int k = 0; k < NW; ++k) {
                        const uint32_t meta = none ? 0u : km[k / WPG], v = kw[k];
                        const int c = 4 * k + a;
                        unsigned char* at = kb + (c >> 3) * S::KATOM + kmajor_off(FINE ? row & (TH - 1) : row, c & 7);
                        if (FINE) {
                            const float2 sm = __half22float2(u2h(meta));
                            uint4 hi, lo;
                            split2(codes2<false>(v), sm, hi.x, lo.x);
                            split2(codes2<true>(v), sm, hi.y, lo.y);
                            split2(codes2<false>(v >> 8), sm, hi.z, lo.z);
                            split2(codes2<true>(v >> 8), sm, hi.w, lo.w);
                            *reinterpret_cast<uint4*>(at) = hi;
                            *reinterpret_cast<uint4*>(at + S::K / 2) = lo;
                        } else {
                            const __half2 s2 = u2h(__byte_perm(meta, 0, 0x1010)), m2 = u2h(__byte_perm(meta, 0, 0x3232));
                            *reinterpret_cast<uint4*>(at) =
                                make_uint4(h2u(__hfma2(codes2<false>(v), s2, m2)), h2u(__hfma2(codes2<true>(v), s2, m2)),
                                           h2u(__hfma2(codes2<false>(v >> 8), s2, m2)), h2u(__hfma2(codes2<true>(v >> 8), s2, m2)));
                        }
                    }
                    if (i & 1) {
                        __syncwarp();
                        if (lane == 0 && !dead) mbar_arrive(&B.rempty[slot]);
                    }
                    if (i == 3 || (FINE && i == 1)) {
                        fence_async_smem();
                        mbar_arrive(&B.kfull[st]);
                    }
                }
            }
        }
    } else if (w < 16) {
        // ============================================================== V of a tile, lanes by tokens
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsOperands));
        // panels wv and wv + 4, half a panel (eight tokens, pairs 4 hh .. + 4) at a time: lane (j group of
        // lanes, b of its quads); with heads of 64 both halves at once
        constexpr int STEPS = D == 128 ? 4 : 2;
        const int wv = w - 12, b = lane & 7, j = D == 128 ? lane >> 3 : (lane >> 3) & 1;
        uint32_t n_tile = 0;
        while (sg.u < sg.ue) {
            const int n = sg.here(), first = sg.ui, seq = sg.rq.seq;
            sg.skip(P, n);
            for (int it = 0; it < n; ++it, ++n_tile) {
                const int st = n_tile & 1;
                wait_idle(&B.vempty[st], (n_tile >> 1) + 1);
                // the flags of the tile four behind have been read by every row that sees it: the products of the
                // tile two behind have ended, which its weights come before, or, where a row tile has none,
                // a wait for `noted`
                {
                    const int f = (n_tile + 4) & (kFlags - 1);
                    vbad[f][tid - 384] = 0;
                    if (tid == 384) any_bad[f] = 0;
                }
                unsigned char* vb = smem + S::off_v + st * S::V;
                const bool tail = (first + it + 1) * TN > seq;
                #pragma unroll 1
                for (int i = 0; i < STEPS; ++i) {
                    const int p = wv + 4 * (D == 128 ? i >> 1 : i), hh = D == 128 ? i & 1 : lane >> 4;
                    const uint32_t g = 8 * n_tile + p, slot = g % RING;
                    const unsigned char* pan = smem + S::off_ring + slot * PANEL;
                    if (D == 64 || (i & 1) == 0) wait(&B.rfull[slot], g / RING);
                    uint32_t vw[4], vm[8];
                    #pragma unroll
                    for (int k = 0; k < 4; ++k)
                        vw[k] = *reinterpret_cast<const uint32_t*>(pan + 8 * D + (4 * hh + k) * D + b * (D / 8) + 4 * j);
                    if constexpr (NG == 1) {
                        uint32_t (&lo)[4] = *reinterpret_cast<uint32_t (*)[4]>(vm), (&hi)[4] = *reinterpret_cast<uint32_t (*)[4]>(vm + 4);
                        load_words(pan + v_meta_offset(D, GRP) + 32 * hh, lo);
                        load_words(pan + v_meta_offset(D, GRP) + 32 * hh + 16, hi);
                    } else {
                        #pragma unroll
                        for (int k = 0; k < 8; ++k)
                            vm[k] = *reinterpret_cast<const uint32_t*>(pan + v_meta_offset(D, GRP) + ((8 * hh + k) * NG + j / WPG) * 4);
                    }
                    const int hp = 2 * p + hh;                // chunk of eight tokens of the tile
                    if (tail) {                               // behind the last token: zeros
                        #pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if ((first + it) * TN + 8 * hp + k >= seq) vm[k] = 0u;
                    }
                    // a NaN scale counts as nothing here: a weight of 0 must not spread it. The rows that see
                    // its token are told by flags
                    uint32_t s2[4], m2[4];                    // of the pairs of tokens
                    auto pair_up = [&]() {
                        #pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            s2[k] = __byte_perm(vm[2 * k], vm[2 * k + 1], 0x5410);
                            m2[k] = __byte_perm(vm[2 * k], vm[2 * k + 1], 0x7632);
                        }
                    };
                    pair_up();
                    __half2 nan = u2h(0u);                    // 0, or NaN (scales are finite otherwise)
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) nan = __hfma2(u2h(s2[k]), u2h(0u), nan);
                    if (__any_sync(0xffffffffu, (h2u(nan) & 0x7fff7fffu) != 0u)) {
                        const int f = n_tile & (kFlags - 1);
                        #pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            if ((vm[k] & 0x7fffu) < 0x7c00u) continue;
                            const int tok = 8 * hp + k;
                            vm[k] = 0u;
                            atomicOr(reinterpret_cast<unsigned*>(&vbad[f][tok & ~3]), (1u << (j / WPG)) << (8 * (tok & 3)));
                            any_bad[f] = 1;
                        }
                        pair_up();
                    }
                    uint32_t out[4][4];                       // [lane of the quad][pair of tokens]
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t v = vw[k];
                        const __half2 sk = u2h(s2[k]), mk = u2h(m2[k]);
                        out[0][k] = h2u(__hfma2(codes2<false>(v), sk, mk));
                        out[1][k] = h2u(__hfma2(codes2<true>(v), sk, mk));
                        out[2][k] = h2u(__hfma2(codes2<false>(v >> 8), sk, mk));
                        out[3][k] = h2u(__hfma2(codes2<true>(v >> 8), sk, mk));
                    }
                    #pragma unroll
                    for (int q = 0; q < 4; ++q)               // lane 32 j + 4 b + q is row 32 j + 8 q + b, chunk hp
                        *reinterpret_cast<uint4*>(vb + (hp >> 3) * S::VATOM + kmajor_off(32 * j + 8 * q + b, hp & 7)) =
                            make_uint4(out[q][0], out[q][1], out[q][2], out[q][3]);
                    if (D == 64 || (i & 1)) {
                        __syncwarp();
                        if (lane == 0 && !dead) mbar_arrive(&B.rempty[slot]);
                    }
                }
                fence_async_smem();
                mbar_arrive(&B.vfull[st]);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsProducts));
        if (__shfl_sync(0xffffffffu, w, 0) < 18) {
        // ============================================================== the products of row tile x
        // the whole warp keeps step, one lane issues: what the instructions need is then uniform
        const int x = __shfl_sync(0xffffffffu, w, 0) - 16;
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const bool one = elect_one();
        constexpr uint32_t ID_S = idesc_f16(TM, TH, false, false), ID_PV = idesc_f16(TM, D, false, false);
        const uint64_t DESC = sw128_desc(0, 16, 1024);
        const uint32_t aq = smem_u32(smem + S::off_q + x * S::Q) >> 4, ak = smem_u32(smem + S::off_k) >> 4, av = smem_u32(smem + S::off_v) >> 4;
        uint32_t n_tile = 0, n_s = 0, n_pv = 0, n_q = 0;      // stored tiles; halves scored; halves summed
        uint32_t s_end = 0, pv_end = 0;                       // one behind the last that was issued
        // S of half `half` of the k-th tile of the CTA, into the buffer of its turn
        auto score = [&](uint32_t k, int half) {
            const int st = FINE ? half : k & 1;
            if (FINE || half == 0) wait(&B.kfull[st], FINE ? k : k >> 1);
            tc_after();
            const uint32_t ah = ak + ((st * S::K + (FINE ? 0 : half * TH * 128)) >> 4);
            if (one && !dead) {
                #pragma unroll
                for (int e = 0; e < (FINE ? 2 : 1) * (D / 16); ++e) {
                    const int f = e % (D / 16);               // (then what K's rounding left, FINE)
                    const uint32_t sq = ((f >> 2) * S::QATOM + (f & 3) * 32) >> 4;
                    const uint32_t sk = ((f >> 2) * S::KATOM + (f & 3) * 32 + (e / (D / 16)) * (S::K / 2)) >> 4;
                    mma_f16(tm + s_col(x, n_s & 1), DESC + (aq + sq), DESC + (ah + sk), ID_S, e > 0 ? 1u : 0u);
                }
                mma_commit(&B.sfull[x][n_s & 1]);
                if (FINE || half) mma_commit(&B.kempty[st]);
                s_end = n_s + 1;
            }
            __syncwarp();
            ++n_s;
        };
        while (sg.u < sg.ue) {
            const int n = sg.here();
            if (sg.rb * CROWS + x * TM >= sg.rq.ql * P.G) {   // no rows: the operands are passed on
                if (n_q) wait(&B.noted[x], n_q - 1);          // V may write over the flags of this row tile's last
                for (int i = 0; i < n; ++i, ++n_tile) {
                    const int st = n_tile & 1;
                    for (int half = 0; half < (FINE ? 2 : 1); ++half) {
                        const int ks = FINE ? half : st;
                        wait(&B.kfull[ks], FINE ? n_tile : n_tile >> 1);
                        if (one) mbar_arrive(&B.kempty[ks]);
                    }
                    wait(&B.vfull[st], n_tile >> 1);
                    if (one) mbar_arrive(&B.vempty[st]);
                }
                sg.skip(P, n);
                continue;
            }
            wait(&B.qfull[x], n_q);                           // (O of the segment before is read, P consumed)
            ++n_q;
            for (int i = -1; i < 2 * n; ++i) {
                if (i + 1 < 2 * n) {                          // the next half's scores, once P of the half before this
                    if (i > 0) wait(&B.pvdone[x][(n_pv - 1) & 1], (n_pv - 1) >> 1);   // one has been read from their buffer
                    score(n_tile + ((i + 1) >> 1), (i + 1) & 1);
                }
                if (i < 0) continue;
                const uint32_t k = n_tile + (i >> 1);
                const int st = k & 1, half = i & 1;
                if (half == 0) wait(&B.vfull[st], k >> 1);
                wait(&B.pfull[x][n_pv & 1], n_pv >> 1);
                tc_after();
                const uint32_t ah = av + ((st * S::V + half * S::VATOM) >> 4);
                if (one && !dead) {
                    #pragma unroll
                    for (int e = 0; e < TH / 16; ++e)
                        mma_f16_ts(tm + o_col(x), tm + s_col(x, n_pv & 1) + 8 * e, DESC + (ah + 2 * e), ID_PV,
                                   (i > 0 || e > 0) ? 1u : 0u);
                    mma_commit(&B.pvdone[x][n_pv & 1]);
                    if (half) mma_commit(&B.vempty[st]);
                    pv_end = n_pv + 1;
                }
                __syncwarp();
                ++n_pv;
            }
            n_tile += n;
            sg.skip(P, n);
        }
        // every product has ended before the tensor memory is freed (their operands are read, too)
        if (s_end) mbar_wait(&B.sfull[x][(s_end - 1) & 1], ((s_end - 1) >> 1) & 1u);
        if (pv_end) mbar_wait(&B.pvdone[x][(pv_end - 1) & 1], ((pv_end - 1) >> 1) & 1u);
        } else if (w == 18) {
            // ========================================================== the stored panels, one each of lanes 0 to 7
            uint32_t g = lane, fills = 0;                     // panels of the CTA; how often place `lane` has been filled
            while (sg.u < sg.ue) {
                const int n = sg.here(), first = sg.ui, seq = sg.rq.seq, h = sg.h, r = sg.r;
                sg.skip(P, n);
                int id = panels_of(P, r, h, first, seq, lane);
                for (int it = 0; it < n; ++it, g += 8) {
                    bool filled = false;
                    const int next = it + 1 < n ? panels_of(P, r, h, first + it + 1, seq, lane) : kNoPanel;
                    if (lane < 8) {
                        const uint32_t slot = g % RING;
                        wait_idle(&B.rempty[slot], g / RING + 1);
                        unsigned char* pan = smem + S::off_ring + slot * PANEL;
                        if (!dead) {                          // (a place that never came free is left as it is)
                            filled = true;
                            if (id >= 0) {
                                mbar_expect_tx(&B.rfull[slot], PANEL);
                                bulk_g2s(pan, P.cache + int64_t(id) * PANEL, PANEL, &B.rfull[slot]);
                            } else {
                                if (id == kBadPanel) {        // NaN keys: so are the rows that see them
                                    report(P.status, TTKV_STATUS_BLOCK_RANGE);
                                    for (int k = 0; k < 2 * 16 * NG; ++k)
                                        reinterpret_cast<uint32_t*>(pan + k_meta_offset(D))[k] = k < 16 * NG ? 0x7e00u : 0u;
                                    fence_async_smem();
                                }
                                mbar_arrive(&B.rfull[slot]);  // (behind the last token nothing is read but codes)
                            }
                        }
                    }
                    id = next;
                    // (in step: no lane a tile ahead of another's place) place `lane` is the k-th of these eight
                    const uint32_t k = (lane + RING - (g - lane) % RING) % RING, all = __ballot_sync(0xffffffffu, filled);
                    fills += lane < RING && k < 8 && (all >> k & 1u);
                }
            }
            // every copy has landed: the operands' warps have waited for it, or where a wait ran out that is
            // made up for. (One whose wait ran out gives no place back, so only a place's last copy can be out)
            if (fills) mbar_wait(&B.rfull[lane], (fills - 1) & 1u);
        }
    }
    __syncwarp();
    tc_before();
    __syncthreads();
    tc_after();
    if (w == 16) tmem_dealloc(tmem_base, kTmemCols);
}

// ------------------------------------------------------------------ the merge
// Row block begun in CTA c and cut: its parts in c and in the CTAs behind it (one or two as a rule). A
// CTA of the merge takes 32 rows of it, a thread four lanes of four rows, whose loads are in flight
// together.
constexpr int kMergeRows = 32, kMergeEach = 4;

template <int D>
__global__ void __launch_bounds__(kMergeRows / kMergeEach * (D / 4)) q4_chunk_merge_kernel(const AttnParams P) {
    constexpr int STEP = kMergeRows / kMergeEach;
    pdl_wait();
    const int c0 = blockIdx.x;
    const int4 a = *reinterpret_cast<const int4*>(P.rec + 8 * c0), b = *reinterpret_cast<const int4*>(P.rec + 8 * c0 + 4);
    if (a.x < 0) return;
    const int r = a.x, h = a.y, rb = a.z, u0 = a.w, U = b.x, share = b.y;
    const int i0 = blockIdx.y * kMergeRows + threadIdx.x / (D / 4), ln = 4 * (threadIdx.x % (D / 4));
    const int c1 = (u0 + U - 1) / share;
    auto place = [&](int c) { return (int64_t(c) * 2 + (c * share >= u0 ? 0 : 1)) * CROWS + i0; };
    float m[kMergeEach], l[kMergeEach];
    float4 o[kMergeEach];
    #pragma unroll
    for (int k = 0; k < kMergeEach; ++k) {
        m[k] = -INFINITY;
        l[k] = 0.f;
        o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const Req rq = request(P, r, false);
    const int n_rows = rq.ql * P.G - rb * CROWS;              // rows of the block (the parts of others are not written)
    for (int c = c0; c <= c1; ++c) {
        const int64_t s = place(c);
        float2 ml[kMergeEach];
        float4 v[kMergeEach];
        #pragma unroll
        for (int k = 0; k < kMergeEach; ++k) {
            const bool in = i0 + k * STEP < n_rows;
            ml[k] = in ? *reinterpret_cast<const float2*>(P.part_ml + 2 * (s + k * STEP)) : make_float2(-INFINITY, 0.f);
            v[k] = in ? *reinterpret_cast<const float4*>(P.part_o + (s + k * STEP) * D + ln) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        #pragma unroll
        for (int k = 0; k < kMergeEach; ++k) {
            const float M = fmaxf(m[k], ml[k].x), wo = part_weight(m[k], M), wn = part_weight(ml[k].x, M);
            m[k] = M;
            l[k] = l[k] * wo + ml[k].y * wn;
            o[k].x = o[k].x * wo + v[k].x * wn;
            o[k].y = o[k].y * wo + v[k].y * wn;
            o[k].z = o[k].z * wo + v[k].z * wn;
            o[k].w = o[k].w * wo + v[k].w * wn;
        }
    }
    #pragma unroll
    for (int k = 0; k < kMergeEach; ++k)
        if (i0 + k * STEP < n_rows)                           // (sums of 0 are NaN, as above)
            store_out(P, rq, h, rb * CROWS + i0 + k * STEP, D, ln, o[k], l[k] == 0.f ? __int_as_float(0x7fc00000) : l[k]);
}

template <int D, int GRP, bool FINE>
int launch_chunk(const AttnParams& P, cudaStream_t st) {
    auto k = q4_chunk_kernel<D, GRP, FINE>;
    if (int e = raise_smem_limit(reinterpret_cast<const void*>(k), "q4_chunk_kernel")) return e;
    cudaFuncAttributes fa{};
    if (cudaFuncGetAttributes(&fa, k) != cudaSuccess || fa.numRegs != kRegsLaunch) {
        cudaGetLastError();
        return fail(TTKV_ERR_CUDA, "q4_chunk_kernel: built with %d registers a thread, its roles share %d", fa.numRegs, kRegsLaunch);
    }
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(P.n_ctas));
    cfg.blockDim = dim3(kChunkThreads);
    cfg.dynamicSmemBytes = ChunkSmem<D, GRP, FINE>::BYTES;
    cfg.stream = st;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, k, P);
    if (e != cudaSuccess) { cudaGetLastError(); return fail(TTKV_ERR_CUDA, "q4_chunk_kernel: %s", cudaGetErrorString(e)); }
    cfg.gridDim = dim3(unsigned(P.n_ctas), CROWS / kMergeRows);
    cfg.blockDim = dim3(kMergeRows / kMergeEach * (D / 4));
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, q4_chunk_merge_kernel<D>, P);
    if (e != cudaSuccess) { cudaGetLastError(); return fail(TTKV_ERR_CUDA, "q4_chunk_merge_kernel: %s", cudaGetErrorString(e)); }
    return TTKV_OK;
}

}  // namespace

namespace q4 {

size_t chunk_workspace_bytes(int d) {
    return size_t(kMaxCtas) * (8 * sizeof(int32_t) + 2 * CROWS * size_t(d + 2) * sizeof(float));
}

int run_chunk(const ttkv_q4_cache_t* c, AttnParams P, void* ws, size_t ws_bytes, cudaStream_t st) {
    if (!ws || ws_bytes < chunk_workspace_bytes(c->d))
        return fail(TTKV_ERR_WORKSPACE, "4-bit prefill: workspace of %zu bytes, %zu needed", ws ? ws_bytes : 0,
                    chunk_workspace_bytes(c->d));
    if (reinterpret_cast<uintptr_t>(ws) & 15) return fail(TTKV_ERR_ALIGN, "4-bit read: workspace not 16-byte aligned");
    int sms = 0;
    if (int e = sm_count(&sms)) return e;
    P.n_ctas = std::min(sms, kMaxCtas);
    P.rec = static_cast<int32_t*>(ws);
    P.part_ml = reinterpret_cast<float*>(P.rec + 8 * kMaxCtas);
    P.part_o = P.part_ml + size_t(kMaxCtas) * 2 * CROWS * 2;
#define TTKV_Q4_CHUNK(D, GRP)                                                                      \
    if (c->d == D && c->group == GRP)                                                              \
        return P.dtype == TTKV_F16 ? launch_chunk<D, GRP, true>(P, st) : launch_chunk<D, GRP, false>(P, st);
    TTKV_Q4_CHUNK(64, 32) TTKV_Q4_CHUNK(64, 64) TTKV_Q4_CHUNK(128, 32) TTKV_Q4_CHUNK(128, 64) TTKV_Q4_CHUNK(128, 128)
#undef TTKV_Q4_CHUNK
    return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: geometry");
}

}  // namespace q4
}  // namespace ttkv
