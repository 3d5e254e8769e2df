// Attention over the 4-bit paged cache: one query token per request (ttkv_q4_decode) or a chunk of
// them (ttkv_q4_prefill).
//
//   o = sum_t p_t V_t / sum_t p_t,   p_t = exp(scale q . K_t),   K_t = m_t + s_t c_t (V alike)
//
// q4_stream_kernel reads every stored byte once per block of 8 NT (query, head) rows. 64 requests of up to
// 14402 tokens (8 KV heads of 128 lanes, 3 query heads each, groups of 128; 477 MB) take 110 us, 4.3 TB/s
// or 66 percent of a measured copy, and 1110 instructions a unit of 64 tokens: three warps a scheduler
// (their registers allow no more) issue in 57 percent of the cycles, half of them on the half-rate pipe
// of the masks. 131071 tokens of 2 KV heads take 26 us, 8 requests of 4322 tokens 21, one of 257 9: there
// launch, schedule and the first copies' latency come before the bytes. The codes c are never turned into values: they are exact operands of the tensor cores,
// and scales and minima act on the products,
//
//   q . K_t = s_t (q . c_t) + m_t sum(q)
//   o       = sum_t (p_t s_t) (c_t - 7.5) + sum_t p_t (m_t + 7.5 s_t).
//
// A code in the low bits of an fp16 is the subnormal c 2^-24, so one mask makes two operands of a
// word (the next nibble's come out as c 2^-20: q is stored with the factor, o divided by it); eight
// values cost five instructions. p_t s_t is rounded to fp16, an operand of the matrix product, after
// scaling by a power of two that keeps the largest near 2^14. It multiplies c - 7.5 (the second sum
// takes the rounded weight's share of 7.5: sum p' of a unit comes from one more product, with 15s), so
// the rounding error is that of weights on centred values: 2^-11 of each term at most.
#include <algorithm>
#include <cmath>

#include "ttkv_q4_attn.cuh"

namespace ttkv {
namespace {

using namespace q4;

constexpr int kUnit = 64;                   // tokens of a unit of work: one softmax step of a warp

__device__ __forceinline__ int units_of(const Req& a) { return a.ql > 0 ? (a.seq + kUnit - 1) / kUnit : 0; }

// ------------------------------------------------------------------ warp-level products
// D += A (16 x 16, row) . B (16 x 8, column), fp16 operands and fp32 sums. (Not volatile, nor is the
// transposition: in their written order they take 20 registers more.)
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// ------------------------------------------------------------------ one warp's rows
// Fragment places of lane (b = lane / 4, a = lane % 4): stored tokens b and b + 8 of a panel as rows
// of S^T, rows 2 a and 2 a + 1 of each block of 8 (query, head) rows as its columns; output lanes
// 32 j + 4 b + (0..3) as rows of O^T.
//
// Weights are taken against a maximum that is looked for only when it has to move: in a segment's first
// unit, and when a lane's sum of a unit's weights passes 2^9. V scales are brought into [2^5, 2^6) by a
// power of two, so the products that become fp16 stay below 2^15 and keep their precision down to
// weights of 2^-19 of the largest; the power falls when a larger scale comes.
//
// The tensor cores do not round a product of a subnormal, they cut it toward zero near 2^-18 of the
// step's largest, and over a long row cuts of products that are all positive show: 4e-4 of the output
// at 131071 tokens. So odd panels go in as -p' (15 - c), whose cuts are to the other side, and what is
// left to centre is 7.5 times the difference of even and odd weights.
constexpr float kWeightsMost = 512.f;

// Exponent field of a stored scale, 0 for a NaN's.
__device__ __forceinline__ uint32_t scale_field(uint32_t meta) {
    const uint32_t e = (meta >> 10) & 31u;
    return e == 31u ? 0u : e;
}

template <int D, int GRP, int NT, bool MANY>
struct WarpRows {
    static constexpr int NW = D / 32, NG = D / GRP, WPG = GRP / 32, ROWS = 8 * NT, PANEL = panel_bytes(D, GRP);
    uint32_t qf[NT][2 * NW][2];         // q 2^e as B fragments, lanes 8 a + (0..7) of each 32
    float q1[NT][2][NG], qm[NT][2];     // sums of q 2^e over each group; 2^-e scale log2(e)
    int lim[NT][2], min_lim;            // tokens each row sees; the fewest any row of the block does
    float m[NT][2], l[NT][2];           // maximum so far (base 2) and this lane's share of the sum
    float o[2 * NW][NT][4];             // (p s 2^vn) . (c - 7.5), 2^-24 of it or (rows + 8 of a fragment) 2^-20
    float dsum[NT][2][NG];              // this lane's share of 2^vn p (m + 7.5 s)
    uint32_t vexp;                      // fp16 exponent field of the largest V scale so far (5 bits); vn = 20 - that. Above
                                        // them 5 bits a row: how far its own largest lies under it (not 0 behind a unit
                                        // that some row does not see to the end, which only such units follow)
    bool fresh;                         // no unit yet

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
            const uint16_t* src = static_cast<const uint16_t*>(P.q) + int64_t(rq.q0 + j) * P.q_stride + int64_t(h * P.G + g) * D + 8 * a;
            uint4 raw[NW];
            if (P.q_vec) {
                #pragma unroll
                for (int w = 0; w < NW; ++w) raw[w] = *reinterpret_cast<const uint4*>(src + 32 * w);
            } else {
                #pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const uint16_t* e = src + 32 * w;
                    raw[w] = make_uint4(e[0] | (uint32_t(e[1]) << 16), e[2] | (uint32_t(e[3]) << 16),
                                        e[4] | (uint32_t(e[5]) << 16), e[6] | (uint32_t(e[7]) << 16));
                }
            }
            float x[NW][8], big = 0.f;
            #pragma unroll
            for (int w = 0; w < NW; ++w) {
                const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 f = P.dtype == TTKV_BF16 ? make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u))
                                                    : __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                    if (!live) f = make_float2(0.f, 0.f);
                    x[w][2 * i] = f.x;
                    x[w][2 * i + 1] = f.y;
                    big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
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
            // a row with an infinity is NaN, also where its scores all come out as -inf (whose weights would be 0)
            const float fac = big == INFINITY ? __int_as_float(0x7fc00000)
                                              : P.scale * kLog2e * __uint_as_float(uint32_t(max(127 - e, 1)) << 23);
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
        min_lim = __reduce_min_sync(0xffffffffu, min_lim);
        vexp = 0;
        fresh = true;
    }

    __device__ __forceinline__ uint32_t own_shift(int nt, int c) const { return MANY ? (vexp >> (5 + 10 * nt + 5 * c)) & 31u : 0u; }

    // Tokens [t0, t0 + 64) of the request, four panels one behind the other. Panels behind the last token
    // hold whatever was there: codes are finite whatever their bits, and scales of tokens that a row does
    // not see are not used.
    __device__ __forceinline__ void step(const uint8_t* unit, int t0, int seq, int lane) {
        const int b = lane >> 2, a = lane & 3;
        const bool tail = t0 + kUnit > min_lim;                   // some row does not see all of them
        const uint8_t* kp = unit + b * (D / 2) + a * (D / 8);
        const uint8_t* vp = unit + 8 * D + a * D + b * (D / 8);
        const uint8_t* mp = unit + k_meta_offset(D) + b * NG * 4;
        constexpr int VM = v_meta_offset(D, GRP) - k_meta_offset(D);

        bool moved = false;
        float s[4][NT][4], ls[NT][2], corr[NT][2];
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt) corr[nt][0] = corr[nt][1] = 1.f;
        for (bool raise = fresh;; raise = true) {
            #pragma unroll
            for (int p = 0; p < 4; ++p) {
                uint32_t lo[NW], hi[NW], sm[2][NG];
                load_words(kp + p * PANEL, lo);
                load_words(kp + p * PANEL + 8 * (D / 2), hi);
                load_words(mp + p * PANEL, sm[0]);
                load_words(mp + p * PANEL + 8 * NG * 4, sm[1]);
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
                        f[i][g].x *= 16777216.f;                  // 2^24 of the codes
                    }
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = i & 1;
                        float x = f[i >> 1][0].y * q1[nt][c][0];
                        x = fmaf(f[i >> 1][0].x, acc[0][nt][i], x);
                        #pragma unroll
                        for (int g = 1; g < NG; ++g) {
                            x = fmaf(f[i >> 1][g].y, q1[nt][c][g], x);
                            x = fmaf(f[i >> 1][g].x, acc[g][nt][i], x);
                        }
                        s[p][nt][i] = x * qm[nt][c];
                    }
                if (tail) {
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        #pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t0 + 16 * p + b + 8 * (i >> 1) >= lim[nt][i & 1]) s[p][nt][i] = -INFINITY;
                }
            }
            if (raise) {
                moved = true;
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = -INFINITY;
                        #pragma unroll
                        for (int p = 0; p < 4; ++p) mx = fmaxf(mx, fmaxf(s[p][nt][c], s[p][nt][2 + c]));
                        #pragma unroll
                        for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
                        mx = fmaxf(mx, m[nt][c]);
                        corr[nt][c] = m[nt][c] == -INFINITY ? 1.f : ex2(m[nt][c] - mx);
                        m[nt][c] = mx;
                    }
            }
            bool over = false;
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float mm = m[nt][c] == -INFINITY ? 0.f : m[nt][c];  // a row that sees nothing has weights of 0
                    float t = 0.f;
                    #pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        s[p][nt][c] = ex2(s[p][nt][c] - mm);
                        s[p][nt][2 + c] = ex2(s[p][nt][2 + c] - mm);
                        t += s[p][nt][c] + s[p][nt][2 + c];
                    }
                    ls[nt][c] = t;
                    over |= t > kWeightsMost;
                }
            if (raise || !__any_sync(0xffffffffu, over)) break;
        }
        fresh = false;
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int c = 0; c < 2; ++c) l[nt][c] = fmaf(l[nt][c], corr[nt][c], ls[nt][c]);
        // the V scales of this lane's tokens (each token's lanes hold the same); the largest's exponent. A NaN's
        // (field 31) is none: its rows are NaN whatever the power, the other groups and rows need theirs
        uint32_t vm[4][2][NG], vmax = 0;
        #pragma unroll
        for (int p = 0; p < 4; ++p)
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                load_words(mp + p * PANEL + VM + i * 8 * NG * 4, vm[p][i]);
                if (tail && t0 + 16 * p + b + 8 * i >= seq) {
                    #pragma unroll
                    for (int g = 0; g < NG; ++g) vm[p][i][g] = 0u;
                }
                #pragma unroll
                for (int g = 0; g < NG; ++g) vmax = __vmaxu2(vmax, vm[p][i][g]);
            }
        vmax = __reduce_max_sync(0xffffffffu, (vmax >> 10) & 31u);
        if (vmax == 31u) {
            vmax = 0u;
            #pragma unroll
            for (int p = 0; p < 4; ++p)
                #pragma unroll
                for (int i = 0; i < 2; ++i)
                    #pragma unroll
                    for (int g = 0; g < NG; ++g) vmax = max(vmax, scale_field(vm[p][i][g]));
            vmax = __reduce_max_sync(0xffffffffu, vmax);
        }
        const uint32_t old = MANY ? vexp & 31u : vexp, ve = max(old, vmax);
        const float vfall = __uint_as_float((127u + old - ve) << 23);         // 2^(old - new)
        moved |= ve != old;
        const uint32_t was = vexp;
        vexp = ve;
        const float vn = __uint_as_float((127u + 20u - ve) << 23);
        if (MANY && tail) {
            // a token's scale must not cost the rows that do not see it their bits: each row's weights go by
            // the largest scale that it has seen, a power of two above the common one
            moved = true;
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t x = (was >> (5 + 10 * nt + 5 * c)) & 31u;
                    uint32_t e = old - x;
                    #pragma unroll
                    for (int p = 0; p < 4; ++p)
                        #pragma unroll
                        for (int i = 0; i < 2; ++i)
                            #pragma unroll
                            for (int g = 0; g < NG; ++g)
                                if (t0 + 16 * p + b + 8 * i < lim[nt][c]) e = max(e, scale_field(vm[p][i][g]));
                    #pragma unroll
                    for (int k = 4; k < 32; k <<= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, k));
                    vexp |= (ve - e) << (5 + 10 * nt + 5 * c);
                    corr[nt][c] *= __uint_as_float((127u + ve - e - x) << 23);
                    const float up = __uint_as_float((127u + ve - e) << 23);
                    #pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        s[p][nt][c] *= up;
                        s[p][nt][2 + c] *= up;
                    }
                }
        }

        if (moved) {                                              // (the same in every lane)
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int c = 0; c < 2; ++c) {
                    corr[nt][c] *= vfall;
                    #pragma unroll
                    for (int g = 0; g < NG; ++g) dsum[nt][c][g] *= corr[nt][c];
                }
            #pragma unroll
            for (int i = 0; i < 2 * NW; ++i)
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) o[i][nt][k] *= corr[nt][k & 1];
        }
        float psum[NG][NT][4];                                    // 15 times the unit's signed sum of p'
        #pragma unroll
        for (int g = 0; g < NG; ++g)
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int i = 0; i < 4; ++i) psum[g][nt][i] = 0.f;
        constexpr uint32_t L = 0x000f000fu, H = 0x00f000f0u;
        #pragma unroll
        for (int p = 0; p < 4; ++p) {
            uint32_t pf[NG][NT][2];
            #pragma unroll
            for (int g = 0; g < NG; ++g)
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&vm[p][i][g]));
                    const float sv = sm.x * (p & 1 ? -vn : vn), mid = fmaf(p & 1 ? -7.5f : 7.5f, sv, sm.y * vn);
                    #pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float p0 = s[p][nt][2 * i], p1 = s[p][nt][2 * i + 1];
                        float w0 = p0 * sv, w1 = p1 * sv, d0 = p0 * mid, d1 = p1 * mid;
                        if (tail) {                               // a weight of 0 on a NaN counts as none
                            const int t = t0 + 16 * p + b + 8 * i;
                            if (t >= lim[nt][0]) w0 = d0 = 0.f;
                            if (t >= lim[nt][1]) w1 = d1 = 0.f;
                        }
                        dsum[nt][0][g] += d0;
                        dsum[nt][1][g] += d1;
                        pf[g][nt][i] = transpose8x8(half2_bits(w0, w1));
                    }
                }
            #pragma unroll
            for (int g = 0; g < NG; ++g)
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma16816(psum[g][nt], L, H, L, H, pf[g][nt][0], pf[g][nt][1]);
            uint32_t lo[NW], hi[NW];                              // tokens 2 a, 2 a + 1 and those + 8
            load_words(vp + p * PANEL, lo);
            load_words(vp + p * PANEL + 4 * D, hi);
            #pragma unroll
            for (int w = 0; w < NW; ++w) {
                if (p & 1) { lo[w] = ~lo[w]; hi[w] = ~hi[w]; }
                const uint32_t l8 = lo[w] >> 8, h8 = hi[w] >> 8;
                #pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t b0 = pf[w / WPG][nt][0], b1 = pf[w / WPG][nt][1];
                    mma16816(o[2 * w][nt], lo[w] & L, lo[w] & H, hi[w] & L, hi[w] & H, b0, b1);
                    mma16816(o[2 * w + 1][nt], l8 & L, l8 & H, h8 & L, h8 & H, b0, b1);
                }
            }
        }
        #pragma unroll
        for (int i = 0; i < 2 * NW; ++i)
            #pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                #pragma unroll
                for (int k = 0; k < 4; ++k) o[i][nt][k] = fmaf(-0.5f, psum[i / 2 / WPG][nt][k], o[i][nt][k]);
    }

    // Sums over the lanes that share columns; o becomes sum p V relative to m, l the whole sum.
    __device__ __forceinline__ void finish() {
        float back[NT][2];
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                back[nt][c] = __uint_as_float((127u + (vexp & 31u) - own_shift(nt, c) - 20u) << 23);
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
                    o[i][nt][k] = fmaf(o[i][nt][k], k < 2 ? 16777216.f : 1048576.f, dsum[nt][k & 1][i / 2 / WPG]) * back[nt][k & 1];
    }

    __device__ __forceinline__ float4 four(int nt, int c, int k) const {      // output lanes 32 k + 4 b + (0..3)
        return make_float4(o[2 * k][nt][c], o[2 * k][nt][2 + c], o[2 * k + 1][nt][c], o[2 * k + 1][nt][2 + c]);
    }

    // As a part: [ROWS][D] of o, then (m, l) of each row.
    __device__ __forceinline__ void put_part(float* part, int lane) const {
        const int b = lane >> 2, a = lane & 3;
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int i = 8 * nt + 2 * a + c;
                #pragma unroll
                for (int k = 0; k < NW; ++k) *reinterpret_cast<float4*>(part + i * D + 32 * k + 4 * b) = four(nt, c, k);
                if (b == 0) *reinterpret_cast<float2*>(part + ROWS * D + 2 * i) = make_float2(m[nt][c], l[nt][c]);
            }
    }

    // As outputs.
    __device__ __forceinline__ void put_out(const AttnParams& P, const Req& rq, int h, int rb, int lane) const {
        const int b = lane >> 2, a = lane & 3;
        #pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = rb * ROWS + 8 * nt + 2 * a + c;
                if (row >= rq.ql * P.G) continue;
                const int j = row / P.G, g = row - j * P.G;
                const int64_t at = int64_t(rq.q0 + j) * P.out_stride + int64_t(h * P.G + g) * D + 4 * b;
                const float inv = l[nt][c] == 0.f ? 0.f : 1.f / l[nt][c];
                #pragma unroll
                for (int k = 0; k < NW; ++k) {
                    const float4 v = four(nt, c, k);
                    store4(P, at + 32 * k, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
    }
};

// ------------------------------------------------------------------ the streaming kernel
// The work is the list of (request, KV head, row block, 64-token unit), shared out in order: of T units CTA c of
// n owns [c S, (c + 1) S), S = ceil(T / n), each of its warps an equal part of that. A warp's run crosses from
// one (request, head, row block) to the next; what a run holds of one is a segment. Starting and ending
// a segment costs about as much as a unit (its queries, its sums), so each one counts as a unit more.
// A segment that is whole writes its output; the others meet in shared memory at the end of the CTA,
// and what is still a part then goes to the workspace for q4_merge_kernel (at most the CTA's first and
// its last).
//
// Every warp streams its own run through its own ring of two or three units in shared memory, filled by
// bulk copies (a panel is one contiguous piece of memory), ahead of the one that is worked on, so no warp
// waits for another and an SM keeps about 100 to 140 KB in flight, more than its share of bandwidth times
// latency (44 GB/s x 1 us). As many warps as their registers allow without spilling: 64 requests of 6000
// tokens with 3 query heads a KV head take 122 us with 8 warps and 108 with 12 (d = 128, groups of 128),
// 132 and 122 (groups of 64), 99 and 89 (d = 64, groups of 64), 110 and 99 (groups of 32); groups of 32 at
// d = 128 spill with 10 (155 and 181), as do two fragments of rows with 12 (194 and 263).
template <int D, int GRP, int NT>
struct Stream {
    static constexpr int PANEL = panel_bytes(D, GRP), UNIT = 4 * PANEL;
    static constexpr int WARPS = NT == 1 && (D == 64 || GRP > 32) ? 12 : 8;
    static constexpr int RING = 3 * UNIT * WARPS <= 216 * 1024 ? 3 : 2;
    static constexpr int THREADS = 32 * WARPS, ROWS = 8 * NT, SLOTS = 2 * WARPS;
    static constexpr int PART = ROWS * (D + 2);                                 // floats of a part: o, then (m, l)
    static constexpr int RING_BYTES = WARPS * RING * UNIT;
    static constexpr int SMEM = std::max(WARPS * PART * 4, RING_BYTES) + WARPS * RING * 8;
};

// A place in the work list: unit ui of the U (and one more that counts for the segment) of row block rb
// of KV head h of request r.
struct Cursor {
    int r, h, rb, ui, U, nrb, seq;
};

__device__ __forceinline__ void load_request(const AttnParams& P, Cursor& c, int rows) {
    const Req a = request(P, c.r, false);
    c.seq = a.seq;
    c.U = units_of(a);
    c.nrb = row_blocks(a, P.G, rows);
}

__device__ __forceinline__ int list_units(const Req& a, int G, int rows) {      // of one KV head
    const int U = units_of(a);
    return U ? row_blocks(a, G, rows) * (U + 1) : 0;
}

// To the next row block; the run is not over, so there is one.
__device__ __forceinline__ void next_block(const AttnParams& P, Cursor& c, int rows) {
    c.ui = 0;
    if (++c.rb < c.nrb) return;
    c.rb = 0;
    if (++c.h < P.H) return;
    c.h = 0;
    do {
        ++c.r;
        load_request(P, c, rows);
    } while (c.U == 0);
}

// MANY: requests may have several queries. The treatment of rows that see different tokens takes registers in every
// unit: 64 requests of 6000 tokens with 3 query heads a KV head take 109 us without and 112 with it (d = 128).
template <int D, int GRP, int NT, bool MANY>
__global__ void __launch_bounds__(Stream<D, GRP, NT>::THREADS, 1) q4_stream_kernel(const AttnParams P) {
    using Rows = WarpRows<D, GRP, NT, MANY>;
    using S = Stream<D, GRP, NT>;
    constexpr int ROWS = S::ROWS, SLOTS = S::SLOTS, WARPS = S::WARPS, THREADS = S::THREADS, PANEL = S::PANEL, RING = S::RING;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::SMEM - WARPS * RING * 8);
    __shared__ int pre[THREADS + 1];
    __shared__ long long wsum[WARPS];
    __shared__ int pid[SLOTS];                           // first unit of the slot's (request, head, row block), -1: none
    __shared__ int pr[SLOTS], ph[SLOTS], prb[SLOTS];
    __shared__ float pm[SLOTS][ROWS], pl[SLOTS][ROWS];   // max and sum of the parts' rows

    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    const bool tell = blockIdx.x == 0;
    uint8_t* ring = smem + w * RING * S::UNIT;
    uint64_t* bar = bars + w * RING;
    if (lane < RING) mbar_init(bar + lane, 1);
    pdl_wait();

    // ---- units of the requests before each thread's share of them
    const int per = (P.n_reqs + THREADS - 1) / THREADS;
    const int rlo = min(tid * per, P.n_reqs), rhi = min(rlo + per, P.n_reqs);
    long long sum = 0;
    for (int r = rlo; r < rhi; ++r) sum += (long long)P.H * list_units(request(P, r, tell), P.G, ROWS);
    long long inc = sum;
    #pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, k);
        if (lane >= k) inc += y;
    }
    if (lane == 31) wsum[w] = inc;
    if (tid < SLOTS) pid[tid] = -1;
    __syncthreads();
    for (int i = 0; i < w; ++i) inc += wsum[i];
    pre[tid] = int(inc - sum);
    if (tid == THREADS - 1) {
        // 2^31 units would read 2^37 tokens: reported, and nothing done
        const bool vast = inc > 0x7fff0000;
        pre[THREADS] = vast ? 0 : int(inc);
        if (vast && tell) report(P.status, TTKV_STATUS_SEQ_BOUND);
    }
    __syncthreads();
    const int T = pre[THREADS], share = share_size(T, P.n_ctas);
    pdl_trigger();
    const int ca = min(int(blockIdx.x) * share, T), cb = min(ca + share, T);
    if (ca == cb) return;

    // ---- this warp's run
    Rows R;
    bool held = false;
    int u = ca + w * (cb - ca) / WARPS;
    const int ue = ca + (w + 1) * (cb - ca) / WARPS;
    if (u < ue) {
        Cursor c;
        {
            int lo = 0, hi = THREADS - 1;                // the last chunk of requests that begins at or before u
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (pre[mid] <= u) lo = mid; else hi = mid - 1;
            }
            int off = u - pre[lo];
            for (c.r = lo * per;; ++c.r) {
                load_request(P, c, ROWS);
                const int all = c.U ? P.H * c.nrb * (c.U + 1) : 0;
                if (off < all) break;
                off -= all;
            }
            const int pair = off / (c.U + 1);
            c.ui = off - pair * (c.U + 1);
            c.h = pair / c.nrb;
            c.rb = pair - c.h * c.nrb;
        }
        // fetching: lanes 0 to 3 each know the block of one panel of unit f, the next to be issued
        Cursor f = c;
        int uf = u, f_blk = 0;
        uint32_t n_f = 0, i_f = 0;                       // units issued, and the next one's place
        const int ppb = P.block_size / kPanelTokens;     // panels of a block
        auto block_of = [&](int t) { return P.bs_shift >= 0 ? t >> P.bs_shift : t / P.block_size; };
        auto look_up = [&]() {                           // f to a unit, and its blocks
            while (uf < ue && f.ui >= f.U) {
                if (++uf < ue) next_block(P, f, ROWS);
            }
            const int t = f.ui * kUnit + 16 * lane;
            if (uf < ue && lane < 4 && t < f.seq) f_blk = P.block_table[int64_t(f.r) * P.bt_stride + block_of(t)];
        };
        auto issue = [&]() {
            if (uf >= ue) return;
            const int t = f.ui * kUnit + 16 * lane;
            const bool mine = lane < 4 && t < f.seq, good = mine && f_blk >= 0 && f_blk < P.n_blocks;
            const uint32_t goods = __ballot_sync(0xffffffffu, good);
            uint8_t* dst = ring + i_f * S::UNIT + lane * PANEL;
            if (__any_sync(0xffffffffu, mine && !good)) {
                if (mine && !good) {                     // NaN scales: the request's rows come out as NaN
                    report(P.status, TTKV_STATUS_BLOCK_RANGE);
                    uint32_t* d = reinterpret_cast<uint32_t*>(dst);
                    for (int k = 4 * D; k < PANEL / 4; ++k) d[k] = 0x00007e00u;
                    fence_async_smem();
                }
                __syncwarp();
            }
            if (lane == 0) mbar_expect_tx(bar + i_f, __popc(goods) * PANEL);
            if (good) {
                const int64_t pan = (int64_t(f_blk) * P.H + f.h) * ppb + ((t - block_of(t) * P.block_size) >> 4);
                bulk_g2s(dst, P.cache + pan * PANEL, PANEL, bar + i_f);
            }
            ++n_f;
            i_f = i_f + 1 == RING ? 0 : i_f + 1;
            ++f.ui;
            ++uf;
            look_up();
        };
        look_up();
        #pragma unroll 1
        for (int i = 1; i < RING; ++i) issue();
        uint32_t n_c = 0, i_c = 0, ph_c = 0;             // units consumed, the place of the next and its phase
        bool late = false;
        while (u < ue) {
            const int n_list = min(c.U + 1 - c.ui, ue - u), n_here = min(c.U - c.ui, n_list), begin = c.ui;
            u += n_list;
            if (n_here > 0) {
                const Req rq = request(P, c.r, false);
                R.start(P, rq, c.h, c.rb, lane);
                for (int i = 0; i < n_here; ++i) {
                    issue();                             // a unit, into the place of the one before this
                    const bool ok = late || mbar_wait(bar + i_c, ph_c);
                    if (!__all_sync(0xffffffffu, ok)) {  // a copy never came: wait for the others, issue no more
                        late = true;
                        if (lane == 0) report(P.status, TTKV_STATUS_TIMEOUT);
                        for (uint32_t k = n_c + 1; k < n_f; ++k) mbar_wait(bar + k % RING, (k / RING) & 1u);
                        uf = ue;
                    }
                    R.step(ring + i_c * S::UNIT, (begin + i) * kUnit, rq.seq, lane);
                    __syncwarp();                        // every lane has read the unit
                    ++n_c;
                    if (++i_c == RING) { i_c = 0; ph_c ^= 1u; }
                }
                R.finish();
                if (begin == 0 && n_here == c.U) {       // whole
                    R.put_out(P, rq, c.h, c.rb, lane);
                } else {
                    // a part: the run's last stays in registers until the rings are free, its first goes
                    // to the workspace
                    held = u == ue;
                    if (lane == 0) {
                        const int e = 2 * w + (held ? 1 : 0);
                        pid[e] = u - n_list - begin;
                        pr[e] = c.r;
                        ph[e] = c.h;
                        prb[e] = c.rb;
                    }
                    if (!held) R.put_part(P.first + (int64_t(blockIdx.x) * WARPS + w) * S::PART, lane);
                }
            }
            if (u < ue) next_block(P, c, ROWS);
        }
    }
    __syncthreads();                                     // every copy has landed and been read
    if (held) R.put_part(reinterpret_cast<float*>(smem) + w * S::PART, lane);
    __syncthreads();

    // ---- what the warps hold of the same (request, head, row block), joined
    auto part_of = [&](int e) -> const float* {
        return (e & 1) ? reinterpret_cast<const float*>(smem) + (e >> 1) * S::PART
                       : P.first + (int64_t(blockIdx.x) * WARPS + (e >> 1)) * S::PART;
    };
    for (int k = tid; k < SLOTS * ROWS; k += THREADS) {
        const int e = k / ROWS, i = k % ROWS;
        if (pid[e] >= 0) {
            const float2 ml = *reinterpret_cast<const float2*>(part_of(e) + ROWS * D + 2 * i);
            pm[e][i] = ml.x;
            pl[e][i] = ml.y;
        }
    }
    __syncthreads();
    static_assert(SLOTS <= 32, "a slot a lane");
    const int mine = lane < SLOTS ? pid[lane] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, mine);
    for (uint32_t heads = __ballot_sync(0xffffffffu, mine >= 0 && (same & ((1u << lane) - 1u)) == 0u); heads; heads &= heads - 1u) {
        const int s0 = __ffs(heads) - 1, id = __shfl_sync(0xffffffffu, mine, s0);
        const uint32_t slots = __shfl_sync(0xffffffffu, same, s0);
        const int s1 = 32 - __clz(slots);
        const Req rq = request(P, pr[s0], false);
        const int h = ph[s0], rb = prb[s0], live = min(ROWS, rq.ql * P.G - rb * ROWS);
        const bool whole = id >= ca && id + units_of(rq) <= cb;
        const int64_t g0 = (int64_t(blockIdx.x) * 2 + (ca >= id ? 0 : 1)) * ROWS;
        for (int e = tid; e < live * (D / 4); e += THREADS) {
            const int i = e / (D / 4), ln = 4 * (e - i * (D / 4));
            float M = -INFINITY;
            for (int k = s0; k < s1; ++k)
                if (slots >> k & 1u) M = fmaxf(M, pm[k][i]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
            #pragma unroll 4
            for (int k = s0; k < s1; ++k) {
                if (!(slots >> k & 1u)) continue;
                const float wt = part_weight(pm[k][i], M);
                const float4 x = *reinterpret_cast<const float4*>(part_of(k) + i * D + ln);
                l = fmaf(wt, pl[k][i], l);
                o.x = fmaf(wt, x.x, o.x); o.y = fmaf(wt, x.y, o.y); o.z = fmaf(wt, x.z, o.z); o.w = fmaf(wt, x.w, o.w);
            }
            if (whole) {
                store_out(P, rq, h, rb * ROWS + i, D, ln, o, l);
            } else {
                *reinterpret_cast<float4*>(P.part_o + (g0 + i) * D + ln) = o;
                if (ln == 0) *reinterpret_cast<float2*>(P.part_ml + (g0 + i) * 2) = make_float2(M, l);
            }
        }
    }
}

// ------------------------------------------------------------------ the merge
// One CTA per (request, KV head, row): the parts that the CTAs left of its (request, head, row block),
// found from the shares; also the zeros of an empty request. D / 4 threads take four lanes each of
// one part, the CTA's thread groups different parts. It is launched early and finds its place in the
// list, a sum over the requests as in the streaming kernel, while that one still runs.
constexpr int kMergeThreads = 256;

__global__ void __launch_bounds__(kMergeThreads) q4_merge_kernel(const AttnParams P, int D, int rows_block) {
    __shared__ float4 so[kMergeThreads];
    __shared__ float2 sml[kMergeThreads / 16];
    __shared__ long long sbefore[kMergeThreads / 32], sall[kMergeThreads / 32];
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const Req rq = request(P, r, false);
    const int per_head = P.max_q * P.G;
    const int h = blockIdx.x / per_head, row = blockIdx.x - h * per_head;
    if (rq.ql <= 0 || row >= rq.ql * P.G) {
        pdl_wait();                                              // this grid ends after the streaming kernel
        return;
    }
    const int lanes = D / 4, grp = tid / lanes, ngrp = kMergeThreads / lanes, ln = 4 * (tid - grp * lanes);
    const int U = units_of(rq);
    const int nrb = row_blocks(rq, P.G, rows_block), rb = row / rows_block, i = row - rb * rows_block;
    long long before = 0, all = 0;
    for (int k = tid; k < P.n_reqs; k += kMergeThreads) {
        const long long n = (long long)P.H * list_units(request(P, k, false), P.G, rows_block);
        all += n;
        before += k < r ? n : 0;
    }
    #pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, k);
        before += __shfl_xor_sync(0xffffffffu, before, k);
    }
    if (lane == 0) {
        sbefore[tid >> 5] = before;
        sall[tid >> 5] = all;
    }
    __syncthreads();
    before = all = 0;
    #pragma unroll
    for (int k = 0; k < kMergeThreads / 32; ++k) {
        before += sbefore[k];
        all += sall[k];
    }
    pdl_wait();
    if (U == 0) {
        if (grp == 0) store_out(P, rq, h, row, D, ln, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
        return;
    }
    if (all > 0x7fff0000) return;                                // (refused, as the streaming kernel has reported)
    const int share = share_size(int(all), P.n_ctas), u0 = int(before) + (h * nrb + rb) * (U + 1);
    const int c0 = u0 / share, c1 = (u0 + U - 1) / share;
    if (c0 == c1) return;                                        // that CTA has written the output
    // a part lies in its CTA's first place unless the CTA's share began before it
    auto place = [&](int c) { return (int64_t(c) * 2 + (c * share >= u0 ? 0 : 1)) * rows_block + i; };
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    #pragma unroll 4
    for (int c = c0 + grp; c <= c1; c += ngrp) {
        const int64_t s = place(c);
        const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + 2 * s);
        const float4 x = *reinterpret_cast<const float4*>(P.part_o + s * D + ln);
        const float M = fmaxf(m, ml.x), wo = part_weight(m, M), wn = part_weight(ml.x, M);
        m = M;
        l = l * wo + ml.y * wn;
        o.x = o.x * wo + x.x * wn; o.y = o.y * wo + x.y * wn; o.z = o.z * wo + x.z * wn; o.w = o.w * wo + x.w * wn;
    }
    so[tid] = o;
    if (ln == 0) sml[grp] = make_float2(m, l);
    __syncthreads();
    if (grp) return;
    for (int k = 0; k < ngrp; ++k) m = fmaxf(m, sml[k].x);
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < ngrp; ++k) {
        const float wt = part_weight(sml[k].x, m);
        const float4 x = so[k * lanes + tid];
        l = fmaf(wt, sml[k].y, l);
        o.x = fmaf(wt, x.x, o.x); o.y = fmaf(wt, x.y, o.y); o.z = fmaf(wt, x.z, o.z); o.w = fmaf(wt, x.w, o.w);
    }
    store_out(P, rq, h, row, D, ln, o, l);
}

// ------------------------------------------------------------------ host

// Fragments of 8 (query, head) rows that a streaming warp takes at once: two above 8 rows, but at d = 128 only
// where that leaves none empty, and in groups of 32 there not at all, since two spill. 64 requests of 6000
// tokens, 8 KV heads, us with two and with one:
//   d, group   16 rows    24         32
//   64, 32     176/197    305/283    322/369   (and ragged, 1 to 20 rows: 36/38)
//   64, 64     158/176    270/254    283/330
//   128, 128   203/219    348/315    369/410
//   128, 64    229/244    399/352    422/459
//   128, 32    350/317    637/463    649/606
int stream_nt(int d, int group, int64_t rows) {
    if (d == 64) return rows > 8 ? 2 : 1;
    return group == 32 || (rows + 7) / 8 % 2 ? 1 : 2;
}

// Workspace: two parts a CTA for the merge, a part a warp.
struct StreamWs {
    size_t part_ml, first, bytes;
};

StreamWs stream_ws(int d, int nt) {
    StreamWs w;
    const size_t rows = size_t(kMaxCtas) * 2 * 8 * nt;
    w.part_ml = rows * d * sizeof(float);
    w.first = w.part_ml + rows * 2 * sizeof(float);
    w.bytes = w.first + size_t(kMaxCtas) * (nt == 1 ? Stream<128, 128, 1>::WARPS : Stream<128, 128, 2>::WARPS) * 8 * nt * (d + 2) * sizeof(float);
    return w;
}

int check_attn(const ttkv_q4_attn_args_t* a) {
    if (!a) return fail(TTKV_ERR_ARG, "4-bit read: null arguments");
    if (int e = check_cache(&a->cache)) return e;
    if (a->n_reqs < 0 || a->bt_cols < 0) return fail(TTKV_ERR_ARG, "4-bit read: batch");
    if (a->n_reqs > 65535) return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: %d requests in one call", a->n_reqs);
    if (a->n_reqs > 0 && (!a->seq_lens || !a->q || !a->out || (a->bt_cols > 0 && !a->block_table)))
        return fail(TTKV_ERR_ARG, "4-bit read: null pointer");
    if (a->HQ < a->cache.H || a->HQ % a->cache.H) return fail(TTKV_ERR_ARG, "HQ=%d is not a multiple of H=%d", a->HQ, a->cache.H);
    if (a->dtype != TTKV_F16 && a->dtype != TTKV_BF16)
        return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: queries and outputs are fp16 or bf16");
    if (!std::isfinite(a->scale)) return fail(TTKV_ERR_ARG, "4-bit read: a scale of %g", double(a->scale));
    if (a->q_stride < 0 || a->out_stride < 0) return fail(TTKV_ERR_ARG, "4-bit read: a negative stride");
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 1)
        return fail(TTKV_ERR_ALIGN, "4-bit read: q or out at an odd address");
    return TTKV_OK;
}

template <int D, int GRP, int NT>
int launch_stream(const AttnParams& P, cudaStream_t st) {
    using S = Stream<D, GRP, NT>;
    const auto k = P.q_len ? q4_stream_kernel<D, GRP, NT, true> : q4_stream_kernel<D, GRP, NT, false>;
    if (int e = raise_smem_limit(reinterpret_cast<const void*>(k), "q4_stream_kernel")) return e;
    // both may start while the kernel before them runs and wait for it themselves
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(P.n_ctas));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, k, P);
    if (e != cudaSuccess) { cudaGetLastError(); return fail(TTKV_ERR_CUDA, "q4_stream_kernel: %s", cudaGetErrorString(e)); }
    cfg.gridDim = dim3(unsigned(P.H * P.max_q * P.G), unsigned(P.n_reqs));
    cfg.blockDim = dim3(kMergeThreads);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, q4_merge_kernel, P, D, 8 * NT);
    if (e != cudaSuccess) { cudaGetLastError(); return fail(TTKV_ERR_CUDA, "q4_merge_kernel: %s", cudaGetErrorString(e)); }
    return TTKV_OK;
}

int run_stream(const ttkv_q4_cache_t* c, AttnParams P, void* ws, size_t ws_bytes, cudaStream_t st) {
    const int nt = stream_nt(c->d, c->group, int64_t(P.max_q) * P.G);
    const StreamWs w = stream_ws(c->d, nt);
    if (!ws || ws_bytes < w.bytes)
        return fail(TTKV_ERR_WORKSPACE, "4-bit read: workspace of %zu bytes, %zu needed", ws ? ws_bytes : 0, w.bytes);
    if (reinterpret_cast<uintptr_t>(ws) & 15) return fail(TTKV_ERR_ALIGN, "4-bit read: workspace not 16-byte aligned");
    int sms = 0;
    if (int e = sm_count(&sms)) return e;
    P.n_ctas = std::min(sms, kMaxCtas);
    char* base = static_cast<char*>(ws);
    P.part_o = reinterpret_cast<float*>(base);
    P.part_ml = reinterpret_cast<float*>(base + w.part_ml);
    P.first = reinterpret_cast<float*>(base + w.first);
#define TTKV_Q4_STREAM(D, GRP)                                                                     \
    if (c->d == D && c->group == GRP) return nt == 2 ? launch_stream<D, GRP, 2>(P, st) : launch_stream<D, GRP, 1>(P, st);
    TTKV_Q4_STREAM(64, 32) TTKV_Q4_STREAM(64, 64) TTKV_Q4_STREAM(128, 64) TTKV_Q4_STREAM(128, 128)
    if (c->d == 128 && c->group == 32) return launch_stream<128, 32, 1>(P, st);
#undef TTKV_Q4_STREAM
    return fail(TTKV_ERR_UNSUPPORTED, "4-bit read: geometry");
}

AttnParams attn_params(const ttkv_q4_attn_args_t* a) {
    const ttkv_q4_cache_t* c = &a->cache;
    AttnParams P{};
    P.cache = c->base; P.n_blocks = c->n_blocks; P.H = c->H; P.G = a->HQ / c->H; P.block_size = c->block_size;
    P.bs_shift = -1;
    for (int b = 0; b < 31; ++b)
        if (c->block_size == (1 << b)) P.bs_shift = b;
    P.block_table = a->block_table; P.bt_stride = a->bt_stride; P.bt_cols = a->bt_cols; P.seq_lens = a->seq_lens;
    P.n_reqs = a->n_reqs; P.q = a->q; P.dtype = a->dtype; P.q_stride = a->q_stride; P.scale = a->scale;
    P.out = a->out; P.out_stride = a->out_stride; P.status = a->status;
    P.q_vec = rows_aligned(a->q, a->dtype, a->q_stride);
    P.out_vec = rows_aligned(a->out, a->dtype, a->out_stride) ? 2
              : (reinterpret_cast<uintptr_t>(a->out) & 7) == 0 && (a->out_stride & 3) == 0;
    return P;
}

// Whether chunks of `rows` (query, head) rows a KV head are streamed, the cache read and its codes fed to
// the tensor cores once per 16 rows (8 in groups of 32 at d = 128, `narrow`), or go to the chunk kernel,
// whose tiles of 256 rows each dequantise the cache once. Streamed against chunked, d = 128 in groups of 128,
// 8 KV heads, bf16 (chunks of fp16 queries take 11 to 16 percent more), us:
//   requests x tokens   16 rows      24           32           48           64
//   64 x 130            56 / 73      73 / 77      91 / 77      128 / 77     159 / 79
//   16 x 500            32 / 36      36 / 36      42 / 34      52 / 36      67 / 36
//   64 x 1500           96 / 206     136 / 216    169 / 200    241 / 208    310 / 204
//   64 x 6000           202 / 550    316 / 579    370 / 531    531 / 552    693 / 548
//   4 x 3000            28 / 50      30 / 54      34 / 50      40 / 54      50 / 50
//   1 x 130             19 / 26      17 / 28      19 / 28      22 / 28      22 / 28
//   1 x 16000           30 / 77      32 / 87      38 / 85      42 / 89      46 / 87
// and in groups of 32:
//   64 x 1500           128 / 206    177 / 216    232 / 202    331 / 210    447 / 204
//   64 x 6000           318 / 544    466 / 566    607 / 533    896 / 556    1183 / 560
//   4 x 3000            30 / 50      34 / 54      44 / 50      52 / 54      62 / 52
// (d = 64 as the first, with 325 / 423 and 286 / 421 at 64 x 6000 and 32 rows). So up to 24 rows always, up to
// 32 over long rows unless narrow, up to 64 where few (request, head) pairs leave most of the chunk kernel's time
// to latency. Many short requests of 17 to 24 rows are the worst of it (64 x 130: up to 18 percent).
bool streams(int64_t rows, int64_t pairs, int max_seq, bool narrow) {
    return rows <= 24 || (rows <= 32 && max_seq >= 1536 && !narrow) || (rows <= 64 && pairs <= 32);
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" size_t ttkv_q4_decode_workspace_bytes(int32_t d, int32_t n_reqs, int32_t group_heads) {
    return n_reqs < 0 ? 0 : stream_ws(d, group_heads > 8 ? 2 : 1).bytes;      // (two fragments need more than one)
}

extern "C" int ttkv_q4_decode(const ttkv_q4_attn_args_t* args) {
    if (int e = check_attn(args)) return e;
    if (args->n_reqs == 0) return TTKV_OK;
    AttnParams P = attn_params(args);
    P.n_rows = args->n_reqs;
    P.max_q = 1;
    P.max_seq = kMaxSeq;
    return run_stream(&args->cache, P, args->workspace, args->workspace_bytes, static_cast<cudaStream_t>(args->stream));
}

extern "C" size_t ttkv_q4_prefill_workspace_bytes(int32_t d, int32_t n_reqs, int32_t group_heads, int32_t max_q_len) {
    if (n_reqs < 0 || max_q_len < 0) return 0;
    const int64_t rows = int64_t(max_q_len) * group_heads;
    const bool some = streams(rows, 0, INT32_MAX, false), all = streams(rows, INT64_MAX, 0, true);    // are streamed
    return std::max(some ? stream_ws(d, rows > 8 ? 2 : 1).bytes : 0, all ? 0 : chunk_workspace_bytes(d));
}

extern "C" int ttkv_q4_prefill(const ttkv_q4_attn_args_t* args) {
    if (int e = check_attn(args)) return e;
    if (args->max_q_len < 0 || args->max_seq_len < 0 || args->n_rows < 0) return fail(TTKV_ERR_ARG, "4-bit prefill: a negative size");
    if (args->n_reqs > 0 && (!args->q_start || !args->q_len)) return fail(TTKV_ERR_ARG, "4-bit prefill: q_start or q_len missing");
    if (args->n_reqs == 0 || args->n_rows == 0 || args->max_q_len == 0) return TTKV_OK;
    if (int64_t(args->max_q_len) * args->HQ > 0x7fffffff)
        return fail(TTKV_ERR_UNSUPPORTED, "4-bit prefill: %d queries of %d heads", args->max_q_len, args->HQ);
    AttnParams P = attn_params(args);
    P.q_start = args->q_start; P.q_len = args->q_len; P.n_rows = args->n_rows; P.max_q = args->max_q_len;
    P.max_seq = std::min(args->max_seq_len, kMaxSeq);
    const cudaStream_t st = static_cast<cudaStream_t>(args->stream);
    const bool narrow = args->cache.d == 128 && args->cache.group == 32;
    return streams(int64_t(args->max_q_len) * P.G, int64_t(args->n_reqs) * P.H, P.max_seq, narrow)
        ? run_stream(&args->cache, P, args->workspace, args->workspace_bytes, st)
        : run_chunk(&args->cache, P, args->workspace, args->workspace_bytes, st);
}
