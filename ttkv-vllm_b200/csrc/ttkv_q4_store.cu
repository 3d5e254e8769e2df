// The 4-bit paged cache: quantise and scatter (ttkv_q4_write), gather and dequantise (ttkv_q4_read).
//
// Bound: memory. A token of one head moves 4 d bytes of 16-bit K and V and d + 8 d / group packed
// bytes, each once. d / 8 consecutive lanes of a warp own a (token, head) row, eight values a lane
// (one 16-byte load of each 16-bit row): the group's minimum and maximum are shuffles within the
// group's lanes, and a lane's eight K codes are one 32-bit word of the panel, its V codes two 16-bit
// ones (the V order pairs tokens, so a lone token's bytes lie apart).
#include "ttkv_async.cuh"
#include "ttkv_q4.cuh"

namespace ttkv {
namespace {

using namespace q4;

constexpr int kStoreThreads = 256;

struct StoreParams {
    uint8_t* cache;
    int64_t n_slots;
    int32_t H, block_size, bs_shift;         // log2 of the block size, -1 where it is no power of two
    const int64_t* slots;
    int32_t n, skip_pad;
    void* k;
    void* v;
    int32_t k_dtype, v_dtype, k_vec, v_vec;
    int64_t k_stride, v_stride;
    int32_t* status;
};

// Scale and minimum of a group whose lanes hold x, and the codes of this lane's eight. G lanes per
// group.
//
// The format rounds the scale once from (hi - lo) / 15 and a code once from (x - m) / s. fp32 settles
// both except next to a border between two results: a scale within 3 units of the middle of the 13
// bits that fp16 drops, a few in ten thousand, which is redone in fp64 out of the way; and a code's
// quotient, off by 5e-6 at most, within 1e-5 of one half. Of 16-bit values one in a few thousand lies
// exactly there, so this is settled in fp32, by the exact remainder x - m - c s: the difference's own
// rounding error is known, and the remainder of a product of 15 bits is exact.
// What bounds a long write is the number of instructions a value.
// Values beyond the limit need no clamp of their own: the ends of the group are clamped, and the
// quotient as a fraction of 15 by its saturation. It is rounded by adding 1.5 2^23, which leaves the
// integer in the low bits of the sum, where eight of them are packed by shifts and adds (the sum's
// high bits, the same in every value, are taken off at the end).
__device__ __noinline__ uint32_t exact_scale(float lo, float hi) {
    // round to odd in fp32 first: its 13 extra bits then decide the fp16 rounding exactly
    const double e = __ddiv_rn(double(hi) - double(lo), 15.0);
    float f = __double2float_rz(e);
    if (double(f) != e) f = __uint_as_float(__float_as_uint(f) | 1u);
    return __half_as_ushort(__float2half_rn(f));
}

// The integer nearest to (x - m) / s, ties to even, c being within one of it; clamped to 0..15.
__device__ __forceinline__ uint32_t exact_code(float x, float m, float s, float c) {
    const float d = x - m, b = d - x, e = (x - (d - b)) - (m + b);      // x - m = d + e exactly
    const float r = fmaf(-c, s, d);                                     // exact
    const float over = (fabsf(r) - 0.5f * s) + copysignf(1.f, r) * e;   // beyond half a step, or 0 at it
    const bool odd = int(c) & 1;
    if (over > 0.f || (over == 0.f && odd)) c += copysignf(1.f, r);
    return uint32_t(fminf(fmaxf(c, 0.f), 15.f));
}

template <int G>
__device__ __forceinline__ uint32_t quantise_group(const float (&x)[8], uint32_t& meta) {
    float lo = x[0], hi = x[0], bad = x[0] * 0.f;             // 0, or NaN where x is not finite
    #pragma unroll
    for (int j = 1; j < 8; ++j) {
        bad = fmaf(x[j], 0.f, bad);
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
    }
    #pragma unroll
    for (int o = 1; o < G; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    constexpr uint32_t MASK = (1u << G) - 1u;                 // (G is 16 at most)
    const bool nan = __ballot_sync(0xffffffffu, bad != bad) & (MASK << (threadIdx.x & 31 & ~(G - 1)));
    lo = fminf(fmaxf(lo, -kLimit), kLimit);
    hi = fminf(fmaxf(hi, -kLimit), kLimit);

    const __half mh = __float2half_rn(lo + 0.f);              // -0 is stored as 0
    const float m = __half2float(mh);
    const float q = (hi - lo) * (1.f / 15.f);
    const uint32_t low = __float_as_uint(q) & 0x1fffu;
    uint32_t sb = __half_as_ushort(__float2half_rn(q));
    if (q < 6.2e-5f || (low >= 0xffdu && low <= 0x1003u)) sb = q == 0.f ? 0u : exact_scale(lo, hi);
    const float s = __half2float(__ushort_as_half(uint16_t(sb)));
    float inv = 0.f;
    if (s > 0.f) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(15.f * s));
    constexpr float MAGIC = 12582912.f;
    uint32_t codes = 0;
    float near = 0.f;
    #pragma unroll
    for (int j = 7; j >= 0; --j) {
        const float t = __saturatef((x[j] - m) * inv), u = fmaf(t, 15.f, MAGIC);
        near = fmaxf(near, fabsf(fmaf(t, 15.f, MAGIC - u)));
        codes = codes * 16u + __float_as_uint(u);
    }
    // the high bits 0x4b400000 of the last three values packed; those of the others were shifted out
    codes -= 0x4b400000u + (0x4b400000u << 4) + (0x4b400000u << 8);
    if (near > 0.49999f) {
        codes = 0;
        #pragma unroll
        for (int j = 0; j < 8; ++j)
            codes |= exact_code(x[j], m, s, fmaf(__saturatef((x[j] - m) * inv), 15.f, MAGIC) - MAGIC) << (4 * j);
    }
    if (nan) codes = 0;
    meta = nan ? 0x7e00u : sb | (uint32_t(__half_as_ushort(mh)) << 16);
    return codes;
}

__device__ __forceinline__ bool slot_ok(const StoreParams& P, int64_t slot, bool first) {
    if (slot >= 0 && slot < P.n_slots) return true;
    if (first && !(slot < 0 && P.skip_pad)) report(P.status, TTKV_STATUS_SLOT_RANGE);
    return false;
}

// Where a slot's token of head h lies: its panel and its place o in it.
__device__ __forceinline__ uint8_t* panel_of(const StoreParams& P, int64_t slot, int h, int panel, int& o) {
    const int64_t blk = P.bs_shift >= 0 ? slot >> P.bs_shift : slot / P.block_size;
    const int off = int(slot - blk * P.block_size);
    o = off % kPanelTokens;
    return P.cache + ((blk * P.H + h) * (P.block_size / kPanelTokens) + off / kPanelTokens) * panel;
}

// A CTA's rows are consecutive tokens of head blockIdx.y, D / 8 threads each: two tokens of a pair lie in
// one warp, whose stores then fill whole sectors. (Two rows a thread, with twice the loads in flight,
// took 62 us against 48 for 16384 tokens: the registers cost more warps than that gives.)
template <int D, int GRP>
__global__ void __launch_bounds__(kStoreThreads) q4_write_kernel(const StoreParams P) {
    constexpr int TPR = D / 8, G = GRP / 8, NG = D / GRP;
    const int i = threadIdx.x % TPR, h = blockIdx.y;
    const int64_t row = int64_t(blockIdx.x) * (kStoreThreads / TPR) + threadIdx.x / TPR;
    const int64_t tok = min(row, int64_t(P.n - 1));  // (rows behind the last token load it again and store nothing)
    pdl_wait();
    pdl_trigger();
    float x[8], y[8];
    const int64_t slot = P.slots[tok];
    load8(P.k, P.k_dtype, tok * P.k_stride + h * D + 8 * i, P.k_vec, x);
    load8(P.v, P.v_dtype, tok * P.v_stride + h * D + 8 * i, P.v_vec, y);
    uint32_t km, vm;
    const uint32_t kc = quantise_group<G>(x, km), vc = quantise_group<G>(y, vm);
    if (row >= P.n || !slot_ok(P, slot, i == 0 && h == 0)) return;
    int o;
    uint8_t* pan = panel_of(P, slot, h, panel_bytes(D, GRP), o);
    // lanes 8 i .. + 8 = 32 w + 8 a: word w of chunk a; = 32 j + 4 b with b = 2 (i % 4) + (0, 1)
    const int w = i / 4, a = i % 4;
    *reinterpret_cast<uint32_t*>(pan + o * (D / 2) + a * (D / 8) + 4 * w) = kc;
    uint8_t* pv = pan + 8 * D + (o / 2) * D + (2 * a) * (D / 8) + 4 * w + 2 * (o & 1);
    *reinterpret_cast<uint16_t*>(pv) = uint16_t(vc & 0xffffu);
    *reinterpret_cast<uint16_t*>(pv + D / 8) = uint16_t(vc >> 16);
    if (i % G == 0) {
        *reinterpret_cast<uint32_t*>(pan + k_meta_offset(D) + (o * NG + i / G) * 4) = km;
        *reinterpret_cast<uint32_t*>(pan + v_meta_offset(D, GRP) + (o * NG + i / G) * 4) = vm;
    }
}

__device__ __forceinline__ void values8(uint32_t codes, uint32_t meta, float (&x)[8]) {
    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&meta));
    #pragma unroll
    for (int j = 0; j < 8; ++j)                      // a code in the low bits of 2^23 is 2^23 + code
        x[j] = fmaf(__uint_as_float(0x4b000000u | ((codes >> (4 * j)) & 15u)) - 8388608.f, sm.x, sm.y);
}

template <int D, int GRP>
__global__ void __launch_bounds__(kStoreThreads) q4_read_kernel(const StoreParams P) {
    constexpr int TPR = D / 8, G = GRP / 8, NG = D / GRP;
    const int i = threadIdx.x % TPR, w = i / 4, a = i % 4, h = blockIdx.y;
    const int64_t tok = int64_t(blockIdx.x) * (kStoreThreads / TPR) + threadIdx.x / TPR;
    pdl_wait();
    pdl_trigger();
    if (tok >= P.n) return;
    const int64_t slot = P.slots[tok];
    if (!slot_ok(P, slot, i == 0 && h == 0)) return;
    int o;
    const uint8_t* pan = panel_of(P, slot, h, panel_bytes(D, GRP), o);
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(pan + o * (D / 2) + a * (D / 8) + 4 * w);
    const uint8_t* pv = pan + 8 * D + (o / 2) * D + (2 * a) * (D / 8) + 4 * w + 2 * (o & 1);
    const uint32_t vc = uint32_t(*reinterpret_cast<const uint16_t*>(pv)) |
                        (uint32_t(*reinterpret_cast<const uint16_t*>(pv + D / 8)) << 16);
    const uint32_t km = *reinterpret_cast<const uint32_t*>(pan + k_meta_offset(D) + (o * NG + i / G) * 4);
    const uint32_t vm = *reinterpret_cast<const uint32_t*>(pan + v_meta_offset(D, GRP) + (o * NG + i / G) * 4);
    float x[8];
    values8(kc, km, x);
    store8(P.k, P.k_dtype, tok * P.k_stride + h * D + 8 * i, P.k_vec, x);
    values8(vc, vm, x);
    store8(P.v, P.v_dtype, tok * P.v_stride + h * D + 8 * i, P.v_vec, x);
}

int check_store(const ttkv_q4_store_args_t* a) {
    if (!a) return fail(TTKV_ERR_ARG, "4-bit store: null arguments");
    if (int e = check_cache(&a->cache)) return e;
    if (a->n < 0 || (a->n > 0 && (!a->slots || !a->k || !a->v)))
        return fail(TTKV_ERR_ARG, "4-bit store: null pointer or a negative count");
    if (a->k_dtype < TTKV_F32 || a->k_dtype > TTKV_BF16 || a->v_dtype < TTKV_F32 || a->v_dtype > TTKV_BF16)
        return fail(TTKV_ERR_ARG, "4-bit store: K or V type");
    const int64_t row = int64_t(a->cache.H) * a->cache.d;
    if (a->n > 1 && (a->k_stride < row || a->v_stride < row)) return fail(TTKV_ERR_ARG, "4-bit store: token strides below H * d");
    if ((reinterpret_cast<uintptr_t>(a->k) & (a->k_dtype == TTKV_F32 ? 3 : 1)) ||
        (reinterpret_cast<uintptr_t>(a->v) & (a->v_dtype == TTKV_F32 ? 3 : 1)))
        return fail(TTKV_ERR_ALIGN, "4-bit store: K or V not aligned to its type");
    return TTKV_OK;
}

template <bool WRITE>
int launch_store(const ttkv_q4_store_args_t* a) {
    if (int e = check_store(a)) return e;
    if (a->n == 0) return TTKV_OK;
    const ttkv_q4_cache_t* c = &a->cache;
    const int32_t n = a->n;
    int shift = -1;
    for (int b = 0; b < 31; ++b)
        if (c->block_size == (1 << b)) shift = b;
    StoreParams P{c->base, c->n_blocks * c->block_size, c->H, c->block_size, shift, a->slots, n, c->flags & TTKV_CACHE_SKIP_PAD,
                  a->k, a->v, a->k_dtype, a->v_dtype, rows_aligned(a->k, a->k_dtype, a->k_stride),
                  rows_aligned(a->v, a->v_dtype, a->v_stride), a->k_stride, a->v_stride, a->status};
    const int per = kStoreThreads / (c->d / 8), ctas = (n + per - 1) / per;
    // may start while the kernel before it runs, and waits for it before its first access
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(ctas), unsigned(c->H));
    cfg.blockDim = dim3(kStoreThreads);
    cfg.stream = static_cast<cudaStream_t>(a->stream);
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    cudaError_t e = cudaErrorInvalidValue;
#define TTKV_Q4_STORE(D, GRP)                                                                      \
    if (c->d == D && c->group == GRP)                                                              \
        e = cudaLaunchKernelEx(&cfg, WRITE ? q4_write_kernel<D, GRP>               \
                                           : q4_read_kernel<D, GRP>, P);
    TTKV_Q4_STORE(64, 32) TTKV_Q4_STORE(64, 64) TTKV_Q4_STORE(128, 32) TTKV_Q4_STORE(128, 64) TTKV_Q4_STORE(128, 128)
#undef TTKV_Q4_STORE
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(TTKV_ERR_CUDA, "%s: %s", WRITE ? "q4_write_kernel" : "q4_read_kernel", cudaGetErrorString(e));
    }
    return TTKV_OK;
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" size_t ttkv_q4_panel_bytes(int32_t d, int32_t group) {
    return q4::geometry_ok(d, group) ? size_t(q4::panel_bytes(d, group)) : 0;
}

extern "C" int ttkv_q4_write(const ttkv_q4_store_args_t* args) { return launch_store<true>(args); }

extern "C" int ttkv_q4_read(const ttkv_q4_store_args_t* args) { return launch_store<false>(args); }
