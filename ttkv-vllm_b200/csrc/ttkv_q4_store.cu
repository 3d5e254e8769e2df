// The 4-bit paged cache: quantise and scatter (ttkv_q4_write), gather and dequantise (ttkv_q4_read).
//
// Bound: memory. A token of one head moves 4 d bytes of 16-bit K and V and d + 8 d / group packed
// bytes, each once. d / 8 consecutive lanes of a warp own a (token, head) row, eight values a lane
// (one 16-byte load of each 16-bit row): the group's minimum and maximum are shuffles within the
// group's lanes, and a lane's eight K codes are one 32-bit word of the panel, its V codes two 16-bit
// ones (the V order pairs tokens, so a lone token's bytes lie apart).
#include "ttkv_q4.cuh"

namespace ttkv {
namespace {

using namespace q4;

constexpr int kStoreThreads = 256;

struct StoreParams {
    uint8_t* cache;
    int64_t n_slots;
    int32_t H, block_size;
    const int64_t* slots;
    int32_t n, skip_pad;
    void* k;
    void* v;
    int32_t k_dtype, v_dtype, k_vec, v_vec;
    int64_t k_stride, v_stride;
    int32_t* status;
};

// Scale and minimum of a group whose lanes hold x (already clamped), and the codes of this lane's
// eight. G lanes per group.
//
// The format rounds the scale once from (hi - lo) / 15 and a code once from (x - m) / s. fp32 settles
// both except next to a border between two results (a scale within 2 units of the 13 bits that fp16
// drops from the middle, a code's quotient within 1e-4 of one half, both a few in ten thousand),
// which are redone in fp64.
template <int G>
__device__ __forceinline__ uint32_t quantise_group(float (&x)[8], uint32_t& meta) {
    float lo = x[0], hi = x[0];
    bool fine = true;
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        fine &= fabsf(x[j]) < INFINITY;
        x[j] = fminf(fmaxf(x[j], -kLimit), kLimit);
        lo = j ? fminf(lo, x[j]) : x[j];
        hi = j ? fmaxf(hi, x[j]) : x[j];
    }
    #pragma unroll
    for (int o = 1; o < G; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    unsigned bad = __ballot_sync(0xffffffffu, !fine);
    bad &= (G == 32 ? 0xffffffffu : ((1u << G) - 1u)) << (threadIdx.x & 31 & ~(G - 1));

    const __half mh = __float2half_rn(lo + 0.f);              // -0 is stored as 0
    const float m = __half2float(mh);
    const float q = __fdiv_rn(hi - lo, 15.f);
    const uint32_t low = __float_as_uint(q) & 0x1fffu;
    __half sh = __float2half_rn(q);
    if (q < 6.2e-5f || (low >= 0xffeu && low <= 0x1002u)) {
        // round to odd in fp32 first: its 13 extra bits then decide the fp16 rounding exactly
        const double e = __ddiv_rn(double(hi) - double(lo), 15.0);
        float f = __double2float_rz(e);
        if (double(f) != e) f = __uint_as_float(__float_as_uint(f) | 1u);
        sh = __float2half_rn(f);
    }
    const float s = __half2float(sh);
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t codes = 0;
    float near = 0.f;
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = (x[j] - m) * inv;
        const float c = rintf(t);
        near = fmaxf(near, fabsf(t - c));
        codes |= uint32_t(fminf(fmaxf(c, 0.f), 15.f)) << (4 * j);
    }
    if (near > 0.4999f && s > 0.f) {
        codes = 0;
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double c = rint(__ddiv_rn(double(x[j]) - double(m), double(s)));
            codes |= uint32_t(fmin(fmax(c, 0.0), 15.0)) << (4 * j);
        }
    }
    if (bad) codes = 0;
    const uint32_t sb = bad ? 0x7e00u : uint32_t(__half_as_ushort(sh)), mb = bad ? 0u : uint32_t(__half_as_ushort(mh));
    meta = sb | (mb << 16);
    return codes;
}

__device__ __forceinline__ bool slot_ok(const StoreParams& P, int64_t slot, bool first) {
    if (slot >= 0 && slot < P.n_slots) return true;
    if (first && !(slot < 0 && P.skip_pad)) report(P.status, TTKV_STATUS_SLOT_RANGE);
    return false;
}

template <int D, int GRP>
__global__ void __launch_bounds__(kStoreThreads) q4_write_kernel(const StoreParams P) {
    constexpr int TPR = D / 8, G = GRP / 8, NG = D / GRP;
    const int64_t row = (int64_t(blockIdx.x) * kStoreThreads + threadIdx.x) / TPR;
    const int i = threadIdx.x % TPR;
    const int64_t tok = row / P.H;
    const int h = int(row - tok * P.H);
    const bool live = tok < P.n;
    const int64_t slot = live ? P.slots[tok] : -1;
    const bool ok = live && slot_ok(P, slot, i == 0 && h == 0);
    float x[8] = {}, y[8] = {};
    if (ok) {                                        // the warp's shuffles below take every lane
        load8(P.k, P.k_dtype, tok * P.k_stride + h * D + 8 * i, P.k_vec, x);
        load8(P.v, P.v_dtype, tok * P.v_stride + h * D + 8 * i, P.v_vec, y);
    }
    uint32_t km, vm;
    const uint32_t kc = quantise_group<G>(x, km), vc = quantise_group<G>(y, vm);
    if (!ok) return;
    const int64_t blk = slot / P.block_size;
    const int off = int(slot - blk * P.block_size), o = off % kPanelTokens;
    uint8_t* pan = P.cache + ((blk * P.H + h) * (P.block_size / kPanelTokens) + off / kPanelTokens) * panel_bytes(D, GRP);
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
    for (int j = 0; j < 8; ++j) x[j] = fmaf(float((codes >> (4 * j)) & 15u), sm.x, sm.y);
}

template <int D, int GRP>
__global__ void __launch_bounds__(kStoreThreads) q4_read_kernel(const StoreParams P) {
    constexpr int TPR = D / 8, G = GRP / 8, NG = D / GRP;
    const int64_t row = (int64_t(blockIdx.x) * kStoreThreads + threadIdx.x) / TPR;
    const int i = threadIdx.x % TPR;
    const int64_t tok = row / P.H;
    const int h = int(row - tok * P.H);
    if (tok >= P.n) return;
    const int64_t slot = P.slots[tok];
    if (!slot_ok(P, slot, i == 0 && h == 0)) return;
    const int64_t blk = slot / P.block_size;
    const int off = int(slot - blk * P.block_size), o = off % kPanelTokens;
    const uint8_t* pan = P.cache + ((blk * P.H + h) * (P.block_size / kPanelTokens) + off / kPanelTokens) * panel_bytes(D, GRP);
    const int w = i / 4, a = i % 4;
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

int check_store(const ttkv_q4_cache_t* c, const int64_t* slots, int32_t n, const void* k, int32_t k_dtype,
                int64_t k_stride, const void* v, int32_t v_dtype, int64_t v_stride) {
    if (int e = check_cache(c)) return e;
    if (n < 0 || (n > 0 && (!slots || !k || !v))) return fail(TTKV_ERR_ARG, "4-bit store: null pointer or a negative count");
    if (k_dtype < TTKV_F32 || k_dtype > TTKV_BF16 || v_dtype < TTKV_F32 || v_dtype > TTKV_BF16)
        return fail(TTKV_ERR_ARG, "4-bit store: K or V type");
    const int64_t row = int64_t(c->H) * c->d;
    if (n > 1 && (k_stride < row || v_stride < row)) return fail(TTKV_ERR_ARG, "4-bit store: token strides below H * d");
    if ((reinterpret_cast<uintptr_t>(k) & (k_dtype == TTKV_F32 ? 3 : 1)) ||
        (reinterpret_cast<uintptr_t>(v) & (v_dtype == TTKV_F32 ? 3 : 1)))
        return fail(TTKV_ERR_ALIGN, "4-bit store: K or V not aligned to its type");
    return TTKV_OK;
}

template <bool WRITE>
int launch_store(const ttkv_q4_cache_t* c, const int64_t* slots, int32_t n, void* k, int32_t k_dtype,
                 int64_t k_stride, void* v, int32_t v_dtype, int64_t v_stride, int32_t* status, void* stream) {
    if (int e = check_store(c, slots, n, k, k_dtype, k_stride, v, v_dtype, v_stride)) return e;
    if (n == 0) return TTKV_OK;
    StoreParams P{c->base, c->n_blocks * c->block_size, c->H, c->block_size, slots, n, c->flags & TTKV_CACHE_SKIP_PAD,
                  k, v, k_dtype, v_dtype, rows_aligned(k, k_dtype, k_stride), rows_aligned(v, v_dtype, v_stride),
                  k_stride, v_stride, status};
    const int64_t threads = int64_t(n) * c->H * (c->d / 8);
    const int64_t ctas = (threads + kStoreThreads - 1) / kStoreThreads;
    if (ctas > 0x7fffffff) return fail(TTKV_ERR_UNSUPPORTED, "4-bit store: %d tokens of %d heads in one call", n, c->H);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define TTKV_Q4_STORE(D, GRP)                                                                      \
    if (c->d == D && c->group == GRP) {                                                            \
        if (WRITE) q4_write_kernel<D, GRP><<<unsigned(ctas), kStoreThreads, 0, st>>>(P);           \
        else q4_read_kernel<D, GRP><<<unsigned(ctas), kStoreThreads, 0, st>>>(P);                  \
    }
    TTKV_Q4_STORE(64, 32) TTKV_Q4_STORE(64, 64) TTKV_Q4_STORE(128, 32) TTKV_Q4_STORE(128, 64) TTKV_Q4_STORE(128, 128)
#undef TTKV_Q4_STORE
    return check_launch(WRITE ? "q4_write_kernel" : "q4_read_kernel");
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" size_t ttkv_q4_panel_bytes(int32_t d, int32_t group) {
    return q4::geometry_ok(d, group) ? size_t(q4::panel_bytes(d, group)) : 0;
}

extern "C" int ttkv_q4_write(const ttkv_q4_cache_t* cache, const int64_t* slots, int32_t n, const void* k,
                             int32_t k_dtype, int64_t k_stride, const void* v, int32_t v_dtype, int64_t v_stride,
                             int32_t* status, void* stream) {
    return launch_store<true>(cache, slots, n, const_cast<void*>(k), k_dtype, k_stride, const_cast<void*>(v), v_dtype,
                              v_stride, status, stream);
}

extern "C" int ttkv_q4_read(const ttkv_q4_cache_t* cache, const int64_t* slots, int32_t n, void* k, int32_t k_dtype,
                            int64_t k_stride, void* v, int32_t v_dtype, int64_t v_stride, int32_t* status, void* stream) {
    return launch_store<false>(cache, slots, n, k, k_dtype, k_stride, v, v_dtype, v_stride, status, stream);
}
