// The 4-bit paged cache: quantise and scatter (ttkv_q4_write), gather and dequantise (ttkv_q4_read).
//
// A token of one head moves 4 d bytes of 16-bit K and V and d + 8 d / group packed bytes, each once.
// Consecutive lanes of a warp own a row of a token and head (16 values a lane in the write, 8 of K and 8
// of V in the read-back), so a group's minimum and maximum are shuffles within its lanes, and a lane's
// codes are whole words of the panel (16-bit halves in V's order, which pairs tokens).
//
// 16384 tokens of 8 heads of 128 bf16 lanes, 86 MB: the write takes 27 us (3.2 TB/s), bound by its
// instructions (20 a value, 80 percent of the issue slots), the read-back 21 (4.1 TB/s), against 13 of
// memory. The write in steps: 38 us with 8 values of K and of V a lane, whose group sums and shuffles are
// done twice as often, at 5 CTAs an SM; 31 with 16 values of one of them at 6; 27 to 29 with a kernel a
// type and unaligned loads out of the way. 8 tokens take 4 us, the launch.
#include "ttkv_async.cuh"
#include "ttkv_q4.cuh"

namespace ttkv {
namespace {

using namespace q4;

constexpr int kStoreThreads = 256, kWriteCtas = 6;

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

// The format rounds the scale once from (hi - lo) / 15 and a code once from (x - m) / s. fp32 settles
// both except next to a border between two results: a scale within 3 units of the middle of the 13
// bits that fp16 drops, a few in ten thousand, which is redone in fp64 out of the way; and a code's
// quotient near one half. x inv - m inv is off by 5e-6 and 15 2^-24 |m inv| at most (m inv is rounded);
// within twice that of one half it is settled by the exact remainder x - m - c s: the difference's own
// rounding error is known, and the remainder of a product of 15 bits is exact. Of 16-bit values one in
// a few thousand lies exactly there.
// Of values beyond the limit the ends of the group are clamped, and the quotient as a fraction of 15 by
// its saturation. 16-bit values need no more: next to the limit they are fp16 numbers, so the minimum is
// exact and the limit's own code 15. In fp32 the minimum may be rounded up, as far as the limit, which
// then has a lower code: there the values are clamped too, where the group has such a one.
// A quotient is rounded by adding 1.5 2^23, which leaves the integer in the low bits of the sum, where
// eight of them are packed by shifts and adds (the sum's high bits, the same in every value, are taken
// off at the end).
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

// Minima and maxima of three, NaN if any is.
__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// a b + c of two pairs at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
        " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// The codes of eight values of a group with minimum m and scale s, inv = 1 / (15 s), mi = m inv.
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], float m, float s, float inv, float mi, float border) {
    constexpr float MAGIC = 12582912.f;
    const float2 fifteen = make_float2(15.f, 15.f), magic = make_float2(MAGIC, MAGIC), minus = make_float2(-1.f, -1.f);
    uint32_t codes = 0;
    float near = 0.f;
    #pragma unroll
    for (int j = 6; j >= 0; j -= 2) {
        const float2 t = make_float2(__saturatef(fmaf(x[j], inv, -mi)), __saturatef(fmaf(x[j + 1], inv, -mi)));
        const float2 u = fma2(t, fifteen, magic), r = fma2(t, fifteen, fma2(u, minus, magic));
        asm("max.abs.f32 %0, %0, %1, %2;" : "+f"(near) : "f"(r.x), "f"(r.y));
        codes = (codes * 16u + __float_as_uint(u.y)) * 16u + __float_as_uint(u.x);
    }
    // the high bits 0x4b400000 of the last three values packed; those of the others were shifted out
    codes -= 0x4b400000u + (0x4b400000u << 4) + (0x4b400000u << 8);
    if (near > border) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = __saturatef((x[j] - m) * inv), c = fmaf(t, 15.f, MAGIC) - MAGIC;
            if (fabsf(fmaf(t, 15.f, -c)) > border)
                codes = (codes & ~(15u << (4 * j))) | exact_code(x[j], m, s, c) << (4 * j);
        }
    }
    return codes;
}

// Scale and minimum of a group whose G lanes hold x and y, and the codes of this lane's sixteen.
template <int G, int DT>
__device__ __forceinline__ uint2 quantise_group(float (&x)[8], float (&y)[8], uint32_t& meta) {
    float lo = min_nan(x[0], y[0]), hi = max_nan(x[0], y[0]);
    #pragma unroll
    for (int j = 1; j < 8; ++j) {
        lo = min3(lo, x[j], y[j]);
        hi = max3(hi, x[j], y[j]);
    }
    #pragma unroll
    for (int o = 1; o < G; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const bool nan = !(fmaxf(-lo, hi) < INFINITY && lo == lo);  // a NaN or an infinity in the group
    if (DT == TTKV_F32 && hi > kLimit) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = fminf(x[j], kLimit);
            y[j] = fminf(y[j], kLimit);
        }
    }
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
    const float mi = m * inv, border = fmaf(fabsf(mi), -1.8e-6f, 0.49999f);
    const uint2 c = make_uint2(codes8(x, m, s, inv, mi, border), codes8(y, m, s, inv, mi, border));
    meta = nan ? 0x7e00u : sb | (uint32_t(__half_as_ushort(mh)) << 16);
    return nan ? make_uint2(0u, 0u) : c;
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

// A CTA's rows are consecutive tokens of K (blockIdx.z + first = 0) or V (1) of head blockIdx.y, of type
// DT, D / 16 threads each: two tokens of a pair lie in one warp, whose stores then fill whole sectors.
template <int D, int GRP, int DT>
__global__ void __launch_bounds__(kStoreThreads, kWriteCtas) q4_write_kernel(const StoreParams P, int first) {
    constexpr int TPR = D / 16, G = GRP / 16, NG = D / GRP;
    const int i = threadIdx.x % TPR, h = blockIdx.y;
    const bool is_v = blockIdx.z + first;
    const int64_t row = int64_t(blockIdx.x) * (kStoreThreads / TPR) + threadIdx.x / TPR;
    const int64_t tok = min(row, int64_t(P.n - 1));  // (rows behind the last token load it again and store nothing)
    pdl_wait();
    pdl_trigger();
    const int64_t slot = P.slots[tok];
    const void* src = is_v ? P.v : P.k;
    const bool vec = is_v ? P.v_vec : P.k_vec;
    const int64_t at = tok * (is_v ? P.v_stride : P.k_stride) + h * D + 16 * i;
    float x[8], y[8];
    load8(src, DT, at, vec, x);
    load8(src, DT, at + 8, vec, y);
    uint32_t meta;
    const uint2 c = quantise_group<G, DT>(x, y, meta);
    if (row >= P.n || !slot_ok(P, slot, i == 0 && h == 0 && blockIdx.z == 0)) return;
    int o;
    uint8_t* pan = panel_of(P, slot, h, panel_bytes(D, GRP), o);
    // lanes 16 i .. + 16 = 32 w + 8 a, a = 2 (i % 2) + (0, 1): word w of chunks a; = 32 j + 4 b, b = 4 (i % 2) + (0..3)
    const int w = i / 2, a = i % 2 * 2;
    if (is_v) {
        uint8_t* pv = pan + 8 * D + (o / 2) * D + (2 * a) * (D / 8) + 4 * w + 2 * (o & 1);
        *reinterpret_cast<uint16_t*>(pv) = uint16_t(c.x & 0xffffu);
        *reinterpret_cast<uint16_t*>(pv + D / 8) = uint16_t(c.x >> 16);
        *reinterpret_cast<uint16_t*>(pv + 2 * (D / 8)) = uint16_t(c.y & 0xffffu);
        *reinterpret_cast<uint16_t*>(pv + 3 * (D / 8)) = uint16_t(c.y >> 16);
    } else {
        uint8_t* pk = pan + o * (D / 2) + a * (D / 8) + 4 * w;
        *reinterpret_cast<uint32_t*>(pk) = c.x;
        *reinterpret_cast<uint32_t*>(pk + D / 8) = c.y;
    }
    if (i % G == 0)
        *reinterpret_cast<uint32_t*>(pan + (is_v ? v_meta_offset(D, GRP) : k_meta_offset(D)) + (o * NG + i / G) * 4) = meta;
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

// A launch of `per_row` threads a token and head, that may start while the kernel before it runs and waits for it
// before its first access.
template <typename... KP, typename... A>
cudaError_t launch_rows(void (*kernel)(KP...), const ttkv_q4_store_args_t* a, int per_row, int parts, const A&... args) {
    const int per = kStoreThreads / per_row;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned((a->n + per - 1) / per), unsigned(a->cache.H), unsigned(parts));
    cfg.blockDim = dim3(kStoreThreads);
    cfg.stream = static_cast<cudaStream_t>(a->stream);
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// K and V in one launch where their types agree.
template <int D, int GRP>
cudaError_t launch_write(const ttkv_q4_store_args_t* a, const StoreParams& P) {
    const int parts = P.k_dtype == P.v_dtype ? 2 : 1;
    for (int first = 0; first < 2; first += parts) {
        const int dt = first ? P.v_dtype : P.k_dtype;
        const cudaError_t e = launch_rows(dt == TTKV_BF16  ? q4_write_kernel<D, GRP, TTKV_BF16>
                                          : dt == TTKV_F16 ? q4_write_kernel<D, GRP, TTKV_F16>
                                                           : q4_write_kernel<D, GRP, TTKV_F32>,
                                          a, D / 16, parts, P, first);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

int store(const ttkv_q4_store_args_t* a, bool write) {
    if (int e = check_store(a)) return e;
    if (a->n == 0) return TTKV_OK;
    const ttkv_q4_cache_t* c = &a->cache;
    int shift = -1;
    for (int b = 0; b < 31; ++b)
        if (c->block_size == (1 << b)) shift = b;
    StoreParams P{c->base, c->n_blocks * c->block_size, c->H, c->block_size, shift, a->slots, a->n, c->flags & TTKV_CACHE_SKIP_PAD,
                  a->k, a->v, a->k_dtype, a->v_dtype, rows_aligned(a->k, a->k_dtype, a->k_stride),
                  rows_aligned(a->v, a->v_dtype, a->v_stride), a->k_stride, a->v_stride, a->status};
    cudaError_t e = cudaErrorInvalidValue;
#define TTKV_Q4_STORE(D, GRP)                                                                      \
    if (c->d == D && c->group == GRP)                                                              \
        e = write ? launch_write<D, GRP>(a, P) : launch_rows(q4_read_kernel<D, GRP>, a, D / 8, 1, P);
    TTKV_Q4_STORE(64, 32) TTKV_Q4_STORE(64, 64) TTKV_Q4_STORE(128, 32) TTKV_Q4_STORE(128, 64) TTKV_Q4_STORE(128, 128)
#undef TTKV_Q4_STORE
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(TTKV_ERR_CUDA, "%s: %s", write ? "q4_write_kernel" : "q4_read_kernel", cudaGetErrorString(e));
    }
    return TTKV_OK;
}

}  // namespace
}  // namespace ttkv

using namespace ttkv;

extern "C" size_t ttkv_q4_panel_bytes(int32_t d, int32_t group) {
    return q4::geometry_ok(d, group) ? size_t(q4::panel_bytes(d, group)) : 0;
}

extern "C" int ttkv_q4_write(const ttkv_q4_store_args_t* args) { return store(args, true); }

extern "C" int ttkv_q4_read(const ttkv_q4_store_args_t* args) { return store(args, false); }
