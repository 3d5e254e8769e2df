// The 4-bit paged cache: geometry and device helpers shared by its write, read-back and attention.
#pragma once

#include "ttkv_common.cuh"

namespace ttkv {
namespace q4 {

constexpr int kPanelTokens = 16;    // tokens of a panel: the M of the read's K fragments
constexpr float kLimit = 57344.f;   // stored values are clamped to it: minimum + 15 scales stays a finite fp16

__host__ __device__ constexpr int panel_bytes(int d, int group) { return kPanelTokens * (d + 8 * (d / group)); }
__host__ __device__ constexpr int k_meta_offset(int d) { return kPanelTokens * d; }
__host__ __device__ constexpr int v_meta_offset(int d, int group) { return kPanelTokens * (d + 4 * (d / group)); }

inline bool geometry_ok(int d, int group) {
    return (d == 64 || d == 128) && (group == 32 || group == 64 || group == 128) && group <= d;
}

// Host checks of a cache shared by every 4-bit entry point.
inline int check_cache(const ttkv_q4_cache_t* c) {
    if (!c) return fail(TTKV_ERR_ARG, "null 4-bit cache");
    if (!geometry_ok(c->d, c->group))
        return fail(TTKV_ERR_UNSUPPORTED, "4-bit cache: d=%d with groups of %d (d 64 or 128, groups of 32, 64 or 128 "
                    "lanes, at most d)", c->d, c->group);
    if (c->H < 1 || c->n_blocks < 0 || (c->n_blocks > 0 && !c->base)) return fail(TTKV_ERR_ARG, "4-bit cache: null or empty");
    if (c->H > 65535) return fail(TTKV_ERR_UNSUPPORTED, "4-bit cache: %d KV heads", c->H);
    if (c->block_size < kPanelTokens || c->block_size % kPanelTokens)
        return fail(TTKV_ERR_UNSUPPORTED, "4-bit cache: block size %d is not a multiple of %d", c->block_size, kPanelTokens);
    if (reinterpret_cast<uintptr_t>(c->base) & 15) return fail(TTKV_ERR_ALIGN, "4-bit cache: base not 16-byte aligned");
    return TTKV_OK;
}

// 16 bytes from an address that is no multiple of 16. Out of line: as predicated code in the aligned
// path it cost the write 12 percent more instructions.
static __device__ __noinline__ uint4 load_bytes16(const uint16_t* p) {
    uint32_t w[4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = uint32_t(p[2 * j]) | (uint32_t(p[2 * j + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// (Ordinary loads, here as in the other kernels that start while the one before them runs: what that one
// writes is not constant for this kernel's whole life, which the read-only path supposes.)
// Eight consecutive elements from element index i of p (fp32, fp16 or bf16). vec: p + i is 16-byte aligned.
__device__ __forceinline__ void load8(const void* p, int dtype, int64_t i, bool vec, float (&x)[8]) {
    auto load = [&](int64_t byte) {
        const uint8_t* b = static_cast<const uint8_t*>(p) + byte;
        return vec ? *reinterpret_cast<const uint4*>(b) : load_bytes16(reinterpret_cast<const uint16_t*>(b));
    };
    if (dtype == TTKV_F32) {
        const uint4 a = load(4 * i), b = load(4 * i + 16);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        #pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]);
        return;
    }
    const uint4 u = load(2 * i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (dtype == TTKV_BF16) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int dtype) {
    if (dtype == TTKV_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store8(void* p, int dtype, int64_t i, bool vec, const float (&x)[8]) {
    if (!vec) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) store_elt(p, dtype, i + j, x[j]);
        return;
    }
    if (dtype == TTKV_F32) {
        float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        f[0] = make_float4(x[0], x[1], x[2], x[3]);
        f[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack2(x[0], x[1], dtype), pack2(x[2], x[3], dtype), pack2(x[4], x[5], dtype), pack2(x[6], x[7], dtype));
}

// Whether every row of [n tokens at stride][H * d] elements of a type starts on 16 bytes.
inline bool rows_aligned(const void* p, int dtype, int64_t stride) {
    const int e = dtype == TTKV_F32 ? 4 : 2;
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * e) % 16 == 0;
}

}  // namespace q4
}  // namespace ttkv
