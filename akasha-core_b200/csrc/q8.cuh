// What the 8-bit operators share: the row quantisation, the alignment and device checks of their entry points.
#pragma once
#include "common.cuh"

namespace ak {

constexpr uint32_t Q8_BS = 16;   // positions per cache block

// AK_OK if `p` is memory that the current device's kernels may be given: its own, managed or mapped host memory. A pointer into another
// device or into pageable host memory would fault in the kernel.
int q8_check_here(const void* p, const char* who);

// AK_OK if these describe a cache that the kernels know, with its pools and scales in place.
int q8_check_cache(const char* who, const void* k_pool, const void* v_pool, const void* k_scales, const void* v_scales, uint32_t heads, uint32_t kv_heads,
                   uint32_t head_dim, uint32_t block_size, uint32_t dtype, uint32_t pool_blocks);

static inline bool q8_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Head sizes that the cache's kernels are built for.
static inline bool q8_head_dim_ok(uint32_t hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128; }

#ifdef __CUDACC__

// A row y is held as q = rint(127 y / max|y|) and s = max|y| / 127. `top` is max|y| as the bits of a non-negative float: ordered as
// unsigned integers these put infinity above every finite value and NaN above infinity, so that neither is lost in a maximum.
// Rows whose largest value is under Q8_ZERO (127 / max would overflow) are zeros, s = 0; a row with an infinity or a NaN has s = NaN
// and q = 0, so that whatever is computed from it is NaN and nothing else is.
constexpr float Q8_ZERO = 1e-30f;
__device__ __forceinline__ void q8_scale(uint32_t top_bits, float& inv, float& s) {
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) { inv = 0.0f; s = __uint_as_float(0x7fc00000u); }
    else if (top < Q8_ZERO) { inv = 0.0f; s = 0.0f; }
    else { inv = 127.0f / top; s = top / 127.0f; }
}
// |y inv| <= 127 (1 + 2^-23): the nearest integer never leaves -127..127. (inv = 0: infinity times 0 is NaN, which converts to 0.)
__device__ __forceinline__ uint32_t q8_of(float y, float inv) { return (uint32_t)__float2int_rn(y * inv) & 0xffu; }
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d, float inv) {
    return q8_of(a, inv) | (q8_of(b, inv) << 8) | (q8_of(c, inv) << 16) | (q8_of(d, inv) << 24);
}
__device__ __forceinline__ bool q8_aligned_dev(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

#endif
}  // namespace ak
