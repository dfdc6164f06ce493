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

// n / d for n below 2^31: (n * mul) >> (31 + shift) with mul = floor(2^(31 + shift) / d) + 1 and 2^shift >= d, whose excess over 2^(31 + shift) / d is
// at most 1, an error of n / 2^(31 + shift) < 2^-shift <= 1 / d.
struct Q8Div {
    uint32_t d, mul, shift;
    Q8Div(uint32_t div) : d(div), shift(0) {
        while ((1ull << shift) < d) shift++;
        mul = (uint32_t)((1ull << (31 + shift)) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> (31 + shift)); }
#endif
};

static inline bool q8_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Head sizes that the cache's kernels are built for.
static inline bool q8_head_dim_ok(uint32_t hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128; }

#ifdef __CUDACC__

// Dynamic shared memory of a kernel, and clusters of 16 CTAs, asked for once on each device (`set`: the kernel's own).
template <typename K>
inline int q8_allow_smem(K* kernel, bool* set, uint32_t bytes, bool wide_clusters = false) {
    int dev = 0;
    AK_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(device_cache_mutex());
    if (!set[dev & 63]) {
        AK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        if (wide_clusters) AK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        set[dev & 63] = true;
    }
    return AK_OK;
}

// A row y is held as q = rint(y f), f = 127 (1 / max|y|), and s = max|y| (1 / 127), every operation rounded to f32. y f is not fused with the rounding to
// an integer: values of bf16 are often half-way between two (y = max|y| / 2 always is), and the error of f alone, up to 2^-23 of it, would decide these
// instead of "half to even" (in 1200 Gaussian bf16 rows of 4096 values 2717 integers of 4.9 million were a step off 127 y / max|y|, 907 are like this).
// `top` is max|y| as the bits of a non-negative float: ordered as
// unsigned integers these put infinity above every finite value and NaN above infinity, so that neither is lost in a maximum.
// Rows whose largest value is under Q8_ZERO are zeros, s = 0; a row with an infinity or a NaN has s = NaN
// and q = 0, so that whatever is computed from it is NaN and nothing else is.
constexpr float Q8_ZERO = 1e-30f;
// f for top from 1e-37 on: the quarter keeps the reciprocal of the largest values out of the subnormal numbers.
__device__ __forceinline__ float q8_inv(float top) { return __fmul_rn(__frcp_rn(top * 0.25f), 31.75f); }
__device__ __forceinline__ void q8_scale(uint32_t top_bits, float& inv, float& s) {
    const float top = __uint_as_float(top_bits);
    inv = q8_inv(top);
    s = top * (1.0f / 127.0f);   // the constant is off by 2^-28 of its value
    if (top < Q8_ZERO) { inv = 0.0f; s = 0.0f; }
    if (top_bits >= 0x7f800000u) { inv = 0.0f; s = __uint_as_float(0x7fc00000u); }
}
// Two values times `inv` (both halves), each rounded, and the integers nearest to the products in the low bits: adding 1.5 * 2^23 leaves them there.
// mul.rn.f32x2 and an addition behind it are made one fused operation by the assembler, and so is a product that adds a constant -0; `none`, -0 that it
// does not know, keeps the two roundings.
__device__ __forceinline__ void q8_int2(float a, float b, uint64_t inv, uint64_t none, uint32_t& ia, uint32_t& ib) {
    asm("{\n"
        ".reg .b64 t;\n"
        "mov.b64 t, {%2, %3};\n"
        "fma.rn.f32x2 t, t, %4, %5;\n"
        "add.rn.f32x2 t, t, %6;\n"
        "mov.b64 {%0, %1}, t;\n"
        "}\n" : "=r"(ia), "=r"(ib) : "f"(a), "f"(b), "l"(inv), "l"(none), "l"(0x4b4000004b400000ull));
}
// The four integers nearest to y inv, |y inv| <= 127 (1 + 2^-22), as bytes. A value that is not finite (times inv = 0) would leave any bits there:
// `ok` = the row's scale is a number.
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d, float inv, bool ok) {
    uint64_t two, none;
    asm("mov.b64 %0, {%1, %1};" : "=l"(two) : "f"(inv));
    asm("mov.b64 %0, {%1, %1};" : "=l"(none) : "f"(inv * -0.0f));
    uint32_t ia, ib, ic, id;
    q8_int2(a, b, two, none, ia, ib);
    q8_int2(c, d, two, none, ic, id);
    const uint32_t v = __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
    return ok ? v : 0u;
}
__device__ __forceinline__ int8_t q8_of(float y, float inv, bool ok) { return ok ? (int8_t)__float2int_rn(__fmul_rn(y, inv)) : (int8_t)0; }
__device__ __forceinline__ bool q8_aligned_dev(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

#endif
}  // namespace ak
