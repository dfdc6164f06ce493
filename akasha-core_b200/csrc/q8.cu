// The row-wise 8-bit operators: RMS norm (or the plain rows) quantised per token, the cache append that rotates and quantises as it
// writes, and reading cached rows back. All are bound by HBM.
#include "q8.cuh"
#include "kernels.h"

namespace ak {

int q8_check_here(const void* p, const char* who) {
    cudaPointerAttributes at{};
    int dev = 0;
    AK_CUDA(cudaGetDevice(&dev));
    AK_CUDA(cudaPointerGetAttributes(&at, p));
    AK_REQUIRE(at.type != cudaMemoryTypeUnregistered, AK_ERR_INVALID_ARG, "%s: %p is not memory that the device can read", who, p);
    AK_REQUIRE(at.type != cudaMemoryTypeDevice || at.device == dev, AK_ERR_INVALID_ARG, "%s: %p is memory of device %d, the current device is %d", who, p,
               at.device, dev);
    return AK_OK;
}

// ============================================================================ norm + quantisation
// h = x (+ residual, written back), y = h / sqrt(mean(h^2) + eps) * w (w == nullptr: y = h), q = rint(127 y / max|y|), s = max|y| / 127.
// One pass: a row lives in the registers of its threads between the two reductions (sum of squares, largest magnitude), so that every
// input byte is read once and every output byte written once. `tpr` threads share a row, each holding NV groups of 4 consecutive values.
//
// RAG: size % 4 != 0. All the arrays of a row start at the same element offset, so groups are cut where the ADDRESS is a multiple of 4
// elements: the first and last group of a row are partial (element by element), all others are whole vectors.
template <typename T> struct Q8Vec;
template <> struct Q8Vec<float> {
    static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    }
};
template <> struct Q8Vec<bf16> {
    static __device__ __forceinline__ void load(const bf16* p, float (&v)[4]) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
        v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
    }
};

constexpr uint32_t NQ_MAX_WARPS = 32;

template <typename T, bool RAG, int NV>
__global__ void __launch_bounds__(1024)
norm_q8_kernel(T* __restrict__ x, const float* __restrict__ residual, const float* __restrict__ w, int8_t* __restrict__ q, float* __restrict__ scales,
               uint32_t rows, uint32_t size, float eps, uint32_t w_vec) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s_sum[NQ_MAX_WARPS];
    __shared__ uint32_t s_top[NQ_MAX_WARPS];
    const uint32_t tpr = blockDim.x, t = threadIdx.x, lane = t & 31, wid = t >> 5, warps = tpr >> 5;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;   // blockDim.y > 1 only with one warp per row
    if (row >= rows) return;
    const size_t off = (size_t)row * size;
    const uint32_t shift = RAG ? (uint32_t)(off & 3) : 0;
    const uint32_t groups = (shift + size + 3) >> 2;
    float v[NV][4];
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const uint32_t g = t + c * tpr;
        v[c][0] = v[c][1] = v[c][2] = v[c][3] = 0.0f;
        if (g >= groups) continue;
        const int32_t e0 = (int32_t)(4 * g - shift);
        if (!RAG || (e0 >= 0 && (uint32_t)e0 + 4 <= size)) {
            T* xp = x + off + e0;
            Q8Vec<T>::load(xp, v[c]);
            if constexpr (sizeof(T) == 4) {
                if (residual) {
                    float r[4];
                    Q8Vec<float>::load(residual + off + e0, r);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[c][e] += r[e];
                    *reinterpret_cast<float4*>(xp) = make_float4(v[c][0], v[c][1], v[c][2], v[c][3]);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int32_t i = e0 + e;
                if (i < 0 || (uint32_t)i >= size) continue;
                v[c][e] = Cvt<T>::to_f(x[off + i]);
                if constexpr (sizeof(T) == 4) {
                    if (residual) { v[c][e] += residual[off + i]; x[off + i] = v[c][e]; }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) ss += v[c][e] * v[c][e];
    }
    if (w) {
        ss = warp_sum(ss);
        if (warps > 1) {
            if (lane == 0) s_sum[wid] = ss;
            __syncthreads();
            ss = warp_sum(lane < warps ? s_sum[lane] : 0.0f);   // the same order in every warp
        }
        const float rs = 1.0f / sqrtf(ss / (float)size + eps);
#pragma unroll
        for (int c = 0; c < NV; c++) {
            const uint32_t g = t + c * tpr;
            if (g >= groups) continue;
            const int32_t e0 = (int32_t)(4 * g - shift);
            if (w_vec && (!RAG || (shift == 0 && (uint32_t)e0 + 4 <= size))) {
                float ww[4];
                Q8Vec<float>::load(w + e0, ww);
#pragma unroll
                for (int e = 0; e < 4; e++) v[c][e] = v[c][e] * rs * ww[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (e0 + e >= 0 && (uint32_t)(e0 + e) < size) v[c][e] = v[c][e] * rs * w[e0 + e];
            }
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < NV; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, abs_bits(v[c][e]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (warps > 1) {
        if (lane == 0) s_top[wid] = top;
        __syncthreads();
        top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
    }
    float inv, s;
    q8_scale(top, inv, s);
    if (t == 0) scales[row] = s;
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const uint32_t g = t + c * tpr;
        if (g >= groups) continue;
        const int32_t e0 = (int32_t)(4 * g - shift);
        if (!RAG || (e0 >= 0 && (uint32_t)e0 + 4 <= size)) {
            *reinterpret_cast<uint32_t*>(q + off + e0) = q8_pack4(v[c][0], v[c][1], v[c][2], v[c][3], inv);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e0 + e >= 0 && (uint32_t)(e0 + e) < size) q[off + e0 + e] = (int8_t)q8_of(v[c][e], inv);
        }
    }
}

// Rows that do not fit the registers of a block (over 32768 values), and buffers that are not aligned for vectors: a block per row, three
// passes over it (the second and third read what the first wrote back). y is computed twice by the same operations, hence with the same bits.
template <typename T>
__global__ void __launch_bounds__(1024)
norm_q8_any_kernel(T* x, const float* residual, const float* __restrict__ w, int8_t* __restrict__ q, float* __restrict__ scales, uint32_t size, float eps) {
    pdl_wait();
    pdl_trigger();
    __shared__ float s_sum[NQ_MAX_WARPS];
    __shared__ uint32_t s_top[NQ_MAX_WARPS];
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const size_t off = (size_t)blockIdx.x * size;
    float ss = 0.0f;
    for (uint32_t i = threadIdx.x; i < size; i += blockDim.x) {
        float v = Cvt<T>::to_f(x[off + i]);
        if constexpr (sizeof(T) == 4) {
            if (residual) { v += residual[off + i]; x[off + i] = v; }
        }
        ss += v * v;
    }
    float rs = 1.0f;
    if (w) {
        ss = warp_sum(ss);
        if (lane == 0) s_sum[wid] = ss;
        __syncthreads();
        ss = warp_sum(lane < warps ? s_sum[lane] : 0.0f);
        rs = 1.0f / sqrtf(ss / (float)size + eps);
    }
    auto value = [&](uint32_t i) { return w ? Cvt<T>::to_f(x[off + i]) * rs * w[i] : Cvt<T>::to_f(x[off + i]); };   // written by this thread
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x; i < size; i += blockDim.x) top = max(top, abs_bits(value(i)));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[wid] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
    float inv, s;
    q8_scale(top, inv, s);
    if (threadIdx.x == 0) scales[blockIdx.x] = s;
    for (uint32_t i = threadIdx.x; i < size; i += blockDim.x) q[off + i] = (int8_t)q8_of(value(i), inv);
}

template <typename T, bool RAG, int NV>
static int norm_q8_launch(cudaStream_t st, T* x, const float* residual, const float* w, int8_t* q, float* scales, uint32_t rows, uint32_t size, float eps,
                          uint32_t tpr) {
    const uint32_t rpb = tpr == 32 ? 4 : 1;
    return launch_k(norm_q8_kernel<T, RAG, NV>, dim3(cdiv(rows, rpb)), dim3(tpr, rpb), 0, st, NO_CLUSTER, x, residual, w, q, scales, rows, size, eps,
                    (uint32_t)q8_aligned(w, 16));
}

template <typename T>
static int norm_q8(cudaStream_t st, T* x, const float* residual, const float* w, int8_t* q, float* scales, uint32_t rows, uint32_t size, float eps) {
    const uint32_t groups = (size + 3) / 4 + (size % 4 ? 1 : 0);   // of a row, at most
    if (groups > 8192 || !q8_aligned(x, 4 * sizeof(T)) || !q8_aligned(residual, 16) || !q8_aligned(q, 4))
        return launch_k(norm_q8_any_kernel<T>, dim3(rows), dim3(512), 0, st, NO_CLUSTER, x, residual, w, q, scales, size, eps);
    uint32_t nv = 1;
    if (rows > 2 * B200_SMS) nv = groups <= 64 ? 2 : (groups <= 1024 ? 4 : 8);
    while (groups > nv * 1024) nv *= 2;
    const uint32_t tpr = cdiv(groups, nv * 32) * 32;
#define AK_NORM_Q8(NV)                                                                                     \
    return size % 4 ? norm_q8_launch<T, true, NV>(st, x, residual, w, q, scales, rows, size, eps, tpr)    \
                    : norm_q8_launch<T, false, NV>(st, x, residual, w, q, scales, rows, size, eps, tpr)
    switch (nv) {
        case 1: AK_NORM_Q8(1);
        case 2: AK_NORM_Q8(2);
        case 4: AK_NORM_Q8(4);
        default: AK_NORM_Q8(8);
    }
#undef AK_NORM_Q8
}

// ============================================================================ split + RoPE + quantised append
// qkv row of a token: `heads` query heads, kv_heads key heads, kv_heads value heads. A group of HD / 4 lanes (HD = 96: 24 of 32) takes one
// head: one float4 per lane, its two pairs rotated, the largest magnitude of the head by shuffles inside the group, 4 bytes out.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
rope_kv_append_q8_kernel(const float* __restrict__ qkv, const float4* __restrict__ rope, uint32_t rope_len, const int32_t* __restrict__ positions,
                         const int32_t* __restrict__ slots, T* __restrict__ q_out, int8_t* __restrict__ k_pool, int8_t* __restrict__ v_pool,
                         float* __restrict__ k_scales, float* __restrict__ v_scales, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t pool_slots) {
    constexpr uint32_t LANES = HD / 4, GROUP = HD == 96 ? 32 : LANES;   // lanes at work / lanes set aside for a head
    pdl_wait();
    pdl_trigger();
    const uint32_t total_heads = heads + 2 * kv_heads;
    const uint64_t item = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) / GROUP;
    const uint32_t l = threadIdx.x % GROUP;
    const uint32_t t = (uint32_t)(item / total_heads), h = (uint32_t)(item % total_heads);
    const bool on = t < tokens && l < LANES;
    int32_t pos = -1, slot = -1;
    if (on) { pos = positions[t]; slot = slots[t]; }
    const bool live = on && (uint32_t)pos < rope_len;   // a token at another position is left out
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        x = *reinterpret_cast<const float4*>(qkv + ((uint64_t)t * total_heads + h) * HD + 4 * l);
        if (h < heads + kv_heads) {
            const float4 f = rope[(uint64_t)pos * (HD / 4) + l];   // (cos, sin) of pairs 2l and 2l + 1
            rope_rotate(x.x, x.y, f.x, f.y, x.x, x.y);
            rope_rotate(x.z, x.w, f.z, f.w, x.z, x.w);
        }
    }
    uint32_t top = max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w)));
#pragma unroll
    for (uint32_t o = GROUP / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) return;
    if (h < heads) {
        T* dst = q_out + ((uint64_t)t * heads + h) * HD + 4 * l;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(dst) = x;
        } else {
            const bf162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
            *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
        return;
    }
    if ((uint32_t)slot >= pool_slots) return;   // not cached
    const bool is_v = h >= heads + kv_heads;
    const uint32_t kh = h - heads - (is_v ? kv_heads : 0);
    const uint64_t at = ((uint64_t)((uint32_t)slot / Q8_BS) * kv_heads + kh) * Q8_BS + (uint32_t)slot % Q8_BS;
    float inv, s;
    q8_scale(top, inv, s);
    *reinterpret_cast<uint32_t*>((is_v ? v_pool : k_pool) + at * HD + 4 * l) = q8_pack4(x.x, x.y, x.z, x.w, inv);
    if (l == 0) (is_v ? v_scales : k_scales)[at] = s;
}

// ============================================================================ cached rows as numbers
// A thread takes 16 bytes of output (VEC values) of the key row and of the value row of one (token, head).
template <typename T>
__global__ void __launch_bounds__(256)
kv_read_q8_kernel(const int8_t* __restrict__ k_pool, const int8_t* __restrict__ v_pool, const float* __restrict__ k_scales, const float* __restrict__ v_scales,
                  const int32_t* __restrict__ slots, T* __restrict__ k_out, T* __restrict__ v_out, uint32_t tokens, uint32_t kv_heads, uint32_t hd,
                  uint32_t pool_slots) {
    constexpr uint32_t VEC = 16 / sizeof(T);
    pdl_wait();
    pdl_trigger();
    const uint32_t chunks = hd / VEC;
    const uint64_t idx = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= (uint64_t)tokens * kv_heads * chunks) return;
    const uint32_t c = (uint32_t)(idx % chunks);
    const uint64_t th = idx / chunks;
    const uint32_t h = (uint32_t)(th % kv_heads), t = (uint32_t)(th / kv_heads);
    const uint32_t slot = (uint32_t)slots[t];
    const bool have = slot < pool_slots;
    const uint64_t at = have ? ((uint64_t)(slot / Q8_BS) * kv_heads + h) * Q8_BS + slot % Q8_BS : 0;
#pragma unroll
    for (int side = 0; side < 2; side++) {
        T* out = side ? v_out : k_out;
        if (!out) continue;
        alignas(16) T o[VEC];
        uint32_t words[VEC / 4];
        float s = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < VEC / 4; i++) words[i] = 0;
        if (have) {
            const int8_t* src = (side ? v_pool : k_pool) + at * hd + c * VEC;
            s = (side ? v_scales : k_scales)[at];
            if constexpr (VEC == 8) {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                words[0] = u.x; words[1] = u.y;
            } else {
                words[0] = *reinterpret_cast<const uint32_t*>(src);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < VEC; i++) o[i] = Cvt<T>::from_f((float)(int8_t)(words[i / 4] >> (8 * (i % 4))) * s);
        *reinterpret_cast<uint4*>(out + idx * VEC) = *reinterpret_cast<const uint4*>(o);
    }
}

template <typename T, int HD>
static int append_q8(cudaStream_t st, const float* qkv, const float* rope, uint32_t rope_len, const int32_t* positions, const int32_t* slots, void* q_out,
                     int8_t* k_pool, int8_t* v_pool, float* k_scales, float* v_scales, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t pool_slots) {
    constexpr uint32_t GROUP = HD == 96 ? 32 : HD / 4;
    const uint64_t threads = (uint64_t)tokens * (heads + 2 * kv_heads) * GROUP;
    AK_REQUIRE(cdiv64(threads, 256) <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "ak_rope_kv_append_q8: %u tokens x %u heads are too many for one call", tokens,
               heads + 2 * kv_heads);
    return launch_k(rope_kv_append_q8_kernel<T, HD>, dim3((unsigned)cdiv64(threads, 256)), dim3(256), 0, st, NO_CLUSTER, qkv,
                    reinterpret_cast<const float4*>(rope), rope_len, positions, slots, (T*)q_out, k_pool, v_pool, k_scales, v_scales, tokens, heads, kv_heads,
                    pool_slots);
}

// The cache's own numbers, checked alike by everything that touches it.
int q8_check_cache(const char* who, const void* k_pool, const void* v_pool, const void* k_scales, const void* v_scales, uint32_t heads, uint32_t kv_heads,
                   uint32_t head_dim, uint32_t block_size, uint32_t dtype, uint32_t pool_blocks) {
    AK_REQUIRE(k_pool && v_pool && k_scales && v_scales, AK_ERR_INVALID_ARG, "%s: null pointer", who);
    AK_REQUIRE(dtype <= AK_BF16, AK_ERR_INVALID_ARG, "%s: dtype must be f32 or bf16", who);
    AK_REQUIRE(block_size == Q8_BS, AK_ERR_UNSUPPORTED, "%s: block_size must be 16", who);
    AK_REQUIRE(q8_head_dim_ok(head_dim), AK_ERR_UNSUPPORTED, "%s: head_dim must be 32, 64, 96 or 128 (got %u)", who, head_dim);
    AK_REQUIRE(kv_heads >= 1 && heads % kv_heads == 0 && heads >= kv_heads && heads <= 65536, AK_ERR_INVALID_ARG,
               "%s: heads (%u) must be a positive multiple of kv_heads (%u), at most 65536", who, heads, kv_heads);
    AK_REQUIRE(pool_blocks >= 1 && pool_blocks <= (1u << 27), AK_ERR_INVALID_ARG, "%s: pool_blocks must be 1 to 2^27 (got %u)", who, pool_blocks);
    AK_REQUIRE(q8_aligned(k_pool, 16) && q8_aligned(v_pool, 16) && q8_aligned(k_scales, 16) && q8_aligned(v_scales, 16), AK_ERR_INVALID_ARG,
               "%s: pools and scales must be 16-byte aligned", who);
    return AK_OK;
}

}  // namespace ak

using namespace ak;
extern "C" {

int ak_rmsnorm_q8(void* stream, void* x, uint32_t in_dtype, const float* residual, const float* w, int8_t* q, float* scales, ak_norm_meta m) {
    AK_REQUIRE(x && q && scales, AK_ERR_INVALID_ARG, "ak_rmsnorm_q8: null pointer");
    AK_REQUIRE(in_dtype <= AK_BF16, AK_ERR_INVALID_ARG, "ak_rmsnorm_q8: in_dtype must be f32 or bf16");
    AK_REQUIRE(!residual || in_dtype == AK_F32, AK_ERR_INVALID_ARG, "ak_rmsnorm_q8: a residual is added to f32 rows only");
    AK_REQUIRE(q8_aligned(x, in_dtype == AK_F32 ? 4 : 2) && q8_aligned(residual, 4) && q8_aligned(w, 4) && q8_aligned(scales, 4), AK_ERR_INVALID_ARG,
               "ak_rmsnorm_q8: a pointer is not aligned to its elements");
    AK_REQUIRE(m.size <= 0x7ffffff0u && m.seq_len <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "ak_rmsnorm_q8: %u rows of %u values are too large", m.seq_len, m.size);
    if (m.seq_len == 0 || m.size == 0) return AK_OK;
    AK_TRY(q8_check_here(q, "ak_rmsnorm_q8"));
    if (in_dtype == AK_F32) return norm_q8<float>(as_stream(stream), (float*)x, residual, w, q, scales, m.seq_len, m.size, m.eps);
    return norm_q8<bf16>(as_stream(stream), (bf16*)x, nullptr, w, q, scales, m.seq_len, m.size, m.eps);
}

int ak_rope_kv_append_q8(void* stream, const float* qkv, const float* rope_table, uint32_t rope_len, const int32_t* positions, const int32_t* slots, void* q_out,
                         int8_t* k_pool, int8_t* v_pool, float* k_scales, float* v_scales, uint32_t tokens, uint32_t heads, uint32_t kv_heads,
                         uint32_t head_dim, uint32_t block_size, uint32_t q_dtype, uint32_t pool_blocks) {
    const char* who = "ak_rope_kv_append_q8";
    AK_REQUIRE(qkv && rope_table && positions && slots && q_out, AK_ERR_INVALID_ARG, "%s: null pointer", who);
    AK_TRY(q8_check_cache(who, k_pool, v_pool, k_scales, v_scales, heads, kv_heads, head_dim, block_size, q_dtype, pool_blocks));
    AK_REQUIRE(rope_len >= 1, AK_ERR_INVALID_ARG, "%s: the RoPE table is empty", who);
    AK_REQUIRE(q8_aligned(qkv, 16) && q8_aligned(rope_table, 16) && q8_aligned(q_out, 16) && q8_aligned(positions, 4) && q8_aligned(slots, 4),
               AK_ERR_INVALID_ARG, "%s: qkv, q_out and the RoPE table must be 16-byte aligned, positions and slots 4-byte", who);
    if (tokens == 0) return AK_OK;
    AK_TRY(q8_check_here(k_pool, who));
#define AK_APPEND_Q8(T, HD)                                                                                                                              \
    return append_q8<T, HD>(as_stream(stream), qkv, rope_table, rope_len, positions, slots, q_out, k_pool, v_pool, k_scales, v_scales, tokens, heads, \
                            kv_heads, pool_blocks * Q8_BS)
#define AK_APPEND_Q8_HD(T)                       \
    switch (head_dim) {                          \
        case 32: AK_APPEND_Q8(T, 32);            \
        case 64: AK_APPEND_Q8(T, 64);            \
        case 96: AK_APPEND_Q8(T, 96);            \
        default: AK_APPEND_Q8(T, 128);           \
    }
    if (q_dtype == AK_F32) { AK_APPEND_Q8_HD(float) }
    AK_APPEND_Q8_HD(bf16)
#undef AK_APPEND_Q8_HD
#undef AK_APPEND_Q8
}

int ak_kv_read_q8(void* stream, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales, const int32_t* slots, void* k_out,
                  void* v_out, uint32_t tokens, uint32_t kv_heads, uint32_t head_dim, uint32_t block_size, uint32_t out_dtype, uint32_t pool_blocks) {
    const char* who = "ak_kv_read_q8";
    AK_REQUIRE(slots && (k_out || v_out), AK_ERR_INVALID_ARG, "%s: null pointer", who);
    AK_TRY(q8_check_cache(who, k_pool, v_pool, k_scales, v_scales, kv_heads, kv_heads, head_dim, block_size, out_dtype, pool_blocks));
    AK_REQUIRE(q8_aligned(k_out, 16) && q8_aligned(v_out, 16) && q8_aligned(slots, 4), AK_ERR_INVALID_ARG, "%s: the outputs must be 16-byte aligned, slots 4-byte", who);
    if (tokens == 0) return AK_OK;
    AK_TRY(q8_check_here(k_pool, who));
    const uint64_t threads = (uint64_t)tokens * kv_heads * (head_dim / (out_dtype == AK_F32 ? 4 : 8));
    AK_REQUIRE(cdiv64(threads, 256) <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "%s: %u tokens x %u heads are too many for one call", who, tokens, kv_heads);
    const dim3 grid((unsigned)cdiv64(threads, 256));
    if (out_dtype == AK_F32)
        return launch_k(kv_read_q8_kernel<float>, grid, dim3(256), 0, as_stream(stream), NO_CLUSTER, k_pool, v_pool, k_scales, v_scales, slots, (float*)k_out,
                        (float*)v_out, tokens, kv_heads, head_dim, pool_blocks * Q8_BS);
    return launch_k(kv_read_q8_kernel<bf16>, grid, dim3(256), 0, as_stream(stream), NO_CLUSTER, k_pool, v_pool, k_scales, v_scales, slots, (bf16*)k_out,
                    (bf16*)v_out, tokens, kv_heads, head_dim, pool_blocks * Q8_BS);
}
}
