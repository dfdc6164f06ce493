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
// The root divides every value of a row alike: q = rint(127 h w / max|h w|) does without it, and the sum of squares and the largest |h w| are taken
// together, in one pass and with one exchange between the row's threads. A row lives in their registers from then on: every input byte is read
// once, every output byte written once. `tpr` threads share a row.
//
// What bounds it: the bytes (with a residual 1.0 of the copy bandwidth, 16384 x 2048 f32 26.5 us = 0.97, 4001 x 8192 26.2 = 0.96, in the
// ring), and instructions where these are few (4001 x 8192 bf16 with weights 21.5 us = 0.70, rows of 2047 39.7 us = 0.65). With y itself and two
// reductions, one after the other: 31, 38, 26.6 and 50 us. Of these 0.1 to 0.5 us (32768 x 320 f32 1.2 of 11.9) are the exact reciprocal's and the
// rounded products', see q8_scale.
template <typename T> struct Q8Vec {
    static constexpr int V = 16 / sizeof(T);   // values of a group: a 16-byte load
    static __device__ __forceinline__ void load(const T* p, float (&v)[V]) {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < V; e++) {
            if constexpr (sizeof(T) == 4) v[e] = __uint_as_float(w[e]);
            else v[e] = __uint_as_float((e & 1) ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        }
    }
};

constexpr uint32_t NQ_MAX_WARPS = 32;

// The largest of |a|, |b| and |c|, NaN if one is NaN.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The sum (`norm`: if it is wanted) and the largest of the non-negative values of a row's threads, the same in every one. `both`: the row's warps' values.
struct RowWarps {
    float sum[NQ_MAX_WARPS];
    uint32_t top[NQ_MAX_WARPS];
};
__device__ __forceinline__ void row_reduce(bool norm, float& sum, float& top, RowWarps& both, uint32_t warps, uint32_t wid, uint32_t lane) {
    if (norm) sum = warp_sum(sum);
    uint32_t bits = __reduce_max_sync(0xffffffffu, abs_bits(top));
    if (warps > 1) {
        if (lane == 0) { both.sum[wid] = sum; both.top[wid] = bits; }
        __syncthreads();
        if (norm) sum = warp_sum(lane < warps ? both.sum[lane] : 0.0f);
        bits = __reduce_max_sync(0xffffffffu, lane < warps ? both.top[lane] : 0u);
    }
    top = __uint_as_float(bits);
}
// What a row's values h w (without weights: h) are multiplied by, and the row's scale, from the largest magnitude `top`: y = rs h w is larger by rs, which the
// quotients do not see, so that the sum of squares and the largest value take one pass and one exchange.
struct RowScale {
    float inv, s;
    bool ok;   // s is a number
};
// A mean square (with eps) under 1e-36 or a sum beyond f32's largest number says nothing of the row any more, whose scale is NaN then. (The sum once more in
// 64 bits for such rows, behind a branch that none else takes, cost bf16 rows 5 to 14 % of their time by its registers, wherever it stood.)
__device__ __forceinline__ RowScale row_scale(bool norm, float sum, float top, float inv_size, float eps) {
    const float square = sum * inv_size + eps;
    const bool none = top < 1e-36f;   // (127 / top is below 2^127, and products h w keep 2^-30 of their largest)
    const float y = none || !norm ? top : square >= 1e-36f && sum < INFINITY ? top * rsqrtf(square) : INFINITY;
    const bool some = y >= Q8_ZERO && !none;
    RowScale o;
    o.ok = y < INFINITY;
    o.inv = some && o.ok ? q8_inv(top) : 0.0f;
    o.s = !o.ok ? __uint_as_float(0x7fc00000u) : some ? y * (1.0f / 127.0f) : 0.0f;
    return o;
}

// Rows of whole vectors: a thread holds NV groups of V consecutive values (16 bytes of input).
template <typename T, int NV>
__global__ void __launch_bounds__(1024)
norm_q8_kernel(T* __restrict__ x, const float* __restrict__ residual, const float* __restrict__ w, int8_t* __restrict__ q, float* __restrict__ scales,
               uint32_t rows, uint32_t size, float inv_size, float eps) {
    constexpr int V = Q8Vec<T>::V;
    pdl_wait();
    pdl_trigger();
    __shared__ RowWarps both;
    const uint32_t tpr = blockDim.x, t = threadIdx.x, lane = t & 31, wid = t >> 5, warps = tpr >> 5, groups = size / V;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;   // blockDim.y > 1 only with one warp per row
    if (row >= rows) return;
    x += (size_t)row * size;
    q += (size_t)row * size;
    float y[NV][V];
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const uint32_t g = t + c * tpr;
#pragma unroll
        for (int e = 0; e < V; e++) y[c][e] = 0.0f;
        if (g < groups) Q8Vec<T>::load(x + V * g, y[c]);
    }
    if constexpr (sizeof(T) == 4) {
        if (residual) {
            residual += (size_t)row * size;
#pragma unroll
            for (int c = 0; c < NV; c++) {
                const uint32_t g = t + c * tpr;
                if (g >= groups) continue;
                float r[4];
                Q8Vec<float>::load(residual + V * g, r);
#pragma unroll
                for (int e = 0; e < 4; e++) y[c][e] += r[e];
                *reinterpret_cast<float4*>(x + V * g) = make_float4(y[c][0], y[c][1], y[c][2], y[c][3]);
            }
        }
    }
    float sum = 0.0f;
    if (w) {
#pragma unroll
        for (int c = 0; c < NV; c++) {
            const uint32_t g = t + c * tpr;
#pragma unroll
            for (int e = 0; e < V; e++) sum += y[c][e] * y[c][e];
            if (g >= groups) continue;
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                float ww[4];
                Q8Vec<float>::load(w + V * g + k, ww);
#pragma unroll
                for (int e = 0; e < 4; e++) y[c][k + e] *= ww[e];
            }
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < NV; c++)
#pragma unroll
        for (int e = 0; e < V; e += 2) top = max_abs(top, y[c][e], y[c][e + 1]);
    row_reduce(w, sum, top, both, warps, wid, lane);
    const RowScale sc = row_scale(w, sum, top, inv_size, eps);
    if (t == 0) scales[row] = sc.s;
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const uint32_t g = t + c * tpr;
        if (g >= groups) continue;
        uint32_t o[V / 4];
#pragma unroll
        for (int k = 0; k < V / 4; k++) o[k] = q8_pack4(y[c][4 * k], y[c][4 * k + 1], y[c][4 * k + 2], y[c][4 * k + 3], sc.inv, sc.ok);
        if constexpr (V == 8) *reinterpret_cast<uint2*>(q + V * g) = make_uint2(o[0], o[1]);
        else *reinterpret_cast<uint32_t*>(q + V * g) = o[0];
    }
}

constexpr uint32_t NQ_RING_BYTES = 226 * 1024;
// Many rows: resident blocks walk over them, a block's next row on its way into shared memory while one is worked on, the weights in registers. A thread
// copies what it reads itself: nobody waits for anybody's copy.
// ODD: rows of any size. All the arrays of a row start at the same element offset, so groups are cut where the ADDRESS is a multiple of V elements, and
// the first and the last group of a row may be partial. The blocks' stride is a multiple of V rows, so that a block sees one shift only, and which
// of a thread's groups are partial is settled once.
template <typename T, int NV, bool ODD, bool RES>
__global__ void __launch_bounds__(1024)
norm_q8_ring_kernel(T* __restrict__ x, const float* __restrict__ residual, const float* __restrict__ w, int8_t* __restrict__ q, float* __restrict__ scales,
                    uint32_t rows, uint32_t size, float inv_size, float eps) {
    constexpr int V = Q8Vec<T>::V, KINDS = RES ? 2 : 1;
    pdl_wait();
    pdl_trigger();
    extern __shared__ __align__(16) uint8_t ring[];       // [2][x, residual][group of a thread][thread] of 16 bytes
    __shared__ RowWarps both[2];
    const uint32_t tpr = blockDim.x, t = threadIdx.x, lane = t & 31, wid = t >> 5, warps = tpr >> 5;
    const uint32_t step = gridDim.x;                        // ODD: a multiple of V, or there is no second row
    const uint32_t shift = ODD ? (uint32_t)(((size_t)blockIdx.x * size) & (V - 1)) : 0, groups = (shift + size + V - 1) / V;
    auto inside = [&](uint32_t i) { return i - shift < size; };   // i: from the row's group 0 on
    auto there = [&](int c) { return t + c * tpr < groups; };
    float ww[NV][V];
    uint32_t part = 0;   // bit c: group c is partial
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const uint32_t i = V * (t + c * tpr);
#pragma unroll
        for (int e = 0; e < V; e++) ww[c][e] = 0.0f;
        if (ODD && there(c) && !(inside(i) && inside(i + V - 1))) part |= 1u << c;
        if (!w || !there(c)) continue;
        if constexpr (ODD) {
#pragma unroll
            for (int e = 0; e < V; e++)
                if (inside(i + e)) ww[c][e] = w[i + e - shift];
        } else {
#pragma unroll
            for (int k = 0; k < V; k += 4) Q8Vec<float>::load(w + i + k, *reinterpret_cast<float(*)[4]>(&ww[c][k]));
        }
    }
    const uint32_t my = smem_u32(ring) + t * 16;
    const size_t stride = (size_t)step * size, off0 = (size_t)blockIdx.x * size - shift + V * t;
    // (a partial group is read whole, with neighbouring rows' values that are dropped, but not past the last row: the one before it has V values behind it)
    auto ask = [&](uint32_t row, size_t off, uint32_t half) {
        if (row < rows) {
#pragma unroll
            for (int c = 0; c < NV; c++) {
                if (!there(c)) continue;
                uint32_t bytes = 16;
                if (ODD && part && row + 1 == rows) bytes = min(16u, (shift + size - V * (t + c * tpr)) * (uint32_t)sizeof(T));
#pragma unroll
                for (int k = 0; k < KINDS; k++) {
                    const void* src = k ? (const void*)(residual + off + c * V * tpr) : (const void*)(x + off + c * V * tpr);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(my + ((half * KINDS + k) * NV + c) * tpr * 16), "l"(src), "r"(bytes) : "memory");
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ask(blockIdx.x, off0, 0);
    size_t off = off0;
    uint32_t half = 0;
    for (uint32_t row = blockIdx.x; row < rows; row += step, off += stride, half ^= 1) {
        ask(row + step, off + stride, half ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        float y[NV][V];
#pragma unroll
        for (int c = 0; c < NV; c++) {
            const uint8_t* src = ring + t * 16 + ((half * KINDS) * NV + c) * tpr * 16;
#pragma unroll
            for (int e = 0; e < V; e++) y[c][e] = 0.0f;
            if (!there(c)) continue;
            Q8Vec<T>::load(reinterpret_cast<const T*>(src), y[c]);
            if constexpr (RES) {
                float r[4];
                Q8Vec<float>::load(reinterpret_cast<const float*>(src + NV * tpr * 16), r);
#pragma unroll
                for (int e = 0; e < 4; e++) y[c][e] += r[e];
                if (!ODD || !(part >> c & 1u)) *reinterpret_cast<float4*>(x + off + c * V * tpr) = make_float4(y[c][0], y[c][1], y[c][2], y[c][3]);
            }
        }
        if (ODD && part) {
#pragma unroll
            for (int c = 0; c < NV; c++)
                if (part >> c & 1u) {
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        if (!inside(V * (t + c * tpr) + e)) y[c][e] = 0.0f;
                        else if constexpr (RES) x[off + c * V * tpr + e] = y[c][e];
                    }
                }
        }
        float sum = 0.0f, top = 0.0f;
        if (w) {
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int e = 0; e < V; e++) {
                    sum += y[c][e] * y[c][e];
                    y[c][e] *= ww[c][e];
                }
        }
#pragma unroll
        for (int c = 0; c < NV; c++)
#pragma unroll
            for (int e = 0; e < V; e += 2) top = max_abs(top, y[c][e], y[c][e + 1]);
        row_reduce(w, sum, top, both[half], warps, wid, lane);   // two: a warp may be a row ahead of another that still reads
        const RowScale sc = row_scale(w, sum, top, inv_size, eps);
        if (t == 0) scales[row] = sc.s;
        uint32_t o[NV][V / 4];
#pragma unroll
        for (int c = 0; c < NV; c++) {
#pragma unroll
            for (int k = 0; k < V / 4; k++) o[c][k] = q8_pack4(y[c][4 * k], y[c][4 * k + 1], y[c][4 * k + 2], y[c][4 * k + 3], sc.inv, sc.ok);
            if (!there(c) || (ODD && (part >> c & 1u))) continue;
            int8_t* dst = q + off + c * V * tpr;
            if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(o[c][0], o[c][1]);
            else *reinterpret_cast<uint32_t*>(dst) = o[c][0];
        }
        if (ODD && part) {
#pragma unroll
            for (int c = 0; c < NV; c++)
                if (part >> c & 1u) {
#pragma unroll
                    for (int e = 0; e < V; e++)
                        if (inside(V * (t + c * tpr) + e)) q[off + c * V * tpr + e] = (int8_t)(o[c][e / 4] >> (8 * (e % 4)));
                }
        }
    }
}

// Rows that do not fit the registers of a block, rows shorter than a vector, and buffers that are not aligned for vectors: a block per row, two passes over it (the second reads what
// the first wrote back).
template <typename T>
__global__ void __launch_bounds__(1024)
norm_q8_any_kernel(T* x, const float* residual, const float* __restrict__ w, int8_t* __restrict__ q, float* __restrict__ scales, uint32_t size, float inv_size, float eps) {
    pdl_wait();
    pdl_trigger();
    __shared__ RowWarps both;
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const size_t off = (size_t)blockIdx.x * size;
    float sum = 0.0f;
    float top = 0.0f;
    for (uint32_t i = threadIdx.x; i < size; i += blockDim.x) {
        float v = Cvt<T>::to_f(x[off + i]);
        if constexpr (sizeof(T) == 4) {
            if (residual) { v += residual[off + i]; x[off + i] = v; }
        }
        sum += v * v;
        top = max_abs(top, w ? v * w[i] : v, 0.0f);
    }
    row_reduce(w, sum, top, both, warps, wid, lane);
    const RowScale sc = row_scale(w, sum, top, inv_size, eps);
    if (threadIdx.x == 0) scales[blockIdx.x] = sc.s;
    for (uint32_t i = threadIdx.x; i < size; i += blockDim.x) {
        const float v = Cvt<T>::to_f(x[off + i]);   // (what this thread wrote back)
        q[off + i] = q8_of(w ? v * w[i] : v, sc.inv, sc.ok);
    }
}

template <typename T>
static int norm_q8(cudaStream_t st, T* x, const float* residual, const float* w, int8_t* q, float* scales, uint32_t rows, uint32_t size, float eps) {
    constexpr uint32_t V = Q8Vec<T>::V, MOST = 32 / V;   // 32 values a thread
    const uint32_t groups = cdiv(size, V) + (size % V ? 1 : 0);   // of a row, at most
    const float inv_size = 1.0f / (float)size;
    const bool vectors = q8_aligned(x, 16) && q8_aligned(residual, 16) && q8_aligned(q, V) && q8_aligned(w, 16);
    if (!vectors || size < V)   // (rows shorter than a vector: those of several rows would reach over the end of the buffer)
        return launch_k(norm_q8_any_kernel<T>, dim3(rows), dim3(size < V ? 32 : 512), 0, st, NO_CLUSTER, x, residual, w, q, scales, size, inv_size, eps);
    const bool few = rows <= 2 * B200_SMS;   // latency: as many threads to a row as there are vectors
    const bool odd = size % V != 0;
    // The ring: any odd size; with weights, rows of more than 24 values a lane of one warp (16384 x 1024 f32 14.6 us, in the other kernel 17.4, but 768 12.5
    // and 12.3), enough of them to keep the resident blocks busy (1000 x 4096 f32 4.3 and 4.1). A residual or no weights leave nothing
    // to keep, and then blocks that come and go are as good or better (16384 x 2048 f32 with a residual 65 us, 72 in the ring).
    if (odd || (w && !residual && rows >= 16 * B200_SMS && size > 768)) {
        // 16 values a thread, few rows or short ones fewer
        const uint32_t n = groups <= (few ? 1024 : 32) ? 1 : groups <= (few ? 2048 : 64) ? 2 : 16 / V, tpr = cdiv(groups, n * 32) * 32;
        const uint32_t bytes = 2 * n * tpr * 16 * (residual ? 2 : 1);   // of shared memory
        if (tpr <= 1024 && bytes <= NQ_RING_BYTES) {
#define AK_NORM_Q8(N, ODD, RES)                                                                                                                                \
    do {                                                                                                                                                       \
        static bool set[64] = {};                                                                                                                              \
        AK_TRY(q8_allow_smem(norm_q8_ring_kernel<T, N, ODD, RES>, set, NQ_RING_BYTES));                                                                        \
        uint32_t most = B200_SMS / V * V;                                                                                                                      \
        if (rows > most) {   /* resident blocks */                                                                                                             \
            int occ = 0;                                                                                                                                       \
            AK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, norm_q8_ring_kernel<T, N, ODD, RES>, (int)tpr, bytes));                                \
            most = B200_SMS * (uint32_t)(occ < 1 ? 1 : occ) / V * V;                                                                                           \
        }                                                                                                                                                      \
        return launch_k(norm_q8_ring_kernel<T, N, ODD, RES>, dim3(rows < most ? rows : most), dim3(tpr), bytes, st, NO_CLUSTER, x, residual, w, q, scales,     \
                        rows, size, inv_size, eps);                                                                                                            \
    } while (0)
#define AK_NORM_Q8_ODD(N)                                       \
    do {                                                        \
        if constexpr (V == 4) {                                 \
            if (residual) AK_NORM_Q8(N, true, true);            \
        }                                                       \
        AK_NORM_Q8(N, true, false);                             \
    } while (0)
            if (!odd) AK_NORM_Q8(16 / V, false, false);
            if (n == 1) AK_NORM_Q8_ODD(1);
            if (n == 2) AK_NORM_Q8_ODD(2);
            if constexpr (V == 4) AK_NORM_Q8_ODD(4);
#undef AK_NORM_Q8_ODD
#undef AK_NORM_Q8
        }
    }
    if (odd || groups > 1024 * MOST)
        return launch_k(norm_q8_any_kernel<T>, dim3(rows), dim3(512), 0, st, NO_CLUSTER, x, residual, w, q, scales, size, inv_size, eps);
    // Many rows: a warp each up to 32 values a thread (16384 x 768 f32 12 us, with 64 threads a row 19), but not with a residual, whose loads want more
    // threads (26 against 32 us); long ones 16 values a thread, or 8 with a residual (16384 x 2048: 65.0 us, with 16 65.8).
    uint32_t n = few ? 1 : residual ? 2 : groups <= 32 * MOST ? cdiv(groups, 32) : 16 / V;
    if (n == 5 || n == 7) n++;
    while (groups > n * 1024) n *= 2;
    const uint32_t tpr = cdiv(groups, n * 32) * 32;
    const dim3 block(tpr, tpr == 32 && !few ? 4 : 1);
#define AK_NORM_Q8(N) \
    case N: return launch_k(norm_q8_kernel<T, N>, dim3(cdiv(rows, block.y)), block, 0, st, NO_CLUSTER, x, residual, w, q, scales, rows, size, inv_size, eps)
    switch (n) {
        AK_NORM_Q8(1);
        AK_NORM_Q8(2);
        AK_NORM_Q8(3);
        AK_NORM_Q8(4);
    }
    if constexpr (MOST == 8) {
        switch (n) {
            AK_NORM_Q8(6);
            AK_NORM_Q8(8);
        }
    }
#undef AK_NORM_Q8
    set_error("ak_rmsnorm_q8: no kernel for rows of %u", size);
    return AK_ERR_UNSUPPORTED;
}

// ============================================================================ split + RoPE + quantised append
// qkv row of a token: `heads` query heads, kv_heads key heads, kv_heads value heads. A few lanes take a head, 16 values each (HD = 96: 12) as four
// pieces of 4 that lie HD / 4 apart, so that the lanes of a piece read and write neighbouring bytes; the pairs of a piece are rotated, the largest
// magnitude of the head goes round by shuffles, 4 bytes a piece go out. The (token, head) rows of a block's tokens lie one behind the other in qkv
// and are dealt out in turns of one row a group of lanes.
//
// With 4 values a lane the hundred instructions that a row takes besides its bytes (addresses, scale, shuffles) were the bound: 16001 tokens, bf16, 12 + 2 x
// 12 heads of 64 58 us then, 35.6 now (0.85 of the copy bandwidth); 5 + 2 x 5 of 64, f32 49 and 20.6; 32 + 2 x 8 of 128 97 and 84 (1.02, 8 pieces
// 95); 64 tokens of 12 + 2 x 12 heads of 64 2.0 and 1.7.
constexpr uint32_t AP_THREADS = 256;
template <int HD> struct ApCfg {
    static constexpr uint32_t PIECES = HD == 96 ? 3 : 4;       // of four values that a lane holds of a head
    static constexpr uint32_t LANES = HD / (4 * PIECES);       // of a head
    static constexpr uint32_t GROUPS = AP_THREADS / LANES;     // rows of a turn
};

template <typename T, int HD>
__global__ void __launch_bounds__(AP_THREADS)
rope_kv_append_q8_kernel(const float* __restrict__ qkv, const float4* __restrict__ rope, uint32_t rope_len, const int32_t* __restrict__ positions,
                         const int32_t* __restrict__ slots, T* __restrict__ q_out, int8_t* __restrict__ k_pool, int8_t* __restrict__ v_pool,
                         float* __restrict__ k_scales, float* __restrict__ v_scales, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t pool_slots,
                         uint32_t per_block, const Q8Div total) {
    using C = ApCfg<HD>;
    constexpr uint32_t P = C::PIECES, STEP = 4 * C::LANES;   // values between a lane's pieces
    pdl_wait();
    pdl_trigger();
    const uint32_t group = threadIdx.x / C::LANES, l = threadIdx.x % C::LANES;
    const uint32_t t0 = blockIdx.x * per_block, items = min(per_block, tokens - t0) * total.d;
    const float* rows = qkv + (uint64_t)t0 * total.d * HD + 4 * l;
    // whole blocks go round together: the shuffles want every lane of a group
    for (uint32_t base = 0; base < items; base += C::GROUPS) {
        const uint32_t i = base + group, of_block = total.of(i), tok = t0 + of_block, head = i - of_block * total.d;
        float4 x[P];
        int32_t pos = -1, slot = -1;
#pragma unroll
        for (uint32_t c = 0; c < P; c++) x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < items) {
#pragma unroll
            for (uint32_t c = 0; c < P; c++) x[c] = *reinterpret_cast<const float4*>(rows + (uint64_t)i * HD + c * STEP);
            pos = positions[tok];
            if (head >= heads) slot = slots[tok];
        }
        const bool live = (uint32_t)pos < rope_len;   // a token at another position is left out
        float4 f[P];   // (cos, sin) of the pieces' pairs
#pragma unroll
        for (uint32_t c = 0; c < P; c++) {
            f[c] = make_float4(1.f, 0.f, 1.f, 0.f);
            if (live && head < heads + kv_heads) f[c] = rope[(uint64_t)pos * (HD / 4) + c * C::LANES + l];
        }
        if (head < heads + kv_heads) {
#pragma unroll
            for (uint32_t c = 0; c < P; c++) {
                rope_rotate(x[c].x, x[c].y, f[c].x, f[c].y, x[c].x, x[c].y);
                rope_rotate(x[c].z, x[c].w, f[c].z, f[c].w, x[c].z, x[c].w);
            }
        }
        if (live && head < heads) {
            T* dst = q_out + ((uint64_t)tok * heads + head) * HD + 4 * l;
#pragma unroll
            for (uint32_t c = 0; c < P; c++) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(dst + c * STEP) = x[c];
                } else {
                    const bf162 a = __floats2bfloat162_rn(x[c].x, x[c].y), b = __floats2bfloat162_rn(x[c].z, x[c].w);
                    *reinterpret_cast<uint2*>(dst + c * STEP) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                }
            }
        }
        const bool kept = live && (uint32_t)slot < pool_slots;   // a key or value head with a place
        if (!__any_sync(0xffffffffu, kept)) continue;
        uint32_t top = 0;
#pragma unroll
        for (uint32_t c = 0; c < P; c++) top = max(top, max(max(abs_bits(x[c].x), abs_bits(x[c].y)), max(abs_bits(x[c].z), abs_bits(x[c].w))));
#pragma unroll
        for (uint32_t o = C::LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (kept) {
            const bool is_v = head >= heads + kv_heads;
            const uint64_t at = ((uint64_t)((uint32_t)slot / Q8_BS) * kv_heads + (head - heads - (is_v ? kv_heads : 0))) * Q8_BS + (uint32_t)slot % Q8_BS;
            float inv, s;
            q8_scale(top, inv, s);
            int8_t* dst = (is_v ? v_pool : k_pool) + at * HD + 4 * l;
#pragma unroll
            for (uint32_t c = 0; c < P; c++) *reinterpret_cast<uint32_t*>(dst + c * STEP) = q8_pack4(x[c].x, x[c].y, x[c].z, x[c].w, inv, s == s);
            if (l == 0) (is_v ? v_scales : k_scales)[at] = s;
        }
    }
}

// ============================================================================ cached rows as numbers
// 16 bytes of output (VEC values) of the key row and of the value row of one (token, head) a thread, RD_AHEAD of them in flight: two (65000 tokens x 8
// heads of 128 to bf16 68 us = 0.91 of the copy bandwidth, with one 80, with four 69), or one where the blocks fit the SMs twice over (64 x 12 heads
// of 64 1.7 us, with two 1.9, with four 2.6; 2000 x 12 heads of 64 3.5 and 4.2).
constexpr uint32_t RD_THREADS = 256;
template <typename T, int HD, int RD_AHEAD> struct RdCfg {
    static constexpr uint32_t VEC = 16 / sizeof(T), CHUNKS = HD / VEC;
    static constexpr uint32_t ROWS = RD_THREADS * RD_AHEAD / CHUNKS;   // (token, head) rows of a block
};

template <typename T, int HD, int RD_AHEAD>
__global__ void __launch_bounds__(RD_THREADS)
kv_read_q8_kernel(const int8_t* __restrict__ k_pool, const int8_t* __restrict__ v_pool, const float* __restrict__ k_scales, const float* __restrict__ v_scales,
                  const int32_t* __restrict__ slots, T* __restrict__ k_out, T* __restrict__ v_out, uint32_t rows, const Q8Div kv_heads, uint32_t pool_slots) {
    using C = RdCfg<T, HD, RD_AHEAD>;
    pdl_wait();
    pdl_trigger();
    uint32_t row[RD_AHEAD], words[RD_AHEAD][2][C::VEC / 4];
    float s[RD_AHEAD][2];
#pragma unroll
    for (uint32_t j = 0; j < RD_AHEAD; j++) {
        const uint32_t item = j * RD_THREADS + threadIdx.x, c = item % C::CHUNKS;
        row[j] = blockIdx.x * C::ROWS + item / C::CHUNKS;
        if (item / C::CHUNKS >= C::ROWS || row[j] >= rows) row[j] = 0xffffffffu;
        uint32_t slot = 0xffffffffu, h = 0;
        if (row[j] != 0xffffffffu) {
            const uint32_t t = kv_heads.of(row[j]);
            h = row[j] - t * kv_heads.d;
            slot = (uint32_t)slots[t];
        }
        const bool have = slot < pool_slots;
        const uint64_t at = have ? ((uint64_t)(slot / Q8_BS) * kv_heads.d + h) * Q8_BS + slot % Q8_BS : 0;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            s[j][side] = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < C::VEC / 4; i++) words[j][side][i] = 0;
            if (!have || !(side ? v_out : k_out)) continue;
            const int8_t* src = (side ? v_pool : k_pool) + at * HD + c * C::VEC;
            s[j][side] = (side ? v_scales : k_scales)[at];
            if constexpr (C::VEC == 8) {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                words[j][side][0] = u.x; words[j][side][1] = u.y;
            } else {
                words[j][side][0] = *reinterpret_cast<const uint32_t*>(src);
            }
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < RD_AHEAD; j++) {
        const uint32_t c = (j * RD_THREADS + threadIdx.x) % C::CHUNKS;
        if (row[j] == 0xffffffffu) continue;
#pragma unroll
        for (int side = 0; side < 2; side++) {
            T* out = side ? v_out : k_out;
            if (!out) continue;
            alignas(16) T o[C::VEC];
#pragma unroll
            for (uint32_t i = 0; i < C::VEC; i++) o[i] = Cvt<T>::from_f((float)(int8_t)(words[j][side][i / 4] >> (8 * (i % 4))) * s[j][side]);
            *reinterpret_cast<uint4*>(out + (uint64_t)row[j] * HD + c * C::VEC) = *reinterpret_cast<const uint4*>(o);
        }
    }
}

template <typename T, int HD>
static int append_q8(cudaStream_t st, const float* qkv, const float* rope, uint32_t rope_len, const int32_t* positions, const int32_t* slots, void* q_out,
                     int8_t* k_pool, int8_t* v_pool, float* k_scales, float* v_scales, uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t pool_slots) {
    const uint32_t total = heads + 2 * kv_heads;
    // Tokens of a block: those of up to 4 turns that leave the fewest groups idle in the last one, while there are three blocks an SM (2000
    // tokens of 20 heads of 128: 6.6 us with one a block, 6.4 with three).
    uint32_t per_block = 1;
    float best = 0.0f;
    for (uint32_t n = 1; n == 1 || (n * total <= 4 * ApCfg<HD>::GROUPS && cdiv(tokens, n) >= 3 * B200_SMS); n++) {
        const float used = (float)(n * total) / (float)(cdiv(n * total, ApCfg<HD>::GROUPS) * ApCfg<HD>::GROUPS);
        if (used > 1.01f * best) { best = used; per_block = n; }
    }
    return launch_k(rope_kv_append_q8_kernel<T, HD>, dim3(cdiv(tokens, per_block)), dim3(AP_THREADS), 0, st, NO_CLUSTER, qkv,
                    reinterpret_cast<const float4*>(rope), rope_len, positions, slots, (T*)q_out, k_pool, v_pool, k_scales, v_scales, tokens, heads, kv_heads,
                    pool_slots, per_block, Q8Div(total));
}

template <typename T, int HD>
static int read_q8(cudaStream_t st, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales, const int32_t* slots, void* k_out,
                   void* v_out, uint32_t tokens, uint32_t kv_heads, uint32_t pool_slots) {
    const uint32_t rows = tokens * kv_heads;
#define AK_READ(AHEAD)                                                                                                                                     \
    return launch_k(kv_read_q8_kernel<T, HD, AHEAD>, dim3(cdiv(rows, RdCfg<T, HD, AHEAD>::ROWS)), dim3(RD_THREADS), 0, st, NO_CLUSTER, k_pool, v_pool, k_scales, \
                    v_scales, slots, (T*)k_out, (T*)v_out, rows, Q8Div(kv_heads), pool_slots)
    if (cdiv(rows, RdCfg<T, HD, 1>::ROWS) <= 16 * B200_SMS) AK_READ(1);
    AK_READ(2);
#undef AK_READ
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
    AK_REQUIRE(rope_len >= 1 && rope_len <= 0x7fffffffu, AK_ERR_INVALID_ARG, "%s: the RoPE table must have 1 to 2^31 - 1 positions (got %u)", who, rope_len);
    AK_REQUIRE(q8_aligned(qkv, 16) && q8_aligned(rope_table, 16) && q8_aligned(q_out, 16) && q8_aligned(positions, 4) && q8_aligned(slots, 4),
               AK_ERR_INVALID_ARG, "%s: qkv, q_out and the RoPE table must be 16-byte aligned, positions and slots 4-byte", who);
    AK_REQUIRE(tokens <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "%s: %u tokens are too many for one call", who, tokens);
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
    AK_REQUIRE((uint64_t)tokens * kv_heads <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "%s: %u tokens x %u heads are too many for one call", who, tokens, kv_heads);
#define AK_READ_Q8(T, HD) return read_q8<T, HD>(as_stream(stream), k_pool, v_pool, k_scales, v_scales, slots, k_out, v_out, tokens, kv_heads, pool_blocks * Q8_BS)
#define AK_READ_Q8_HD(T)                         \
    switch (head_dim) {                          \
        case 32: AK_READ_Q8(T, 32);              \
        case 64: AK_READ_Q8(T, 64);              \
        case 96: AK_READ_Q8(T, 96);              \
        default: AK_READ_Q8(T, 128);             \
    }
    if (out_dtype == AK_F32) { AK_READ_Q8_HD(float) }
    AK_READ_Q8_HD(bf16)
#undef AK_READ_Q8_HD
#undef AK_READ_Q8
}
}
