// Attention of the newest tokens of every sequence over the 8-bit paged cache.
//
//   o_r = sum_j softmax_j(scale * ks_j (q_r . k_j)) vs_j v_j,   j < limit_r = kv_len - q_len + i + 1 for query i of its sequence
//
// k_j, v_j are int8 rows, ks_j, vs_j their f32 scales. One pass over the cache with the running maximum and sum of the softmax; the
// bytes of the cache are read once and bound the kernel (132 bytes per position and kv head at head size 64, 264 at 128).
//
// The products run on mma.sync.m16n8k16 in f16: int8 is exact in f16 (1024 + 128 + v is assembled by a byte permute and 1152 taken off),
// and the tile of 16 rows is one more than a group of query heads fills: decode has one query per (sequence, head), so tcgen05, whose
// smallest tile is 64 rows of one K, has nothing to work with. The rows of the A operand:
//   PIECES = 2: 8 queries, rows 0-7 their leading f16 part and rows 8-15 what is left of it (22 bits together), for q and for the
//               weights p * vs alike. Both f32 and bf16 results come out as from f32 arithmetic, and for up to 8 query rows it costs nothing:
//               the other 8 rows would be empty.
//   PIECES = 1: 16 queries (bf16 results, more than 8 query rows per kv head): weights rounded once to f16 (2^-12, the result to 2^-9).
// q is scaled by a power of two per row to below 2^15, the weights by one that follows the largest value scale met so far (below 2^14), so
// that f16's range does not matter: a leading part's last bit is 2^-10 of its value, down to 2^-38 of the largest one.
//
// A CTA of WARPS warps takes one (sequence, kv head, tile of queries, split); each warp has every WARPS-th cache block of the split and a
// ring of cp.async stages of its own, no barrier in the loop. The warps' results are merged in shared memory and the splits', which are
// the CTAs of one cluster, through distributed shared memory in split order: no scratch, no atomics, the same bits every time.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "q8.cuh"
#include "tcgen05.cuh"
namespace cg = cooperative_groups;

namespace ak {

constexpr int AQ_WARPS = 4;
constexpr uint32_t AQ_MAX_SPLITS = 16;   // CTAs of a cluster (8 is the portable limit, 16 is asked for)

template <int HD> struct AqCfg {
    static constexpr int TILE = 16 * HD;                   // bytes of a block's keys (or values) of one head
    static constexpr int STAGE = 2 * TILE + 128;           // keys | values | 16 key scales | 16 value scales
    static constexpr int STAGES = HD >= 96 ? 3 : 4;
    static constexpr int RING = AQ_WARPS * STAGES * STAGE;
};

// Where 16-byte chunk `col` of row `row` sits in a tile. Keys are read 4 chunks of 2 rows at a time, values 32 bytes of every other row:
// the permutations keep either within distinct banks (head sizes 64 and 128; 96 has two-way conflicts).
template <int HD> __device__ __forceinline__ uint32_t k_at(uint32_t row, uint32_t col) {
    if (HD == 128) return row * 128 + ((col ^ ((row & 1) << 2)) << 4);
    return row * HD + (col << 4);
}
template <int HD> __device__ __forceinline__ uint32_t v_at(uint32_t row, uint32_t col) {
    if (HD == 128) return row * 128 + ((col ^ (((row >> 1) & 3) << 1)) << 4);
    if (HD == 64) return (row >> 1) * 128 + (((((row & 1) << 2) | col) ^ (((row >> 1) & 3) << 1)) << 4);
    return row * HD + (col << 4);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
template <int N> __device__ __forceinline__ void lds_words(uint32_t a, uint32_t* w) {
    if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
    else w[0] = lds32(a);
}
__device__ __forceinline__ float2 lds_f2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
    return v;
}

// Two int8 of a word that has had its sign bits flipped (v + 128 as unsigned bytes), as f16: bytes sel of {u, 0x64..} are 1024 + 128 + v.
__device__ __forceinline__ uint32_t half2_of(uint32_t u, uint32_t sel) {
    const uint32_t t = __byte_perm(u, 0x64646464u, sel);
    uint32_t r;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// D(16x8, f32) += A(16x16, f16, row) B(16x8, f16, col)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {   // 2 ulp; 0 for -infinity, NaN for NaN
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

struct AqArgs {
    const void* q;
    const int8_t *k_pool, *v_pool;
    const float *k_scales, *v_scales;
    const int32_t *tables, *lens;
    void* out;
    uint32_t q_len, heads, kv_heads, group, q_tiles, max_blocks, pool_blocks;
    float scale;
};

// The d-index of word w (4 consecutive values) that lane t of a quad holds of a key row: chunk t, then chunk 4 + t (HD 128), 8-byte pieces for
// what is left. The order in which q . k is summed is free as long as q is laid out alike.
template <int HD> __device__ __forceinline__ uint32_t d_of(uint32_t t, int w) {
    if (HD == 32) return 8 * t + 4 * w;
    if (w < 4) return 16 * t + 4 * w;
    if (HD == 96) return 64 + 8 * t + 4 * (w - 4);
    return 64 + 16 * t + 4 * (w - 4);
}
template <int HD> __device__ __forceinline__ void load_key(uint32_t tile, uint32_t row, uint32_t t, uint32_t (&w)[HD / 16]) {
    if constexpr (HD == 32) {
        lds_words<2>(tile + row * 32 + 8 * t, w);
    } else {
        lds_words<4>(tile + k_at<HD>(row, t), w);
        if constexpr (HD == 128) lds_words<4>(tile + k_at<HD>(row, 4 + t), w + 4);
        if constexpr (HD == 96) lds_words<2>(tile + row * 96 + 64 + 8 * t, w + 4);
    }
}
// The HD / 8 values from HD / 8 * g on of a value row
template <int HD> __device__ __forceinline__ void load_value(uint32_t tile, uint32_t row, uint32_t g, uint32_t (&w)[HD / 32]) {
    if constexpr (HD == 128) lds_words<4>(tile + v_at<128>(row, g), w);
    else if constexpr (HD == 64) lds_words<2>(tile + v_at<64>(row, g >> 1) + ((g & 1) << 3), w);
    else if constexpr (HD == 32) w[0] = lds32(tile + row * 32 + 4 * g);
    else {
#pragma unroll
        for (int i = 0; i < 3; i++) w[i] = lds32(tile + row * 96 + 12 * g + 4 * i);
    }
}

template <typename T, int HD, int PIECES>
__global__ void __launch_bounds__(AQ_WARPS * 32)
attn_decode_q8_kernel(const AqArgs a) {
    using C = AqCfg<HD>;
    constexpr int ROWS = PIECES == 2 ? 8 : 16;    // queries of a tile
    constexpr int NR = PIECES == 2 ? 1 : 2;       // of them a lane holds
    constexpr int KW = HD / 16;                   // words of a key row per lane = steps of q . k
    constexpr int NT = HD / 8;                    // 8-wide tiles of the result
    constexpr bool LOW_Q = PIECES == 2 && sizeof(T) == 4;   // bf16 queries have no second part (8 bits)
    constexpr bool HIGH_ROWS_Q = PIECES == 1 || LOW_Q;
    pdl_wait();
    pdl_trigger();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_m[AQ_WARPS][ROWS], s_l[AQ_WARPS][ROWS];
    __shared__ float s_top[ROWS], s_sum[ROWS];

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t qt = blockIdx.x % a.q_tiles, kvh = (blockIdx.x / a.q_tiles) % a.kv_heads, seq = blockIdx.x / (a.q_tiles * a.kv_heads);
    const uint32_t split = blockIdx.z, n_splits = gridDim.z;
    const uint32_t total_rows = a.q_len * a.group;
    const int32_t cap = (int32_t)(a.max_blocks * Q8_BS);
    const int32_t len = a.lens[seq];

    // positions that row r of the tile may see
    auto limit_of = [&](uint32_t r) -> int32_t {
        const uint32_t rr = qt * ROWS + r;
        if (rr >= total_rows) return 0;
        const int64_t lim = (int64_t)len - a.q_len + rr / a.group + 1;
        return lim < 0 ? 0 : (int32_t)(lim < cap ? lim : cap);
    };
    auto q_index = [&](uint32_t r) -> size_t {   // first value of row r's query (and result)
        const uint32_t rr = qt * ROWS + r;
        return (((size_t)seq * a.q_len + rr / a.group) * a.heads + (size_t)kvh * a.group + rr % a.group) * HD;
    };
    const uint32_t last = min((uint32_t)ROWS, total_rows - qt * ROWS) - 1;
    const int32_t lim_min = limit_of(0), lim_max = limit_of(last);   // limits grow with the row
    int32_t lim[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) lim[r] = limit_of(g + 8 * r);

    // ---- queries: A operand rows g (and g + 8), scaled to below 2^15 by a power of two
    uint32_t qa[KW][HIGH_ROWS_Q ? 4 : 2];
    float row_scale[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const bool have = qt * ROWS + g + 8 * r < total_rows;
        const T* qp = reinterpret_cast<const T*>(a.q) + (have ? q_index(g + 8 * r) : 0);
        float x[KW][4];
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < KW; w++) {
            const uint32_t d = d_of<HD>(t, w);
            if constexpr (sizeof(T) == 4) {
                const float4 v = *reinterpret_cast<const float4*>(qp + d);
                x[w][0] = v.x; x[w][1] = v.y; x[w][2] = v.z; x[w][3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(qp + d);
                x[w][0] = __uint_as_float(v.x << 16); x[w][1] = __uint_as_float(v.x & 0xffff0000u);
                x[w][2] = __uint_as_float(v.y << 16); x[w][3] = __uint_as_float(v.y & 0xffff0000u);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (!have) x[w][e] = 0.0f;
                top = max(top, abs_bits(x[w][e]));
            }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = (int)(top >> 23) - 127;              // floor(log2 max|q|)
        const bool finite = top < 0x7f800000u;
        const int ef = 13 - (e < -100 ? -100 : e);   // q * 2^ef is below 2^14
        const float f = pow2i(finite ? ef : 0);
        // scores in the base-2 domain; a query with an infinity or a NaN has NaN for every score
        row_scale[r] = finite ? a.scale * 1.4426950408889634f * pow2i(-ef) : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int w = 0; w < KW; w++) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = finite ? x[w][i] * f : 0.0f;
            const uint32_t h0 = pack_half2(y[0], y[1]), h1 = pack_half2(y[2], y[3]);
            if (r == 0) { qa[w][0] = h0; qa[w][1] = h1; }
            else { qa[w][HIGH_ROWS_Q ? 2 : 0] = h0; qa[w][HIGH_ROWS_Q ? 3 : 0] = h1; }
            if constexpr (LOW_Q) {
                const float2 b0 = unpack_half2(h0), b1 = unpack_half2(h1);
                qa[w][2] = pack_half2(y[0] - b0.x, y[1] - b0.y);
                qa[w][3] = pack_half2(y[2] - b1.x, y[3] - b1.y);
            }
        }
    }

    // ---- this split's blocks, this warp's share of them
    const uint32_t nblk = ((uint32_t)lim_max + Q8_BS - 1) / Q8_BS;
    const uint32_t per = (nblk + n_splits - 1) / n_splits;
    const uint32_t b_begin = min(split * per, nblk), b_end = min(b_begin + per, nblk);
    const uint32_t first = b_begin + warp;
    const uint32_t mine = first < b_end ? (b_end - first + AQ_WARPS - 1) / AQ_WARPS : 0;
    const int32_t* table = a.tables + (size_t)seq * a.max_blocks;
    const uint32_t ring = smem_u32(smem) + warp * (C::STAGES * C::STAGE);

    uint32_t ids = 0xffffffffu;   // lane j: the cache block of this warp's tile (i & ~31) + j
    auto request = [&](uint32_t i) {
        if (i < mine) {
            if ((i & 31u) == 0) ids = i + lane < mine ? (uint32_t)table[first + (i + lane) * AQ_WARPS] : 0xffffffffu;
            const uint32_t blk = __shfl_sync(0xffffffffu, ids, i & 31u);
            if (blk < a.pool_blocks) {
                const uint32_t dst = ring + (i % C::STAGES) * C::STAGE;
                const size_t at = (size_t)blk * a.kv_heads + kvh;
                const int8_t *ks = a.k_pool + at * C::TILE, *vs = a.v_pool + at * C::TILE;
#pragma unroll
                for (uint32_t j = 0; j < (uint32_t)HD; j += 32) {
                    const uint32_t c = j + lane, row = c / (HD / 16), col = c % (HD / 16);
                    cp_async16(dst + k_at<HD>(row, col), ks + c * 16);
                    cp_async16(dst + C::TILE + v_at<HD>(row, col), vs + c * 16);
                }
                if (lane < 8) cp_async16(dst + 2 * C::TILE + lane * 16, (lane < 4 ? a.k_scales : a.v_scales) + at * Q8_BS + (lane & 3) * 4);
            }
        }
        cp_commit();
    };
    // Which tiles were requested: a block outside the pool holds no positions. (The ids of tile i are still in the window of tile i + STAGES
    // only while both share a group of 32, so validity travels as a bit.)
    uint32_t valid_bits = 0;
    auto request_at = [&](uint32_t i) {
        request(i);
        const bool ok = i < mine && __shfl_sync(0xffffffffu, ids, i & 31u) < a.pool_blocks;
        valid_bits = (valid_bits & ~(1u << (i % C::STAGES))) | ((ok ? 1u : 0u) << (i % C::STAGES));
    };
#pragma unroll
    for (uint32_t i = 0; i + 1 < (uint32_t)C::STAGES; i++) request_at(i);

    float m_run[NR], l_run[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) { m_run[r] = -INFINITY; l_run[r] = 0.0f; }
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    int v_exp = -110;   // weights are p * vs * 2^(13 - v_exp), v_exp >= log2 of every finite value scale so far

    for (uint32_t i = 0; i < mine; i++) {
        request_at(i + C::STAGES - 1);
        cp_wait<C::STAGES - 1>();
        __syncwarp();
        if ((valid_bits >> (i % C::STAGES)) & 1u) {
            const uint32_t ksm = ring + (i % C::STAGES) * C::STAGE, vsm = ksm + C::TILE, sks = vsm + C::TILE, svs = sks + 64;
            const int32_t pos0 = (int32_t)((first + i * AQ_WARPS) * Q8_BS);
            // ---- S = q . K^T: columns 2t, 2t + 1 of positions 0-7 and 8-15
            float sc[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
                uint32_t w[KW];
                load_key<HD>(ksm, 8 * n + g, t, w);
#pragma unroll
                for (int k = 0; k < KW; k++) {
                    const uint32_t u = w[k] ^ 0x80808080u;
                    const uint32_t b0 = half2_of(u, 0x4140), b1 = half2_of(u, 0x4342);
                    if constexpr (HIGH_ROWS_Q) mma_f16(sc[n], qa[k][0], qa[k][2], qa[k][1], qa[k][3], b0, b1);
                    else mma_f16(sc[n], qa[k][0], 0u, qa[k][1], 0u, b0, b1);
                }
            }
            const float2 ka = lds_f2(sks + 8 * t), kb = lds_f2(sks + 32 + 8 * t);
            const float2 va = lds_f2(svs + 8 * t), vb = lds_f2(svs + 32 + 8 * t);
            const float kscale[4] = {ka.x, ka.y, kb.x, kb.y};
            float vscale[4] = {va.x, va.y, vb.x, vb.y};
            const bool whole = pos0 + (int32_t)Q8_BS <= lim_min;   // every row sees the whole tile
            // ---- exponent of the weights: follows the largest value scale that any row of the tile sees
            float vtop = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int32_t pos = pos0 + (c >> 1) * 8 + 2 * (int32_t)t + (c & 1);
                const float v = fabsf(vscale[c]);
                if (pos < lim_max && v < INFINITY) vtop = fmaxf(vtop, v);
            }
            vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 1));
            vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 2));
            const int ve = (int)(__float_as_uint(vtop) >> 23) - 126;   // vtop < 2^ve
            float regrade = 1.0f;
            if (ve > v_exp) { regrade = ve - v_exp > 120 ? 0.0f : pow2i(v_exp - ve); v_exp = ve; }   // warp-uniform
            const float vf = pow2i(13 - v_exp > 126 ? 126 : 13 - v_exp);
            // ---- running maximum and sum, weights
            uint32_t pw[4];   // A operand of P . V
            float corr[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                float s[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float dot = PIECES == 2 ? sc[c >> 1][c & 1] + sc[c >> 1][2 + (c & 1)] : sc[c >> 1][2 * r + (c & 1)];
                    s[c] = dot * (row_scale[r] * kscale[c]);
                }
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int32_t pos = pos0 + (c >> 1) * 8 + 2 * (int32_t)t + (c & 1);
                        if (pos >= lim[r]) { s[c] = -INFINITY; }
                    }
                }
                float mb = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
                mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
                mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
                const float m_new = fmaxf(m_run[r], mb);
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;   // a row that has seen nothing yet
                corr[r] = ex2(m_run[r] - m_use);
                m_run[r] = m_new;
                float wgt[4], sum = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float p = ex2(s[c] - m_use);
                    sum += p;
                    const int32_t pos = pos0 + (c >> 1) * 8 + 2 * (int32_t)t + (c & 1);
                    // positions a row does not see may hold anything, a NaN for a scale included
                    wgt[c] = whole || pos < lim[r] ? p * (vscale[c] * vf) : 0.0f;
                }
                l_run[r] = l_run[r] * corr[r] + sum;   // this lane's positions only: the quad is added up at the end
                const uint32_t h0 = pack_half2(wgt[0], wgt[1]), h1 = pack_half2(wgt[2], wgt[3]);
                pw[r] = h0; pw[2 + r] = h1;
                if constexpr (PIECES == 2) {
                    const float2 b0 = unpack_half2(h0), b1 = unpack_half2(h1);
                    pw[1] = pack_half2(wgt[0] - b0.x, wgt[1] - b0.y);
                    pw[3] = pack_half2(wgt[2] - b1.x, wgt[3] - b1.y);
                }
            }
            const float c0 = corr[0] * regrade, c1 = corr[NR - 1] * regrade;
            if (__any_sync(0xffffffffu, c0 != 1.0f || c1 != 1.0f)) {
#pragma unroll
                for (int j = 0; j < NT; j++) { acc[j][0] *= c0; acc[j][1] *= c0; acc[j][2] *= c1; acc[j][3] *= c1; }
            }
            // ---- O += P . V
            uint32_t w0[HD / 32], w1[HD / 32], w2[HD / 32], w3[HD / 32];
            load_value<HD>(vsm, 2 * t, g, w0);
            load_value<HD>(vsm, 2 * t + 1, g, w1);
            load_value<HD>(vsm, 8 + 2 * t, g, w2);
            load_value<HD>(vsm, 9 + 2 * t, g, w3);
#pragma unroll
            for (int i4 = 0; i4 < HD / 32; i4++) {
                const uint32_t a0 = w0[i4] ^ 0x80808080u, a1 = w1[i4] ^ 0x80808080u, a2 = w2[i4] ^ 0x80808080u, a3 = w3[i4] ^ 0x80808080u;
                const uint32_t lo01 = __byte_perm(a0, a1, 0x5140), lo23 = __byte_perm(a0, a1, 0x7362);   // (d, d+1) and (d+2, d+3), position pairs
                const uint32_t hi01 = __byte_perm(a2, a3, 0x5140), hi23 = __byte_perm(a2, a3, 0x7362);
                mma_f16(acc[4 * i4 + 0], pw[0], pw[1], pw[2], pw[3], half2_of(lo01, 0x4140), half2_of(hi01, 0x4140));
                mma_f16(acc[4 * i4 + 1], pw[0], pw[1], pw[2], pw[3], half2_of(lo01, 0x4342), half2_of(hi01, 0x4342));
                mma_f16(acc[4 * i4 + 2], pw[0], pw[1], pw[2], pw[3], half2_of(lo23, 0x4140), half2_of(hi23, 0x4140));
                mma_f16(acc[4 * i4 + 3], pw[0], pw[1], pw[2], pw[3], half2_of(lo23, 0x4342), half2_of(hi23, 0x4342));
            }
        }
        __syncwarp();
    }
    cp_wait<0>();

    // ---- the warps' results, in true units, over the ring: [warp][row][HD]
#pragma unroll
    for (int r = 0; r < NR; r++) {
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
        if (t == 0) { s_m[warp][g + 8 * r] = m_run[r]; s_l[warp][g + 8 * r] = l_run[r]; }
    }
    __syncthreads();   // every warp is done with its ring
    float* part = reinterpret_cast<float*>(smem);
    {
        const float un = pow2i(v_exp - 13 < -126 ? -126 : v_exp - 13);
        float* wp = part + (size_t)warp * ROWS * HD;
        // accumulator columns 2t, 2t + 1 of tile j are n = 2t, 2t + 1: values HD / 8 * n + j
#pragma unroll
        for (int j = 0; j < NT; j++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const uint32_t d = (HD / 8) * (2 * t + c) + j;
                if (PIECES == 2) wp[g * HD + d] = (acc[j][c] + acc[j][2 + c]) * un;
                else {
                    wp[g * HD + d] = acc[j][c] * un;
                    wp[(g + 8) * HD + d] = acc[j][2 + c] * un;
                }
            }
        }
    }
    __syncthreads();
    // ---- merged over the warps into [row][HD] (in place of warp 0's)
    for (uint32_t i = threadIdx.x; i < (last + 1) * HD; i += AQ_WARPS * 32) {
        const uint32_t r = i / HD;
        float M = s_m[0][r];
#pragma unroll
        for (int w = 1; w < AQ_WARPS; w++) M = fmaxf(M, s_m[w][r]);
        const float use = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < AQ_WARPS; w++) {
            const float f = ex2(s_m[w][r] - use);
            L += s_l[w][r] * f;
            o += part[w * ROWS * HD + i] * f;
        }
        part[i] = o;
        if (i % HD == 0) { s_top[r] = M; s_sum[r] = L; }
    }
    T* out = reinterpret_cast<T*>(a.out);
    if (n_splits == 1) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < (last + 1) * HD; i += AQ_WARPS * 32) {
            const uint32_t r = i / HD;
            const float L = s_sum[r];
            out[q_index(r) + i % HD] = Cvt<T>::from_f(L == 0.0f ? 0.0f : part[i] / L);   // a row that sees nothing is zero
        }
        return;
    }
    // ---- and over the splits: every CTA of the cluster finishes its share of the values
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (uint32_t i = split * (AQ_WARPS * 32) + threadIdx.x; i < (last + 1) * HD; i += n_splits * AQ_WARPS * 32) {
        const uint32_t r = i / HD;
        float M = -INFINITY;
        for (uint32_t s = 0; s < n_splits; s++) M = fmaxf(M, *cluster.map_shared_rank(&s_top[r], s));
        const float use = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, o = 0.0f;
        for (uint32_t s = 0; s < n_splits; s++) {
            const float f = ex2(*cluster.map_shared_rank(&s_top[r], s) - use);
            L += *cluster.map_shared_rank(&s_sum[r], s) * f;
            o += *cluster.map_shared_rank(&part[i], s) * f;
        }
        out[q_index(r) + i % HD] = Cvt<T>::from_f(L == 0.0f ? 0.0f : o / L);
    }
    cluster.sync();   // nobody leaves while a peer may still read its results
}

// Splits: as many CTAs as two for every SM, but no fewer than 8 blocks (two a warp) each.
static uint32_t aq_pick_splits(uint64_t units, uint32_t max_blocks) {
    uint32_t s = 1;
    while (s < AQ_MAX_SPLITS && units * s * 2 <= 2 * B200_SMS && max_blocks / (2 * s) >= 8) s *= 2;
    return s;
}

template <typename T, int HD, int PIECES>
static int aq_launch(cudaStream_t st, AqArgs a, uint32_t rows, uint32_t n_splits) {
    constexpr uint32_t ROWS = PIECES == 2 ? 8 : 16;
    using C = AqCfg<HD>;
    constexpr size_t merge = (size_t)AQ_WARPS * ROWS * HD * 4;
    constexpr size_t smem = merge > (size_t)C::RING ? merge : (size_t)C::RING;
    a.q_tiles = cdiv(a.q_len * a.group, ROWS);
    const uint64_t units = (uint64_t)rows * a.kv_heads * a.q_tiles;
    AK_REQUIRE(units <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "ak_attn_decode_paged_q8: %u rows x %u heads x %u tiles of queries are too many for one call", rows,
               a.kv_heads, a.q_tiles);
    if (!n_splits) n_splits = aq_pick_splits(units, a.max_blocks);
    while (n_splits & (n_splits - 1)) n_splits &= n_splits - 1;   // a cluster of a power of two of CTAs
    {
        static bool attr_set[64] = {};
        int dev = 0;
        AK_CUDA(cudaGetDevice(&dev));
        std::lock_guard<std::mutex> lock(device_cache_mutex());
        if (!attr_set[dev & 63]) {
            AK_CUDA(cudaFuncSetAttribute(attn_decode_q8_kernel<T, HD, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            AK_CUDA(cudaFuncSetAttribute(attn_decode_q8_kernel<T, HD, PIECES>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            attr_set[dev & 63] = true;
        }
    }
    return launch_k(attn_decode_q8_kernel<T, HD, PIECES>, dim3((unsigned)units, 1, n_splits), dim3(AQ_WARPS * 32), smem, st,
                    n_splits > 1 ? dim3(1, 1, n_splits) : NO_CLUSTER, a);
}

}  // namespace ak

using namespace ak;
extern "C" int ak_attn_decode_paged_q8(void* stream, const void* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scales, const float* v_scales,
                                       const int32_t* block_tables, const int32_t* kv_lens, void* out, ak_attn_q8_params p) {
    const char* who = "ak_attn_decode_paged_q8";
    AK_REQUIRE(q && block_tables && kv_lens && out, AK_ERR_INVALID_ARG, "%s: null pointer", who);
    AK_TRY(q8_check_cache(who, k_pool, v_pool, k_scales, v_scales, p.heads, p.kv_heads, p.head_dim, p.block_size, p.dtype, p.pool_blocks));
    AK_REQUIRE(q8_aligned(q, 16) && q8_aligned(out, 16) && q8_aligned(block_tables, 4) && q8_aligned(kv_lens, 4), AK_ERR_INVALID_ARG,
               "%s: q and out must be 16-byte aligned, tables and lengths 4-byte", who);
    AK_REQUIRE(p.q_len >= 1 && p.q_len <= 65536, AK_ERR_INVALID_ARG, "%s: q_len must be 1 to 65536 (got %u)", who, p.q_len);
    AK_REQUIRE(p.max_blocks_per_seq >= 1 && p.max_blocks_per_seq <= (1u << 26), AK_ERR_INVALID_ARG, "%s: max_blocks_per_seq must be 1 to 2^26 (got %u)", who,
               p.max_blocks_per_seq);
    AK_REQUIRE(p.n_splits <= AQ_MAX_SPLITS, AK_ERR_INVALID_ARG, "%s: n_splits must be at most %u (got %u)", who, AQ_MAX_SPLITS, p.n_splits);
    if (p.rows == 0) return AK_OK;
    AK_TRY(q8_check_here(out, who));
    const uint32_t group = p.heads / p.kv_heads;
    const AqArgs a{q, k_pool, v_pool, k_scales, v_scales, block_tables, kv_lens, out, p.q_len, p.heads, p.kv_heads, group, 1, p.max_blocks_per_seq,
                   p.pool_blocks, p.scale};
    const bool two = p.dtype == AK_F32 || (uint64_t)p.q_len * group <= 8;
#define AK_ATTN_Q8(HD)                                                                                         \
    return p.dtype == AK_F32 ? aq_launch<float, HD, 2>(as_stream(stream), a, p.rows, p.n_splits)              \
           : two             ? aq_launch<bf16, HD, 2>(as_stream(stream), a, p.rows, p.n_splits)               \
                             : aq_launch<bf16, HD, 1>(as_stream(stream), a, p.rows, p.n_splits)
    switch (p.head_dim) {
        case 32: AK_ATTN_Q8(32);
        case 64: AK_ATTN_Q8(64);
        case 96: AK_ATTN_Q8(96);
        default: AK_ATTN_Q8(128);
    }
#undef AK_ATTN_Q8
}
