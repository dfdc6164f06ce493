// Attention of the newest tokens of every sequence over the 8-bit paged cache.
//
//   o_r = sum_j softmax_j(scale * ks_j (q_r . k_j)) vs_j v_j,   j < limit_r = kv_len - q_len + i + 1 for query i of its sequence
//
// k_j, v_j are int8 rows, ks_j, vs_j their f32 scales. One pass over the cache with the running maximum and sum of the softmax; the
// bytes of the cache are read once and bound the kernel (136 bytes per position and kv head at head size 64, 264 at 128).
//
// Decode has one query per (sequence, head), a group of heads or a few drafted tokens at most 16 or so. mma.sync takes the cache as its 16-row operand and
// the queries as the 8-column one, which with one query per kv head is enough for the bytes (0.96). Groups would fill a tcgen05 tile, 128 positions
// by the digits of 16 queries, with each score in a register once; that form is not built, and instructions hold 16 query rows at 0.57 of the bytes.
// A column pair is one query in two parts, so that the 8 columns are 4 queries:
//   S^T = K q   m16n8k32 on int8 as it lies in the cache. A query is held as integers X = rint(q F), F = 127 * 256^(D - 1) / max|q|, in
//               D signed base-256 digits: 2 for bf16 (16 bits of the head's largest value), 3 for f32 (24 bits). Sums of digits are exact.
//   O^T = V p   m16n8k16 on f16, in which int8 is exact (1024 + 128 + v is put together by a byte permute and 1152 taken off). A weight
//               w = p vs is its leading f16 part and what is left of it, times 2^11 (22 bits together, TWO), or, for bf16 results and more than 4 query
//               rows, the leading part alone (11 bits; the result has 8) with two queries to a column pair.
// What the fewer bits buy: three digits for bf16 too took 1 to 10 % more time (64 x 16 x 128 77.0 us instead of 76.0, 64 x 12 x 64 up to 512 positions 11.6
// instead of 10.5), weights in two parts for 16 query rows 115 us instead of 69. In 64 x 16 x 128 bf16 results differ from those of f32 arithmetic by 3.8e-4 (by
// neighbouring bf16 numbers; 5e-5 with three digits), in 16 query rows by 8e-4 (4.5e-4 with weights in two parts); against 64 bits, whose distance is the
// results' own rounding, all of them are off by 1.7e-3.
// Scores come out with lanes holding positions g, g + 8 of one query, and turn into the second product's operand by a transposition of 8 x 8
// blocks (movmatrix). With the queries as the 16-row operand of f16 products (and keys converted like values) a tile took 370 instructions and 168
// registers instead of 280 and 117, and 64 x 16 heads x 2048 positions x 128 113 us instead of 86.
//
// Weights are 2^(s - m) with a reference m that follows the running maximum only when a score is more than 8 above it: up to then weights
// grow to 2^8, which f16 has room for (they are scaled by a power of two, below 2^13, that follows the largest value scale that the query has met so
// far), and no reduction over the lanes stands between the two products.
//
// Measured (graph of launches on three sets of inputs, cold L2): 64 sequences x 16 heads x 128, 64 to 4096 positions 90 us = 0.96 of the copy
// bandwidth, 2048 each 86 to 91 us; 64 x 12 heads x 64 x 1024, f32 23.4 us = 0.70: bound by instructions there (some 210 a tile of 2176 bytes, issue
// slots three quarters busy); 2 sequences of 60000 x 8 kv heads x 16 query rows 64 us = 0.57: few CTAs, instructions; one sequence of 300 x 5 heads
// 5.7 us, a chain of latencies (the shortest launch takes 1.3).
//
// A CTA takes one (sequence, kv head, tile of queries, split); each warp has every n-th cache block of the split and a ring of cp.async
// stages of its own, no barrier in the loop. The warps' results are merged in shared memory and the splits', which are the CTAs of one
// cluster, through distributed shared memory in split order: no scratch, no atomics, the same bits every time.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <atomic>

#include "kernels.h"
#include "q8.cuh"
#include "tcgen05.cuh"
namespace cg = cooperative_groups;

namespace ak {

constexpr uint32_t AQ_MAX_WARPS = 8;
constexpr uint32_t AQ_MAX_SPLITS = 16;   // CTAs of a cluster (8 is the portable limit, 16 is asked for)

template <int HD> struct AqCfg {
    static constexpr int TILE = 16 * HD;                   // bytes of a block's keys (or values) of one head
    static constexpr int STAGE = 2 * TILE + 128;           // keys | values | 16 key scales | 16 value scales
    static constexpr int STAGES = HD == 128 ? 3 : 4;       // of a warp's ring (3, 4 and 6 are the same to a microsecond at 128: latency is not what bounds it)
    static constexpr int CTAS = HD >= 96 ? 2 : 3;          // of AQ_MAX_WARPS warps that an SM holds: 16 warps (128 registers), 24 (80) up to head size 64
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
__device__ __forceinline__ float lds_f(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
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

// D(16x8, s32) += A(16x32, s8, row) B(32x8, s8, col)
__device__ __forceinline__ void mma_s8(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_first(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
// the transpose of the 8 x 8 block of which lane (g, t) holds row g, columns 2t and 2t + 1
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
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

// The d-index of word w (4 consecutive values) that lane t of a quad holds of a key row: chunk t, then chunk 4 + t (HD 128), an 8-byte piece
// where there are no four chunks. The order in which q . k is summed is free as long as q is laid out alike.
template <int HD> __device__ __forceinline__ uint32_t d_of(uint32_t t, int w) {
    if (HD == 32) return 8 * t + 4 * w;
    if (w < 4) return 16 * t + 4 * w;
    if (HD == 96) return 64 + 8 * t + 4 * (w - 4);
    return 64 + 16 * t + 4 * (w - 4);
}
// A lane's offsets in a tile, the same for every tile. 8 rows further is 8 HD bytes further whatever the permutation.
template <int HD> struct AqLane {
    uint32_t key, key2;       // its first chunk of row g, and its second piece
    uint32_t val, val2;       // its HD / 8 values of rows 2t and 2t + 1
    uint32_t put_k, put_v;    // where it puts the first 16 bytes that it copies
    __device__ __forceinline__ AqLane(uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3, row = lane / (HD / 16), col = lane % (HD / 16);
        key = HD == 32 ? g * 32 + 8 * t : k_at<HD>(g, t);
        key2 = HD == 128 ? k_at<HD>(g, 4 + t) : g * HD + 64 + 8 * t;
        const uint32_t byte = (HD / 8) * g;
        val = HD == 128 || HD == 64 ? v_at<HD>(2 * t, byte >> 4) + (byte & 15) : 2 * t * HD + byte;
        val2 = HD == 128 || HD == 64 ? v_at<HD>(2 * t + 1, byte >> 4) + (byte & 15) : (2 * t + 1) * HD + byte;
        put_k = k_at<HD>(row, col);
        put_v = v_at<HD>(row, col);
    }
    __device__ __forceinline__ void load_key(uint32_t tile, uint32_t (&w)[HD / 16]) const {
        if constexpr (HD == 32) lds_words<2>(tile + key, w);
        else lds_words<4>(tile + key, w);
        if constexpr (HD == 128) lds_words<4>(tile + key2, w + 4);
        if constexpr (HD == 96) lds_words<2>(tile + key2, w + 4);
    }
    __device__ __forceinline__ void load_value(uint32_t at, uint32_t (&w)[HD / 32]) const {
        if constexpr (HD == 96) {
#pragma unroll
            for (int i = 0; i < 3; i++) w[i] = lds32(at + 4 * i);
        } else {
            lds_words<HD / 32>(at, w);
        }
    }
};

template <typename T, int HD, int NQ, bool TWO>
__global__ void __launch_bounds__(AQ_MAX_WARPS * 32, AqCfg<HD>::CTAS)
attn_decode_q8_kernel(const AqArgs a) {
    using C = AqCfg<HD>;
    constexpr int STAGES = C::STAGES;
    // Tiles of a turn of the loop: two share its votes, waits and addresses where the registers allow it (64 x 12 heads x 64 x 1024, f32 24.4 -> 22.6 us,
    // 128 x 5 heads x 32 36.8 -> 33.9; at head size 128 four stages leave room for 12 warps on an SM: 90 -> 101 us).
    constexpr int TURN = HD == 128 || (HD == 64 && NQ == 2) ? 1 : 2;
    constexpr float REST = 2048.0f;                  // what is left of a weight is held times this: at most 2^12, and f16's smallest numbers are of no account
    constexpr int ROWS = 4 * NQ;                     // queries of a tile: NQ column blocks of 4
    constexpr int DIGITS = sizeof(T) == 4 ? 3 : 2;   // of a query
    constexpr int KW = HD / 16, KS = HD / 32;        // words of a key row per lane, steps of K q
    constexpr int NP = TWO ? NQ : NQ / 2;            // column blocks of V p
    constexpr int MT = HD / 16;                      // 16-row tiles of the result
    pdl_wait();
    pdl_trigger();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_m[AQ_MAX_WARPS][ROWS], s_l[AQ_MAX_WARPS][ROWS];
    __shared__ float s_f[AQ_MAX_SPLITS][ROWS];            // factors of the warps' (then of the splits') results
    __shared__ float s_top[AQ_MAX_SPLITS][ROWS], s_sum[AQ_MAX_SPLITS][ROWS], s_unit[ROWS];
    __shared__ uint64_t s_at[ROWS];                       // where a row's query and result begin
    __shared__ __align__(16) int8_t s_q[ROWS][DIGITS == 3 ? 4 : 2][HD];   // digits, the last plane of four is zero

    const uint32_t warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t qt = blockIdx.x % a.q_tiles, kvh = (blockIdx.x / a.q_tiles) % a.kv_heads, seq = blockIdx.x / (a.q_tiles * a.kv_heads);
    const uint32_t split = blockIdx.z, n_splits = gridDim.z;
    const uint32_t total_rows = a.q_len * a.group;
    const int32_t cap = (int32_t)(a.max_blocks * Q8_BS);
    const int32_t* table = a.tables + (size_t)seq * a.max_blocks;
    // Lane j: the cache block of this warp's tile (i & ~31) + j. Without splits the first ones are known before the length is.
    uint32_t ids = 0xffffffffu;
    if (n_splits == 1 && warp + lane * warps < a.max_blocks) ids = (uint32_t)table[warp + lane * warps];
    const int32_t len = a.lens[seq];
    // The first queries are on their way while the length is.
    constexpr int QV = HD / 8;       // values of a row that a thread takes, 8 threads a row
    uint32_t qraw[QV * (int)sizeof(T) / 4];
    auto q_row = [&](uint32_t r) -> uint64_t {   // where row r's query and result begin (row 0's for a row that is not there)
        const uint32_t rr = qt * ROWS + r < total_rows ? qt * ROWS + r : qt * ROWS;
        return (((uint64_t)seq * a.q_len + rr / a.group) * a.heads + (uint64_t)kvh * a.group + rr % a.group) * HD;
    };
    auto q_load = [&](uint64_t at) {
        const uint8_t* qp = reinterpret_cast<const uint8_t*>(a.q) + at * sizeof(T);
        if constexpr (QV * sizeof(T) % 16 == 0) {
#pragma unroll
            for (int e = 0; e < QV * (int)sizeof(T) / 16; e++) {
                const uint4 v = reinterpret_cast<const uint4*>(qp)[e];
                qraw[4 * e] = v.x; qraw[4 * e + 1] = v.y; qraw[4 * e + 2] = v.z; qraw[4 * e + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < QV * (int)sizeof(T) / 8; e++) {
                const uint2 v = reinterpret_cast<const uint2*>(qp)[e];
                qraw[2 * e] = v.x; qraw[2 * e + 1] = v.y;
            }
        }
    };
    uint64_t my_at = 0;
    if (threadIdx.x < ROWS * 8) { my_at = q_row(threadIdx.x >> 3); q_load(my_at + (threadIdx.x & 7) * QV); }


    // ---- positions that row r of the tile may see
    auto limit_of = [&](uint32_t r) -> int32_t {
        const uint32_t rr = qt * ROWS + r;
        if (rr >= total_rows) return 0;
        const int64_t lim = (int64_t)len - a.q_len + rr / a.group + 1;
        return lim < 0 ? 0 : (int32_t)(lim < cap ? lim : cap);
    };
    const uint32_t last = min((uint32_t)ROWS, total_rows - qt * ROWS) - 1;
    const int32_t lim_min = limit_of(0), lim_max = limit_of(last);   // limits grow with the row
    int32_t lim[NQ];
#pragma unroll
    for (int u = 0; u < NQ; u++) lim[u] = limit_of(4 * u + t);

    if (n_splits > 1) cluster_arrive_all();   // "this CTA runs", waited for before the first access to a peer
    // ---- this split's blocks, this warp's share of them
    const uint32_t nblk = ((uint32_t)lim_max + Q8_BS - 1) / Q8_BS;
    const uint32_t per = (nblk + n_splits - 1) / n_splits;
    const uint32_t b_begin = min(split * per, nblk), b_end = min(b_begin + per, nblk);
    const uint32_t first = b_begin + warp;
    const uint32_t mine = first < b_end ? (b_end - first + warps - 1) / warps : 0;
    const uint32_t ring = smem_u32(smem) + warp * (STAGES * C::STAGE);

    // The next tile is asked for, into the next stage of the ring. A block outside the pool holds no positions: bit j of `there` says whether the
    // j-th newest tile is there.
    const AqLane<HD> at_lane(lane);
    const int8_t *my_k = a.k_pool + lane * 16, *my_v = a.v_pool + lane * 16;
    const float* my_s = (lane < 4 ? a.k_scales : a.v_scales) + (lane & 3) * 4;
    uint32_t there = 0, asked = 0, put = ring;
    auto request = [&]() {
        there <<= 1;
        if (asked < mine) {
            if ((asked & 31u) == 0 && (asked > 0 || n_splits > 1)) ids = asked + lane < mine ? (uint32_t)table[first + (asked + lane) * warps] : 0xffffffffu;
            const uint32_t blk = __shfl_sync(0xffffffffu, ids, asked & 31u);
            asked++;
            if (blk < a.pool_blocks) {
                there |= 1u;
                const uint64_t at = (uint64_t)blk * a.kv_heads + kvh;
                const int8_t *ks = my_k + at * C::TILE, *vs = my_v + at * C::TILE;
#pragma unroll
                for (int j = 0; j < HD / 32; j++) {
                    cp_async16(put + at_lane.put_k + 512 * j, ks + 512 * j);
                    cp_async16(put + C::TILE + (HD == 128 ? at_lane.put_v ^ ((j & 1) << 6) : at_lane.put_v) + 512 * j, vs + 512 * j);
                }
                if (lane < 8) cp_async16(put + 2 * C::TILE + lane * 16, my_s + at * Q8_BS);
            }
        }
        put = put == ring + (STAGES - 1) * C::STAGE ? ring : put + C::STAGE;
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - TURN; i++) request();

    // ---- queries: digits into shared memory, for every warp
    for (uint32_t i = threadIdx.x; i < ROWS * 8; i += blockDim.x) {   // whole groups of 8: blockDim.x and ROWS * 8 are multiples of 32
        const uint32_t r = i >> 3, d = (i & 7) * QV;
        const bool have = qt * ROWS + r < total_rows;
        if (i >= blockDim.x) { my_at = q_row(r); q_load(my_at + d); }
        float x[QV];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < QV; e++) {
            if constexpr (sizeof(T) == 4) x[e] = __uint_as_float(qraw[e]);
            else x[e] = __uint_as_float((e & 1) ? qraw[e / 2] & 0xffff0000u : qraw[e / 2] << 16);
            top = max(top, abs_bits(x[e]));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (!have) top = 0;
        // |q| under 1e-30 counts as 0 (F would overflow); a query with an infinity or a NaN has NaN for every score
        const float most = __uint_as_float(top), full = DIGITS == 3 ? 8323072.0f : 32512.0f;   // 127 * 256^(D - 1)
        const bool finite = top < 0x7f800000u, some = finite && most >= Q8_ZERO;
        const float F = some ? full / most : 0.0f;
        if ((i & 7) == 0) {
            s_unit[r] = !finite ? __uint_as_float(0x7fc00000u) : some ? most / full * (a.scale * 1.4426950408889634f) : 0.0f;   // scores in the base-2 domain
            s_at[r] = my_at;
        }
#pragma unroll
        for (int e = 0; e < QV; e += 4) {
            uint32_t dg[3] = {0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int32_t X = some ? __float2int_rn(x[e + j] * F) : 0;
                // signed digits: the low byte as it is, what is left a multiple of 256
#pragma unroll
                for (int k = DIGITS - 1; k > 0; k--) {
                    const int32_t low = (int8_t)X;
                    dg[k] |= ((uint32_t)low & 0xffu) << (8 * j);
                    X = (X - low) >> 8;
                }
                dg[0] |= ((uint32_t)X & 0xffu) << (8 * j);
            }
#pragma unroll
            for (int k = 0; k < DIGITS; k++) *reinterpret_cast<uint32_t*>(&s_q[r][k][d + e]) = dg[k];
            if constexpr (DIGITS == 3) *reinterpret_cast<uint32_t*>(&s_q[r][3][d + e]) = 0;
        }
    }
    __syncthreads();
    // operand lane (g, t): column g = digit g & 1 of query g >> 1 of each block (3 digits: of a second block, digits 2 and the zeros)
    constexpr int QK = DIGITS == 3 ? 2 : 1;
    uint32_t qb[NQ][KS][2 * QK];
    float row_scale[NQ];
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        row_scale[u] = s_unit[4 * u + t];
#pragma unroll
        for (int w = 0; w < KW; w++)
#pragma unroll
            for (int k = 0; k < (DIGITS == 3 ? 2 : 1); k++)
                qb[u][w >> 1][2 * k + (w & 1)] = *reinterpret_cast<const uint32_t*>(&s_q[4 * u + (g >> 1)][2 * k + (g & 1)][d_of<HD>(t, w)]);
    }

    float m_ref[NQ], l_run[NQ];
    int v_exp[NQ];   // a query's weights are p * vs * 2^(5 - v_exp) with vs < 2^v_exp for every finite value scale that it has seen so far
#pragma unroll
    for (int u = 0; u < NQ; u++) {
        const bool sees = lim[u] > 0;   // one that does not never asks for a reference, or a power of two
        m_ref[u] = sees ? -INFINITY : 0.0f;
        v_exp[u] = sees ? -110 : 127;
        if (!sees) row_scale[u] = 0.0f;
        l_run[u] = 0.0f;
    }
    uint32_t get = ring;
    int32_t pos0 = (int32_t)(first * Q8_BS);
    float acc[NP][MT][4];
#pragma unroll
    for (int u = 0; u < NP; u++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[u][j][0] = acc[u][j][1] = acc[u][j][2] = acc[u][j][3] = 0.0f;

    for (uint32_t i = 0; i < mine; i += TURN) {
#pragma unroll
        for (int b = 0; b < TURN; b++) request();
        cp_wait<STAGES - TURN>();
        __syncwarp();
        uint32_t tile[TURN];    // where the turn's tiles are
        int32_t pos[TURN];      // this lane's first position of each (its second is 8 further); none that anybody sees for a tile that is not there
#pragma unroll
        for (int b = 0; b < TURN; b++) {
            tile[b] = get;
            get = get == ring + (STAGES - 1) * C::STAGE ? ring : get + C::STAGE;
            pos[b] = (there >> (STAGES - 1 - b)) & 1u ? pos0 + (int32_t)g : 1 << 30;
            pos0 += (int32_t)(warps * Q8_BS);
        }
        // every row sees all of every tile
        const bool whole = pos0 + (int32_t)(Q8_BS - warps * Q8_BS) <= lim_min && ((there >> (STAGES - TURN)) & ((1u << TURN) - 1)) == (1u << TURN) - 1;
        // ---- S^T = K q: positions g, g + 8 of query t
        int32_t dot[TURN][NQ][QK][4];
        float ks[TURN][2], vs[TURN][2];
#pragma unroll
        for (int b = 0; b < TURN; b++) {
            uint32_t k0[KW], k1[KW];
            at_lane.load_key(tile[b], k0);
            at_lane.load_key(tile[b] + 8 * HD, k1);
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int u = 0; u < NQ; u++)
#pragma unroll
                    for (int d = 0; d < QK; d++) {
                        if (k == 0) mma_s8_first(dot[b][u][d], k0[0], k1[0], k0[1], k1[1], qb[u][0][2 * d], qb[u][0][2 * d + 1]);
                        else mma_s8(dot[b][u][d], k0[2 * k], k1[2 * k], k0[2 * k + 1], k1[2 * k + 1], qb[u][k][2 * d], qb[u][k][2 * d + 1]);
                    }
            const uint32_t sks = tile[b] + 2 * C::TILE + 4 * g;
            ks[b][0] = lds_f(sks); ks[b][1] = lds_f(sks + 32);
            vs[b][0] = lds_f(sks + 64); vs[b][1] = lds_f(sks + 96);
        }
        if (!whole) {   // behind the last row's end may be anything, a NaN for a scale included: nothing of it may move a reference, or the results' last bits
#pragma unroll
            for (int b = 0; b < TURN; b++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (pos[b] + 8 * h >= lim_max) ks[b][h] = vs[b][h] = 0.0f;
        }
        float x[TURN][NQ][2], p[TURN][NQ][2], most = -INFINITY, v_most = 0.0f;   // q . k without scales; exponents 2^..; the largest of these; of the value scales
#pragma unroll
        for (int b = 0; b < TURN; b++) {
            v_most = fmaxf(v_most, fmaxf(fabsf(vs[b][0]), fabsf(vs[b][1])));
#pragma unroll
            for (int u = 0; u < NQ; u++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int32_t two = dot[b][u][0][2 * h] * 256 + dot[b][u][0][2 * h + 1];
                    x[b][u][h] = QK == 2 ? fmaf((float)two, 256.0f, (float)dot[b][u][QK - 1][2 * h]) : (float)two;
                    // (a row without a reference yet has +infinity here for every score)
                    p[b][u][h] = fmaf(x[b][u][h], row_scale[u] * ks[b][h], -m_ref[u]);
                    most = fmaxf(most, p[b][u][h]);
                }
        }
        // A score more than 8 above its row's reference, or a value scale that a row's power of two does not cover yet. (Also by positions that not
        // every row sees: the branch looks again, so that what a row does not see neither moves its reference nor takes bits from its weights.)
        int v_least = v_exp[0];
#pragma unroll
        for (int u = 1; u < NQ; u++) v_least = min(v_least, v_exp[u]);
        if (__any_sync(0xffffffffu, most > 8.0f || v_most >= pow2i(v_least))) {
            float corr[NQ];
#pragma unroll
            for (int u = 0; u < NQ; u++) {
                float mb = -INFINITY, vtop = 0.0f;
#pragma unroll
                for (int b = 0; b < TURN; b++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        p[b][u][h] = x[b][u][h] * (row_scale[u] * ks[b][h]);
                        if (pos[b] + 8 * h < lim[u]) {
                            mb = fmaxf(mb, p[b][u][h]);
                            if (fabsf(vs[b][h]) < INFINITY) vtop = fmaxf(vtop, fabsf(vs[b][h]));
                        }
                    }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
                    vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, o));
                }
                const int ve = (int)(__float_as_uint(vtop) >> 23) - 126;   // vtop < 2^ve
                float regrade = 1.0f;
                if (ve > v_exp[u]) { regrade = ve - v_exp[u] > 120 ? 0.0f : pow2i(v_exp[u] - ve); v_exp[u] = ve; }
                const float m_new = fmaxf(m_ref[u], mb);
                corr[u] = m_new == -INFINITY ? 1.0f : ex2(m_ref[u] - m_new);
                m_ref[u] = m_new;
#pragma unroll
                for (int b = 0; b < TURN; b++)
#pragma unroll
                    for (int h = 0; h < 2; h++) p[b][u][h] -= m_new;
                l_run[u] *= corr[u];
                corr[u] *= regrade;
            }
#pragma unroll
            for (int u = 0; u < NP; u++) {
                const float c0 = TWO ? corr[u] : corr[(2 * u) % NQ], c1 = TWO ? corr[u] : corr[(2 * u + 1) % NQ];
#pragma unroll
                for (int j = 0; j < MT; j++) { acc[u][j][0] *= c0; acc[u][j][1] *= c1; acc[u][j][2] *= c0; acc[u][j][3] *= c1; }
            }
        }
        float w[TURN][NQ][2], vf[NQ];
#pragma unroll
        for (int u = 0; u < NQ; u++) vf[u] = pow2i(5 - v_exp[u]);
#pragma unroll
        for (int b = 0; b < TURN; b++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int u = 0; u < NQ; u++) {
                    p[b][u][h] = ex2(p[b][u][h]);
                    w[b][u][h] = p[b][u][h] * (vs[b][h] * vf[u]);
                }
        if (!whole) {   // positions that a row does not see
#pragma unroll
            for (int b = 0; b < TURN; b++)
#pragma unroll
                for (int u = 0; u < NQ; u++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        if (pos[b] + 8 * h >= lim[u]) p[b][u][h] = w[b][u][h] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < TURN; b++)
#pragma unroll
            for (int u = 0; u < NQ; u++) l_run[u] += p[b][u][0] + p[b][u][1];   // this lane's positions only: added up over the lanes at the end
#pragma unroll
        for (int b = 0; b < TURN; b++) {
            uint32_t pw[NP][2];
#pragma unroll
            for (int u = 0; u < NP; u++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (TWO) {
                        const float lead = __half2float(__float2half_rn(w[b][u][h]));
                        pw[u][h] = transpose8(pack_half2(lead, (w[b][u][h] - lead) * REST));
                    } else {
                        pw[u][h] = transpose8(pack_half2(w[b][(2 * u) % NQ][h], w[b][(2 * u + 1) % NQ][h]));
                    }
                }
            // ---- O^T += V p (a tile that is not there has weights of 0, and int8 is finite whatever its stage holds)
            const uint32_t vsm = tile[b] + C::TILE;
            uint32_t w0[HD / 32], w1[HD / 32], w2[HD / 32], w3[HD / 32];
            at_lane.load_value(vsm + at_lane.val, w0);
            at_lane.load_value(vsm + at_lane.val2, w1);
            at_lane.load_value(vsm + at_lane.val + 8 * HD, w2);
            at_lane.load_value(vsm + at_lane.val2 + 8 * HD, w3);
#pragma unroll
            for (int j = 0; j < HD / 32; j++) {
                const uint32_t a0 = w0[j] ^ 0x80808080u, a1 = w1[j] ^ 0x80808080u, a2 = w2[j] ^ 0x80808080u, a3 = w3[j] ^ 0x80808080u;
                // bytes of two positions side by side: values 4j, 4j + 1 and 4j + 2, 4j + 3 of the lane's HD / 8
                const uint32_t lo01 = __byte_perm(a0, a1, 0x5140), lo23 = __byte_perm(a0, a1, 0x7362);
                const uint32_t hi01 = __byte_perm(a2, a3, 0x5140), hi23 = __byte_perm(a2, a3, 0x7362);
                const uint32_t x0 = half2_of(lo01, 0x4140), x1 = half2_of(lo01, 0x4342), x2 = half2_of(hi01, 0x4140), x3 = half2_of(hi01, 0x4342);
                const uint32_t y0 = half2_of(lo23, 0x4140), y1 = half2_of(lo23, 0x4342), y2 = half2_of(hi23, 0x4140), y3 = half2_of(hi23, 0x4342);
#pragma unroll
                for (int u = 0; u < NP; u++) {
                    mma_f16(acc[u][2 * j], x0, x1, x2, x3, pw[u][0], pw[u][1]);
                    mma_f16(acc[u][2 * j + 1], y0, y1, y2, y3, pw[u][0], pw[u][1]);
                }
            }
        }
        __syncwarp();
    }
    cp_wait<0>();

    // ---- the warps' results, in true units, over the ring: [warp][row][HD]
#pragma unroll
    for (int u = 0; u < NQ; u++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l_run[u] += __shfl_xor_sync(0xffffffffu, l_run[u], o);
        if (g == 0) { s_m[warp][4 * u + t] = m_ref[u]; s_l[warp][4 * u + t] = l_run[u]; }
    }
    __syncthreads();   // every warp is done with its ring
    float* part = reinterpret_cast<float*>(smem);
    {
        float un[NQ];
#pragma unroll
        for (int u = 0; u < NQ; u++) un[u] = pow2i(v_exp[u] - 5);
        float* wp = part + (size_t)warp * ROWS * HD + (HD / 8) * g;
        // rows g and g + 8 of tile j are values 2j and 2j + 1 of the lane's HD / 8, columns 2t and 2t + 1 the parts of a query or two queries
#pragma unroll
        for (int u = 0; u < NP; u++)
#pragma unroll
            for (int j = 0; j < MT; j++) {
                if constexpr (TWO) {
                    *reinterpret_cast<float2*>(wp + (4 * u + t) * HD + 2 * j) =
                        make_float2(fmaf(acc[u][j][1], 1.0f / REST, acc[u][j][0]) * un[u], fmaf(acc[u][j][3], 1.0f / REST, acc[u][j][2]) * un[u]);
                } else {
                    *reinterpret_cast<float2*>(wp + (8 * u + t) * HD + 2 * j) = make_float2(acc[u][j][0] * un[(2 * u) % NQ], acc[u][j][2] * un[(2 * u) % NQ]);
                    *reinterpret_cast<float2*>(wp + (8 * u + 4 + t) * HD + 2 * j) = make_float2(acc[u][j][1] * un[(2 * u + 1) % NQ], acc[u][j][3] * un[(2 * u + 1) % NQ]);
                }
            }
    }
    __syncthreads();
    if (n_splits > 1) cluster_wait_all();
    // ---- merged over the warps, and stored or (with splits) put in place of warp 0's
    if (threadIdx.x < ROWS) {
        const uint32_t r = threadIdx.x;
        float M = s_m[0][r], L = 0.0f;
        for (uint32_t w = 1; w < warps; w++) M = fmaxf(M, s_m[w][r]);
        const float use = M == -INFINITY ? 0.0f : M;
        for (uint32_t w = 0; w < warps; w++) L += s_l[w][r] * ex2(s_m[w][r] - use);
        const float norm = n_splits > 1 ? 1.0f : (L == 0.0f ? 0.0f : 1.0f / L);   // a row that sees nothing is zero
        for (uint32_t w = 0; w < warps; w++) s_f[w][r] = ex2(s_m[w][r] - use) * norm;
        if (n_splits > 1) {   // to every CTA of the cluster (which all run by now: see the arrival above)
            cg::cluster_group cluster = cg::this_cluster();
            for (uint32_t k = 0; k < n_splits; k++) {
                *cluster.map_shared_rank(&s_top[split][r], k) = M;
                *cluster.map_shared_rank(&s_sum[split][r], k) = L;
            }
        }
    }
    __syncthreads();
    T* out = reinterpret_cast<T*>(a.out);
    auto store = [&](uint32_t r, uint32_t d, float4 o) {
        T* dst = out + s_at[r] + d;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(dst) = o;
        } else {
            const bf162 x = __floats2bfloat162_rn(o.x, o.y), y = __floats2bfloat162_rn(o.z, o.w);
            *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
        }
    };
    for (uint32_t i = threadIdx.x; i < (last + 1) * (HD / 4); i += blockDim.x) {
        const uint32_t r = i / (HD / 4);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t w = 0; w < warps; w++) {
            const float4 v = *reinterpret_cast<const float4*>(part + w * ROWS * HD + 4 * i);
            const float f = s_f[w][r];
            o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
        }
        if (n_splits == 1) store(r, 4 * i % HD, o);
        else *reinterpret_cast<float4*>(part + 4 * i) = o;
    }
    if (n_splits == 1) return;
    // ---- and over the splits: every CTA of the cluster finishes its share of the values
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < ROWS) {
        const uint32_t r = threadIdx.x;
        float M = -INFINITY, L = 0.0f;
        for (uint32_t k = 0; k < n_splits; k++) M = fmaxf(M, s_top[k][r]);
        const float use = M == -INFINITY ? 0.0f : M;
        for (uint32_t k = 0; k < n_splits; k++) {
            s_f[k][r] = ex2(s_top[k][r] - use);
            L += s_sum[k][r] * s_f[k][r];
        }
        s_l[0][r] = L == 0.0f ? 0.0f : 1.0f / L;
    }
    __syncthreads();
    for (uint32_t i = split * blockDim.x + threadIdx.x; i < (last + 1) * (HD / 4); i += n_splits * blockDim.x) {
        const uint32_t r = i / (HD / 4);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t k = 0; k < n_splits; k++) {
            const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part + 4 * i, k));
            const float f = s_f[k][r];
            o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
        }
        const float norm = s_l[0][r];
        store(r, 4 * i % HD, make_float4(o.x * norm, o.y * norm, o.z * norm, o.w * norm));
    }
    cluster.sync();   // nobody leaves while a peer may still read its results
}

// ============================================================================ launch
constexpr uint32_t AQ_ALONE = 120 * 1024;   // bytes of shared memory with which a CTA has an SM to itself

template <typename T, int HD, int NQ, bool TWO> struct AqForm {
    static constexpr uint32_t ROWS = 4 * NQ;
    using C = AqCfg<HD>;
    static constexpr size_t MERGE = (size_t)ROWS * HD * 4, RING = (size_t)C::STAGES * C::STAGE, PER_WARP = MERGE > RING ? MERGE : RING;
    static constexpr size_t MOST = PER_WARP * AQ_MAX_WARPS > AQ_ALONE ? PER_WARP * AQ_MAX_WARPS : AQ_ALONE;
    static size_t smem(uint32_t warps, bool alone) { return alone && PER_WARP * warps < AQ_ALONE ? AQ_ALONE : PER_WARP * warps; }

    // Clusters of n CTAs of 8 warps that the device holds at once (asked for once; `alone`: one CTA on an SM).
    static int room(int dev, uint32_t n, bool alone, uint32_t& clusters) {
        static std::atomic<int> known[64][2][AQ_MAX_SPLITS + 1] = {};   // one more than the number
        int k = known[dev & 63][alone][n].load(std::memory_order_relaxed);
        if (!k) {
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
            attr.val.clusterDim.z = n;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(B200_SMS, 1, n);
            cfg.blockDim = dim3(AQ_MAX_WARPS * 32);
            cfg.dynamicSmemBytes = smem(AQ_MAX_WARPS, alone);
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int num = 0;
            AK_CUDA(cudaOccupancyMaxActiveClusters(&num, attn_decode_q8_kernel<T, HD, NQ, TWO>, &cfg));
            known[dev & 63][alone][n].store(k = num + 1, std::memory_order_relaxed);
        }
        clusters = (uint32_t)(k - 1);
        return AK_OK;
    }
};

// Warps of a CTA, splits of a sequence, and whether its CTAs get an SM each.
//
// 8 warps instead of 4 where the sequences are long (128 blocks and more: the CTAs' starts and ends weigh less; 64 x 16 heads x 128 up to
// 4096 positions 90 against 95 us, but 64 x 12 heads x 64 up to 512 16.4 against 13.0) or where all of them fit at once (8 x 12 heads 6.0 against
// 6.6 us).
//
// Splits: the number with the shortest estimate, in us, for sequences that fill half of their tables, fitted to 1 to 24 sequences of 500 to
// 60000 positions: a wave of k CTAs on an SM takes 5 (clusters 6 and 0.06 for every CTA), and for each of a warp's tiles 0.2 + 0.002 HD times k
// (1.15 for one alone: latency), or what its bytes take at 6.5 MB/us (once for all tiles of queries). Clusters share SMs before all are taken: `alone`
// keeps a second CTA off an SM where all clusters find room like that. Measured whole and in what it picks: 1 x 12 heads x 64 x 4000 18.3 and
// 8.4 us (8), 2 x 5 x 32 x 9000 9.0 (9), 5 x 8 kv heads x 128 x 30000 120 and 53 (3; 60 in 4), 24 x 8 x 128 x 6000 52 whole, 63 in 2. Over 108 shapes
// it is 4 % from the best number on average, 19 % at most (4 x 12 x 64 x 8000).
// Tables much wider than the sequences cost: 100 positions each in tables of 4096 and more instead of 112, 1 x 12 heads x 64 6.8 us instead of 4.9 and
// 4 x 12 7.9 instead of 5.0 (splits without work), 64 x 12 12.3 instead of 6.6 (8 warps instead of 4); 1000 positions 64 x 12 22.6 instead of 18.8. The
// lengths are on the device, where a launch cannot be shaped by them.
template <typename F, int HD>
static int aq_plan(uint64_t units, uint32_t q_tiles, uint32_t max_blocks, uint32_t& warps, uint32_t& n_splits, bool& alone) {
    const uint32_t cap = F::C::CTAS * B200_SMS;   // CTAs of 8 warps on all SMs
    warps = max_blocks >= 128 || units <= cap ? 8 : 4;
    alone = false;
    if (n_splits == 1 || (n_splits == 0 && warps == 4)) { n_splits = 1; return AK_OK; }
    const float tile = 0.2f + 0.002f * HD, bytes = 8.0f * F::C::STAGE / (6.5e6f * (float)q_tiles);
    const uint32_t blocks = (max_blocks + 1) / 2;
    int dev = 0;
    AK_CUDA(cudaGetDevice(&dev));
    float best = 1e30f;
    uint32_t pick = 1;
    for (uint32_t n = n_splits ? n_splits : 1; n <= (n_splits ? n_splits : AQ_MAX_SPLITS) && (n == 1 || n_splits || blocks >= n * 8); n++) {
        uint32_t room = cap, lone = 0;
        if (n > 1) {
            AK_TRY(F::room(dev, n, true, lone));
            AK_TRY(F::room(dev, n, false, room));
            if (room == 0) continue;
        }
        const bool one = n > 1 && units <= lone;
        const float tiles = (float)cdiv(blocks, n * warps), fixed = n == 1 ? 5.0f : 6.0f + 0.06f * n;
        auto wave = [&](uint64_t u) {
            const uint32_t deep = (uint32_t)((u * n + B200_SMS - 1) / B200_SMS), k = one ? 1 : n > 1 && deep < 2 ? 2 : deep;
            const float work = tile * (k > 1 ? (float)k : 1.15f), flow = bytes * (float)(u * n);
            return fixed + tiles * (work > flow ? work : flow);
        };
        const uint64_t full = units / room;
        const float t = (float)full * wave(room) + (units % room ? wave(units % room) : 0.0f);
        if (t < 0.97f * best) { best = t; pick = n; alone = one; }
    }
    n_splits = pick;
    return AK_OK;
}

template <typename T, int HD, int NQ, bool TWO>
static int aq_launch(cudaStream_t st, AqArgs a, uint32_t rows, uint32_t n_splits) {
    using F = AqForm<T, HD, NQ, TWO>;
    a.q_tiles = cdiv(a.q_len * a.group, F::ROWS);
    const uint64_t units = (uint64_t)rows * a.kv_heads * a.q_tiles;
    AK_REQUIRE(units <= 0x7fffffffu, AK_ERR_UNSUPPORTED, "ak_attn_decode_paged_q8: %u rows x %u heads x %u tiles of queries are too many for one call", rows,
               a.kv_heads, a.q_tiles);
    static bool set[64] = {};
    AK_TRY(q8_allow_smem(attn_decode_q8_kernel<T, HD, NQ, TWO>, set, (uint32_t)F::MOST, true));
    uint32_t warps;
    bool alone;
    AK_TRY((aq_plan<F, HD>(units, a.q_tiles, a.max_blocks, warps, n_splits, alone)));
    return launch_k(attn_decode_q8_kernel<T, HD, NQ, TWO>, dim3((unsigned)units, 1, n_splits), dim3(warps * 32), F::smem(warps, alone), st,
                    n_splits > 1 ? dim3(1, 1, n_splits) : NO_CLUSTER, a);
}

// The query rows of a kv head choose the form: f32, and up to 4 rows, go 4 to a CTA with weights in two parts, bf16 with more rows 8 to a CTA with the
// leading part. Further tiles of queries read the cache again, from L2 mostly: 16 rows as one tile (168 registers, 12 warps on an SM)
// took 71 us where two tiles of 8 take 63 (2 sequences of 60000, 8 kv heads x 128).
template <int HD>
static int aq_form(cudaStream_t st, const AqArgs& a, const ak_attn_q8_params& p) {
    if (p.dtype == AK_F32) return aq_launch<float, HD, 1, true>(st, a, p.rows, p.n_splits);
    if ((uint64_t)a.q_len * a.group <= 4) return aq_launch<bf16, HD, 1, true>(st, a, p.rows, p.n_splits);
    return aq_launch<bf16, HD, 2, false>(st, a, p.rows, p.n_splits);
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
    AK_REQUIRE(p.q_len >= 1 && (uint64_t)p.q_len * p.heads <= (1u << 24), AK_ERR_INVALID_ARG, "%s: q_len (%u) must be positive, q_len * heads at most 2^24", who,
               p.q_len);
    AK_REQUIRE(p.max_blocks_per_seq >= 1 && p.max_blocks_per_seq <= (1u << 26), AK_ERR_INVALID_ARG, "%s: max_blocks_per_seq must be 1 to 2^26 (got %u)", who,
               p.max_blocks_per_seq);
    AK_REQUIRE(p.n_splits <= AQ_MAX_SPLITS, AK_ERR_INVALID_ARG, "%s: n_splits must be at most %u (got %u)", who, AQ_MAX_SPLITS, p.n_splits);
    if (p.rows == 0) return AK_OK;
    AK_TRY(q8_check_here(out, who));
    const uint32_t group = p.heads / p.kv_heads;
    const AqArgs a{q, k_pool, v_pool, k_scales, v_scales, block_tables, kv_lens, out, p.q_len, p.heads, p.kv_heads, group, 1, p.max_blocks_per_seq,
                   p.pool_blocks, p.scale};
    switch (p.head_dim) {
        case 32: return aq_form<32>(as_stream(stream), a, p);
        case 64: return aq_form<64>(as_stream(stream), a, p);
        case 96: return aq_form<96>(as_stream(stream), a, p);
        default: return aq_form<128>(as_stream(stream), a, p);
    }
}
