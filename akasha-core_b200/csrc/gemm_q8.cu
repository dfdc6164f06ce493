// 8-bit tensor-core product for sm_100a:  C[m,n] (op)= (sum_k A[m,k] W[n,k]) * sa[m] * sw[n],  A and W int8, sums exact in 32-bit integers.
//
// tcgen05.mma.kind::i8: one MMA takes 32 values of K, so a 128-byte row of a staged tile is 128 values, and everything that moves bytes is as in
// the bf16 product: both operands K-major, tiles staged by TMA with the 128-byte swizzle (the tensor maps see pairs of int8 as one 16-bit
// element), accumulators in TMEM, read back with tcgen05.ld. A sum of k products is at most 2^14 k in size: exact for k up to 131056 (the
// largest multiple of 16 below 2^17). It is converted to f32 (one rounding above 2^24), multiplied by the row's and then the column's scale.
//
// Two kernels: a CTA pair on 256 x 256 tiles, persistent, for large m; one CTA per tile of 128 rows and 16 to 256 columns, K split over the CTAs of a
// cluster, for the rest.
// Integer sums do not depend on their order: a row's result is the same whatever shares the launch, split or not.
//
// Nothing is read before griddepcontrol.wait: the weights may be the result of the kernel just before (ak_rmsnorm_q8 quantises them as well).
// Every mbarrier wait is bounded; where one runs out a status word is set and the CTA leaves through the common exit, which frees its TMEM.
#include "gemm_epi.cuh"
#include "kernels.h"
#include "q8.cuh"
#include "tcgen05.cuh"
#include "tma.h"

#include <cooperative_groups.h>
namespace cg = cooperative_groups;

namespace ak {

__device__ unsigned int g_gemm_q8_status = 0;

constexpr uint32_t I8_M = 128;         // rows of a CTA's tile
constexpr uint32_t I8_KB = 128;        // values (= bytes) of K per block
constexpr uint32_t I8_MAX_STAGES = 12;
constexpr uint32_t I8_THREADS = 192;

struct I8Scales {
    const float *a, *w;   // [m], [n]
};

// The scales of W consecutive columns from `col` on, 0 past n (col % 4 == 0). `vec`: the array is 16-byte aligned.
template <int W>
__device__ __forceinline__ void col_scales(const float* w, uint32_t col, uint32_t n, bool vec, float (&s)[W]) {
    if (vec && col + W <= n) {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(w + col + j);
            s[j] = v.x; s[j + 1] = v.y; s[j + 2] = v.z; s[j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; j++) s[j] = col + j < n ? w[col + j] : 0.0f;
    }
}

// The sum of products to f32, times the row's and then the column's scale, every operation rounded: none of them is fused with an addition behind it, so that
// a result has the same bits whichever way it takes to memory (the tensor memory accelerator's addition, a vector, one element).
__device__ __forceinline__ float i8_scaled(int32_t sum, float sa, float sw) { return __fmul_rn(__fmul_rn((float)sum, sa), sw); }

// One result, with the epilogue's operation; `old` is what it is added to.
template <int EPI>
__device__ __forceinline__ void store_one(const GemmEpi& ep, uint32_t row, uint32_t col, float v, float old) {
    const size_t at = (size_t)row * ep.ldc + col;
    if constexpr (EPI == AK_EPI_STORE_F32) reinterpret_cast<float*>(ep.c)[at] = v;
    else if constexpr (EPI == AK_EPI_ADD_F32) reinterpret_cast<float*>(ep.c)[at] = __fadd_rn(v, old);
    else reinterpret_cast<bf16*>(ep.c)[at] = __float2bfloat16_rn(EPI == AK_EPI_SILU_BF16 ? epi_silu(v) : v);
}
// 16 columns of a warp's 32 rows where rows are not aligned for vectors (an odd pitch, the last columns): turned in shared memory (32 x 17 floats) so
// that an instruction writes 16 neighbouring elements of two rows instead of one element of 32 (bf16, 6576 x 82 x 256: 11.2 us that way, 4.3 like
// this; 8000 x 8001 x 1024: 631 and 119, and 64 through TMA with a pitch of 8008). 32 columns at a time, whose rows rotate instead of being padded,
// cost 6 % more.
template <int EPI>
__device__ __forceinline__ void store_rows16(const GemmEpi& ep, float* buf, uint32_t row0, uint32_t m, uint32_t col0, uint32_t n, const float* v, uint32_t lane) {
    const uint32_t r0 = row0 + (lane >> 4), col = col0 + (lane & 15);
    float old[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; i++) {   // all asked for before the first is needed
        old[i] = 0.0f;
        if constexpr (EPI == AK_EPI_ADD_F32)
            if (r0 + 2 * i < m && col < n) old[i] = reinterpret_cast<const float*>(ep.c)[(size_t)(r0 + 2 * i) * ep.ldc + col];
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; j++) buf[lane * 17 + j] = v[j];
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 16; i++)
        if (r0 + 2 * i < m && col < n) store_one<EPI>(ep, r0 + 2 * i, col, buf[((lane >> 4) + 2 * i) * 17 + (lane & 15)], old[i]);
}

// ============================================================================ one CTA per tile
// grid = (n tiles, m tiles, ks), cluster = (1, 1, ks): the CTAs of a cluster take a part of K each, push the column slice that a peer owns
// into its shared memory, and every one adds up and stores its own slice.
// Warp 0 = TMA producer, warp 1 = MMA issuer (+ TMEM), warps 2-5 = epilogue, one TMEM lane quadrant each.
template <int EPI, bool SPLIT>
__global__ void __launch_bounds__(I8_THREADS)
gemm_q8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmEpi ep, const I8Scales sc, uint32_t m, uint32_t n,
               uint32_t k, uint32_t bn, uint32_t stages, uint32_t tmem_cols, uint32_t a_rows, uint32_t a_box) {
    // bn: columns of the tile, a multiple of 16 up to 256. a_rows: rows of an activation slot. The MMA reads 128 rows from its start; what
    // follows the box feeds accumulator rows that are never stored.
    const uint32_t B_BYTES = bn * I8_KB;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[I8_MAX_STAGES], empty_bar[I8_MAX_STAGES], acc_bar, xch_bar;
    __shared__ uint32_t tmem_base_sm, fail_flag;

    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ks = SPLIT ? cluster.num_blocks() : 1u, rank = SPLIT ? cluster.block_rank() : 0u;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t a_bytes = a_rows * I8_KB, stage_tx = a_box * I8_KB + B_BYTES;
    uint8_t* const b_base = smem + (size_t)stages * a_bytes;
    const uint32_t overrun = (I8_M - a_rows) * I8_KB, b_total = stages * B_BYTES;
    int32_t* red = reinterpret_cast<int32_t*>(b_base + b_total + (overrun > b_total ? overrun - b_total : 0u));   // exchange buffer [ks][a_rows][bn / ks]
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t m0 = blockIdx.y * I8_M, n0 = blockIdx.x * bn;
    const uint32_t kb_total = (k + I8_KB - 1) / I8_KB, per = (kb_total + ks - 1) / ks;
    const uint32_t kb_begin = min(rank * per, kb_total), num_kb = min(per, kb_total - kb_begin);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < stages; s++) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        mbar_init(&acc_bar, 1);
        mbar_init(&xch_bar, 1);
        fail_flag = 0;
        mbar_fence_init();
        // the slices that the peers will push: bn / ks columns of every valid row from each of them (armed before the start barrier)
        if (SPLIT) mbar_expect_tx(&xch_bar, (ks - 1) * min(m - m0, I8_M) * (bn / ks) * 4u);
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_sm, tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    if (SPLIT) cluster_arrive_all();   // "this CTA runs"; waited for right before the exchange
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_sm;
    pdl_trigger();
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (uint32_t i = 0; i < num_kb; i++) {
                if (i >= stages && !mbar_wait(&empty_bar[s], ph ^ 1u)) { atomicExch(&fail_flag, 1u); break; }
                mbar_expect_tx(&full_bar[s], stage_tx);
                const int32_t kx = (int32_t)((kb_begin + i) * (I8_KB / 2));   // in 16-bit elements
                tma_load_2d(smem + (size_t)s * a_bytes, &tmA, kx, (int32_t)m0, &full_bar[s]);
                tma_load_2d(b_base + (size_t)s * B_BYTES, &tmB, kx, (int32_t)n0, &full_bar[s]);
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        const uint32_t idesc = make_idesc_i8(I8_M, bn);
        uint32_t s = 0, ph = 0;
        const uint64_t da0 = make_smem_desc(smem_u32(smem)), db0 = make_smem_desc(smem_u32(b_base));
        const uint32_t da_step = a_bytes >> 4;
        for (uint32_t i = 0; i < num_kb; i++) {
            if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], ph))) { if (lane == 0) atomicExch(&fail_flag, 2u); break; }
            tc_fence_after();
            const uint64_t da = da0 + s * da_step, db = db0 + s * (B_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
                for (uint32_t kk = 0; kk < I8_KB / 32; kk++)   // 32 values = 32 bytes along K: +2 in the descriptor's address field
                    tc_mma_i8(tmem_base, da + (uint64_t)(kk * 2), db + (uint64_t)(kk * 2), idesc, (i == 0 && kk == 0) ? 0u : 1u);
                if (num_kb > stages) tc_commit(&empty_bar[s]);
                if (i + 1 == num_kb) tc_commit(&acc_bar);
            }
            __syncwarp();
            if (++s == stages) { s = 0; ph ^= 1u; }
        }
        if (num_kb == 0 && lane == 0) mbar_arrive(&acc_bar);   // no part of K is left for this CTA: it contributes zeros
    }

    const uint32_t quad = warp & 3u, trow = quad * 32 + lane, row = m0 + trow;
    const bool vec = q8_aligned_dev(sc.w);
    bool got = true;
    float sw[16];   // the next columns' scales are on their way while these are used
    const float sa = (warp >= 2 && row < m) ? sc.a[row] : 0.0f;
    if (warp >= 2) {
        if (!SPLIT) col_scales<16>(sc.w, n0, n, vec, sw);
        got = mbar_wait(&acc_bar, 0);
        if (!got && lane == 0) atomicExch(&fail_flag, 3u);
        got = __all_sync(0xffffffffu, got);
        tc_fence_after();
    }
    if (!SPLIT) {
        if (warp >= 2 && got) {
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < bn; c0 += 16) {
                uint32_t r[16];
                float v[16];
                tmem_ld16(tmem_base + ((quad * 32u) << 16) + c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = i8_scaled((int32_t)r[j], sa, sw[j]);
                if (c0 + 16 < bn) col_scales<16>(sc.w, n0 + c0 + 16, n, vec, sw);
                // (the ring's first 16 KB are free by now: every MMA has read its operands)
                if (n0 + c0 + 16 <= n && (ep.ldc & 7u) == 0) epi_store16<EPI>(ep, row, row < m, n0 + c0, v, n, lane);
                else store_rows16<EPI>(ep, reinterpret_cast<float*>(smem) + quad * (32 * 17), m0 + quad * 32, m, n0 + c0, n, v, lane);
            }
        }
    } else {
        const uint32_t SL = bn / ks;   // columns of a slice, a multiple of 4
        cluster_wait_all();                      // every peer runs
        if (warp >= 2 && got) {
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < bn; c0 += 16) {
                uint32_t r[16];
                if (num_kb > 0) {
                    tmem_ld16(tmem_base + ((quad * 32u) << 16) + c0, r);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j++) r[j] = 0u;
                }
                if (row < m) {
#pragma unroll
                    for (uint32_t j = 0; j < 16; j += 4) {
                        const uint32_t col = c0 + j, dest = col / SL, off = col - dest * SL;
                        int32_t* slot = red + ((size_t)rank * a_rows + trow) * SL + off;
                        if (dest == rank) *reinterpret_cast<uint4*>(slot) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                        else st_async_v4(map_to_cta(smem_u32(slot), dest), r[j], r[j + 1], r[j + 2], r[j + 3], map_to_cta(smem_u32(&xch_bar), dest));
                    }
                }
            }
            // a CTA leaves after it has received everything addressed to it, or through cluster_leave_after_failure: nobody writes into one that is gone
            bool landed = mbar_wait(&xch_bar, 0);
            if (!landed && lane == 0) atomicExch(&fail_flag, 6u);
            got = __all_sync(0xffffffffu, landed);
            const bool vectors = (ep.ldc & 3u) == 0;
            if (got && vectors && row < m) {
#pragma unroll 1
                for (uint32_t j = 0; j < SL; j += 4) {
                    int4 acc = make_int4(0, 0, 0, 0);
                    for (uint32_t src = 0; src < ks; src++) {
                        const int4 p = *reinterpret_cast<const int4*>(red + ((size_t)src * a_rows + trow) * SL + j);
                        acc.x += p.x; acc.y += p.y; acc.z += p.z; acc.w += p.w;
                    }
                    const uint32_t col = n0 + rank * SL + j;
                    float s4[4];
                    col_scales<4>(sc.w, col, n, vec, s4);
                    const float v[4] = {i8_scaled(acc.x, sa, s4[0]), i8_scaled(acc.y, sa, s4[1]), i8_scaled(acc.z, sa, s4[2]), i8_scaled(acc.w, sa, s4[3])};
                    epi_store<EPI, 4>(ep, row, col, v, n);
                }
            }
            if (got && !vectors) {   // an odd pitch: neighbouring lanes take neighbouring columns, of rows that other lanes have put down
                __syncwarp();
#pragma unroll 1
                for (uint32_t i = 0, r = lane / SL, c = lane % SL; i < SL; i++) {
                    const float s_row = __shfl_sync(0xffffffffu, sa, r & 31u);
                    const uint32_t col = n0 + rank * SL + c;
                    const uint32_t row_i = m0 + quad * 32 + r;
                    if (row_i < m && col < n) {
                        int32_t acc = 0;
                        for (uint32_t src = 0; src < ks; src++) acc += red[((size_t)src * a_rows + quad * 32 + r) * SL + c];
                        const float old = EPI == AK_EPI_ADD_F32 ? reinterpret_cast<const float*>(ep.c)[(size_t)row_i * ep.ldc + col] : 0.0f;
                        store_one<EPI>(ep, row_i, col, i8_scaled(acc, s_row, sc.w[col]), old);
                    }
                    for (c += 32; c >= SL; c -= SL) r++;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && fail_flag) atomicExch(&g_gemm_q8_status, fail_flag);
    if (SPLIT && fail_flag) cluster_leave_after_failure(&xch_bar);
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, tmem_cols);
    }
}

// ============================================================================ CTA pair
// Measured (graph of launches): 16384 x 8192 x 2048 184 us = 2990 TOPS with bf16 results, 192 with SiLU, 4001 x 2048 x 8192 added to f32 50 us (128 tiles
// are two turns of 74 pairs, the second one not full); the tensor pipe is busy for 75 % of the cycles, and the power limit takes
// a fifth of the clock in longer runs. What feeds it is the L2: a K block of 64 KB takes a pair 0.39 us, its MMAs 0.27. Below K = 1024 the results
// bound it, 3 us a tile (16 epilogue warps and five stages instead of 8 and six: the same there, 4 % slower for long K): 8000 x 8008 x 1024 bf16 62 us, 0.63 of
// the rate. With 168 registers, 32 of them the columns' scales, the epilogue of bf16 results without an activation spills 4 (16 bytes stored, 44 loaded).
//
// A cluster of two CTAs walks over [256 x 256] tiles: each stages its 128 rows of A and its half (128 rows) of the weight tile per K block, the
// leader issues MMAs of 256 x 256 x 32 that read both CTAs' shared memory, rows 0-127 accumulate in its TMEM and rows 128-255 in the peer's.
// Two accumulator buffers of 256 columns: the epilogue drains one tile while the MMAs of the next run.
//   full[s]       leader's barrier, both CTAs' loads are counted on it;       empty[s]      one per CTA, committed by the leader;
//   acc_full[b]   one per CTA, committed after a tile's last MMA;             acc_empty[b]  leader's, 16 arrivals (8 epilogue warps of each CTA).
constexpr int I8P_BN = 256;
constexpr int I8P_EPI_WARPS = 8;
constexpr int I8P_EPI_COLS = I8P_BN / (I8P_EPI_WARPS / 4);   // of a tile, for each of a lane quadrant's warps
constexpr int I8P_THREADS = 128 + I8P_EPI_WARPS * 32;   // the first warpgroup holds the TMA and the MMA warp
constexpr uint32_t I8P_A_BYTES = I8_M * I8_KB, I8P_STAGE = I8P_A_BYTES + (I8P_BN / 2) * I8_KB;
constexpr uint32_t I8P_OUT_WARP = 32 * 128;             // an epilogue warp's staged piece: 32 rows x 128 bytes

template <int EPI>
__global__ void __launch_bounds__(I8P_THREADS, 1)
gemm_q8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC, const GemmEpi ep,
                    const I8Scales sc, uint32_t m, uint32_t n, uint32_t k, uint32_t stages, uint32_t tiles_n, uint32_t tiles_total, uint32_t tma_out) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[I8_MAX_STAGES], empty_bar[I8_MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base_sm, fail_flag;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t num_kb = (k + I8_KB - 1) / I8_KB;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < stages; s++) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (uint32_t b = 0; b < 2; b++) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * I8P_EPI_WARPS); }
        fail_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        tmem_alloc2(&tmem_base_sm, 2 * I8P_BN);
        tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();   // both hold their TMEM and barriers before either touches the other's
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_sm;
    pdl_trigger();
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0, s = 0, ph = 0;
            bool ok = true;
            for (uint32_t t = pair; t < tiles_total && ok; t += n_pairs) {
                const int32_t m0 = (int32_t)(((t / tiles_n) * 2 + rank) * I8_M), nb0 = (int32_t)((t % tiles_n) * I8P_BN + rank * (I8P_BN / 2));
                for (uint32_t kb = 0; kb < num_kb; kb++, it++) {
                    if (it >= stages && !mbar_wait(&empty_bar[s], ph ^ 1u)) { atomicExch(&fail_flag, 1u); ok = false; break; }
                    uint8_t* dst = smem + (size_t)s * I8P_STAGE;
                    const uint32_t bar = map_to_cta(smem_u32(&full_bar[s]), 0);
                    if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * I8P_STAGE);
                    const int32_t kx = (int32_t)(kb * (I8_KB / 2));
                    tma_load_2d_pair(dst, &tmA, kx, m0, bar);
                    tma_load_2d_pair(dst + I8P_A_BYTES, &tmB, kx, nb0, bar);
                    if (++s == stages) { s = 0; ph ^= 1u; }
                }
            }
            // every commit that the leader addressed to this CTA's empty barriers has landed before the CTA may leave (the last
            // min(it, stages) uses, oldest first)
            if (ok && it > 0) {
                const bool wrapped = it >= stages;
                uint32_t ds = wrapped ? s : 0u, dph = wrapped ? (ph ^ 1u) : 0u;
                for (uint32_t j = 0, cnt = wrapped ? stages : it; j < cnt; j++) {
                    if (!mbar_wait(&empty_bar[ds], dph)) { atomicExch(&fail_flag, 5u); break; }
                    if (++ds == stages) { ds = 0; dph ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc = make_idesc_i8(2 * I8_M, I8P_BN);
            uint32_t tc = 0, s = 0, ph = 0;
            bool ok = true;
            const uint64_t d0 = make_smem_desc(smem_u32(smem));
            const uint32_t empty0 = map_to_cta(smem_u32(&empty_bar[0]), 0), empty1 = map_to_cta(smem_u32(&empty_bar[0]), 1);
            const uint32_t acc_full0 = map_to_cta(smem_u32(&acc_full[0]), 0), acc_full1 = map_to_cta(smem_u32(&acc_full[0]), 1);
            for (uint32_t t = pair; t < tiles_total && ok; t += n_pairs, tc++) {
                const uint32_t buf = tc & 1u, acc_col = tmem_base + buf * I8P_BN;
                if (tc >= 2 && !__all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((tc >> 1) & 1u) ^ 1u))) {
                    if (lane == 0) atomicExch(&fail_flag, 4u);
                    break;
                }
                tc_fence_after();
                for (uint32_t kb = 0; kb < num_kb; kb++) {
                    if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], ph))) { if (lane == 0) atomicExch(&fail_flag, 2u); ok = false; break; }
                    tc_fence_after();
                    const uint64_t da = d0 + s * (uint32_t)(I8P_STAGE >> 4), db = da + (uint32_t)(I8P_A_BYTES >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = 0; kk < I8_KB / 32; kk++)
                            tc_mma2_i8(acc_col, da + (uint64_t)(kk * 2), db + (uint64_t)(kk * 2), idesc, (kb == 0 && kk == 0) ? 0u : 1u);
                        tc_commit2(empty0 + s * 8);   // the stage is reusable in both CTAs once these MMAs have read it
                        tc_commit2(empty1 + s * 8);
                        if (kb + 1 == num_kb) {
                            tc_commit2(acc_full0 + buf * 8);
                            tc_commit2(acc_full1 + buf * 8);
                        }
                    }
                    __syncwarp();
                    if (++s == stages) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp >= 4) {
        // Two warps per lane quadrant, half of the columns each. `tma_out`: pieces of 32 rows x 128 bytes go through a swizzled buffer and
        // leave as TMA stores (or adds into f32); otherwise (pitch of C not a multiple of 16 bytes) from registers.
        const uint32_t quad = warp & 3u, part = (warp - 4) >> 2;
        constexpr bool OUT_BF16 = (EPI == AK_EPI_STORE_BF16 || EPI == AK_EPI_SILU_BF16);
        constexpr uint32_t CW = OUT_BF16 ? 64 : 32;
        uint8_t* const stage_sm = smem + (size_t)stages * I8P_STAGE + (size_t)(warp - 4) * I8P_OUT_WARP;
        const bool vec = q8_aligned_dev(sc.w);
        uint32_t tc = 0;
        for (uint32_t t = pair; t < tiles_total; t += n_pairs, tc++) {
            const uint32_t row0 = ((t / tiles_n) * 2 + rank) * I8_M + quad * 32, row = row0 + lane;
            const uint32_t n0 = (t % tiles_n) * I8P_BN + part * I8P_EPI_COLS;
            const uint32_t acc0 = tmem_base + ((quad * 32u) << 16) + (tc & 1u) * I8P_BN + part * I8P_EPI_COLS;
            const float sa = row < m ? sc.a[row] : 0.0f;
            float sw[32];   // the next columns' scales are on their way while these are used
            col_scales<32>(sc.w, n0, n, vec, sw);
            bool got = mbar_wait(&acc_full[tc & 1u], (tc >> 1) & 1u);
            if (!got && lane == 0) atomicExch(&fail_flag, 3u);
            if (!__all_sync(0xffffffffu, got)) break;
            tc_fence_after();
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < (uint32_t)I8P_EPI_COLS; c0 += 32) {
                uint32_t r[32];
                float v[32];
                tmem_ld32(acc0 + c0, r);
                tmem_ld_wait();
                if (c0 + 32 == (uint32_t)I8P_EPI_COLS) {   // this warp has read its part: the buffer may be written again
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[tc & 1u]), 0));
                }
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = i8_scaled((int32_t)r[j], sa, sw[j]);
                if (c0 + 32 < (uint32_t)I8P_EPI_COLS) col_scales<32>(sc.w, n0 + c0 + 32, n, vec, sw);
                const uint32_t col = n0 + (OUT_BF16 ? (c0 & ~32u) : c0);   // first column of the staged piece
                // a store is clipped at n in whole 16-byte units only: a ragged last piece is stored from registers
                if (!tma_out || (col + CW > n && (n * (OUT_BF16 ? 2u : 4u)) % 16u != 0)) {
                    if (lane == 0) tma_store_wait_read<0>();   // the staging buffer may still be read by an earlier piece's store
#pragma unroll
                    for (int j = 0; j < 32; j += 16) {
                        if (n0 + c0 + j + 16 <= n && (ep.ldc & 7u) == 0) epi_store16<EPI>(ep, row, row < m, n0 + c0 + j, v + j, n, lane);
                        else store_rows16<EPI>(ep, reinterpret_cast<float*>(stage_sm), row0, m, n0 + c0 + j, n, v + j, lane);
                    }
                    continue;
                }
                const bool first_part = !OUT_BF16 || (c0 & 32u) == 0;
                if (first_part) {   // the previous piece has been read out of the buffer
                    if (lane == 0) tma_store_wait_read<0>();
                    __syncwarp();
                }
                uint8_t* const srow = stage_sm + lane * 128;
                if (OUT_BF16) {
#pragma unroll
                    for (int q4 = 0; q4 < 4; q4++) {
                        uint32_t pk[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float t0 = v[8 * q4 + 2 * e], t1 = v[8 * q4 + 2 * e + 1];
                            const bf162 o = (EPI == AK_EPI_SILU_BF16) ? __floats2bfloat162_rn(epi_silu(t0), epi_silu(t1)) : __floats2bfloat162_rn(t0, t1);
                            pk[e] = *reinterpret_cast<const uint32_t*>(&o);
                        }
                        const uint32_t ch = (c0 & 32u) / 8 + q4;
                        *reinterpret_cast<uint4*>(srow + ((ch ^ (lane & 7u)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                    }
                    if (first_part) continue;
                } else {
#pragma unroll
                    for (uint32_t ch = 0; ch < 8; ch++)
                        *reinterpret_cast<float4*>(srow + ((ch ^ (lane & 7u)) << 4)) = make_float4(v[4 * ch], v[4 * ch + 1], v[4 * ch + 2], v[4 * ch + 3]);
                }
                tma_store_fence();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < m && col < n) {
                        if (EPI == AK_EPI_ADD_F32) tma_reduce_add_2d(&tmC, stage_sm, (int32_t)col, (int32_t)row0);
                        else tma_store_2d(&tmC, stage_sm, (int32_t)col, (int32_t)row0);
                    }
                    tma_store_commit();
                }
            }
        }
        if (tma_out && lane == 0) tma_store_wait<0>();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && fail_flag) atomicExch(&g_gemm_q8_status, fail_flag);
    cluster_sync_all();   // nobody frees TMEM or leaves while the pair may still use this CTA's memory
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc2(tmem_base, 2 * I8P_BN);
    }
}

// ============================================================================ launch
constexpr uint32_t I8_SMEM_TWO = 112 * 1024;    // two CTAs fit one SM below this
constexpr uint32_t I8_SMEM_ONE = 220 * 1024;
constexpr uint32_t I8_SMEM_PAIR = 226 * 1024;

struct I8Plan { uint32_t bn, ks, stages; };   // bn = 0: the pair kernel

// Rows of the activation box: a small batch fills only part of the 128-row tile, rows that the box does not fetch cost nothing.
static uint32_t i8_box_rows(uint32_t m) { return m >= I8_M ? I8_M : (m > 64 ? m : (m > 32 ? 64 : (m > 16 ? 32 : 16))); }
static uint32_t i8_slot_rows(uint32_t m) { return (i8_box_rows(m) + 7) / 8 * 8; }   // whole swizzle atoms
static size_t i8_smem(uint32_t stages, uint32_t bn, uint32_t a_rows, bool split) {
    const size_t overrun = (size_t)(I8_M - a_rows) * I8_KB, b_total = (size_t)stages * bn * I8_KB;
    return (size_t)stages * (a_rows + bn) * I8_KB + (overrun > b_total ? overrun - b_total : 0) + (split ? (size_t)a_rows * bn * 4 : 0) + 1024;
}

// Stages of the ring: what is left of an SM, or of half of one, up to the whole part of K.
static uint32_t i8_stages(uint32_t bn, uint32_t ks, uint32_t per, uint32_t a_rows, uint64_t ctas) {
    const size_t room = ctas <= B200_SMS ? I8_SMEM_ONE : I8_SMEM_TWO, stage = (a_rows + bn) * I8_KB, fixed = i8_smem(0, bn, a_rows, ks > 1);
    uint32_t st = fixed < room ? (uint32_t)((room - fixed) / stage) + (uint32_t)((I8_M - a_rows) / bn) : 0;   // weight slots double as the overrun
    if (st > I8_MAX_STAGES) st = I8_MAX_STAGES;
    if (st > per) st = per;
    while (st > 1 && i8_smem(st, bn, a_rows, ks > 1) > room) st--;
    return st;
}

// The shortest of the tile widths, K splits and the pair kernel by what a launch takes, in us. Fitted to 250 measurements of 26 shapes from
// 1 x 2304 x 768 to 2048^3 and 1500 x 1000 x 4000 (a graph of launches, weights of three sets; over these the choice loses 1.2 % on average
// against the best of all, 10 % at most: 64 x 6144 x 2048 7.9 us with tiles of 32 columns, 7.2 with 48; over 80 further shapes of 1 to 128 rows 2 % and 17 %),
// and, between tile and pair, to 291 of 200 to 5000 rows, three epilogues (0.4 % on average, 31 % at most: 5000 x 1000 x 256).
//   tile   2.1, the epilogue 0.01 a column, and per K block of b KB (activation and weight tile) 0.17 + b / 168, the rate of one TMA stream
//          from L2; two CTAs on an SM share 121 KB/us, and every further pair of them starts anew. A split adds its exchange. With several tiles
//          of rows, a million results takes 1.05, a third of the loads' time less; where they are added, 1.6.
//   pair   4.4, and per turn of the 74 pairs 0.40 per K block and what of a tile's 3 us of results that does not cover.
//   Weights come from HBM at 5.5 MB/us at most.
static I8Plan i8_plan(uint32_t m, uint32_t n, uint32_t k, bool add) {
    const uint32_t kb = cdiv(k, I8_KB), mt = cdiv(m, I8_M), ar = i8_slot_rows(m);
    const float rows = (float)(m < I8_M ? m : I8_M), stream = (float)n * k / 5.5e6f;
    I8Plan p{};
    float best = 1e30f;
    if (m > I8_M && n > 128) {
        const float rest = 3.0f - 0.24f * kb;
        best = 4.4f + (float)cdiv64((uint64_t)cdiv(m, 2 * I8_M) * cdiv(n, I8P_BN), B200_SMS / 2) * (kb * 0.40f + (rest > 0.0f ? rest : 0.0f));
    }
    const float out = (float)m * n * (add ? 1.5f : 1.0f) / 0.95e6f;
    for (uint32_t ks = 1; ks <= 8; ks *= 2) {
        const uint32_t per = cdiv(kb, ks), unit = ks > 4 ? 32 : 16;   // a slice of bn / ks columns is whole groups of 4
        if (ks > 1 && (ks - 1) * per >= kb) break;                    // every CTA of a cluster gets work
        for (uint32_t bn = unit; bn <= 256 && bn < n + 16; bn += bn < 128 ? unit : 32) {
            const uint64_t ctas = (uint64_t)mt * cdiv(n, bn) * ks, turns = (ctas + 2 * B200_SMS - 1) / (2 * B200_SMS);
            if (ks > 1 && i8_stages(bn, ks, per, ar, ctas) < (per < 4 ? per : 4)) continue;   // the exchange buffer leaves no ring
            const float b = (float)(ar + bn) * I8_KB * 1e-3f, one = 0.17f + b / 168.0f, two = b / 60.5f;
            const float load = per * (ctas <= B200_SMS ? one : (float)turns * (one > two ? one : two) * (mt > 1 ? 1.08f : 1.0f));
            float t = 2.1f + 0.01f * bn + (float)(turns - 1) * 0.9f + (load > stream ? load + 0.15f * stream : stream + 0.15f * load);
            const float hidden = add ? 0.0f : 0.35f * load;
            if (mt > 1 && out > hidden) t += out - hidden;
            if (ks > 1) t += 0.8f + rows * bn * 4e-3f * (float)(ks - 1) / (float)ks / 7.9f;
            if (t < best) { best = t; p.bn = bn; p.ks = ks; }
        }
    }
    if (!p.bn) return p;
    p.stages = i8_stages(p.bn, p.ks, cdiv(kb, p.ks), ar, (uint64_t)mt * cdiv(n, p.bn) * p.ks);
    return p;
}

template <int EPI, bool SPLIT>
static int i8_launch_tile(cudaStream_t st, const CUtensorMap& tmA, const CUtensorMap& tmB, const GemmEpi& ep, const I8Scales& sc, uint32_t m, uint32_t n, uint32_t k,
                          const I8Plan& p) {
    static bool set[64] = {};
    AK_TRY(q8_allow_smem(gemm_q8_kernel<EPI, SPLIT>, set, I8_SMEM_ONE));
    const uint32_t ar = i8_slot_rows(m);
    uint32_t cols = 32;
    while (cols < p.bn) cols *= 2;
    return launch_k(gemm_q8_kernel<EPI, SPLIT>, dim3(cdiv(n, p.bn), cdiv(m, I8_M), p.ks), dim3(I8_THREADS), i8_smem(p.stages, p.bn, ar, SPLIT), st,
                    dim3(1, 1, p.ks), tmA, tmB, ep, sc, m, n, k, p.bn, p.stages, cols, ar, i8_box_rows(m));
}

template <int EPI>
static int i8_launch_epi(cudaStream_t st, const void* a, const void* wt, const GemmEpi& ep, const I8Scales& sc, uint32_t m, uint32_t n, uint32_t k) {
    CUtensorMap tmA, tmB;
    const I8Plan p = i8_plan(m, n, k, EPI == AK_EPI_ADD_F32);
    if (!p.bn) {
        static bool set[64] = {};
        AK_TRY(q8_allow_smem(gemm_q8_pair_kernel<EPI>, set, I8_SMEM_PAIR));
        constexpr uint32_t OUT = I8P_EPI_WARPS * I8P_OUT_WARP, STAGES = (I8_SMEM_PAIR - 1024 - OUT) / I8P_STAGE;
        static_assert(STAGES >= 2 && STAGES <= I8_MAX_STAGES, "ring of the pair kernel");
        AK_TRY(make_tmap_2d(&tmA, a, 2, k / 2, m, k, I8_KB / 2, I8_M, TMA_SWIZZLE_128B));
        AK_TRY(make_tmap_2d(&tmB, wt, 2, k / 2, n, k, I8_KB / 2, I8P_BN / 2, TMA_SWIZZLE_128B));
        constexpr uint32_t esz = (EPI == AK_EPI_STORE_BF16 || EPI == AK_EPI_SILU_BF16) ? 2 : 4;
        const uint32_t tma_out = ((uint64_t)ep.ldc * esz) % 16 == 0;
        CUtensorMap tmC = tmA;
        if (tma_out) AK_TRY(make_tmap_2d(&tmC, ep.c, esz, n, m, (uint64_t)ep.ldc * esz, 128 / esz, 32, TMA_SWIZZLE_128B));
        const uint32_t tiles_n = cdiv(n, I8P_BN), tiles = tiles_n * cdiv(m, 2 * I8_M), pairs = tiles < B200_SMS / 2 ? tiles : B200_SMS / 2;
        return launch_k(gemm_q8_pair_kernel<EPI>, dim3(2 * pairs), dim3(I8P_THREADS), STAGES * I8P_STAGE + OUT + 1024, st, dim3(2, 1, 1), tmA, tmB, tmC, ep, sc, m,
                        n, k, STAGES, tiles_n, tiles, tma_out);
    }
    AK_TRY(make_tmap_2d(&tmA, a, 2, k / 2, m, k, I8_KB / 2, i8_box_rows(m), TMA_SWIZZLE_128B));
    AK_TRY(make_tmap_2d(&tmB, wt, 2, k / 2, n, k, I8_KB / 2, p.bn, TMA_SWIZZLE_128B));
    return p.ks > 1 ? i8_launch_tile<EPI, true>(st, tmA, tmB, ep, sc, m, n, k, p) : i8_launch_tile<EPI, false>(st, tmA, tmB, ep, sc, m, n, k, p);
}

int gemm_q8_status(unsigned int* out) {
    AK_CUDA(cudaMemcpyFromSymbol(out, g_gemm_q8_status, sizeof(unsigned int)));
    return AK_OK;
}

}  // namespace ak

using namespace ak;
extern "C" int ak_gemm_q8(void* stream, const int8_t* a, const float* a_scales, const int8_t* wt, const float* w_scales, void* c, ak_matmul_meta m,
                          uint32_t epilogue, uint32_t ldc) {
    const char* who = "ak_gemm_q8";
    AK_REQUIRE(a && a_scales && wt && w_scales && c, AK_ERR_INVALID_ARG, "%s: null pointer", who);
    AK_REQUIRE(m.k >= 16 && m.k % 16 == 0 && m.k <= 131056, AK_ERR_UNSUPPORTED, "%s: k (%u) must be a multiple of 16 from 16 to 131056", who, m.k);
    AK_REQUIRE(epilogue <= AK_EPI_SILU_BF16, AK_ERR_INVALID_ARG, "%s: unknown epilogue %u", who, epilogue);
    AK_REQUIRE(ldc >= m.n, AK_ERR_INVALID_ARG, "%s: ldc (%u) must be at least n (%u)", who, ldc, m.n);
    AK_REQUIRE(m.m <= 65535u * I8_M && m.n <= (1u << 30) && ldc <= (1u << 30), AK_ERR_UNSUPPORTED, "%s: %u x %u (pitch %u) is too large", who, m.m, m.n, ldc);
    AK_REQUIRE(q8_aligned(a, 16) && q8_aligned(wt, 16) && q8_aligned(c, 16) && q8_aligned(a_scales, 4) && q8_aligned(w_scales, 4), AK_ERR_INVALID_ARG,
               "%s: operands and output must be 16-byte aligned, scales 4-byte", who);
    if (m.m == 0 || m.n == 0) return AK_OK;
    AK_TRY(q8_check_here(c, who));
    GemmEpi ep{};
    ep.c = c;
    ep.ldc = ldc;
    const I8Scales sc{a_scales, w_scales};
    switch (epilogue) {
        case AK_EPI_STORE_F32: return i8_launch_epi<AK_EPI_STORE_F32>(as_stream(stream), a, wt, ep, sc, m.m, m.n, m.k);
        case AK_EPI_ADD_F32: return i8_launch_epi<AK_EPI_ADD_F32>(as_stream(stream), a, wt, ep, sc, m.m, m.n, m.k);
        case AK_EPI_STORE_BF16: return i8_launch_epi<AK_EPI_STORE_BF16>(as_stream(stream), a, wt, ep, sc, m.m, m.n, m.k);
        default: return i8_launch_epi<AK_EPI_SILU_BF16>(as_stream(stream), a, wt, ep, sc, m.m, m.n, m.k);
    }
}
