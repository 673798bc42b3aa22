// Products of few int8 tokens (up to 128) and a large int8 weight: C[m, n] = sum_k A[m, k] B[n, k], scaled per token and channel.
//
// With so few tokens the weight's bytes are most of the work, and the job is to keep enough of them under way on every
// SM, from the first cycle to the last.  A CTA owns groups of weight rows, as many per group as it takes for the groups to
// cover the SMs once (or a whole number of times); one thread streams them by TMA into a ring that fills the shared
// memory, across the ends of groups, so that no epilogue interrupts the stream.  Between weights of 117 and 176 MB
// that runs at 6.5 TB/s, the rate of a copy; 4 us are spent around it.  What multiplies depends on the tokens:
//
//   up to 16 (or 32)  eight warps with mma.m16n8k32, weight rows as M and tokens as N; they share a stage's KB blocks of K and
//                     its strips of 16 rows, and the sums, whole numbers, are added in shared memory in any order;
//   up to 128         one thread with tcgen05 (kind::i8), tokens as M and weight rows as N, into TMEM.
//
// Against the tiles that serve more tokens (128 x 256 and the like, with K split over a cluster) this saves the padding to 128
// rows, the SMs that 256-row tiles leave without one, and the reduction: 1 x 6144 x 4096 6.8 us (11.0), 16 x 28672 x 4096 21.7
// (26.6), 64 x 6144 x 4096 9.1 (15.9), 128 x 2112 x 7168 12.9 (17.6), 128 x 7168 x 2048 7.3 (18.7); bf16 results, in a stream,
// inputs rotated through more than L2 (the first takes 5.3 to 6.4 where two to four weights take turns).
//
// K is a sum, so its order is free: with mma.m16n8k32, lane (g, t) of a warp takes bytes [32 t, 32 t + 32) of a block's rows,
// for the weight and the tokens alike, as two 16-byte loads without bank conflicts, not the 4-byte pieces that the
// instruction's layout names.
#include <cuda.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "ptx_sm100.cuh"
#include "store_rows.cuh"

using namespace fgptx;

namespace {

constexpr int WARPS = 8;  // that multiply; one more fetches
constexpr int THREADS = 32 * (WARPS + 1);
constexpr int BLOCK_K = 128;
constexpr int MAX_ROWS = 256;
constexpr int MAX_TOKENS = 128;
constexpr int MAX_STAGES = 16;
constexpr int SMEM_BYTES = 224 * 1024;         // ring, sums and alignment
constexpr int STREAM_SMEM_BYTES = 220 * 1024;  // ring, rows behind it and alignment; 5 KB are static

struct StreamArgs {
    FgSkinny p;
    int rows;    // per group, a multiple of 16
    int groups;
    int stages;
    int token_rows;  // int8_stream_kernel: rows of the tokens' box, a multiple of 8
    int c_align;     // int8_stream_kernel: what the rows of p.c begin at multiples of (fg_row_align)
    int wide;  // one load brings all KB blocks of a stage (K a multiple of 128); otherwise each has its own
    // Grouped (int8_skinny_kernel): p.b holds n_experts weights of p.N rows, rows [offs[e - 1], offs[e]) of p.a are expert e's,
    // and an item of work is a group of weight rows of an expert that has rows; groups counts those of one weight.
    const int32_t* offs;
    int n_experts;
    int64_t bias_stride;  // values between the bias rows of consecutive experts (0: one row)
    unsigned int* status;
};

__device__ __forceinline__ float load_bias(const void* p, int dtype, int64_t i) {
    if (dtype == FG_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    if (dtype == FG_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    return reinterpret_cast<const float*>(p)[i];
}

__device__ __forceinline__ float rounded(float v, int dtype) {
    if (dtype == FG_DTYPE_BF16) return __bfloat162float(__float2bfloat16_rn(v));
    if (dtype == FG_DTYPE_F16) return __half2float(__float2half_rn(v));
    return v;
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A barrier of THREADS threads that also tells all of them whether any of them failed.
template <int THREADS>
__device__ __forceinline__ bool any_failed(bool failed) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)failed), "n"(THREADS) : "memory");
    return r != 0u;
}

// A wait ran out somewhere: what is still under way lands before the CTA ends.
__device__ void drain(uint64_t* full_bar, int stages, int issued) {
    uint32_t alone = 0u;
    for (int j = issued > stages ? issued - stages : 0; j < issued; ++j)
        mbar_wait(&full_bar[j % stages], (uint32_t)(j / stages) & 1u, &alone, nullptr, 0, 100000000ull);
}

// `cols` values, a multiple of eight, to a 16-byte boundary.
__device__ __forceinline__ void store_row(uint8_t* to, const float (&v)[32], int cols, int dtype) {
    uint4* o = reinterpret_cast<uint4*>(to);
    if (dtype == FG_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (4 * i < cols) o[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = fg_pair_of(v[8 * i + 2 * j], v[8 * i + 2 * j + 1], dtype);
        if (8 * i < cols) o[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The experts that have rows (up to MOST), in order, into shared memory; returns their number.  Every CTA finds the same.
template <int MOST>
__device__ int experts_with_rows(const int32_t* offs, int n_experts, int rows, int (&id)[MOST], int (&first)[MOST], int (&count)[MOST],
                                 int (&warp_count)[WARPS + 1]) {
    constexpr int EACH = 4;  // experts per lane: up to 1024 by eight warps
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lo[EACH], n[EACH];
    unsigned have[EACH];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int e = (warp * EACH + i) * 32 + lane;
        const bool in = warp < WARPS && e < n_experts;
        lo[i] = in && e > 0 ? min(max(offs[e - 1], 0), rows) : 0;
        n[i] = in ? min(max(offs[e], 0), rows) - lo[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        have[i] = __ballot_sync(0xffffffffu, n[i] > 0);
        mine += __popc(have[i]);
    }
    if (lane == 0) warp_count[warp] = mine;
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) at += warp_count[w];
        all += warp_count[w];
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int to = at + __popc(have[i] & ((1u << lane) - 1u));
        if (n[i] > 0 && to < MOST) {
            id[to] = (warp * EACH + i) * 32 + lane;
            first[to] = lo[i];
            count[to] = n[i];
        }
        at += __popc(have[i]);
    }
    __syncthreads();
    return min(all, MOST);
}

// NT: tiles of eight tokens.  KB: blocks of K per stage; 8 / KB warps share the strips of 16 rows of a block, up to SPW
// each.  Every warp passes every stage, in order.
template <int NT, int SPW, int KB, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 1) int8_skinny_kernel(const __grid_constant__ CUtensorMap tm_w,
                                                                 const __grid_constant__ CUtensorMap tm_x, const StreamArgs a) {
    constexpr int TOKENS = 8 * NT, WS = WARPS / KB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES];
    __shared__ uint32_t abort_word;
    __shared__ float sa_s[TOKENS];
    const FgSkinny& p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w_block = a.rows * BLOCK_K, w_bytes = KB * w_block, stage_bytes = w_bytes + KB * TOKENS * BLOCK_K;
    int* sums = reinterpret_cast<int*>(ring + (size_t)a.stages * stage_bytes);  // [TOKENS][rows]
    volatile uint32_t* abort_flag = &abort_word;
    const int steps = ((int)p.K + KB * BLOCK_K - 1) / (KB * BLOCK_K);  // stages per group
    if (!GROUPED && a.wide && warp == WARPS && lane == 0) {
        // While the kernel before this one drains, the first stages of the weight come as far as L2.
        for (int step = 0; step < min(a.stages, steps); ++step) tma_prefetch_3d(&tm_w, 0, blockIdx.x * a.rows, step * KB);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], WARPS);
        }
        abort_word = 0u;
        fence_mbar_init();
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
    }
    for (int i = threadIdx.x; i < TOKENS * a.rows; i += THREADS) sums[i] = 0;
    __syncthreads();
    fg_pdl_wait();
    __shared__ int ex_id[TOKENS], ex_first[TOKENS], ex_count[TOKENS], warp_count[WARPS + 1];
    int items = a.groups;
    if constexpr (GROUPED) items *= experts_with_rows(a.offs, a.n_experts, (int)p.M, ex_id, ex_first, ex_count, warp_count);

    if (warp == WARPS) {
        if (lane == 0) {
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
                const int ex = GROUPED ? item / a.groups : 0;
                const int w_row = GROUPED ? ex_id[ex] * (int)p.N + item % a.groups * a.rows : item * a.rows, x_row = GROUPED ? ex_first[ex] : 0;
                for (int step = 0; step < steps; ++step) {
                    ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, a.status, 20);
                    if (!ok) break;
                    uint8_t* to = ring + (size_t)stage * stage_bytes;
                    mbar_arrive_expect_tx(&full_bar[stage], (uint32_t)stage_bytes);
                    if (a.wide) {
                        tma_load_3d(to, &tm_w, &full_bar[stage], 0, w_row, step * KB);
                        tma_load_3d(to + w_bytes, &tm_x, &full_bar[stage], 0, x_row, step * KB);
                    } else {
#pragma unroll 1
                        for (int b = 0; b < KB; ++b) {
                            tma_load_3d(to + b * w_block, &tm_w, &full_bar[stage], (step * KB + b) * BLOCK_K, w_row, 0);
                            tma_load_3d(to + w_bytes + b * TOKENS * BLOCK_K, &tm_x, &full_bar[stage], (step * KB + b) * BLOCK_K, x_row, 0);
                        }
                    }
                    ++issued;
                    if (++stage == a.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (*abort_flag) drain(full_bar, a.stages, issued);
        }
        __syncwarp();
        fg_pdl_trigger();  // every load has been issued
    } else {
        const int g = lane >> 2, t = lane & 3, ws = warp % WS, wk = warp / WS;  // strips, block of the stage
        const int strips = a.rows / 16;
        const int off0 = ((2 * t) ^ g) << 4, off1 = ((2 * t + 1) ^ g) << 4;  // the 128-byte swizzle of the copies
        if ((int)threadIdx.x < TOKENS) sa_s[threadIdx.x] = p.sa[p.sa_mode == FG_SCALE_VECTOR && (int)threadIdx.x < p.M ? threadIdx.x : 0];
        const int r = threadIdx.x;  // the row of the group that this thread finishes
        int stage = 0;
        uint32_t phase = 0;
        if constexpr (GROUPED) {  // rows behind the last group are zeros
            const int esz = p.out_dtype == FG_DTYPE_F32 ? 4 : 2;
            for (int64_t row = min(max(a.offs[a.n_experts - 1], 0), (int)p.M) + (int64_t)blockIdx.x; row < p.M; row += gridDim.x) {
                uint16_t* to = reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(p.c) + row * p.ld_c * esz);
                for (int64_t i = threadIdx.x; i < p.N * (esz / 2); i += 32 * WARPS) to[i] = 0;
            }
        }
        for (int item = blockIdx.x; item < items; item += gridDim.x) {
            const int ex = GROUPED ? item / a.groups : 0, expert = GROUPED ? ex_id[ex] : 0, m0 = GROUPED ? ex_first[ex] : 0;
            const int tokens = GROUPED ? ex_count[ex] : (int)p.M;
            const int64_t n = (int64_t)(GROUPED ? item % a.groups : item) * a.rows + r;
            const bool mine = r < a.rows && n < p.N;
            const float sb = mine ? p.sb[p.sb_mode == FG_SCALE_VECTOR ? expert * p.N + n : 0] : 0.0f;
            const float bias = mine && p.bias ? load_bias(p.bias, p.bias_dtype, expert * a.bias_stride + n) : 0.0f;
            int acc[SPW][NT][4];
#pragma unroll
            for (int s = 0; s < SPW; ++s)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[s][j][i] = 0;
            bool ok = true;
            for (int step = 0; step < steps; ++step) {
                ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, a.status, 21));
                if (!ok) break;
                const uint8_t* tile = ring + (size_t)stage * stage_bytes + g * BLOCK_K;
                const uint8_t* w_tile = tile + wk * w_block;
                const uint8_t* x_tile = tile + w_bytes + wk * TOKENS * BLOCK_K;
                uint4 x[NT][2];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    x[j][0] = *reinterpret_cast<const uint4*>(x_tile + 8 * j * BLOCK_K + off0);
                    x[j][1] = *reinterpret_cast<const uint4*>(x_tile + 8 * j * BLOCK_K + off1);
                }
#pragma unroll
                for (int s = 0; s < SPW; ++s) {
                    const int strip = s * WS + ws;
                    if (strip >= strips) break;
                    const uint8_t* lo = w_tile + strip * 16 * BLOCK_K;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 u = *reinterpret_cast<const uint4*>(lo + (i ? off1 : off0));
                        const uint4 v = *reinterpret_cast<const uint4*>(lo + 8 * BLOCK_K + (i ? off1 : off0));
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            mma_s8(acc[s][j], u.x, v.x, u.y, v.y, x[j][i].x, x[j][i].y);
                            mma_s8(acc[s][j], u.z, v.z, u.w, v.w, x[j][i].z, x[j][i].w);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[stage]);
                if (++stage == a.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
#pragma unroll
            for (int s = 0; s < SPW; ++s) {
                const int strip = s * WS + ws;
                if (strip >= strips) break;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int m = 8 * j + 2 * t + (i & 1);
                        if (m < tokens) atomicAdd(&sums[m * a.rows + 16 * strip + 8 * (i >> 1) + g], acc[s][j][i]);
                    }
            }
            if (any_failed<32 * WARPS>(!ok)) break;
            if (r < a.rows) {
                for (int m = 0; m < tokens; ++m) {
                    float v = sb * (sa_s[m0 + m] * (float)sums[m * a.rows + r]);
                    sums[m * a.rows + r] = 0;  // also where the group reaches beyond the weight
                    if (!mine) continue;
                    if (p.bias) v = (p.bias_after_round ? rounded(v, p.out_dtype) : v) + bias;
                    const int64_t at = (int64_t)(m0 + m) * p.ld_c + n;
                    if (p.out_dtype == FG_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
                    else if (p.out_dtype == FG_DTYPE_F16) reinterpret_cast<__half*>(p.c)[at] = __float2half_rn(v);
                    else reinterpret_cast<float*>(p.c)[at] = v;
                }
            }
            if (item + (int)gridDim.x < items) any_failed<32 * WARPS>(false);  // the sums are zeros again
        }
    }
    __syncthreads();
}

// The same stream for more tokens, multiplied by tcgen05 (kind::i8): tokens are the 128 rows of the accumulator in TMEM, the
// group's weight rows its columns.  Only the token rows that exist are fetched; the instruction reads 128, and what the
// others hold reaches accumulator rows that nobody reads.  Warp 0 fetches, warp 1 multiplies, warps 4 to 7 finish a
// group (two accumulators: the next group is multiplied meanwhile).
template <int KB>
__global__ void __launch_bounds__(256, 1) int8_stream_kernel(const __grid_constant__ CUtensorMap tm_w,
                                                             const __grid_constant__ CUtensorMap tm_x, const StreamArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full_bar[MAX_STAGES], empty_bar[MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t abort_word, tmem_slot;
    __shared__ __align__(16) float col_scale[2][MAX_ROWS];
    __shared__ float col_bias[2][MAX_ROWS];
    const FgSkinny& p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int x_block = a.token_rows * BLOCK_K, w_block = a.rows * BLOCK_K, stage_bytes = KB * (x_block + w_block);
    const int steps = ((int)p.K + KB * BLOCK_K - 1) / (KB * BLOCK_K);
    const int quads = ((int)p.M + 31) / 32;                         // warps of the epilogue that hold tokens
    const int acc_cols = (a.rows + 31) / 32 * 32;                   // of one accumulator
    const uint32_t tmem_cols = 2 * acc_cols <= 64 ? 64 : 2 * acc_cols <= 128 ? 128 : 2 * acc_cols <= 256 ? 256 : 512;
    volatile uint32_t* abort_flag = &abort_word;
    if (warp == 0 && lane == 0) {
        if (a.wide)  // as above: as far as L2 while the kernel before this one drains
            for (int step = 0; step < min(a.stages, steps); ++step) tma_prefetch_3d(&tm_w, 0, blockIdx.x * a.rows, step * KB);
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], quads);
        }
        abort_word = 0u;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    fg_pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int grp = blockIdx.x; grp < a.groups && ok; grp += gridDim.x)
                for (int step = 0; step < steps; ++step) {
                    ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, a.status, 22);
                    if (!ok) break;
                    uint8_t* to = ring + (size_t)stage * stage_bytes;
                    mbar_arrive_expect_tx(&full_bar[stage], (uint32_t)stage_bytes);
                    if (a.wide) {
                        tma_load_3d(to, &tm_x, &full_bar[stage], 0, 0, step * KB);
                        tma_load_3d(to + KB * x_block, &tm_w, &full_bar[stage], 0, grp * a.rows, step * KB);
                    } else {
#pragma unroll 1
                        for (int b = 0; b < KB; ++b) {
                            tma_load_3d(to + b * x_block, &tm_x, &full_bar[stage], (step * KB + b) * BLOCK_K, 0, 0);
                            tma_load_3d(to + KB * x_block + b * w_block, &tm_w, &full_bar[stage], (step * KB + b) * BLOCK_K, grp * a.rows, 0);
                        }
                    }
                    ++issued;
                    if (++stage == a.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            if (*abort_flag) drain(full_bar, a.stages, issued);
        }
        __syncwarp();
        fg_pdl_trigger();  // every load has been issued
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_s8_s32(128, a.rows);
        int stage = 0;
        uint32_t phase = 0, round = 0;
        bool ok = true, ready = false;  // ready: the next stage had come when it was last looked at
        for (int grp = blockIdx.x; grp < a.groups && ok; grp += gridDim.x, ++round) {
            const uint32_t buf = round & 1u, d = tmem + buf * acc_cols;
            ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((round >> 1) & 1u) ^ 1u, abort_flag, a.status, 23));
            if (!ok) break;
            tc_fence_after_sync();
            for (int step = 0; step < steps; ++step) {
                ok = __all_sync(0xffffffffu, ready || mbar_wait(&full_bar[stage], phase, abort_flag, a.status, 24));
                if (!ok) break;
                uint64_t* this_empty = &empty_bar[stage];
                const uint32_t x_addr = smem_u32(ring + (size_t)stage * stage_bytes);
                if (++stage == a.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
                ready = mbar_test_wait(&full_bar[stage], phase);  // answered while the instructions are issued
                if (elect_one()) {
                    const uint32_t w_addr = x_addr + KB * x_block;
#pragma unroll
                    for (int b = 0; b < KB; ++b) {
                        const uint64_t x_desc = umma_desc_k_sw128(x_addr + b * x_block), w_desc = umma_desc_k_sw128(w_addr + b * w_block);
#pragma unroll
                        for (int k = 0; k < BLOCK_K / 32; ++k)
                            umma_i8(d, x_desc + (uint64_t)(2 * k), w_desc + (uint64_t)(2 * k), idesc, step > 0 || b > 0 || k > 0 ? 1u : 0u);
                    }
                    umma_commit(this_empty);
                    if (step == steps - 1) umma_commit(&acc_full[buf]);
                }
                __syncwarp();
            }
        }
    } else if (warp >= 4) {
        const int quad = warp & 3, tid = (int)threadIdx.x - 128, m = quad * 32 + lane;
        const bool tokens = quad < quads, mine = m < p.M;
        const float sa = p.sa[p.sa_mode == FG_SCALE_VECTOR && mine ? m : 0];
        const int esz = p.out_dtype == FG_DTYPE_F32 ? 4 : 2;
        uint8_t* out = reinterpret_cast<uint8_t*>(p.c) + m * p.ld_c * esz;
        const FgRows rows = fg_rows(out, mine, lane, p.ld_c * esz);
        // Behind the ring, where the instructions read what reaches no row that counts.
        uint8_t* staging = ring + (size_t)a.stages * stage_bytes + quad * 2048;
        uint32_t round = 0;
        bool ok = true;
        for (int grp = blockIdx.x; grp < a.groups; grp += gridDim.x, ++round) {
            const uint32_t buf = round & 1u;
            const int64_t n0 = (int64_t)grp * a.rows;
            for (int r = tid; r < a.rows; r += 128) {
                const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;
                col_scale[buf][r] = p.sb[p.sb_mode == FG_SCALE_VECTOR ? n : 0];
                col_bias[buf][r] = p.bias ? load_bias(p.bias, p.bias_dtype, n) : 0.0f;
            }
            if (any_failed<128>(!ok)) break;
            if (!tokens) continue;
            ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (round >> 1) & 1u, abort_flag, a.status, 25));
            if (!ok) continue;
            tc_fence_after_sync();
            const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * acc_cols;
            for (int c = 0; c < a.rows; c += 32) {
                uint32_t raw[32];
                tmem_ld_32x32b_x32(acc + c, raw);
                tmem_ld_wait();
                const int cols = (int)min((int64_t)min(32, a.rows - c), p.N - n0 - c);
                if (cols <= 0) break;
                float v[32];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 s = *reinterpret_cast<const float4*>(&col_scale[buf][c + 4 * q]);
                    v[4 * q] = s.x * (sa * (float)(int)raw[4 * q]);
                    v[4 * q + 1] = s.y * (sa * (float)(int)raw[4 * q + 1]);
                    v[4 * q + 2] = s.z * (sa * (float)(int)raw[4 * q + 2]);
                    v[4 * q + 3] = s.w * (sa * (float)(int)raw[4 * q + 3]);
                }
                if (p.bias) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = (p.bias_after_round ? rounded(v[i], p.out_dtype) : v[i]) + col_bias[buf][c + i];
                }
                // Whole pieces of aligned rows by their own lanes: there is little to write, and its end is waited for (64 x 9472 x 4096
                // 10.8 us, 11.4 through shared memory; 64 x 9471 12.3, by their own lanes 17).
                if (a.c_align == 16 && cols % 8 == 0) {
                    if (mine) store_row(out + (n0 + c) * esz, v, cols, p.out_dtype);
                } else {
                    fg_store_rows(staging, lane, v, rows, p.ld_c * esz, (n0 + c) * esz, cols, p.out_dtype, a.c_align);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, tmem_cols);
    }
}

int byte_maps(StreamArgs& a, int kb, int token_rows, CUtensorMap* tm_w, CUtensorMap* tm_x) {
    const FgSkinny& p = a.p;
    a.wide = p.K % BLOCK_K == 0;
    const uint64_t w_rows = (uint64_t)p.N * (uint64_t)(a.offs ? a.n_experts : 1);
    int rc;
    if (a.wide) {  // blocks of 128 bytes as the last dimension
        const uint64_t blocks = (uint64_t)(p.K / BLOCK_K);
        rc = fg_byte_map(tm_w, p.b, BLOCK_K, w_rows, blocks, (uint64_t)p.ld_b, BLOCK_K, (uint32_t)a.rows, 3, (uint32_t)kb);
        if (rc == FG_OK) rc = fg_byte_map(tm_x, p.a, BLOCK_K, (uint64_t)p.M, blocks, (uint64_t)p.ld_a, BLOCK_K, (uint32_t)token_rows, 3, (uint32_t)kb);
    } else {
        rc = fg_byte_map(tm_w, p.b, (uint64_t)p.K, w_rows, 1, (uint64_t)p.ld_b, (uint64_t)p.ld_b * w_rows, (uint32_t)a.rows, 3);
        if (rc == FG_OK) rc = fg_byte_map(tm_x, p.a, (uint64_t)p.K, (uint64_t)p.M, 1, (uint64_t)p.ld_a, (uint64_t)p.ld_a * p.M, (uint32_t)token_rows, 3);
    }
    return rc;
}

template <int KB>
int launch_stream(StreamArgs& a, cudaStream_t st) {
    const FgSkinny& p = a.p;
    auto kernel = int8_stream_kernel<KB>;
    static bool attr_done[64];
    static std::mutex mu;
    {
        std::lock_guard<std::mutex> lock(mu);
        bool& done = attr_done[fg_device_index()];
        if (!done) {
            FG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, STREAM_SMEM_BYTES));
            done = true;
        }
    }
    const int grid = a.groups < fg_num_sms() ? a.groups : fg_num_sms();
    const int64_t stage = (int64_t)KB * (a.rows + a.token_rows) * BLOCK_K;
    const int64_t all = fg_cdiv(p.K, KB * BLOCK_K) * fg_cdiv(a.groups, grid);
    const int64_t pad = 128 * BLOCK_K;  // the instruction reads 128 rows of tokens from the last stage too
    int64_t stages = (STREAM_SMEM_BYTES - 1024 - pad) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (stages > all) stages = all;
    FG_REQUIRE(stages >= 1, FG_ERR_UNSUPPORTED, "a stage of %lld bytes does not fit", (long long)stage);
    a.stages = (int)stages;
    CUtensorMap tm_w, tm_x;
    const int rc = byte_maps(a, KB, a.token_rows, &tm_w, &tm_x);
    if (rc != FG_OK) return rc;
    FG_CUDA(fg_launch(kernel, (unsigned)grid, 256, (size_t)(stages * stage + pad + 1024), st, 1, tm_w, tm_x, a));
    return FG_OK;
}

template <int NT, int SPW, int KB, bool GROUPED>
int launch(StreamArgs& a, cudaStream_t st) {
    const FgSkinny& p = a.p;
    auto kernel = int8_skinny_kernel<NT, SPW, KB, GROUPED>;
    static bool attr_done[64];
    static std::mutex mu;
    {
        std::lock_guard<std::mutex> lock(mu);
        bool& done = attr_done[fg_device_index()];
        if (!done) {
            FG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
            done = true;
        }
    }
    const int64_t items = (int64_t)a.groups * (GROUPED ? (p.M < a.n_experts ? p.M : a.n_experts) : 1);  // at most
    const int grid = items < fg_num_sms() ? (int)items : fg_num_sms();
    const int64_t stage = (int64_t)KB * (a.rows + 8 * NT) * BLOCK_K;
    const int64_t all = fg_cdiv(p.K, KB * BLOCK_K) * fg_cdiv(items, grid);
    const int64_t sums = (int64_t)8 * NT * a.rows * sizeof(int) + 1024;
    int64_t stages = (SMEM_BYTES - sums) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (stages > all) stages = all;
    FG_REQUIRE(stages >= 1, FG_ERR_UNSUPPORTED, "a stage of %lld bytes does not fit", (long long)stage);
    a.stages = (int)stages;
    CUtensorMap tm_w, tm_x;
    const int rc = byte_maps(a, KB, 8 * NT, &tm_w, &tm_x);
    if (rc != FG_OK) return rc;
    const size_t smem = (size_t)(stages * stage + sums);
    FG_CUDA(fg_launch(kernel, (unsigned)grid, THREADS, smem, st, 1, tm_w, tm_x, a));
    return FG_OK;
}

// Stages of 19 to 48 KB (64 with 17 to 32 tokens and 32 rows): the lower a group, the more blocks of K.
template <bool GROUPED>
int launch_registers(StreamArgs& a, cudaStream_t st) {
    auto by_rows = [&](auto nt) -> int {
        constexpr int NT = decltype(nt)::value;
        if (a.rows <= 16) return launch<NT, 1, 8, GROUPED>(a, st);
        if (a.rows <= 32) return launch<NT, 2, 8, GROUPED>(a, st);
        if constexpr (NT <= 2) {
            if (a.rows <= 64) return launch<NT, 2, 4, GROUPED>(a, st);
            if (a.rows <= 128) return launch<NT, 2, 2, GROUPED>(a, st);
            return launch<NT, 2, 1, GROUPED>(a, st);
        }
        fg_set_error("groups of %d rows are built for up to 16 tokens", a.rows);
        return FG_ERR_UNSUPPORTED;
    };
    if (a.p.M <= 8) return by_rows(std::integral_constant<int, 1>());
    if (a.p.M <= 16) return by_rows(std::integral_constant<int, 2>());
    if constexpr (!GROUPED) return by_rows(std::integral_constant<int, 4>());
    fg_set_error("at most 16 rows");
    return FG_ERR_UNSUPPORTED;
}

int launch_tensor_memory(StreamArgs& a, cudaStream_t st) {
    a.token_rows = (int)((a.p.M + 7) / 8 * 8);
    a.c_align = fg_row_align(a.p.c, a.p.ld_c * (a.p.out_dtype == FG_DTYPE_F32 ? 4 : 2));
    const int rows = a.rows + a.token_rows;
    // Four blocks of K per stage while three such stages fit: 4096 x 14336 with 80 tokens 21.2 us, 24.5 with two blocks.  Three blocks
    // take 11.4 us where two take 10.8 (9472 x 4096 with 65).
    return rows <= 128 ? launch_stream<4>(a, st) : rows <= 192 ? launch_stream<2>(a, st) : launch_stream<1>(a, st);
}

// Rows per group: as few rounds of groups as their height allows, and in those all groups of one height.
int group_rows(int64_t N) {
    const int64_t rounds = fg_cdiv(N, (int64_t)MAX_ROWS * fg_num_sms());
    return (int)(fg_cdiv(fg_cdiv(N, rounds * fg_num_sms()), 16) * 16);
}

// A tcgen05 instruction takes 64 cycles for its 128 rows of tokens however few they are and however low the group is, 142 ns
// per block of K, where the registers' instructions take what tokens and rows cost; those run out above (0.4 PFLOP/s).
// Measured, registers / TMEM: 2112 x 7168 5.6 / 10.7 us with 16 tokens, 7.2 / 10.6 with 32; 6144 x 4096 7.6 / 8.9 with 16,
// 9.5 / 8.9 with 32; 24576 x 7168 33.3 / 33.1 and 39.1 / 33.2; 4096 x 14336 15.7 / 20.2 with 32, 21.8 / 19.7 with 33.
bool in_registers(int64_t M, int rows) { return M <= 16 || (M <= 32 && rows <= 32); }

}  // namespace

bool fg_int8_is_skinny(int64_t M) { return M <= MAX_TOKENS; }

// Where the stream of the weight does not bound it: a block of K takes what the instruction and the ring take, or the bytes that an SM
// takes in, 113 per ns.
int64_t fg_int8_skinny_time(int64_t M, int64_t N, int64_t K) {
    const int rows = group_rows(N);
    if (in_registers(M, rows)) return 0;  // nothing is faster
    const int64_t bytes = (rows + fg_cdiv(M, 8) * 8) * BLOCK_K, ring = bytes <= 128 * BLOCK_K ? 150 : 178;
    return 3000 + fg_cdiv(fg_cdiv(N, rows), fg_num_sms()) * fg_cdiv(K, BLOCK_K) * (bytes / 113 > ring ? bytes / 113 : ring);
}

int fg_int8_skinny(const FgSkinny& p, cudaStream_t st) {
    FG_REQUIRE(p.M > 0 && p.N > 0 && p.M <= MAX_TOKENS && p.K > 0 && p.K % 16 == 0, FG_ERR_UNSUPPORTED, "bad sizes");
    StreamArgs a{};
    a.p = p;
    a.status = fg_status_word_device_ptr();
    a.rows = group_rows(p.N);
    a.groups = (int)fg_cdiv(p.N, a.rows);
    return in_registers(p.M, a.rows) ? launch_registers<false>(a, st) : launch_tensor_memory(a, st);
}

// The same for experts: rows [offs[e - 1], offs[e]) of up to 16 in all times weight e.  One launch without tables of tiles, and groups
// of weight rows that fit the SMs whatever the number of experts.  Measured against two launches and 128-row tiles: 1 row x 4096 x
// 14336 11.4 us (43.2), 8 rows in 256 experts x 4096 x 7168 40.8 (45.7; the weights alone 35.9), x 7168 x 2048 23.9 (30.4), 16 rows in 8
// experts x 28672 x 4096 131.6 (136.0).  From 17 rows on the tiles are as fast (84 us both, 90 % of the weights' stream).
int fg_int8_skinny_grouped(const FgSkinny& p, const int32_t* offs, int n_experts, int64_t bias_stride, cudaStream_t st) {
    FG_REQUIRE(fg_int8_is_skinny_grouped(p.M, p.N, n_experts) && p.M > 0 && p.N > 0 && p.K > 0 && p.K % 16 == 0, FG_ERR_UNSUPPORTED, "bad sizes");
    StreamArgs a{};
    a.p = p;
    a.offs = offs;
    a.n_experts = n_experts;
    a.bias_stride = bias_stride;
    a.status = fg_status_word_device_ptr();
    // The height whose groups, over as many experts as can have rows, take the least time on an SM: their weight rows, the tokens'
    // rows beside them, and an epilogue that is worth 64 KB of the weight.
    const int64_t experts = p.M < n_experts ? p.M : n_experts;
    int64_t least = INT64_MAX;
    for (int rows = MAX_ROWS; rows >= 16; rows -= 16) {
        const int64_t most = fg_cdiv(fg_cdiv(p.N, rows) * experts, fg_num_sms()) * (rows + (p.M <= 8 ? 8 : 16) + 65536 / p.K);
        if (most < least) {
            least = most;
            a.rows = rows;
        }
    }
    a.groups = (int)fg_cdiv(p.N, a.rows);
    return launch_registers<true>(a, st);
}

bool fg_int8_is_skinny_grouped(int64_t M, int64_t N, int n_experts) {
    return M <= 16 && n_experts <= 1024 && N * n_experts < (1ll << 31) - MAX_ROWS;
}
