// Products of few int8 tokens and a large int8 weight: C[m, n] = sum_k A[m, k] B[n, k], scaled per token and channel.
//
// With so few tokens the weight's bytes are all the work, and the job is to keep enough of them under way on every
// SM, from the first cycle to the last.  A CTA owns groups of weight rows, as many per group as it takes for the groups to
// cover the SMs once (or a whole number of times); one thread streams them by TMA into a ring that fills the shared
// memory, across the ends of groups, so that no epilogue interrupts the stream.  Eight warps multiply with mma.m16n8k32
// (weight rows as M, tokens as N): they share a stage's KB blocks of K and its strips of 16 rows, and the sums, whole
// numbers, are added in shared memory in any order.  The tensor cores of tcgen05 would be idle here whatever they are
// fed with, and need the tokens padded to 128 rows and the weight cut in tiles of 256 rows, which leaves SMs without one.
//
// K is a sum, so its order is free: lane (g, t) of a warp takes bytes [32 t, 32 t + 32) of a block's rows, for the weight
// and the tokens alike, as two 16-byte loads without bank conflicts, not the 4-byte pieces that the instruction's layout names.
#include <cuda.h>

#include <mutex>

#include "common.cuh"
#include "ptx_sm100.cuh"

using namespace fgptx;

namespace {

constexpr int WARPS = 8;  // that multiply; one more fetches
constexpr int THREADS = 32 * (WARPS + 1);
constexpr int BLOCK_K = 128;
constexpr int MAX_ROWS = 256;
constexpr int MAX_STAGES = 16;
constexpr int SMEM_BYTES = 224 * 1024;  // ring, sums and alignment

struct StreamArgs {
    FgSkinny p;
    int rows;    // per group, a multiple of 16
    int groups;
    int stages;
    int wide;  // one load brings all KB blocks of a stage (K a multiple of 128); otherwise each has its own
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

// A barrier of the multiplying warps that also tells all of them whether any of them failed.
__device__ __forceinline__ bool any_failed(bool failed) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)failed), "n"(32 * WARPS) : "memory");
    return r != 0u;
}

// NT: tiles of eight tokens.  KB: blocks of K per stage; 8 / KB warps share the strips of 16 rows of a block, up to SPW
// each.  Every warp passes every stage, in order.
template <int NT, int SPW, int KB>
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
    if (warp == WARPS && lane == 0) {
        // While the kernel before this one drains, the first stages of the weight come as far as L2.
        if (a.wide)
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

    if (warp == WARPS) {
        if (lane == 0) {
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int grp = blockIdx.x; grp < a.groups && ok; grp += gridDim.x)
                for (int step = 0; step < steps; ++step) {
                    ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, a.status, 20);
                    if (!ok) break;
                    uint8_t* to = ring + (size_t)stage * stage_bytes;
                    mbar_arrive_expect_tx(&full_bar[stage], (uint32_t)stage_bytes);
                    if (a.wide) {
                        tma_load_3d(to, &tm_w, &full_bar[stage], 0, grp * a.rows, step * KB);
                        tma_load_3d(to + w_bytes, &tm_x, &full_bar[stage], 0, 0, step * KB);
                    } else {
#pragma unroll 1
                        for (int b = 0; b < KB; ++b) {
                            tma_load_3d(to + b * w_block, &tm_w, &full_bar[stage], (step * KB + b) * BLOCK_K, grp * a.rows, 0);
                            tma_load_3d(to + w_bytes + b * TOKENS * BLOCK_K, &tm_x, &full_bar[stage], (step * KB + b) * BLOCK_K, 0, 0);
                        }
                    }
                    ++issued;
                    if (++stage == a.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            if (*abort_flag) {  // a wait ran out somewhere: what is still under way lands before the CTA ends
                uint32_t alone = 0u;
                for (int j = issued > a.stages ? issued - a.stages : 0; j < issued; ++j)
                    mbar_wait(&full_bar[j % a.stages], (uint32_t)(j / a.stages) & 1u, &alone, nullptr, 0, 100000000ull);
            }
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
        for (int grp = blockIdx.x; grp < a.groups; grp += gridDim.x) {
            const int64_t n = (int64_t)grp * a.rows + r;
            const bool mine = r < a.rows && n < p.N;
            const float sb = mine ? p.sb[p.sb_mode == FG_SCALE_VECTOR ? n : 0] : 0.0f;
            const float bias = mine && p.bias ? load_bias(p.bias, p.bias_dtype, n) : 0.0f;
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
                        if (m < p.M) atomicAdd(&sums[m * a.rows + 16 * strip + 8 * (i >> 1) + g], acc[s][j][i]);
                    }
            }
            if (any_failed(!ok)) break;
            if (mine) {
                for (int m = 0; m < p.M; ++m) {
                    float v = sb * (sa_s[m] * (float)sums[m * a.rows + r]);
                    sums[m * a.rows + r] = 0;
                    if (p.bias) v = (p.bias_after_round ? rounded(v, p.out_dtype) : v) + bias;
                    const int64_t at = m * p.ld_c + n;
                    if (p.out_dtype == FG_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p.c)[at] = __float2bfloat16_rn(v);
                    else if (p.out_dtype == FG_DTYPE_F16) reinterpret_cast<__half*>(p.c)[at] = __float2half_rn(v);
                    else reinterpret_cast<float*>(p.c)[at] = v;
                }
            }
            if (grp + gridDim.x < a.groups) any_failed(false);  // the sums are zeros again
        }
    }
    __syncthreads();
}

template <int NT, int SPW, int KB>
int launch(StreamArgs& a, cudaStream_t st) {
    const FgSkinny& p = a.p;
    auto kernel = int8_skinny_kernel<NT, SPW, KB>;
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
    const int grid = a.groups < fg_num_sms() ? a.groups : fg_num_sms();
    const int64_t stage = (int64_t)KB * (a.rows + 8 * NT) * BLOCK_K;
    const int64_t all = fg_cdiv(p.K, KB * BLOCK_K) * fg_cdiv(a.groups, grid);
    const int64_t sums = (int64_t)8 * NT * a.rows * sizeof(int) + 1024;
    int64_t stages = (SMEM_BYTES - sums) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (stages > all) stages = all;
    FG_REQUIRE(stages >= 1, FG_ERR_UNSUPPORTED, "a stage of %lld bytes does not fit", (long long)stage);
    a.stages = (int)stages;
    a.wide = p.K % BLOCK_K == 0;
    CUtensorMap tm_w, tm_x;
    int rc;
    if (a.wide) {  // blocks of 128 bytes as the last dimension
        const uint64_t blocks = (uint64_t)(p.K / BLOCK_K);
        rc = fg_byte_map(&tm_w, p.b, BLOCK_K, (uint64_t)p.N, blocks, (uint64_t)p.ld_b, BLOCK_K, (uint32_t)a.rows, 3, KB);
        if (rc == FG_OK) rc = fg_byte_map(&tm_x, p.a, BLOCK_K, (uint64_t)p.M, blocks, (uint64_t)p.ld_a, BLOCK_K, 8 * NT, 3, KB);
    } else {
        rc = fg_byte_map(&tm_w, p.b, (uint64_t)p.K, (uint64_t)p.N, 1, (uint64_t)p.ld_b, (uint64_t)p.ld_b * p.N, (uint32_t)a.rows, 3);
        if (rc == FG_OK) rc = fg_byte_map(&tm_x, p.a, (uint64_t)p.K, (uint64_t)p.M, 1, (uint64_t)p.ld_a, (uint64_t)p.ld_a * p.M, 8 * NT, 3);
    }
    if (rc != FG_OK) return rc;
    const size_t smem = (size_t)(stages * stage + sums);
    FG_CUDA(fg_launch(kernel, (unsigned)grid, THREADS, smem, st, 1, tm_w, tm_x, a));
    return FG_OK;
}

// Stages of 20 to 48 KB: the lower a group, the more blocks of K.
template <int NT>
int launch_rows(StreamArgs& a, cudaStream_t st) {
    if (a.rows <= 16) return launch<NT, 1, 8>(a, st);
    if (a.rows <= 32) return launch<NT, 2, 8>(a, st);
    if (a.rows <= 64) return launch<NT, 2, 4>(a, st);
    if constexpr (NT < 8) {
        if (a.rows <= 128) return launch<NT, 2, 2>(a, st);
        return launch<NT, 2, 1>(a, st);
    }
    fg_set_error("groups of %d rows are built for up to 32 tokens", a.rows);
    return FG_ERR_UNSUPPORTED;
}

// Rows per group, as many groups as that gives: as few rounds of groups as their height allows, and in those all
// groups of one height.
int group_rows(int64_t N) {
    const int64_t rounds = fg_cdiv(N, (int64_t)MAX_ROWS * fg_num_sms());
    return (int)(fg_cdiv(fg_cdiv(N, rounds * fg_num_sms()), 16) * 16);
}

}  // namespace

// Up to 32 tokens the weight streams at the rate of HBM (6.5 TB/s between a 117 MB and a 176 MB weight, and 4 us around
// that); above, mma.sync runs out (0.4 PFLOP/s): with groups of up to 64 rows, where the tiles of tcgen05 are
// slower still, up to 64 tokens.  Measured, this against the tcgen05 tiles: M = 1, N x K = 6144 x 4096 6.3 / 11.0 us, 28672 x 4096
// 21.4 / 25.5, 24576 x 7168 31.0 / 36.8; M = 32 9.4 / 13.4, 25.2 / 26.5, 37.6 / 37.9; M = 64 14.7 / 15.9, 38.8 / 27.1,
// 56.0 / 38.8.
bool fg_int8_is_skinny(int64_t M, int64_t N) { return M <= 32 || (M <= 64 && group_rows(N) <= 64); }

int fg_int8_skinny(const FgSkinny& p, cudaStream_t st) {
    FG_REQUIRE(p.M > 0 && p.N > 0 && fg_int8_is_skinny(p.M, p.N) && p.K > 0 && p.K % 16 == 0, FG_ERR_UNSUPPORTED, "bad sizes");
    StreamArgs a{};
    a.p = p;
    a.status = fg_status_word_device_ptr();
    a.rows = group_rows(p.N);
    a.groups = (int)fg_cdiv(p.N, a.rows);
    return p.M <= 8 ? launch_rows<1>(a, st) : p.M <= 16 ? launch_rows<2>(a, st) : p.M <= 32 ? launch_rows<4>(a, st) : launch_rows<8>(a, st);
}
