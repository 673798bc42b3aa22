// Tokens sorted by expert and back: the permutation itself, the copy of the tokens' rows into expert order, the
// weighted sum of the experts' rows per token, and the gradients of both.
//
//   rows[row(t, k)] = x[t]                              out[t] = sum_k w[t, k] * rows[row(t, k)]
//   d_x[t] = sum_k d_rows[row(t, k)]                    d_rows[row(t, k)] = w[t, k] * d_out[t]
//                                                       d_w[t, k] = <d_out[t], rows[row(t, k)]>
//
// row_of_slot holds row(t, k), or ~row for a slot without an expert: such slots own the rows behind the last
// expert's, so that every row belongs to exactly one slot and no kernel has to look for rows that nobody names.
#include <cooperative_groups.h>

#include <mutex>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;

struct SortArgs {
    const void* ids;  // [numel]
    int ids_are_i64;
    int64_t numel;
    int num_experts;
    const int32_t* expert_map;  // nullable: the expert of id i is expert_map[i]
    int expert_map_len;
    int32_t* offs;         // [num_experts] ends of the experts' rows
    int32_t* row_of_slot;  // [numel]
    int32_t* slot_of_row;  // [numel]
};

// Expert of slot i, num_experts if it has none.
__device__ __forceinline__ int expert_of(const SortArgs& a, int64_t i) {
    long long id = a.ids_are_i64 ? reinterpret_cast<const int64_t*>(a.ids)[i] : reinterpret_cast<const int32_t*>(a.ids)[i];
    if (a.expert_map) id = id >= 0 && id < a.expert_map_len ? a.expert_map[id] : -1;
    return id >= 0 && id < a.num_experts ? (int)id : a.num_experts;
}

// A counting sort by one cluster, stable like a sort by (expert, slot): every warp owns a contiguous segment of
// the slots and counts it, the counts are scanned over warps, CTAs (distributed shared memory) and experts, and every warp
// walks its segment again in order.  Bucket num_experts takes the slots without an expert.
__global__ void __launch_bounds__(SORT_THREADS, 1) sort_slots_kernel(SortArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    cg::cluster_group cluster = cg::this_cluster();
    const int n_ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int E = a.num_experts, B = E + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    extern __shared__ int32_t smem[];
    int32_t* warp_hist = smem;                    // [SORT_WARPS][B] counts, then the row of the warp's next slot within the CTA
    int32_t* cta_total = smem + SORT_WARPS * B;   // [B] read by the other CTAs
    int32_t* base = cta_total + B;                // [B] first row of this CTA
    __shared__ int32_t scan_tmp[SORT_WARPS];
    for (int i = threadIdx.x; i < SORT_WARPS * B; i += SORT_THREADS) warp_hist[i] = 0;
    __syncthreads();

    const int64_t segments = (int64_t)n_ranks * SORT_WARPS;
    const int64_t seg_len = ((a.numel + segments - 1) / segments + 31) / 32 * 32;
    const int64_t seg_begin = min((rank * (int64_t)SORT_WARPS + warp) * seg_len, a.numel);
    const int64_t seg_end = min(seg_begin + seg_len, a.numel);
    int32_t* my_hist = warp_hist + warp * B;
    for (int64_t i0 = seg_begin; i0 < seg_end; i0 += 32) {
        const int e = i0 + lane < seg_end ? expert_of(a, i0 + lane) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(peers) - 1) my_hist[e] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < B; e += SORT_THREADS) {
        int32_t run = 0;
        for (int w = 0; w < SORT_WARPS; ++w) {
            const int32_t t = warp_hist[w * B + e];
            warp_hist[w * B + e] = run;
            run += t;
        }
        cta_total[e] = run;
    }
    cluster.sync();
    const int e0 = threadIdx.x;  // num_experts <= SORT_THREADS; the last bucket follows all others and needs no scan
    int32_t before = 0, total = 0;
    if (e0 < E) {
        for (int r = 0; r < n_ranks; ++r) {
            const int32_t c = cluster.map_shared_rank(cta_total, r)[e0];
            if (r < rank) before += c;
            total += c;
        }
    }
    int32_t none_before = 0;
    if (threadIdx.x == 0)
        for (int r = 0; r < rank; ++r) none_before += cluster.map_shared_rank(cta_total, r)[E];
    cluster.sync();  // nobody leaves while the others read its counts
    int32_t incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    if (lane == 31) scan_tmp[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int32_t v = scan_tmp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t t = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += t;
        }
        scan_tmp[lane] = v;
    }
    __syncthreads();
    incl += warp > 0 ? scan_tmp[warp - 1] : 0;
    if (e0 < E) {
        base[e0] = incl - total + before;
        if (rank == 0) a.offs[e0] = incl;
    }
    if (threadIdx.x == 0) base[E] = scan_tmp[SORT_WARPS - 1] + none_before;
    __syncthreads();
    for (int64_t i0 = seg_begin; i0 < seg_end; i0 += 32) {
        const int64_t i = i0 + lane;
        const int e = i < seg_end ? expert_of(a, i) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int leader = __ffs(peers) - 1;
        int32_t cur = 0;
        if (e >= 0 && lane == leader) {
            cur = my_hist[e];
            my_hist[e] = cur + __popc(peers);
        }
        cur = __shfl_sync(0xffffffffu, cur, leader);
        if (e >= 0) {
            const int32_t row = base[e] + cur + __popc(peers & ((1u << lane) - 1u));
            a.row_of_slot[i] = e < E ? row : ~row;
            a.slot_of_row[row] = (int32_t)i;
        }
        __syncwarp();
    }
}

// One CTA per token: its row is read once and written to the rows of its slots; rows of slots without an expert
// become zeros (their scales 1).  UNIT: the bytes of a load, 16 where everything is aligned to that.
template <typename UNIT>
__global__ void __launch_bounds__(256) permute_rows_kernel(const UNIT* x, int64_t ld_x, const float* scale, int64_t ld_scale,
                                                           const int32_t* row_of_slot, int topk, int64_t n_rows, UNIT* rows,
                                                           int units, float* row_scale, int scale_cols) {
    fg_pdl_wait();
    fg_pdl_trigger();
    const int64_t t = blockIdx.x;
    for (int v = threadIdx.x; v < units; v += blockDim.x) {
        const UNIT value = x[t * ld_x + v];
        for (int k = 0; k < topk; ++k) {
            const int32_t r = row_of_slot[t * topk + k];
            const int64_t row = r < 0 ? ~r : r;
            if (row < n_rows) rows[row * units + v] = r < 0 ? UNIT{} : value;
        }
    }
    for (int c = threadIdx.x; c < scale_cols; c += blockDim.x) {
        const float value = scale[t * ld_scale + c];
        for (int k = 0; k < topk; ++k) {
            const int32_t r = row_of_slot[t * topk + k];
            const int64_t row = r < 0 ? ~r : r;
            if (row < n_rows) row_scale[row * scale_cols + c] = r < 0 ? 1.0f : value;
        }
    }
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, int64_t i) {
    if (dtype == FG_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
    if (dtype == FG_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(w)[i]);
    return reinterpret_cast<const float*>(w)[i];
}

__device__ __forceinline__ void store_weight(void* w, int dtype, int64_t i, float v) {
    if (dtype == FG_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
    else if (dtype == FG_DTYPE_F16) reinterpret_cast<__half*>(w)[i] = __float2half_rn(v);
    else reinterpret_cast<float*>(w)[i] = v;
}

struct SumArgs {
    const void* rows;  // [n_rows, H], row stride ld_rows
    int64_t ld_rows, n_rows;
    const int32_t* row_of_slot;  // [T, topk]
    const void* weights;         // nullable [T, topk], row stride ld_w
    int w_dtype;
    int64_t ld_w;
    int topk;
    int64_t H;
    void* out;  // [T, H]
    // backward
    const void* d_out;  // [T, H], row stride ld_d_out
    int64_t ld_d_out;
    void* d_rows;  // [n_rows, H]; NULL: not wanted
    void* d_w;     // [T, topk]; NULL: not wanted
};

// One CTA per token; sums in fp32 in slot order.
template <typename T, int V>
__global__ void __launch_bounds__(256) unpermute_kernel(SumArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    const int64_t t = blockIdx.x;
    const T* rows = reinterpret_cast<const T*>(a.rows);
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.H; c += (int64_t)blockDim.x * V) {
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
        for (int k = 0; k < a.topk; ++k) {
            const int32_t r = a.row_of_slot[t * a.topk + k];
            if (r < 0 || r >= a.n_rows) continue;
            const float w = a.weights ? load_weight(a.weights, a.w_dtype, t * a.ld_w + k) : 1.0f;
            float f[V];
            if constexpr (V == 8) fg_load8(rows + r * a.ld_rows + c, f);
            else f[0] = fg_to_float(rows[r * a.ld_rows + c]);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = fmaf(w, f[i], acc[i]);
        }
        T* out = reinterpret_cast<T*>(a.out) + t * a.H + c;
        if constexpr (V == 8) fg_store8(out, acc);
        else out[0] = fg_from_float<T>(acc[0]);
    }
}

// One CTA per token: d_out[t] times the weight into the gradient of every row of the token, and its product
// with the row summed over the CTA into the gradient of the weight.
template <typename T, int V>
__global__ void __launch_bounds__(256) unpermute_backward_kernel(SumArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    __shared__ float part[8];
    const int64_t t = blockIdx.x;
    const T* rows = reinterpret_cast<const T*>(a.rows);
    const T* d_out = reinterpret_cast<const T*>(a.d_out) + t * a.ld_d_out;
    for (int k = 0; k < a.topk; ++k) {
        const int32_t r = a.row_of_slot[t * a.topk + k];
        const int64_t row = r < 0 ? ~r : r;
        const bool inside = row < a.n_rows, real = r >= 0 && inside;
        const float w = real && a.weights ? load_weight(a.weights, a.w_dtype, t * a.ld_w + k) : 1.0f;
        float dot = 0.0f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < a.H; c += (int64_t)blockDim.x * V) {
            float g[V], f[V];
            if constexpr (V == 8) fg_load8(d_out + c, g);
            else g[0] = fg_to_float(d_out[c]);
            if (a.d_w && real) {
                if constexpr (V == 8) fg_load8(rows + row * a.ld_rows + c, f);
                else f[0] = fg_to_float(rows[row * a.ld_rows + c]);
#pragma unroll
                for (int i = 0; i < V; ++i) dot = fmaf(g[i], f[i], dot);
            }
            if (a.d_rows && inside) {
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = real ? w * g[i] : 0.0f;
                T* o = reinterpret_cast<T*>(a.d_rows) + row * a.H + c;
                if constexpr (V == 8) fg_store8(o, g);
                else o[0] = fg_from_float<T>(g[0]);
            }
        }
        if (a.d_w) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
            __syncthreads();
            if (threadIdx.x == 0) {
                float sum = 0.0f;
                for (int i = 0; i < (int)blockDim.x / 32; ++i) sum += part[i];
                store_weight(a.d_w, a.w_dtype, t * a.topk + k, real ? sum : 0.0f);
            }
            __syncthreads();
        }
    }
}

int elem_size(int dtype) { return dtype == FG_DTYPE_F32 ? 4 : 2; }

template <typename F>
int by_type(int dtype, F&& f) {
    switch (dtype) {
        case FG_DTYPE_BF16: return f(__nv_bfloat16());
        case FG_DTYPE_F16: return f(__half());
        case FG_DTYPE_F32: return f(float());
        default: fg_set_error("unsupported dtype code %d", dtype); return FG_ERR_INVALID_ARGUMENT;
    }
}

// Threads of a CTA that walks a row of n pieces: few iterations, no more threads than pieces (in whole warps).
unsigned threads_for(int64_t n) { return n >= 256 ? 256u : (unsigned)(n < 32 ? 32 : (n + 31) / 32 * 32); }

bool aligned16(const void* p, int64_t stride_bytes) { return (uintptr_t)p % 16 == 0 && stride_bytes % 16 == 0; }

}  // namespace

extern "C" {

int fg_moe_permute(void* rows, float* row_scale, int32_t* offs, int32_t* row_of_slot, int32_t* slot_of_row, const void* x,
                   const float* scale, const void* topk_ids, int ids_are_i64, const int32_t* expert_map, int expert_map_len,
                   int64_t T, int topk, int num_experts, int64_t H, int elem_bytes, int64_t ld_x, int64_t scale_cols,
                   int64_t ld_scale, void* stream) {
    FG_REQUIRE(T >= 0 && topk >= 0 && H >= 0 && scale_cols >= 0, FG_ERR_INVALID_ARGUMENT, "negative size");
    FG_REQUIRE(num_experts > 0 && num_experts <= SORT_THREADS, FG_ERR_UNSUPPORTED, "num_experts %d must be in [1, %d]", num_experts,
               SORT_THREADS);
    FG_REQUIRE(elem_bytes == 1 || elem_bytes == 2 || elem_bytes == 4, FG_ERR_INVALID_ARGUMENT, "elements of %d bytes", elem_bytes);
    FG_REQUIRE(T * topk < (1ll << 31) - 1 && H * elem_bytes < (1ll << 31) && scale_cols < (1ll << 31), FG_ERR_UNSUPPORTED, "size too large");
    FG_REQUIRE(expert_map == nullptr || expert_map_len > 0, FG_ERR_INVALID_ARGUMENT, "empty expert_map");
    const int64_t numel = T * topk;
    FG_REQUIRE(offs && (numel == 0 || (topk_ids && row_of_slot && slot_of_row)), FG_ERR_INVALID_ARGUMENT, "null pointer");
    FG_REQUIRE(numel == 0 || H == 0 || (rows && x), FG_ERR_INVALID_ARGUMENT, "null pointer");
    FG_REQUIRE(numel == 0 || scale_cols == 0 || (row_scale && scale), FG_ERR_INVALID_ARGUMENT, "null pointer");
    cudaStream_t st = (cudaStream_t)stream;
    const SortArgs a{topk_ids, ids_are_i64, numel, num_experts, expert_map, expert_map_len, offs, row_of_slot, slot_of_row};
    int ranks = 1;
    while (ranks < 8 && (int64_t)ranks * SORT_THREADS * 4 < numel) ranks *= 2;
    const size_t smem = (size_t)(SORT_WARPS + 2) * (num_experts + 1) * sizeof(int32_t);
    static std::mutex mu;
    static size_t smem_set[64];
    {
        std::lock_guard<std::mutex> lock(mu);
        size_t& have = smem_set[fg_device_index()];
        if (have < 48 * 1024) have = 48 * 1024;
        if (smem > have) {
            FG_CUDA(cudaFuncSetAttribute(sort_slots_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            have = smem;
        }
    }
    FG_CUDA(fg_launch(sort_slots_kernel, (unsigned)ranks, SORT_THREADS, smem, st, (unsigned)ranks, a));
    if (numel == 0 || (H == 0 && scale_cols == 0)) return FG_OK;
    const int64_t row_bytes = H * elem_bytes;
    auto go = [&](auto unit) -> cudaError_t {
        using U = decltype(unit);
        const int64_t units = row_bytes / (int64_t)sizeof(U);
        return fg_launch(permute_rows_kernel<U>, (unsigned)T, threads_for(units), 0, st, 1, (const U*)x,
                         ld_x * elem_bytes / (int64_t)sizeof(U), scale, ld_scale, (const int32_t*)row_of_slot, topk, numel, (U*)rows,
                         (int)units, row_scale, (int)scale_cols);
    };
    const bool vec = aligned16(x, ld_x * elem_bytes) && aligned16(rows, row_bytes);
    FG_CUDA(vec ? go(uint4()) : elem_bytes == 4 ? go(uint32_t()) : elem_bytes == 2 ? go(uint16_t()) : go(uint8_t()));
    return FG_OK;
}

int fg_moe_unpermute(void* out, const void* rows, const int32_t* row_of_slot, const void* weights, int w_dtype, int64_t T,
                     int topk, int64_t n_rows, int64_t H, int64_t ld_rows, int64_t ld_w, int dtype, void* stream) {
    FG_REQUIRE(T >= 0 && topk >= 0 && n_rows >= 0 && H >= 0, FG_ERR_INVALID_ARGUMENT, "negative size");
    FG_REQUIRE(T < (1ll << 31) && n_rows < (1ll << 31), FG_ERR_UNSUPPORTED, "size too large");
    FG_REQUIRE(!weights || w_dtype == FG_DTYPE_BF16 || w_dtype == FG_DTYPE_F16 || w_dtype == FG_DTYPE_F32, FG_ERR_INVALID_ARGUMENT,
               "bad weight dtype %d", w_dtype);
    if (T == 0 || H == 0) return FG_OK;
    FG_REQUIRE(out && (topk == 0 || (row_of_slot && (rows || n_rows == 0))), FG_ERR_INVALID_ARGUMENT, "null pointer");
    SumArgs a{};
    a.rows = rows; a.ld_rows = ld_rows; a.n_rows = n_rows; a.row_of_slot = row_of_slot; a.weights = weights; a.w_dtype = w_dtype;
    a.ld_w = ld_w; a.topk = topk; a.H = H; a.out = out;
    const int es = elem_size(dtype);
    const bool vec = H % 8 == 0 && aligned16(rows, ld_rows * es) && aligned16(out, H * es);
    return by_type(dtype, [&](auto tag) -> int {
        using E = decltype(tag);
        FG_CUDA(vec ? fg_launch(unpermute_kernel<E, 8>, (unsigned)T, threads_for(H / 8), 0, (cudaStream_t)stream, 1, a)
                    : fg_launch(unpermute_kernel<E, 1>, (unsigned)T, threads_for(H), 0, (cudaStream_t)stream, 1, a));
        return FG_OK;
    });
}

int fg_moe_unpermute_backward(void* d_rows, void* d_weights, const void* d_out, const void* rows, const int32_t* row_of_slot,
                              const void* weights, int w_dtype, int64_t T, int topk, int64_t n_rows, int64_t H, int64_t ld_d_out,
                              int64_t ld_rows, int64_t ld_w, int dtype, void* stream) {
    FG_REQUIRE(T >= 0 && topk >= 0 && n_rows >= 0 && H >= 0, FG_ERR_INVALID_ARGUMENT, "negative size");
    FG_REQUIRE(T < (1ll << 31) && n_rows < (1ll << 31), FG_ERR_UNSUPPORTED, "size too large");
    FG_REQUIRE(!(weights || d_weights) || w_dtype == FG_DTYPE_BF16 || w_dtype == FG_DTYPE_F16 || w_dtype == FG_DTYPE_F32,
               FG_ERR_INVALID_ARGUMENT, "bad weight dtype %d", w_dtype);
    if (T == 0 || topk == 0) return FG_OK;
    FG_REQUIRE(row_of_slot && (H == 0 || d_out) && (!d_weights || rows || H == 0), FG_ERR_INVALID_ARGUMENT, "null pointer");
    SumArgs a{};
    a.rows = rows; a.ld_rows = ld_rows; a.n_rows = n_rows; a.row_of_slot = row_of_slot; a.weights = weights; a.w_dtype = w_dtype;
    a.ld_w = ld_w; a.topk = topk; a.H = H; a.d_out = d_out; a.ld_d_out = ld_d_out; a.d_rows = d_rows; a.d_w = d_weights;
    const int es = elem_size(dtype);
    const bool vec = H % 8 == 0 && aligned16(d_out, ld_d_out * es) && (!d_weights || aligned16(rows, ld_rows * es)) && aligned16(d_rows, H * es);
    return by_type(dtype, [&](auto tag) -> int {
        using E = decltype(tag);
        FG_CUDA(vec ? fg_launch(unpermute_backward_kernel<E, 8>, (unsigned)T, threads_for(H / 8), 0, (cudaStream_t)stream, 1, a)
                    : fg_launch(unpermute_backward_kernel<E, 1>, (unsigned)T, threads_for(H), 0, (cudaStream_t)stream, 1, a));
        return FG_OK;
    });
}

}  // extern "C"
