// Tokens sorted by expert and back: the permutation itself, the copy of the tokens' rows into expert order, the
// weighted sum of the experts' rows per token, and the gradients of both.
//
//   rows[row(t, k)] = x[t]                              out[t] = sum_k w[t, k] * rows[row(t, k)]
//   d_x[t] = sum_k d_rows[row(t, k)]                    d_rows[row(t, k)] = w[t, k] * d_out[t]
//                                                       d_w[t, k] = <d_out[t], rows[row(t, k)]>
//
// row_of_slot holds row(t, k), or ~row for a slot without an expert: such slots own the rows behind the last
// expert's, so that every row belongs to exactly one slot and no kernel has to look for rows that nobody names.
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace {

constexpr int MAX_EXPERTS = 1024;

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

// Many slots, first launch: every CTA ranks the slots of one chunk among themselves, stable like a sort by (expert,
// slot).  A warp owns a contiguous part of the chunk and counts it; the counts are scanned over the warps, and the
// warp walks its part again in order.  What the row kernel needs of a chunk goes into `table`:
//   table[e * n_chunks + c] = {slots of expert e in chunk c, slots of experts below e in chunk c}
// The second launch turns them into the first row of every expert and chunk (the first numbers of the chunks before, and
// the second numbers of all chunks); a slot's row is that plus its rank.  One cluster of eight CTAs, with the scans through
// distributed shared memory, took 13 us for 65536 slots where the two launches take 6; without the second launch, every
// token's CTA adding up its slots' rows, the row kernel takes 94 us instead of 88.  Bucket num_experts holds the
// slots without an expert.
constexpr int MAX_CHUNKS = 256;
constexpr int CHUNK_THREADS = 512;
constexpr int CHUNK_WARPS = CHUNK_THREADS / 32;

struct ChunkTable {
    int2* table;
    int n_chunks;
    int chunk;  // slots, a multiple of CHUNK_THREADS
};

__global__ void __launch_bounds__(CHUNK_THREADS) rank_slots_kernel(SortArgs a, ChunkTable ct) {
    fg_pdl_wait();
    fg_pdl_trigger();
    const int E = a.num_experts, B = E + 1, bits = 32 - __clz(E);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    extern __shared__ int32_t warp_hist[];  // [CHUNK_WARPS][B] counts, then the rank of the warp's next slot of the bucket
    __shared__ int32_t scan_tmp[CHUNK_WARPS];
    const int64_t begin = (int64_t)blockIdx.x * ct.chunk + (int64_t)warp * (ct.chunk / CHUNK_WARPS);
    const int64_t end = min(begin + ct.chunk / CHUNK_WARPS, a.numel);
    const int kept = begin + lane < end ? expert_of(a, begin + lane) : -1;
    for (int i = threadIdx.x; i < CHUNK_WARPS * B; i += CHUNK_THREADS) warp_hist[i] = 0;
    __syncthreads();
    int32_t* my_hist = warp_hist + warp * B;
    for (int64_t i = begin + lane; i < end; i += 32) atomicAdd(&my_hist[i < begin + 32 ? kept : expert_of(a, i)], 1);
    __syncthreads();
    // over the warps per bucket, then over the buckets; B may exceed the threads
    int32_t carry = 0;
    for (int e0 = 0; e0 < B; e0 += CHUNK_THREADS) {
        const int e = e0 + (int)threadIdx.x;
        int32_t total = 0;
        if (e < B) {
#pragma unroll
            for (int w = 0; w < CHUNK_WARPS; ++w) {
                const int32_t n = warp_hist[w * B + e];
                warp_hist[w * B + e] = total;
                total += n;
            }
        }
        int32_t incl = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t n = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += n;
        }
        if (lane == 31) scan_tmp[warp] = incl;
        __syncthreads();
        int32_t all = 0;
#pragma unroll
        for (int w = 0; w < CHUNK_WARPS; ++w) {
            if (w < warp) incl += scan_tmp[w];
            all += scan_tmp[w];
        }
        if (e < B) ct.table[(int64_t)e * ct.n_chunks + blockIdx.x] = make_int2(total, carry + incl - total);
        carry += all;
        __syncthreads();
    }
    for (int64_t i0 = begin; i0 < end; i0 += 32) {
        const int64_t i = i0 + lane;
        const int e = i >= end ? -1 : i0 == begin ? kept : expert_of(a, i);
        // lanes of the same bucket, one vote per bit of the bucket's number (a match over 32 lanes of many different
        // buckets takes several times as long)
        unsigned peers = __ballot_sync(0xffffffffu, e >= 0);
        for (int b = 0; b < bits; ++b) {
            const unsigned ones = __ballot_sync(0xffffffffu, (e >> b) & 1);
            peers &= (e >> b) & 1 ? ones : ~ones;
        }
        const int32_t cur = e >= 0 ? my_hist[e] : 0;
        __syncwarp();
        if (e >= 0) {
            const unsigned below = peers & ((1u << lane) - 1u);
            if (below == 0u) my_hist[e] = cur + __popc(peers);
            a.row_of_slot[i] = cur + __popc(below);  // the row kernel makes it a row
        }
        __syncwarp();
    }
}

// A token's row to the rows of its slots; rows of slots without an expert become zeros (their scales 1).
struct RowArgs {
    const void* x;
    int64_t ld_x;  // units
    const float* scale;
    int64_t ld_scale;
    int topk;
    int64_t tokens, n_rows;
    void* rows;
    int units;  // per row
    float* row_scale;
    int scale_cols;
};
constexpr int SLOTS_AT_ONCE = 8;

// The token of a thread: the CTA's, or with SHARED one per threadIdx.y.  With one per CTA it is the same in all threads, what is found
// by it too, and that takes fewer registers: 16381 x 2 fp16 rows of 4096 are summed in 70 us, in 89 with the general form.
template <bool SHARED>
__device__ __forceinline__ int64_t token_of_thread() {
    if constexpr (SHARED) return (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    else return blockIdx.x;
}

struct __align__(32) Unit32 {
    uint4 lo, hi;
};

template <typename UNIT>
__device__ __forceinline__ UNIT load_unit(const UNIT* p) { return *p; }
template <>
__device__ __forceinline__ Unit32 load_unit(const Unit32* p) {
    Unit32 v;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.lo.x), "=r"(v.lo.y), "=r"(v.lo.z), "=r"(v.lo.w), "=r"(v.hi.x), "=r"(v.hi.y), "=r"(v.hi.z), "=r"(v.hi.w)
                 : "l"(p) : "memory");
    return v;
}
template <typename UNIT>
__device__ __forceinline__ void store_unit(UNIT* p, const UNIT& v) { *p = v; }
template <>
__device__ __forceinline__ void store_unit(Unit32* p, const Unit32& v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(v.lo.x), "r"(v.lo.y), "r"(v.lo.z), "r"(v.lo.w), "r"(v.hi.x), "r"(v.hi.y), "r"(v.hi.z), "r"(v.hi.w)
                 : "memory");
}

template <typename UNIT, int N>
__device__ __forceinline__ void load_pieces(const RowArgs& a, int64_t t, int v0, UNIT (&piece)[N]) {
    const UNIT* x = reinterpret_cast<const UNIT*>(a.x) + t * a.ld_x;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int v = v0 + u * (int)blockDim.x;
        piece[u] = v < a.units ? load_unit(x + v) : UNIT{};
    }
}

template <typename UNIT, int N>
__device__ __forceinline__ void store_pieces(const RowArgs& a, int32_t r, int v0, const UNIT (&piece)[N]) {
    const int64_t row = r < 0 ? ~r : r;
    if (row >= a.n_rows) return;
    UNIT* out = reinterpret_cast<UNIT*>(a.rows) + row * a.units;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int v = v0 + u * (int)blockDim.x;
        if (v < a.units) store_unit(out + v, r < 0 ? UNIT{} : piece[u]);
    }
}

__device__ __forceinline__ void store_scales(const RowArgs& a, int64_t t, int k, int32_t r) {
    const int64_t row = r < 0 ? ~r : r;
    if (row >= a.n_rows) return;
    for (int c = threadIdx.x; c < a.scale_cols; c += blockDim.x)
        a.row_scale[row * a.scale_cols + c] = r < 0 ? 1.0f : a.scale[t * a.ld_scale + c];
}

// Many slots, second launch, a warp per bucket: table[e, c].x becomes the first row of expert e's slots in chunk c.
__global__ void __launch_bounds__(256) scan_chunks_kernel(SortArgs s, ChunkTable ct) {
    fg_pdl_wait();
    fg_pdl_trigger();
    const int lane = threadIdx.x & 31, e = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (e > s.num_experts) return;
    int2* of_e = ct.table + (int64_t)e * ct.n_chunks;
    int2 v[MAX_CHUNKS / 32];
    int32_t below = 0;
#pragma unroll
    for (int i = 0; i < MAX_CHUNKS / 32; ++i) {
        const int c = 32 * i + lane;
        v[i] = c < ct.n_chunks ? of_e[c] : make_int2(0, 0);
        below += v[i].y;
    }
    int32_t run = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0 && e > 0) s.offs[e - 1] = run;  // the slots of the experts below e
#pragma unroll
    for (int i = 0; i < MAX_CHUNKS / 32; ++i) {
        const int c = 32 * i + lane;
        int32_t incl = v[i].x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t n = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += n;
        }
        if (c < ct.n_chunks) of_e[c].x = run + incl - v[i].x;
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// Many slots, third launch, one CTA per token, or per several (threadIdx.y) of narrow rows: a row is read once and written slot
// after slot.  Bound by the writes, which are topk times the reads, and by the rate of a copy.  Few registers (and so many CTAs,
// a row each, under way) matter more than pieces per thread, and accesses of 32 bytes more than those of 16: 8192 x 8 rows of
// 14336 bytes take 164 us (6.4 TB/s of the 6.6 of a copy), 178 with two pieces of 16 bytes per thread; rows of 7168 bytes 84,
// 88, and 98 with four pieces and the slots' rows in registers, 91-97 as bulk copies through a ring in shared memory.
// UNIT: the bytes of a load, the most that everything is aligned to.
template <typename UNIT, bool SHARED>
__global__ void __launch_bounds__(512) permute_rows_kernel(SortArgs s, ChunkTable ct, RowArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    constexpr int PIECES = sizeof(UNIT) == 32 ? 1 : 2, SLOTS = 32, MAX_TOKENS = SHARED ? 32 : 1;
    __shared__ int32_t row_s[MAX_TOKENS * SLOTS];
    const int64_t t = token_of_thread<SHARED>(), t0 = SHARED ? t - threadIdx.y : t;
    const int tokens = SHARED ? (int)blockDim.y : 1, units = !SHARED || t < a.tokens ? a.units : 0;
    UNIT piece[PIECES];
    if (units) load_pieces(a, t, threadIdx.x, piece);
    for (int k0 = 0; k0 < a.topk; k0 += SLOTS) {
        const int slots = min(SLOTS, a.topk - k0);
        for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < tokens * slots; i += tokens * blockDim.x) {
            const int y = SHARED ? i / slots : 0, k = i - y * slots;
            if (SHARED && t0 + y >= a.tokens) break;
            const int64_t slot = (t0 + y) * a.topk + k0 + k;
            const int rank = s.row_of_slot[slot], e = expert_of(s, slot);
            const int32_t row = ct.table[(int64_t)e * ct.n_chunks + (int)slot / ct.chunk].x + rank;
            s.slot_of_row[row] = (int32_t)slot;
            row_s[y * SLOTS + k] = s.row_of_slot[slot] = e < s.num_experts ? row : ~row;
        }
        __syncthreads();
        const int32_t* my_rows = row_s + (SHARED ? threadIdx.y * SLOTS : 0);
        for (int v0 = threadIdx.x; v0 < units; v0 += PIECES * blockDim.x) {
            if (v0 >= PIECES * (int)blockDim.x || k0 > 0) load_pieces(a, t, v0, piece);
#pragma unroll 1
            for (int k = 0; k < slots; ++k) store_pieces(a, my_rows[k], v0, piece);
        }
        if (a.scale_cols && (!SHARED || t < a.tokens))
            for (int k = 0; k < slots; ++k) store_scales(a, t, k, my_rows[k]);
        __syncthreads();
    }
}

// Few slots: sorting and copying in one launch.  The CTA of a token counts for each of its slots the slots that come
// before it in (expert, slot) order, which is the slot's row, while the token's row is on its way.  The last
// CTA counts the experts instead.  With few tokens each has several CTAs, for a part of its row each (blockIdx.y).
template <typename UNIT, int PIECES>
__global__ void __launch_bounds__(256) sort_and_permute_kernel(SortArgs s, RowArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    __shared__ int32_t hist[MAX_EXPERTS];
    __shared__ int32_t before[8][SLOTS_AT_ONCE];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int numel = (int)s.numel, E = s.num_experts;
    const int64_t t = blockIdx.x;
    if (t * a.topk >= numel) {
        if (blockIdx.y > 0) return;
        for (int e = threadIdx.x; e < E; e += blockDim.x) hist[e] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < numel; i += blockDim.x) {
            const int e = expert_of(s, i);
            if (e < E) atomicAdd(&hist[e], 1);
        }
        __syncthreads();
        int32_t run = 0;
        for (int e0 = 0; e0 < E; e0 += blockDim.x) {
            const int e = e0 + (int)threadIdx.x;
            int32_t incl = e < E ? hist[e] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) before[warp][0] = incl;
            __syncthreads();
            int32_t all = 0;
            for (int w = 0; w < warps; ++w) {
                if (w < warp) incl += before[w][0];
                all += before[w][0];
            }
            if (e < E) s.offs[e] = run + incl;
            run += all;
            __syncthreads();
        }
        return;
    }
    UNIT piece[PIECES];
    const int v0 = blockIdx.y * PIECES * blockDim.x + threadIdx.x;
    load_pieces(a, t, v0, piece);
    for (int k0 = 0; k0 < a.topk; k0 += SLOTS_AT_ONCE) {
        const int first = (int)t * a.topk + k0;
        // (expert, slot) as one number: below 65536 * 1025
        int32_t key[SLOTS_AT_ONCE], n[SLOTS_AT_ONCE];
#pragma unroll
        for (int k = 0; k < SLOTS_AT_ONCE; ++k) {
            key[k] = k0 + k < a.topk ? expert_of(s, first + k) * numel + first + k : 0;
            n[k] = 0;
        }
#pragma unroll 2
        for (int i = threadIdx.x; i < numel; i += blockDim.x) {
            const int32_t other = expert_of(s, i) * numel + i;
#pragma unroll
            for (int k = 0; k < SLOTS_AT_ONCE; ++k) n[k] += other < key[k];
        }
#pragma unroll
        for (int k = 0; k < SLOTS_AT_ONCE; ++k) {
            const int32_t sum = __reduce_add_sync(0xffffffffu, n[k]);
            if (lane == 0) before[warp][k] = sum;
        }
        __syncthreads();
        int32_t r[SLOTS_AT_ONCE];
#pragma unroll
        for (int k = 0; k < SLOTS_AT_ONCE; ++k) {
            r[k] = 0;
            for (int w = 0; w < warps; ++w) r[k] += before[w][k];
            if (k0 + k >= a.topk) continue;
            const bool none = key[k] >= E * numel;
            if (threadIdx.x == 0 && blockIdx.y == 0) {
                s.slot_of_row[r[k]] = first + k;
                s.row_of_slot[first + k] = none ? ~r[k] : r[k];
            }
            if (none) r[k] = ~r[k];
            store_pieces(a, r[k], v0, piece);
            for (int v = v0 + gridDim.y * PIECES * blockDim.x; v < a.units; v += gridDim.y * PIECES * blockDim.x) {
                UNIT more[PIECES];
                load_pieces(a, t, v, more);
                store_pieces(a, r[k], v, more);
            }
            if (a.scale_cols && blockIdx.y == 0) store_scales(a, t, k0 + k, r[k]);
        }
        __syncthreads();
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
    int64_t tokens, H;
    void* out;  // [T, H]
    // backward
    const void* d_out;  // [T, H], row stride ld_d_out
    int64_t ld_d_out;
    void* d_rows;  // [n_rows, H]; NULL: not wanted
    void* d_w;     // [T, topk]; NULL: not wanted
};

// V consecutive values of a row: one 16-byte load, or one value where rows are not aligned to that.
template <typename T, int V>
struct Piece {
    static_assert(V == 1 || V * sizeof(T) == 16, "one value or 16 bytes");
    using Raw = std::conditional_t<V == 1, T, uint4>;
    static __device__ __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
    static __device__ __forceinline__ Raw load_once(const T* p) {
        if constexpr (V == 1) return *p;
        else return __ldcs(reinterpret_cast<const uint4*>(p));
    }
    static __device__ __forceinline__ void unpack(const Raw& raw, float (&f)[V]) {
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = fg_to_float(e[i]);
    }
    static __device__ __forceinline__ void store(T* p, const float (&f)[V]) {
        Raw raw;
        T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = fg_from_float<T>(f[i]);
        *reinterpret_cast<Raw*>(p) = raw;
    }
};

// Rows and weights of K consecutive slots of token t; row -1: nothing to read.
template <int K>
__device__ __forceinline__ void load_slots(const SumArgs& a, int64_t t, int k0, int32_t (&row)[K], float (&w)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        row[k] = k0 + k < a.topk ? a.row_of_slot[t * a.topk + k0 + k] : -1;
        w[k] = a.weights && k0 + k < a.topk ? load_weight(a.weights, a.w_dtype, t * a.ld_w + k0 + k) : 1.0f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (row[k] < 0 || row[k] >= a.n_rows) row[k] = -1;
}

// One CTA per token and per part of its columns (blockIdx.y), or per several tokens (threadIdx.y), sums in fp32 in slot order.
// A thread has K slots of U pieces in flight, eight loads whatever the number of slots.
template <typename T, int V, int K, bool SHARED>
__global__ void __launch_bounds__(256) unpermute_kernel(SumArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    constexpr int U = K >= 8 ? 1 : 8 / K;
    using P = Piece<T, V>;
    const int64_t t = token_of_thread<SHARED>();
    if (SHARED && t >= a.tokens) return;
    const T* rows = reinterpret_cast<const T*>(a.rows);
    const int64_t step = (int64_t)blockDim.x * V;
    int32_t row[K];
    float w[K];
    load_slots(a, t, 0, row, w);
    for (int64_t c = ((int64_t)blockIdx.y * U * blockDim.x + threadIdx.x) * V; c < a.H; c += gridDim.y * U * step) {
        float acc[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[u][i] = 0.0f;
        for (int k0 = 0;;) {
            typename P::Raw raw[K][U];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (row[k] >= 0 && c + u * step < a.H) raw[k][u] = P::load_once(rows + row[k] * a.ld_rows + c + u * step);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (row[k] < 0) continue;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float f[V];
                    P::unpack(raw[k][u], f);
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[u][i] = fmaf(w[k], f[i], acc[u][i]);
                }
            }
            if (a.topk <= K) break;  // the slots stay in registers
            k0 = k0 + K < a.topk ? k0 + K : 0;
            load_slots(a, t, k0, row, w);
            if (k0 == 0) break;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c + u * step < a.H) P::store(reinterpret_cast<T*>(a.out) + t * a.H + c + u * step, acc[u]);
    }
}

// One CTA per token, or per several (threadIdx.y, whole warps each): d_out[t] times the weight into the gradient of every row of
// the token, and its product with the row into the gradient of the weight, slot after slot. d_out is read once where a row is up
// to four pieces per thread (16 KB), everything else is read and written once; the products are summed in a fixed order: a
// thread's columns, the lanes, the warps.  Bound by HBM: 8192 x 8 bf16 rows of 7168 (2.0 GB) take 307 us, 6.5 TB/s, which is the
// rate of a copy.  More slots in flight per thread cost registers and with them CTAs (404 us with two slots at once); streaming
// loads and stores (.cs) take 315.
template <typename T, int V, bool SHARED>
__global__ void __launch_bounds__(256, 4) unpermute_backward_kernel(SumArgs a) {
    fg_pdl_wait();
    fg_pdl_trigger();
    constexpr int U = 4, K = 32;  // pieces per thread and round, slots whose sums are parked at once
    using P = Piece<T, V>;
    __shared__ float part[8][K];
    const int64_t t = token_of_thread<SHARED>();
    const bool live = !SHARED || t < a.tokens;
    const T* rows = reinterpret_cast<const T*>(a.rows);
    const T* d_out = reinterpret_cast<const T*>(a.d_out) + t * a.ld_d_out;
    T* d_rows = reinterpret_cast<T*>(a.d_rows);
    const int step = (int)blockDim.x * V, first = (int)threadIdx.x * V, H = live ? (int)a.H : 0;
    const int first_warp = SHARED ? (int)(threadIdx.y * blockDim.x) >> 5 : 0;
    const bool one_round = H <= U * step;
    typename P::Raw g[U];
    auto load_g = [&](int c) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c + u * step < H) g[u] = P::load(d_out + c + u * step);
    };
    if (one_round) load_g(first);
    for (int k0 = 0; k0 < a.topk; k0 += K) {
        const int slots = min(K, a.topk - k0);
#pragma unroll 1
        for (int k = 0; k < slots; ++k) {
            const int32_t r = live ? a.row_of_slot[t * a.topk + k0 + k] : -1;
            const int64_t row = r < 0 ? ~r : r;
            const bool real = r >= 0 && row < a.n_rows;
            const float w = real && a.weights ? load_weight(a.weights, a.w_dtype, t * a.ld_w + k0 + k) : 1.0f;
            const T* from = rows + row * a.ld_rows;
            T* to = a.d_rows && row < a.n_rows ? d_rows + row * a.H : nullptr;
            float dot = 0.0f;
            for (int c = first; c < H; c += U * step) {
                if (!one_round) load_g(c);
                typename P::Raw raw[U];
                if (a.d_w && real) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + u * step < H) raw[u] = P::load(from + c + u * step);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (c + u * step >= H) continue;
                    float f[V], x[V];
                    P::unpack(g[u], f);
                    if (a.d_w && real) {
                        P::unpack(raw[u], x);
#pragma unroll
                        for (int i = 0; i < V; ++i) dot = fmaf(f[i], x[i], dot);
                    }
                    if (to) {
#pragma unroll
                        for (int i = 0; i < V; ++i) f[i] = real ? w * f[i] : 0.0f;
                        P::store(to + c + u * step, f);
                    }
                }
            }
            if (a.d_w) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                if ((threadIdx.x & 31) == 0) part[first_warp + (threadIdx.x >> 5)][k] = dot;
            }
        }
        if (a.d_w) {
            __syncthreads();
            if ((int)threadIdx.x < slots && live) {
                float sum = 0.0f;
                for (int i = 0; i < (int)blockDim.x / 32; ++i) sum += part[first_warp + i][threadIdx.x];
                store_weight(a.d_w, a.w_dtype, t * a.topk + k0 + threadIdx.x, sum);
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

// Several tokens share a CTA of 256 threads where one is served by fewer and moves few bytes, while four CTAs per SM are left: the
// chip starts a CTA per 1.1 ns, in which 7 KB are moved.  Measured, a CTA per token / shared: 16384 x 8 rows of 128 bytes permuted in
// 24.0 / 11.5 us and summed in 19.0 / 4.8, 16384 x 2 rows of 1024 bytes 22.9 / 13.7 and 18.8 / 12.8.
dim3 block_of_tokens(unsigned threads, int64_t T, int64_t bytes_per_token) {
    unsigned tokens = 1;
    if (bytes_per_token <= 16384)
        while (2 * tokens * threads <= 256 && tokens < 32 && T >= 8 * (int64_t)tokens * fg_num_sms()) tokens *= 2;
    return dim3(threads, tokens);
}

// The same without whole warps: for kernels whose threads do not speak to each other.
unsigned few_threads_for(int64_t n) { return n > 16 ? threads_for(n) : n > 8 ? 16 : 8; }

bool aligned16(const void* p, int64_t stride_bytes) { return (uintptr_t)p % 16 == 0 && stride_bytes % 16 == 0; }

// Whether every token's CTA looks at all slots for itself, one launch instead of three.  What that costs grows with
// tokens x slots and hides behind the rows that are copied meanwhile.  Measured, one launch against three: 8 experts per
// token and rows of 14 KB, 2048 slots 8.8 / 12.7 us, 4096 slots 16.0 / 17.6, 6144 slots 28.9 / 24.6; 2 and 8 KB: 1024 slots 6.6 /
// 6.8, 2048 slots 12.7 / 8.2; 8 and 1 KB: 512 slots 6.1 / 6.5, 2048 slots 9.2 / 6.8.
constexpr int64_t ONE_LAUNCH_LOOKS = 65536;
bool one_launch(int64_t T, int64_t numel, int64_t row_bytes) {
    const int64_t most = 64 * row_bytes > ONE_LAUNCH_LOOKS ? 64 * row_bytes : ONE_LAUNCH_LOOKS;
    return numel <= 65536 && T * numel <= most;
}

// Chunks of whole rounds of a CTA, no more than MAX_CHUNKS of them.
ChunkTable chunk_table(void* workspace, int64_t numel) {
    int64_t chunk = CHUNK_THREADS;
    if (fg_cdiv(numel, chunk) > MAX_CHUNKS) chunk = fg_cdiv(fg_cdiv(numel, MAX_CHUNKS), CHUNK_THREADS) * CHUNK_THREADS;
    return ChunkTable{reinterpret_cast<int2*>(workspace), (int)fg_cdiv(numel, chunk), (int)chunk};
}

int rank_slots(const SortArgs& a, const ChunkTable& ct, cudaStream_t st) {
    const size_t smem = (size_t)CHUNK_WARPS * (a.num_experts + 1) * sizeof(int32_t);
    static std::mutex mu;
    static size_t smem_set[64];
    {
        std::lock_guard<std::mutex> lock(mu);
        size_t& have = smem_set[fg_device_index()];
        if (have < 48 * 1024) have = 48 * 1024;
        if (smem > have) {
            FG_CUDA(cudaFuncSetAttribute(rank_slots_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            have = smem;
        }
    }
    FG_CUDA(fg_launch(rank_slots_kernel, (unsigned)ct.n_chunks, CHUNK_THREADS, smem, st, 1, a, ct));
    FG_CUDA(fg_launch(scan_chunks_kernel, (unsigned)a.num_experts / 8 + 1, 256, 0, st, 1, a, ct));
    return FG_OK;
}

}  // namespace

extern "C" {

int64_t fg_moe_permute_workspace_bytes(int64_t T, int topk, int num_experts) {
    if (T < 0 || topk < 0 || num_experts <= 0 || T * topk >= (1ll << 31) - 1) return -1;
    return one_launch(T, T * topk, 0) ? 0 : (int64_t)chunk_table(nullptr, T * topk).n_chunks * (num_experts + 1) * (int64_t)sizeof(int2);
}

int fg_moe_permute(void* rows, float* row_scale, int32_t* offs, int32_t* row_of_slot, int32_t* slot_of_row, const void* x,
                   const float* scale, const void* topk_ids, int ids_are_i64, const int32_t* expert_map, int expert_map_len,
                   int64_t T, int topk, int num_experts, int64_t H, int elem_bytes, int64_t ld_x, int64_t scale_cols,
                   int64_t ld_scale, void* workspace, int64_t workspace_bytes, void* stream) {
    FG_REQUIRE(T >= 0 && topk >= 0 && H >= 0 && scale_cols >= 0, FG_ERR_INVALID_ARGUMENT, "negative size");
    FG_REQUIRE(num_experts > 0 && num_experts <= MAX_EXPERTS, FG_ERR_UNSUPPORTED, "num_experts %d must be in [1, %d]", num_experts,
               MAX_EXPERTS);
    FG_REQUIRE(elem_bytes == 1 || elem_bytes == 2 || elem_bytes == 4, FG_ERR_INVALID_ARGUMENT, "elements of %d bytes", elem_bytes);
    FG_REQUIRE(T * topk < (1ll << 31) - 1 && H * elem_bytes < (1ll << 31) && scale_cols < (1ll << 31), FG_ERR_UNSUPPORTED, "size too large");
    FG_REQUIRE(expert_map == nullptr || expert_map_len > 0, FG_ERR_INVALID_ARGUMENT, "empty expert_map");
    const int64_t numel = T * topk;
    FG_REQUIRE(offs && (numel == 0 || (topk_ids && row_of_slot && slot_of_row)), FG_ERR_INVALID_ARGUMENT, "null pointer");
    FG_REQUIRE(numel == 0 || H == 0 || (rows && x), FG_ERR_INVALID_ARGUMENT, "null pointer");
    FG_REQUIRE(numel == 0 || scale_cols == 0 || (row_scale && scale), FG_ERR_INVALID_ARGUMENT, "null pointer");
    cudaStream_t st = (cudaStream_t)stream;
    const SortArgs a{topk_ids, ids_are_i64, numel, num_experts, expert_map, expert_map_len, offs, row_of_slot, slot_of_row};
    const int64_t row_bytes = H * elem_bytes;
    const auto aligned = [&](int to) { return (uintptr_t)x % to == 0 && (uintptr_t)rows % to == 0 && ld_x * elem_bytes % to == 0 && row_bytes % to == 0; };
    const int unit = aligned(16) ? 16 : aligned(8) ? 8 : aligned(4) ? 4 : aligned(2) ? 2 : 1;
    const auto row_args = [&](int unit) {
        return RowArgs{x, ld_x * elem_bytes / unit, scale, ld_scale, topk, T, numel, rows, (int)(row_bytes / unit), row_scale, (int)scale_cols};
    };
    const RowArgs r = row_args(unit);
    const unsigned threads = threads_for(r.units);
    auto by_unit = [&](auto&& go) -> cudaError_t {
        return unit == 16 ? go(uint4()) : unit == 8 ? go(uint2()) : unit == 4 ? go((unsigned int)0) : unit == 2 ? go((unsigned short)0) : go((unsigned char)0);
    };
    if (numel > 0 && one_launch(T, numel, row_bytes)) {
        // A row per CTA, four pieces per thread; with few tokens two pieces, and parts of a row until there are two CTAs per SM.
        const unsigned block = threads < 128 ? 128u : threads;
        unsigned parts = 1;
        while (parts < 32 && T * parts * 2 <= 2 * fg_num_sms() && parts * 2 * block < (unsigned)r.units) parts *= 2;
        const dim3 grid((unsigned)T + 1, parts);
        FG_CUDA(by_unit([&](auto u) {
            using U = decltype(u);
            return parts > 1 ? fg_launch(sort_and_permute_kernel<U, 2>, grid, block, 0, st, 1, a, r)
                             : fg_launch(sort_and_permute_kernel<U, 4>, grid, block, 0, st, 1, a, r);
        }));
        return FG_OK;
    }
    if (numel == 0) {
        FG_CUDA(cudaMemsetAsync(offs, 0, (size_t)num_experts * sizeof(int32_t), st));
        return FG_OK;
    }
    const int64_t need = fg_moe_permute_workspace_bytes(T, topk, num_experts);
    FG_REQUIRE(workspace && (uintptr_t)workspace % 8 == 0 && workspace_bytes >= need, FG_ERR_INVALID_ARGUMENT,
               "workspace holds %lld bytes, needs %lld (8-byte aligned)", (long long)workspace_bytes, (long long)need);
    const ChunkTable ct = chunk_table(workspace, numel);
    const int rc = rank_slots(a, ct, st);
    if (rc != FG_OK) return rc;
    // Early whatever the size of the grid: what it waits for is the scan alone, 3 us (fg_launch keeps grids that fill the chip
    // back because they may wait long, in the way of other streams).
    if (aligned(32)) {
        const RowArgs wide = row_args(32);
        const dim3 block = wide.units > 256 ? dim3(wide.units >= 512 ? 512u : (unsigned)(wide.units + 31) / 32 * 32)
                                            : block_of_tokens(few_threads_for(wide.units), T, row_bytes * (topk + 1));
        FG_CUDA(fg_launch_when(true, block.y > 1 ? permute_rows_kernel<Unit32, true> : permute_rows_kernel<Unit32, false>,
                               (unsigned)fg_cdiv(T, block.y), block, 0, st, 1, a, ct, wide));
        return FG_OK;
    }
    const dim3 block = block_of_tokens(few_threads_for(fg_cdiv(r.units, 2)), T, row_bytes * (topk + 1));
    FG_CUDA(by_unit([&](auto u) {
        using U = decltype(u);
        return fg_launch_when(true, block.y > 1 ? permute_rows_kernel<U, true> : permute_rows_kernel<U, false>, (unsigned)fg_cdiv(T, block.y),
                              block, 0, st, 1, a, ct, r);
    }));
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
    a.ld_w = ld_w; a.topk = topk; a.tokens = T; a.H = H; a.out = out;
    const int es = elem_size(dtype);
    const bool vec = aligned16(rows, ld_rows * es) && aligned16(out, H * es);
    const int slots = topk <= 2 ? 2 : topk <= 4 ? 4 : 8;  // at once
    const int64_t pieces = fg_cdiv(vec ? H * es / 16 : H, 8 / slots);  // per thread: 8 / slots
    // Few tokens: their columns are spread over CTAs, until there are two CTAs per SM or a thread has one round.
    unsigned parts = 1;
    while (parts < 64 && T * parts < 2 * fg_num_sms() && parts * (int64_t)threads_for(pieces) < pieces) parts *= 2;
    const dim3 block = parts > 1 ? dim3(threads_for(pieces)) : block_of_tokens(few_threads_for(pieces), T, H * es * (topk + 1));
    return by_type(dtype, [&](auto tag) -> int {
        using E = decltype(tag);
        auto go = [&](auto kernel) { return fg_launch(kernel, dim3((unsigned)fg_cdiv(T, block.y), parts), block, 0, (cudaStream_t)stream, 1, a); };
        auto of_slots = [&](auto v, auto k) {
            constexpr int V = decltype(v)::value, K = decltype(k)::value;
            return block.y > 1 ? go(unpermute_kernel<E, V, K, true>) : go(unpermute_kernel<E, V, K, false>);
        };
        auto by_slots = [&](auto v) -> cudaError_t {
            return slots == 2 ? of_slots(v, std::integral_constant<int, 2>())
                 : slots == 4 ? of_slots(v, std::integral_constant<int, 4>()) : of_slots(v, std::integral_constant<int, 8>());
        };
        FG_CUDA(vec ? by_slots(std::integral_constant<int, 16 / sizeof(E)>()) : by_slots(std::integral_constant<int, 1>()));
        return FG_OK;
    });
}

int fg_moe_unpermute_backward(void* d_rows, void* d_weights, const void* d_out, const void* rows, const int32_t* row_of_slot,
                              const void* weights, int w_dtype, int64_t T, int topk, int64_t n_rows, int64_t H, int64_t ld_d_out,
                              int64_t ld_rows, int64_t ld_w, int dtype, void* stream) {
    FG_REQUIRE(T >= 0 && topk >= 0 && n_rows >= 0 && H >= 0, FG_ERR_INVALID_ARGUMENT, "negative size");
    FG_REQUIRE(T < (1ll << 31) && n_rows < (1ll << 31) && H < (1ll << 30), FG_ERR_UNSUPPORTED, "size too large");
    FG_REQUIRE(!(weights || d_weights) || w_dtype == FG_DTYPE_BF16 || w_dtype == FG_DTYPE_F16 || w_dtype == FG_DTYPE_F32,
               FG_ERR_INVALID_ARGUMENT, "bad weight dtype %d", w_dtype);
    if (T == 0 || topk == 0) return FG_OK;
    FG_REQUIRE(row_of_slot && (H == 0 || d_out) && (!d_weights || rows || H == 0), FG_ERR_INVALID_ARGUMENT, "null pointer");
    SumArgs a{};
    a.rows = rows; a.ld_rows = ld_rows; a.n_rows = n_rows; a.row_of_slot = row_of_slot; a.weights = weights; a.w_dtype = w_dtype;
    a.ld_w = ld_w; a.topk = topk; a.tokens = T; a.H = H; a.d_out = d_out; a.ld_d_out = ld_d_out; a.d_rows = d_rows; a.d_w = d_weights;
    const int es = elem_size(dtype);
    const bool vec = aligned16(d_out, ld_d_out * es) && (!d_weights || aligned16(rows, ld_rows * es)) && aligned16(d_rows, H * es);
    return by_type(dtype, [&](auto tag) -> int {
        using E = decltype(tag);
        constexpr int V = 16 / sizeof(E);
        const dim3 block = block_of_tokens(threads_for(vec ? H / V : H), T, H * es * (2 * topk + 1));
        auto go = [&](auto kernel) { return fg_launch(kernel, (unsigned)fg_cdiv(T, block.y), block, 0, (cudaStream_t)stream, 1, a); };
        auto of_values = [&](auto v) {
            return block.y > 1 ? go(unpermute_backward_kernel<E, decltype(v)::value, true>) : go(unpermute_backward_kernel<E, decltype(v)::value, false>);
        };
        FG_CUDA(vec ? of_values(std::integral_constant<int, V>()) : of_values(std::integral_constant<int, 1>()));
        return FG_OK;
    });
}

}  // extern "C"
