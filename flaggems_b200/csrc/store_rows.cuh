// Results of a warp that holds a row of up to 32 columns per lane, written row by row.
//
// A lane that stores its own row touches 32 rows per instruction: half a sector each by 16 bytes, a sixteenth by 2 bytes where
// rows have no common alignment.  Through 2 KB of shared memory (64 bytes of each row at a time) an instruction writes 8, 2 or 1
// rows, each in one piece.  int8 products, each lane its row / this: 3859 x 6144 x 4096 in fp32 111 / 75 us,
// 3859 x 6145 x 4096 in bf16 309 / 77 and in fp32 223 / 91, 395 x 2845 x 2240 in bf16 24.1 / 12.6.
#pragma once

#include "common.cuh"

// Two values rounded to bf16 or fp16, the first in the lower half.
__device__ __forceinline__ uint32_t fg_pair_of(float lo, float hi, int dtype) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return dtype == FG_DTYPE_BF16 ? *reinterpret_cast<const uint32_t*>(&b) : *reinterpret_cast<const uint32_t*>(&h);
}

// What the begins of rows `stride` bytes apart are multiples of: 16, 4 or 2.
inline int fg_row_align(const void* c, int64_t stride) {
    const uintptr_t x = (uintptr_t)c | (uintptr_t)stride;
    return x % 16 == 0 ? 16 : x % 4 == 0 ? 4 : 2;
}

// The rows of a warp, one per lane, whose results are written if `ok`.  Found before the results are waited for.
struct FgRows {
    uint8_t* first;  // lane 0's
    unsigned ok;     // a bit per lane
    bool even;       // the rows lie a stride apart
};

__device__ __forceinline__ FgRows fg_rows(uint8_t* row, bool ok, int lane, int64_t stride) {
    FgRows r;
    r.first = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)row, 0));
    r.ok = __ballot_sync(0xffffffffu, ok);
    r.even = __all_sync(0xffffffffu, !ok || row == r.first + lane * stride);
    return r;
}

// v: `cols` columns of the lane's row, from byte `offset` of the row on; the rows are even.  The same in all lanes: cols, offset,
// stride and align (fg_row_align).  stage: 2 KB of the warp's own, 16-byte aligned.
__device__ __forceinline__ void fg_store_rows(uint8_t* stage, int lane, const float (&v)[32], const FgRows& rows, int64_t stride,
                                              int64_t offset, int cols, int dtype, int align) {
    // pieces of 16 bytes are swizzled against bank conflicts
    auto at = [&](int r, int byte) { return stage + r * 64 + (byte ^ (((r >> 1) & 3) << 4)); };
    // `bytes` (up to 64) of every row to its byte `offset`
    auto out = [&](int64_t offset, int bytes) {
        if (align == 16 && bytes == 64) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = (lane >> 2) + 8 * j, byte = (lane & 3) << 4;
                uint8_t* p = rows.first + r * stride + offset + byte;
                if ((rows.ok >> r) & 1u) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(at(r, byte));
            }
        } else if (align >= 4) {
#pragma unroll 4
            for (int j = 0; j < 16; ++j) {
                const int r = (lane >> 4) + 2 * j, byte = (lane & 15) << 2;
                uint8_t* p = rows.first + r * stride + offset + byte;
                if (!((rows.ok >> r) & 1u)) continue;
                if (byte + 4 <= bytes) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(at(r, byte));
                else if (byte < bytes) *reinterpret_cast<uint16_t*>(p) = *reinterpret_cast<const uint16_t*>(at(r, byte));
            }
        } else {
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
                const int byte = lane << 1;
                uint8_t* p = rows.first + r * stride + offset + byte;
                if (((rows.ok >> r) & 1u) && byte < bytes) *reinterpret_cast<uint16_t*>(p) = *reinterpret_cast<const uint16_t*>(at(r, byte));
            }
        }
    };
    auto through = [&](const uint32_t (&w)[16], int64_t offset, int bytes) {
        const int mine = (lane >> 1) & 3;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ mine) << 4)) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        __syncwarp();
        out(offset, bytes);
        __syncwarp();
    };
    uint32_t w[16];
    if (dtype == FG_DTYPE_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (16 * h >= cols) break;
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[16 * h + i]);
            through(w, offset + 64 * h, min(64, 4 * (cols - 16 * h)));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = fg_pair_of(v[2 * i], v[2 * i + 1], dtype);
    through(w, offset, 2 * cols);
}
