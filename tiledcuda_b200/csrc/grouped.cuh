// Device side shared by the kernels of the grouped products: the table of groups in shared memory, conversion of
// accumulators and the way from TMEM to the output.
#pragma once

#include <cuda_bf16.h>

#include "grouped.h"
#include "sm100.cuh"

namespace tcb {

// Per group: first row and number of rows, and the number of row tiles in all groups before it.
struct GroupTable {
    int first[kMaxExperts];
    int len[kMaxExperts];
    int tiles_before[kMaxExperts + 1];
};

// Executed by one whole warp. Offsets are clamped into [0, token_rows] and a decreasing pair makes an empty group, so
// that whatever they hold no access leaves the tensors; `report` lets one CTA of the grid record that.
// fixed_tiles >= 0: every group has that many row tiles (wgrad).
__device__ __forceinline__ void build_group_table(GroupTable* t, const GroupedArgs& a, int fixed_tiles, bool report) {
    const int lane = threadIdx.x & 31;
    if (a.offsets == nullptr) {
        if (lane == 0) {
            t->first[0] = 0;
            t->len[0] = a.token_rows;
            t->tiles_before[0] = 0;
            t->tiles_before[1] = fixed_tiles >= 0 ? fixed_tiles : (a.token_rows + a.tile_rows - 1) / a.tile_rows;
        }
        __syncwarp();
        return;
    }
    int base = 0;
    bool bad = false;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int e = e0 + lane;
        int tiles = 0;
        if (e < a.experts) {
            int64_t lo, hi;
            if (a.offsets_are_int64) {
                lo = static_cast<const int64_t*>(a.offsets)[e];
                hi = static_cast<const int64_t*>(a.offsets)[e + 1];
            } else {
                lo = static_cast<const int32_t*>(a.offsets)[e];
                hi = static_cast<const int32_t*>(a.offsets)[e + 1];
            }
            const int64_t rows = a.token_rows;
            bad |= lo < 0 || hi > rows || hi < lo;
            lo = min(max(lo, static_cast<int64_t>(0)), rows);
            hi = max(lo, min(max(hi, static_cast<int64_t>(0)), rows));
            const int len = static_cast<int>(hi - lo);
            t->first[e] = static_cast<int>(lo);
            t->len[e] = len;
            tiles = fixed_tiles >= 0 ? fixed_tiles : (len + a.tile_rows - 1) / a.tile_rows;
        }
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        if (e < a.experts) t->tiles_before[e] = base + sum - tiles;
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) t->tiles_before[a.experts] = base;
    if (report && __any_sync(0xffffffffu, bad) && lane == 0) atomicMax(a.status, static_cast<uint32_t>(kDevIndexOutOfRange));
    __syncwarp();
}

// One output tile: rows [row0, row0 + rows) of the output (of group e's slice for wgrad), columns from col0 on, summed over
// x in [x0, x0 + x_len). `width` is rows rounded up to 32, the N extent of its MMAs.
struct GroupTile {
    int e, row0, rows, width, col0, x0, x_len;
};

// The tiles of a group are walked in bands of kBandCols column tiles, row tiles outermost inside a band, so that the CTAs
// in flight share operands through L2.
constexpr int kBandCols = 8;

template <bool kRaggedX>
__device__ __forceinline__ GroupTile group_tile(const GroupTable* t, const GroupedArgs& a, int tile, int col_tiles, int tile_cols) {
    const int row_tile_all = tile / col_tiles;
    int lo = 0, hi = a.experts - 1;          // the last group with tiles_before <= row_tile_all
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t->tiles_before[mid] <= row_tile_all) lo = mid;
        else hi = mid - 1;
    }
    GroupTile g;
    g.e = lo;
    const int before = t->tiles_before[lo];
    const int row_tiles = t->tiles_before[lo + 1] - before;
    const int local = tile - before * col_tiles;
    const int per_band = kBandCols * row_tiles;
    const int band = local / per_band;
    const int band_cols = min(kBandCols, col_tiles - band * kBandCols);
    const int in_band = local - band * per_band;
    const int rt = in_band / band_cols;
    const int ct = band * kBandCols + in_band - rt * band_cols;
    g.col0 = ct * tile_cols;
    if (kRaggedX) {
        g.row0 = rt * a.tile_rows;
        g.rows = min(a.tile_rows, a.other - g.row0);
        g.x0 = t->first[lo];
        g.x_len = t->len[lo];
    } else {
        // the rows of a group spread evenly over its tiles, in steps of 32
        const int len = t->len[lo];
        const int step = ((len + row_tiles - 1) / row_tiles + 31) & ~31;
        g.row0 = t->first[lo] + rt * step;
        g.rows = min(step, len - rt * step);
        g.x0 = 0;
        g.x_len = a.other;
    }
    g.width = (g.rows + 31) & ~31;
    return g;
}

__device__ __forceinline__ uint16_t to_half_bits(float v, int type) {
    return type == TC_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// 32 x 32 block of the output, one column per lane and one row per register, through `stage` (4 KiB of this warp) to
// out[row, col] for row < rows and column < cols: rows leave as 64-byte (16-bit types) or 128-byte pieces.
__device__ __forceinline__ void store_block(const float (&v)[32], uint8_t* stage, const GroupedArgs& a, int64_t out_index, int rows,
                                            int cols, int lane) {
    __syncwarp();   // the previous block has left the staging area
    if (a.out_type == TC_F32) {
        float* s = reinterpret_cast<float*>(stage);
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j * 32 + lane] = v[j];
        __syncwarp();
        float* out = static_cast<float*>(a.out) + out_index;
        const int piece = lane & 7;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (r >= rows) break;
            const float4 x = *reinterpret_cast<const float4*>(s + r * 32 + piece * 4);
            float* dst = out + r * a.ldo + piece * 4;
            if (a.vector_out && piece * 4 + 4 <= cols) {
                *reinterpret_cast<float4*>(dst) = x;
            } else {
                const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (piece * 4 + j < cols) dst[j] = e[j];
            }
        }
    } else {
        uint16_t* s = reinterpret_cast<uint16_t*>(stage);
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j * 32 + lane] = to_half_bits(v[j], a.out_type);
        __syncwarp();
        uint16_t* out = static_cast<uint16_t*>(a.out) + out_index;
        const int piece = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2);
            if (r >= rows) break;
            const uint4 x = *reinterpret_cast<const uint4*>(s + r * 32 + piece * 8);
            uint16_t* dst = out + r * a.ldo + piece * 8;
            if (a.vector_out && piece * 8 + 8 <= cols) {
                *reinterpret_cast<uint4*>(dst) = x;
            } else {
                const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (piece * 8 + j < cols) dst[j] = static_cast<uint16_t>(e[j >> 1] >> ((j & 1) * 16));
            }
        }
    }
}

}  // namespace tcb
