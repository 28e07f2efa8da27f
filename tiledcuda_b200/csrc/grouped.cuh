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

// Row range of group e. Offsets are clamped into [0, token_rows] and a decreasing pair makes an empty group, so that
// whatever they hold no access leaves the tensors; `bad` tells that this was needed.
__device__ __forceinline__ void group_range(const GroupedArgs& a, int e, int& first, int& len, bool& bad) {
    int64_t lo = 0, hi = a.token_rows;
    if (a.offsets != nullptr) {
        if (a.offsets_are_int64) {
            lo = static_cast<const int64_t*>(a.offsets)[e];
            hi = static_cast<const int64_t*>(a.offsets)[e + 1];
        } else {
            lo = static_cast<const int32_t*>(a.offsets)[e];
            hi = static_cast<const int32_t*>(a.offsets)[e + 1];
        }
    }
    const int64_t rows = a.token_rows;
    bad |= lo < 0 || hi > rows || hi < lo;
    lo = min(max(lo, static_cast<int64_t>(0)), rows);
    hi = max(lo, min(max(hi, static_cast<int64_t>(0)), rows));
    first = static_cast<int>(lo);
    len = static_cast<int>(hi - lo);
}

// Row tiles of a group: its rows cut evenly, or (wgrad) the same for every group.
template <bool kRaggedX>
__device__ __forceinline__ int group_row_tiles(const GroupedArgs& a, int len) {
    return static_cast<int>((static_cast<uint32_t>(kRaggedX ? a.other : len) + static_cast<uint32_t>(a.tile_rows) - 1) >> a.tile_shift);
}

__device__ __forceinline__ int64_t warp_inclusive_sum(int64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += up;
    }
    return v;
}

// Executed by one whole warp (forward and dgrad); `report` lets one CTA of the grid record bad offsets.
__device__ __forceinline__ void build_group_table(GroupTable* t, const GroupedArgs& a, bool report) {
    const int lane = threadIdx.x & 31;
    int64_t base = 0;
    bool bad = false;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int e = e0 + lane;
        int tiles = 0;
        if (e < a.experts) {
            int first, len;
            group_range(a, e, first, len, bad);
            t->first[e] = first;
            t->len[e] = len;
            tiles = group_row_tiles<false>(a, len);
        }
        const int64_t sum = warp_inclusive_sum(tiles);
        const int64_t most = a.most_row_tiles;
        if (e < a.experts) t->tiles_before[e] = static_cast<int>(min(base + sum - tiles, most));
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) t->tiles_before[a.experts] = static_cast<int>(min(base, static_cast<int64_t>(a.most_row_tiles)));
    if (report && __any_sync(0xffffffffu, bad) && lane == 0) atomicMax(a.status, static_cast<uint32_t>(kDevIndexOutOfRange));
    __syncwarp();
}

// One output tile: rows [row0, row0 + rows) of the output (of group e's slice for wgrad), columns from col0 on, summed over
// x in [x0, x0 + x_len). `width` is rows rounded up to 32 (16 where tiles have 16), the N extent of its MMAs.
struct GroupTile {
    int e, row0, rows, width, col0, x0, x_len;
};

template <bool kRaggedX>
__device__ __forceinline__ GroupTile make_group_tile(const GroupedArgs& a, int e, int first, int len, int rt, int row_tiles, int col0) {
    GroupTile g;
    g.e = e;
    g.col0 = col0;
    if (kRaggedX) {
        g.row0 = rt * a.tile_rows;
        g.rows = min(a.tile_rows, a.other - g.row0);
        g.x0 = first;
        g.x_len = len;
    } else {
        // the rows of a group spread evenly over its tiles, in steps of 32
        const int step = min(a.tile_rows, ((len - 1) / row_tiles + 32) & ~31);
        g.row0 = first + rt * step;
        g.rows = min(step, len - rt * step);
        g.x0 = 0;
        g.x_len = a.other;
    }
    g.width = min(a.tile_rows, (g.rows + 31) & ~31);
    return g;
}

// The tiles of a group are walked in bands of kBandCols column tiles, row tiles outermost inside a band, so that the CTAs in
// flight share operands through L2: neighbours read the same rows of Q at the same time, and a piece of P is read by the few
// row tiles under way. (8192^3 in 8 bits: 337 us with bands of 16, 346 with 8, 342 with 12, 347 with 24, 368 with all 32 column
// tiles in one band, 382 with the column tiles outermost.)
constexpr int kBandCols = 16;

template <bool kRaggedX>
__device__ __forceinline__ GroupTile banded_tile(const GroupedArgs& a, int e, int first, int len, int local, int row_tiles, int col_tiles,
                                                 int tile_cols) {
    const int per_band = kBandCols * row_tiles;
    const int band = local / per_band;
    const int band_cols = min(kBandCols, col_tiles - band * kBandCols);
    const int in_band = local - band * per_band;
    const int rt = in_band / band_cols;
    const int ct = band * kBandCols + in_band - rt * band_cols;
    return make_group_tile<kRaggedX>(a, e, first, len, rt, row_tiles, ct * tile_cols);
}

__device__ __forceinline__ GroupTile group_tile(const GroupTable* t, const GroupedArgs& a, int tile, int col_tiles, int tile_cols) {
    const int row_tile_all = tile / col_tiles;
    int lo = 0, hi = a.experts - 1;          // the last group with tiles_before <= row_tile_all
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t->tiles_before[mid] <= row_tile_all) lo = mid;
        else hi = mid - 1;
    }
    const int before = t->tiles_before[lo];
    return banded_tile<false>(a, lo, t->first[lo], t->len[lo], tile - before * col_tiles, t->tiles_before[lo + 1] - before, col_tiles, tile_cols);
}

// 16-bit operands: the tensor cores cut what they add to an accumulator, at about 2^-24 of it on average in each step of 16
// terms, always towards zero. Over a long sum of one sign that adds up (2^20 terms in one accumulator: 2e-3 of the sum), so an
// accumulator takes 8192 terms at most, 5e-5; the pieces of a longer sum are added in fp32 to nearest, in order, and kept
// in TMEM columns beside the accumulator. An epilogue warp does so for the lanes and columns that it drains.
constexpr int kSumPiece = 8192;

// One piece of a long sum: total = acc for the first, total += acc for those between, acc += total for the last. Of the
// tile's rows (TMEM columns) those that this warp drains: `block` of them (16 or 32) from `first` on, then `step` on.
static __device__ __noinline__ void add_sum_piece(uint32_t acc, uint32_t total, bool is_first, bool is_last, int rows, int first, int step,
                                                  int block) {
    for (int j0 = first; j0 < rows; j0 += step) {
        for (int j = j0; j < min(rows, j0 + block); j += 16) {
            uint32_t v[16];
            __syncwarp();
            tmem_ld_x16(acc + static_cast<uint32_t>(j), v);
            if (!is_first) {
                uint32_t t[16];
                tmem_ld_x16(total + static_cast<uint32_t>(j), t);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(t[i]) + __uint_as_float(v[i]));
            } else {
                tmem_ld_wait();
            }
            tmem_st_x16((is_last ? acc : total) + static_cast<uint32_t>(j), v);
        }
    }
    tmem_st_wait();
}

__device__ __forceinline__ uint16_t to_half_bits(float v, int type) {
    return type == TC_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    return pack_half2(lo, hi);
}

// 16 TMEM lanes by 32 columns: register 4 q + 2 i + b of a thread is lane 8 i + lane / 4, column 8 q + 2 (lane % 4) + b,
// i.e. four 16 x 8 blocks, each in the accumulator fragment layout of the warp-level MMAs.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_block(uint32_t taddr, uint32_t (&r)[2][16]) {
    tmem_ld_16x256b_x4(taddr, r[0]);
    tmem_ld_16x256b_x4(taddr + (16u << 16), r[1]);
}
__device__ __forceinline__ void tmem_ld_block(uint32_t taddr, uint32_t (&r)[2][8]) {
    tmem_ld_16x256b_x2(taddr, r[0]);
    tmem_ld_16x256b_x2(taddr + (16u << 16), r[1]);
}
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_x32(taddr, r); }
__device__ __forceinline__ void tmem_ld_columns(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_x16(taddr, r); }

// Four 8 x 8 blocks of 16-bit values, each stored transposed: lane l gives the address of row l % 8 of block l / 8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What a warp needs of the scales of its part of an 8-bit tile: those of its columns, and of the first 32 rows it takes. Loaded
// while the accumulator is still being computed: read from memory when they are needed, they cost each block of 32 rows a trip
// to L2.
struct TileScales {
    float p[4];   // columns 8 m + lane / 4 where 16-bit results leave as rows; else p[0] is column `lane`
    float q;      // row first + lane
};

__device__ __forceinline__ bool leaves_by_rows(const GroupedArgs& a) { return a.out_type != TC_F32 && a.vector_out; }

template <bool kI8>
__device__ __forceinline__ TileScales load_scales(const GroupTile& t, const GroupedArgs& a, int col, int lane, int first) {
    TileScales s = {};
    if (kI8) {
        const int cols = a.cols - col;
        const float* scale_p = a.scale_p + static_cast<int64_t>(t.e) * a.cols + col;
        const bool by_rows = leaves_by_rows(a);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int c = by_rows ? 8 * m + (lane >> 2) : lane;
            s.p[m] = c < cols && (by_rows || m == 0) ? scale_p[c] : 0.f;
        }
        s.q = first + lane < t.rows ? a.scale_q[t.row0 + first + lane] : 0.f;
    }
    return s;
}

// 16-bit results on 16-byte rows: tcgen05.ld in fragment layout, packed along rows, transposed by stmatrix into
// [row][column] and stored as 64-byte row pieces. A block of 32 rows costs a warp 4 stmatrix instead of 32 stores of 2 bytes
// a lane; the block after it is loaded from TMEM meanwhile.
template <bool kI8, bool kRaggedX, int kRows, bool kBf16>
__device__ __forceinline__ void drain_rows(uint32_t taddr, const GroupTile& t, const GroupedArgs& a, int cols, int64_t out0, uint8_t* staging,
                                           float* row_scales, TileScales scales, bool zero, int lane, int first, int step) {
    const float* scale_q = kI8 ? a.scale_q + t.row0 : nullptr;
    const uint32_t stage = smem_u32(staging);
    // rows of 64 bytes, their 16-byte pieces exchanged so that neither side meets a bank twice
    const int sr = lane & 7, sm = lane >> 3;
    const uint32_t st_addr = stage + static_cast<uint32_t>(sr * 64 + ((sm ^ (sr >> 1)) & 3) * 16);
    const int lr = lane >> 2, lp = lane & 3;
    const uint8_t* ld_addr = staging + lr * 64 + ((lp ^ (lr >> 1)) & 3) * 16;
    uint16_t* out = static_cast<uint16_t*>(a.out) + out0 + lr * a.ldo + lp * 8;
    const int piece_cols = cols - lp * 8;
    uint32_t r[2][kRows / 2];
    tmem_ld_block(taddr + static_cast<uint32_t>(first), r);
    for (int j0 = first; j0 < t.rows; j0 += step) {
        __syncwarp();   // the block before this one has left the staging area
        if (kI8) {
            if (lane < kRows) row_scales[lane] = scales.q;
            scales.q = lane < kRows && j0 + step + lane < t.rows ? scale_q[j0 + step + lane] : 0.f;
        }
        tmem_ld_wait();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kRows / 8; ++q) {
            uint32_t h[4];
            uint64_t sq2 = 0;
            if (kI8) sq2 = *reinterpret_cast<const uint64_t*>(row_scales + 8 * q + 2 * (lane & 3));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const uint32_t u0 = r[m >> 1][4 * q + 2 * (m & 1)], u1 = r[m >> 1][4 * q + 2 * (m & 1) + 1];
                float lo, hi;
                if (kI8) {
                    const uint64_t v = mul2(pack2(__int2float_rn(static_cast<int>(u0)), __int2float_rn(static_cast<int>(u1))), sq2);
                    unpack2(mul2(v, pack2(scales.p[m], scales.p[m])), lo, hi);
                } else {
                    lo = kRaggedX && zero ? 0.f : __uint_as_float(u0);
                    hi = kRaggedX && zero ? 0.f : __uint_as_float(u1);
                }
                h[m] = pack_pair<kBf16>(lo, hi);
            }
            stmatrix_x4_trans(st_addr + static_cast<uint32_t>(q) * 512, h[0], h[1], h[2], h[3]);
        }
        if (j0 + step < t.rows) tmem_ld_block(taddr + static_cast<uint32_t>(j0 + step), r);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kRows / 8; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(ld_addr + i * 512);
            uint16_t* dst = out + static_cast<int64_t>(j0 + i * 8) * a.ldo;
            if (j0 + i * 8 + lr < t.rows) {
                if (piece_cols >= 8) {
                    *reinterpret_cast<uint4*>(dst) = x;
                } else {
                    const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < piece_cols) dst[j] = static_cast<uint16_t>(e[j >> 1] >> ((j & 1) * 16));
                }
            }
        }
    }
}

// Drains the part of an output tile that one warp owns: 32 output columns (TMEM lanes, from column `col` of the output on)
// by the tile's rows (TMEM columns), scaled, converted and stored; of the rows the kRows from `first` on, then `step` on.
// `staging` is kRows * 64 bytes and `row_scales` kRows floats of shared memory of this warp. `zero`: the accumulator holds
// nothing, the sum is empty. 16-bit results on 16-byte rows go through drain_rows; everything else keeps one column per
// lane, and each row of a block is one coalesced store of 32 elements.
template <bool kI8, bool kRaggedX, int kRows>
__device__ __forceinline__ void drain_tile(uint32_t taddr, const GroupTile& t, const GroupedArgs& a, int col, uint8_t* staging,
                                           float* row_scales, TileScales scales, bool zero, int lane, int first, int step) {
    const int cols = a.cols - col;
    if (cols <= 0 || first >= t.rows) return;
    const int64_t out0 = (kRaggedX ? t.e * a.stride_o : 0) + static_cast<int64_t>(t.row0) * a.ldo + col;
    const float* scale_q = kI8 ? a.scale_q + t.row0 : nullptr;
    if (leaves_by_rows(a)) {
        if (a.out_type == TC_BF16) drain_rows<kI8, kRaggedX, kRows, true>(taddr, t, a, cols, out0, staging, row_scales, scales, zero, lane, first, step);
        else drain_rows<kI8, kRaggedX, kRows, false>(taddr, t, a, cols, out0, staging, row_scales, scales, zero, lane, first, step);
    } else {
        for (int j0 = first; j0 < t.rows; j0 += step) {
            uint32_t r[kRows];
            __syncwarp();
            if (kI8) {
                if (lane < kRows) row_scales[lane] = scales.q;
                scales.q = lane < kRows && j0 + step + lane < t.rows ? scale_q[j0 + step + lane] : 0.f;
                __syncwarp();
            }
            tmem_ld_columns(taddr + static_cast<uint32_t>(j0), r);
            tmem_ld_wait();
            if (lane < cols) {
                const int64_t at = out0 + static_cast<int64_t>(j0) * a.ldo + lane;
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    if (j0 + j < t.rows) {
                        const float v = kI8 ? __int2float_rn(static_cast<int>(r[j])) * row_scales[j] * scales.p[0] : kRaggedX && zero ? 0.f : __uint_as_float(r[j]);
                        if (a.out_type == TC_F32) static_cast<float*>(a.out)[at + j * a.ldo] = v;
                        else static_cast<uint16_t*>(a.out)[at + j * a.ldo] = to_half_bits(v, a.out_type);
                    }
                }
            }
        }
    }
    __syncwarp();
}

}  // namespace tcb
