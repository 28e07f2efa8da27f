// What the launchers of the grouped products share. All five products are one form,
//     out[r, c] = sum_x P[c, x] Q[r, x]        (times scale_q[r] scale_p[c] for 8-bit operands)
// over groups that own a range of the tensor rows:
//     forward   r = token (ragged), c = n, x = k:   P = B[e] (x contiguous), Q = A (x contiguous)
//     dgrad     r = token (ragged), c = k, x = n:   P = B[e] (c contiguous), Q = dC (x contiguous)
//     wgrad     r = n, c = k, x = token (ragged):   P = A (c contiguous),   Q = dC (r contiguous)
// P's 128 or 256 columns are the M side of the MMA and the rows its N side, whose width the instruction takes in
// steps of 16 or 32: a group of few rows costs few MMA columns, and the accumulator of a tile has the output's columns
// in TMEM lanes and its rows in TMEM columns.
#pragma once

#include "host.h"

namespace tcb {

constexpr int kMaxExperts = 1024;   // the kernels keep three integers per expert in shared memory

struct GroupedProblem {
    const void* p;
    const void* q;
    const float* scale_p;     // [experts, cols] or null
    const float* scale_q;     // [token_rows] or null
    const void* offsets;      // null: one group of all rows
    int offsets_are_int64;
    void* out;
    int64_t token_rows;       // rows of the tensors that the offsets cut
    int64_t experts;
    int64_t cols;             // extent of c
    int64_t other;            // forward, dgrad: extent of x; wgrad: extent of r
    int64_t ldp, stride_p, ldq, ldo, stride_o;   // elements; stride_o: wgrad only
    int in_type;              // tc_type of P and Q, or kTypeI8
    int out_type;
    bool p_c_contiguous;      // dgrad, wgrad
    bool ragged_x;            // wgrad
};
constexpr int kTypeI8 = 100;

// What the kernels get by value.
struct GroupedArgs {
    const void* offsets;
    const float* scale_p;
    const float* scale_q;
    void* out;
    int64_t ldo, stride_o;
    int offsets_are_int64;
    int token_rows;
    int experts;
    int cols;
    int other;
    int tile_rows;        // most rows of an output tile, a power of two
    int tile_shift;       // its logarithm
    int most_row_tiles;   // row tiles of all groups together; more come out of overlapping offsets only and are left out
    int out_type;
    int vector_out;       // rows of out start on 16-byte boundaries
    uint32_t idesc;       // instruction descriptor without the N field
    uint32_t* status;
};

inline GroupedArgs grouped_args(const GroupedProblem& g, int tile_rows, int64_t row_tiles, const DeviceInfo* dev) {
    GroupedArgs a;
    a.offsets = g.offsets;
    a.scale_p = g.scale_p;
    a.scale_q = g.scale_q;
    a.out = g.out;
    a.ldo = g.ldo;
    a.stride_o = g.stride_o;
    a.offsets_are_int64 = g.offsets_are_int64;
    a.token_rows = static_cast<int>(g.token_rows);
    a.experts = static_cast<int>(g.experts);
    a.cols = static_cast<int>(g.cols);
    a.other = static_cast<int>(g.other);
    a.tile_rows = tile_rows;
    a.tile_shift = 0;
    while ((1 << a.tile_shift) < tile_rows) ++a.tile_shift;
    a.most_row_tiles = static_cast<int>(row_tiles);
    a.out_type = g.out_type;
    const int es = g.out_type == TC_F32 ? 4 : 2;
    a.vector_out = aligned16(g.out) && (g.ldo * es) % 16 == 0 && (g.stride_o * es) % 16 == 0;
    a.idesc = 0;
    a.status = dev->status_word;
    return a;
}

// tcgen05 instruction descriptor without its N field, for M rows of the MMA (sm100.cuh: make_idesc_f16_f32). For kind::i8
// the format fields count otherwise: D 2 = s32, A and B 1 = s8.
uint32_t grouped_idesc(const GroupedProblem& g, int m);

// Tensor maps of the operands, 128-byte swizzle: 128 bytes of the contiguous dimension by box_rows of the other one.
int grouped_map_p(CUtensorMap* map, const GroupedProblem& g, int box_rows);
int grouped_map_q(CUtensorMap* map, const GroupedProblem& g, int box_rows);

// Which kernel runs a problem.
struct GroupedPlan {
    bool pair;        // grouped_pair.cu, else grouped_split.cu
    int tile_rows;    // most rows of an output tile
    int splits;       // pieces of x per tile (split kernel)
    int64_t row_tiles;   // bound on the row tiles of all groups together
    int64_t tiles;    // and on the output tiles
    bool alone;       // one CTA per SM (split kernel)
};

int launch_grouped_pair(const GroupedProblem& g, const GroupedPlan& plan, const DeviceInfo* dev, cudaStream_t stream);
int launch_grouped_split(const GroupedProblem& g, const GroupedPlan& plan, const DeviceInfo* dev, cudaStream_t stream);

}  // namespace tcb
