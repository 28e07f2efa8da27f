// Grouped products on CTA pairs: tiles of 256 output columns (128 per CTA) by up to 256 rows, tcgen05.mma.cta_group::2
// with M = 256 (output columns) and N = the tile's rows rounded up to 32. See grouped.h for the common form.
//   warp 0      TMA producer (both CTAs): per stage 256 bytes of x for 128 columns of P and half of the tile's rows of Q,
//               landing in the issuing CTA's shared memory and completing on the leader's full barrier;
//   warp 1      TMEM owner; in the leader also the MMA issuer;
//   warps 2..17 epilogue (both CTAs), four per TMEM lane quarter: accumulator -> scaled -> converted -> shared memory -> rows
//               of the output, 16 rows at a time. A warp spends most of a block waiting (TMEM, stmatrix, stores), so their
//               number counts: four took 6500 cycles for a 128 x 256 accumulator, more than the MMAs of a short sum, eight
//               4500; sixteen take another 7 to 12 % off a weight gradient of many experts (64 x [2048, 1024]: 97 us from
//               105) and a fifth off 8-bit results on unaligned rows;
//   warp 18     works out the CTA's tiles, 16 at a time (one per lane), into a ring in shared memory: a search and three
//               divisions, about 1000 cycles, which the MMA issuer would otherwise spend between any two tiles;
//   warp 19     wgrad only: the last K step (16 rows of x) of a group may hold rows of the next group, which have to count as
//               zero whatever they hold (NaN included), in both operands. Such a step has a buffer of its own, loaded when
//               the producer starts the tile; this warp overwrites the foreign rows with zeros long before the MMA issuer
//               comes to it. (Cleared in the ring instead, it held up every tile by about 1000 cycles.)
// Persistent over tiles; accumulators are double-buffered in TMEM, except for a tile whose sum is longer than kSumPiece: its
// pieces all go through one accumulator, and the columns of the other one hold their total. Which tiles there are follows from
// the offsets, which every CTA reads from device memory into a table at the start.
#include "grouped.cuh"

namespace tcb {

constexpr int kGpCols = 128;              // output columns per CTA
constexpr int kGpRows = 256;              // most rows per tile
constexpr int kGpStages = 3;
constexpr int kGpOperand = 128 * 256;     // bytes of one operand per stage and CTA: 128 columns / rows x 256 bytes of x
constexpr int kGpChunk = kGpOperand / 2;  // 128 bytes of x (x contiguous), or 64 columns / rows (those contiguous)
constexpr int kGpStageBytes = 2 * kGpOperand;
constexpr int kGpEpilogueWarps = 16;
constexpr int kGpDrainRows = 16;          // rows of a block
constexpr int kGpThreads = 32 * (3 + kGpEpilogueWarps);   // and a warp more for wgrad
constexpr int kGpBatch = 16;              // tiles worked out at a time; the ring holds two batches
constexpr int kGpTailPiece = 16 * 128;    // 16 rows of x for 64 columns / rows
constexpr int kGpTailSlot = 4 * kGpTailPiece;

// Shared memory behind the ring of operand stages.
template <bool kI8, bool kRaggedX>
struct PairSmem {
    static constexpr int kTail = kGpStages * kGpStageBytes;                          // wgrad: two slots
    static constexpr int kStaging = kTail + (kRaggedX ? 2 * kGpTailSlot : 0);
    static constexpr int kScales = kStaging + kGpEpilogueWarps * kGpDrainRows * 64;
    static constexpr int kTiles = kScales + (kI8 ? kGpEpilogueWarps * kGpDrainRows * 4 : 0);
    static constexpr int kBars = kTiles + 2 * kGpBatch * static_cast<int>(sizeof(GroupTile));
    static constexpr int kTable = kBars + 256;                                        // forward, dgrad
    static constexpr int kTotal = kTable + (kRaggedX ? 0 : static_cast<int>(sizeof(GroupTable))) + 1024;
    static_assert(kTotal <= 232448, "shared memory of one CTA");
};

// A role's walk through the CTA's tiles. One thread or one converged warp each.
struct TileCursor {
    const GroupTile* ring;
    uint64_t* bar_full;     // [2]: a batch has been written
    uint64_t* bar_empty;    // [2]: every role has read the last tile of a batch
    volatile uint32_t* abort_word;
    int i;

    // false at the end, or when a wait ran out. kWarp: all lanes call it, lane 0 arrives.
    template <bool kWarp>
    __device__ __forceinline__ bool next(GroupTile& t) {
        const int half = (i / kGpBatch) & 1;
        if (i % kGpBatch == 0) {
            const uint32_t parity = static_cast<uint32_t>(i / (2 * kGpBatch)) & 1u;
            const bool ok = kWarp ? mbar_wait_warp(&bar_full[half], parity, abort_word, kDevTimeoutMma)
                                  : mbar_wait(&bar_full[half], parity, abort_word, kDevTimeoutMma);
            if (!ok) return false;
        }
        t = ring[i % (2 * kGpBatch)];
        if (i % kGpBatch == kGpBatch - 1) {
            if (kWarp) __syncwarp();
            if (!kWarp || (threadIdx.x & 31) == 0) mbar_arrive(&bar_empty[half]);
        }
        ++i;
        return t.rows > 0;
    }
};

__device__ __forceinline__ void umma_i8_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* m, uint32_t bar_cluster_addr, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// The epilogue's part in a tile whose sum comes in `before_last` + 1 pieces: waits for each, adds it to the total, and leaves the
// whole sum in the accumulator. One warp; false when a wait ran out.
static __device__ __noinline__ bool join_pieces(uint32_t acc, uint32_t total, uint64_t* bar_full, uint64_t* bar_empty, uint32_t parity,
                                                int before_last, int rows, int first, volatile uint32_t* abort_word) {
    for (int piece = 0;; ++piece) {
        if (!mbar_wait_warp(bar_full, parity, abort_word, kDevTimeoutEpilogue)) return false;
        tc_fence_after_sync();
        const bool is_last = piece == before_last;
        add_sum_piece(acc, total, piece == 0, is_last, rows, first, kGpEpilogueWarps / 4 * kGpDrainRows, kGpDrainRows);
        if (is_last) return true;
        tc_fence_before_sync();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive_cluster(map_to_cta(smem_u32(bar_empty), 0));
        parity ^= 1u;
    }
}

// kLong: a sum may be longer than kSumPiece (never for 8-bit operands, whose sums are exact).
template <bool kI8, bool kPCols, bool kRaggedX, bool kLong>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kRaggedX ? kGpThreads + 32 : kGpThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                    const __grid_constant__ CUtensorMap tmap_p_small,
                    const __grid_constant__ CUtensorMap tmap_q_small, const GroupedArgs a) {
    constexpr int kBlockX = kI8 ? 256 : 128;   // x elements per stage
    constexpr int kStepX = kBlockX / 8;        // per MMA
    constexpr int kPieceBlocks = kSumPiece / kBlockX;
    static_assert(!(kI8 && kLong));
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    uint8_t* smem_p = smem;
    uint8_t* smem_q = smem + kGpStages * kGpOperand;
    using S = PairSmem<kI8, kRaggedX>;
    uint8_t* smem_tail = smem + S::kTail;
    uint8_t* staging = smem + S::kStaging;
    float* scales = reinterpret_cast<float*>(smem + S::kScales);
    GroupTile* tile_ring = reinterpret_cast<GroupTile*>(smem + S::kTiles);
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem + S::kBars);   // used in the leader
    uint64_t* bar_empty = bar_full + kGpStages;          // one per CTA
    uint64_t* bar_acc_full = bar_empty + kGpStages;      // one per CTA
    uint64_t* bar_acc_empty = bar_acc_full + 2;          // used in the leader
    uint64_t* bar_tail_full = bar_acc_empty + 2;         // one per CTA: its part of a last step has landed
    uint64_t* bar_tail_ready = bar_tail_full + 2;        // used in the leader: both CTAs have cleared the foreign rows
    uint64_t* bar_tail_empty = bar_tail_ready + 2;       // one per CTA
    uint64_t* bar_tiles_full = bar_tail_empty + 2;       // one per CTA
    uint64_t* bar_tiles_empty = bar_tiles_full + 2;      // one per CTA
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_tiles_empty + 2);
    volatile uint32_t* abort_word = tmem_slot + 1;
    GroupTable* table = reinterpret_cast<GroupTable*>(smem + S::kTable);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const uint32_t rank = __shfl_sync(0xffffffffu, cluster_ctarank(), 0);   // 0 = leader
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    const int col_tiles = (a.cols + 2 * kGpCols - 1) / (2 * kGpCols);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kGpStages; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_tail_full[i], 1);
            mbar_init(&bar_tail_ready[i], 2);
            mbar_init(&bar_tail_empty[i], 1);
            mbar_init(&bar_acc_full[i], 1);
            mbar_init(&bar_acc_empty[i], 2 * kGpEpilogueWarps);   // of both CTAs
            mbar_init(&bar_tiles_full[i], 1);
            mbar_init(&bar_tiles_empty[i], 1 + kGpEpilogueWarps + (rank == 0 ? 1 : 0) + (kRaggedX ? 1 : 0));
        }
        *abort_word = 0;
        fence_barrier_init();
    }
    if (warp == 2 && lane == 0) {
        tma_prefetch_desc(&tmap_p);
        tma_prefetch_desc(&tmap_q);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    grid_launch_dependents();
    // Without offsets the tiles follow from the sizes: the table is part of the set-up, which does not wait for the kernel before
    // this one. (Built by the scheduler in that case too, it cost nothing there, but the compiler made the epilogue of all
    // variants 3 to 18 % slower: 7252 x 7426 int8, K = 144, 64 us instead of 55.)
    if (!kRaggedX && a.offsets == nullptr && warp == 0) build_group_table(table, a, false);
    tc_fence_before_sync();
    cluster_sync_all();   // barriers of both CTAs are initialised before anyone signals across the pair
    tc_fence_after_sync();
    // From here on everybody who touches global memory first waits for the kernel before this one (griddepcontrol.wait).
    const uint32_t tmem_base = *tmem_slot;
    TileCursor cursor{tile_ring, bar_tiles_full, bar_tiles_empty, abort_word, 0};
    GroupTile t;

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        const bool leader = elect_one_sync();
        grid_dependency_wait();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        int tails = 0;
        while (ok && cursor.next<true>(t)) {
            const int x_len = kRaggedX ? t.x_len & ~15 : t.x_len;   // what the ring carries
            const int blocks = (x_len + kBlockX - 1) / kBlockX;
            const int col = t.col0 + static_cast<int>(rank) * kGpCols;
            const int half = t.width >> 1;                              // this CTA's rows of Q
            const int row = t.row0 + static_cast<int>(rank) * half;
            if (kRaggedX && x_len != t.x_len) {
                const int slot = tails & 1;
                if (!mbar_wait_warp(&bar_tail_empty[slot], (static_cast<uint32_t>(tails >> 1) & 1u) ^ 1u, abort_word, kDevTimeoutProducer)) break;
                if (leader) {
                    const uint32_t bar_addr = map_to_cta(smem_u32(&bar_tail_full[slot]), rank);
                    uint8_t* dst = smem_tail + slot * kGpTailSlot;
                    mbar_arrive_expect_tx(&bar_tail_full[slot], kGpTailSlot);
                    for (int c = 0; c < 2; ++c) {
                        tma_load_3d_pair(dst + c * kGpTailPiece, &tmap_p_small, bar_addr, col + c * 64, t.x0 + x_len, 0);
                        tma_load_2d_pair(dst + (2 + c) * kGpTailPiece, &tmap_q_small, bar_addr, row + c * 64, t.x0 + x_len);
                    }
                }
                ++tails;
            }
            for (int kb = 0; kb < blocks; ++kb) {
                if (!mbar_wait_warp(&bar_empty[stage], phase ^ 1u, abort_word, kDevTimeoutProducer)) {
                    ok = false;
                    break;
                }
                const int x = kb * kBlockX;
                const int chunks = x_len - x > kBlockX / 2 ? 2 : 1;      // 128-byte pieces of x
                const int q_boxes = (half + 31) >> 5;
                const bool whole_q = t.width == kGpRows;
                const bool two_rows = half > 64;                         // wgrad: 64-row pieces of Q
                // wgrad: of a group's last block only the 16-row steps that it has are fetched
                const int steps = kRaggedX ? min(kBlockX, x_len - x) >> 4 : 8;
                const uint32_t p_bytes = kRaggedX ? steps * 2 * kGpTailPiece : kPCols ? kGpOperand : chunks * kGpChunk;
                const uint32_t q_bytes = kRaggedX ? steps * (two_rows ? 2 : 1) * kGpTailPiece : chunks * (whole_q ? kGpChunk : q_boxes * 4096);
                const uint32_t bar_addr = map_to_cta(smem_u32(&bar_full[stage]), 0);   // counts the bytes of both CTAs
                uint8_t* dst_p = smem_p + stage * kGpOperand;
                uint8_t* dst_q = smem_q + stage * kGpOperand;
                if (leader) {
                    if (rank == 0) mbar_arrive_expect_tx(&bar_full[stage], 2 * (p_bytes + q_bytes));
                    if (kRaggedX) {
                        const int y = t.x0 + x;
                        for (int i = 0; i < (steps < 8 ? steps : 1); ++i) {
                            const CUtensorMap* mp = steps < 8 ? &tmap_p_small : &tmap_p;
                            const CUtensorMap* mq = steps < 8 ? &tmap_q_small : &tmap_q;
                            const int at = i * kGpTailPiece;
                            tma_load_3d_pair(dst_p + at, mp, bar_addr, col, y + i * 16, 0);
                            tma_load_3d_pair(dst_p + kGpChunk + at, mp, bar_addr, col + 64, y + i * 16, 0);
                            tma_load_2d_pair(dst_q + at, mq, bar_addr, row, y + i * 16);
                            if (two_rows) tma_load_2d_pair(dst_q + kGpChunk + at, mq, bar_addr, row + 64, y + i * 16);
                        }
                    } else {
                        if (kPCols) {
                            tma_load_3d_pair(dst_p, &tmap_p, bar_addr, col, x, t.e);
                            tma_load_3d_pair(dst_p + kGpChunk, &tmap_p, bar_addr, col + 64, x, t.e);
                        } else {
                            for (int c = 0; c < chunks; ++c) tma_load_3d_pair(dst_p + c * kGpChunk, &tmap_p, bar_addr, x + c * (kBlockX / 2), col, t.e);
                        }
                        for (int c = 0; c < chunks; ++c) {
                            if (whole_q) {
                                tma_load_2d_pair(dst_q + c * kGpChunk, &tmap_q, bar_addr, x + c * (kBlockX / 2), row);
                            } else {
                                for (int b = 0; b < q_boxes; ++b)
                                    tma_load_2d_pair(dst_q + c * kGpChunk + b * 4096, &tmap_q_small, bar_addr, x + c * (kBlockX / 2), row + b * 32);
                            }
                        }
                    }
                }
                if (++stage == kGpStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader CTA only) ----------------
        if (lane == 0 && rank == 0) {
            const uint32_t desc_hi = smem_desc_hi_sw128(1024);
            const uint32_t p_lo0 = smem_desc_lo(smem_u32(smem_p), kPCols ? kGpChunk : 16);
            const uint32_t q_lo0 = smem_desc_lo(smem_u32(smem_q), kRaggedX ? kGpChunk : 16);
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;   // bit per accumulator
            int tails = 0;
            bool ok = true;
            while (ok && cursor.next<false>(t)) {
                const int x_len = kRaggedX ? t.x_len & ~15 : t.x_len;
                const int blocks = (x_len + kBlockX - 1) / kBlockX;
                const uint32_t idesc = a.idesc | (static_cast<uint32_t>(t.width >> 3) << 17);
                if (!mbar_wait(&bar_acc_empty[acc], ((acc_phase >> acc) & 1u) ^ 1u, abort_word, kDevTimeoutMma)) break;
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kGpRows);
                bool landed = false;   // the next stage was seen full while the MMAs of this one were being issued
                int piece_end = kLong ? kPieceBlocks : blocks;
                for (int kb = 0; kb < blocks; ++kb) {
                    if (kLong && kb == piece_end) {
                        umma_commit_pair_both(smem_u32(&bar_acc_full[acc]));
                        acc_phase ^= 1u << acc;
                        piece_end += kPieceBlocks;
                        if (!mbar_wait(&bar_acc_empty[acc], ((acc_phase >> acc) & 1u) ^ 1u, abort_word, kDevTimeoutMma)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                    }
                    if (!landed && !mbar_wait(&bar_full[stage], phase, abort_word, kDevTimeoutMma)) {
                        ok = false;
                        break;
                    }
                    const int rest = x_len - kb * kBlockX;
                    tc_fence_after_sync();
                    const uint32_t p_lo = p_lo0 + static_cast<uint32_t>(stage) * (kGpOperand >> 4);
                    const uint32_t q_lo = q_lo0 + static_cast<uint32_t>(stage) * (kGpOperand >> 4);
                    const int steps = min(8, (rest + kStepX - 1) / kStepX);
                    const bool wraps = stage + 1 == kGpStages;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (k == 4) landed = kb + 1 < blocks && mbar_test(&bar_full[wraps ? 0 : stage + 1], wraps ? phase ^ 1u : phase);
                        if (k < steps) {
                            // x contiguous: 32 bytes on in the swizzled row, the next chunk after four; else 16 rows of x on
                            const uint32_t off_p = kPCols ? k * (2048u >> 4) : static_cast<uint32_t>(((k >> 2) * kGpChunk + (k & 3) * 32) >> 4);
                            const uint32_t off_q = kRaggedX ? k * (2048u >> 4) : static_cast<uint32_t>(((k >> 2) * kGpChunk + (k & 3) * 32) >> 4);
                            const uint64_t dp = smem_desc_join(p_lo + off_p, desc_hi), dq = smem_desc_join(q_lo + off_q, desc_hi);
                            if (kI8) umma_i8_ss_pair(d_tmem, dp, dq, idesc, (kb | k) != 0);
                            else umma_f16_ss_pair(d_tmem, dp, dq, idesc, kLong && k == 0 ? kb + kPieceBlocks != piece_end : (kb | k) != 0);
                        }
                    }
                    umma_commit_pair_both(smem_u32(&bar_empty[stage]));
                    if (++stage == kGpStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (kRaggedX && x_len != t.x_len) {
                    const int slot = tails & 1;
                    if (!mbar_wait_cluster(&bar_tail_ready[slot], static_cast<uint32_t>(tails >> 1) & 1u, abort_word, kDevTimeoutMma)) break;
                    tc_fence_after_sync();
                    const uint32_t lo = smem_desc_lo(smem_u32(smem_tail), kGpTailPiece) + static_cast<uint32_t>(slot) * (kGpTailSlot >> 4);
                    umma_f16_ss_pair(d_tmem, smem_desc_join(lo, desc_hi), smem_desc_join(lo + (2 * kGpTailPiece >> 4), desc_hi), idesc, blocks > 0);
                    umma_commit_pair_both(smem_u32(&bar_tail_empty[slot]));
                    ++tails;
                }
                umma_commit_pair_both(smem_u32(&bar_acc_full[acc]));
                acc_phase ^= 1u << acc;
                // behind a long sum the same one again: once it is free, so is its total in the other one
                if (!kLong || blocks <= kPieceBlocks) acc ^= 1;
            }
        }
        __syncwarp();
    } else if (warp < 2 + kGpEpilogueWarps) {
        // ---------------- epilogue (both CTAs) ----------------
        grid_dependency_wait();
        const int quarter = warp & 3;
        uint8_t* stage = staging + (warp - 2) * kGpDrainRows * 64;
        float* row_scales = scales + (warp - 2) * kGpDrainRows;
        const int first_row = ((warp - 2) >> 2) * kGpDrainRows;   // its first block of rows; the warps of a quarter take turns
        int acc = 0;
        uint32_t acc_phase = 0;   // bit per accumulator
        while (cursor.next<true>(t)) {
            const int col = t.col0 + static_cast<int>(rank) * kGpCols + quarter * 32;
            const TileScales tile_scales = load_scales<kI8>(t, a, col, lane, first_row);
            const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
            const uint32_t taddr = lanes + static_cast<uint32_t>(acc * kGpRows);
            const int x_len = kRaggedX ? t.x_len & ~15 : t.x_len;   // what goes through the ring
            const bool in_pieces = kLong && x_len > kSumPiece;
            if (in_pieces) {
                if (!join_pieces(taddr, lanes + static_cast<uint32_t>((acc ^ 1) * kGpRows), &bar_acc_full[acc], &bar_acc_empty[acc],
                                 (acc_phase >> acc) & 1u, (x_len - 1) / kSumPiece, t.rows, first_row, abort_word))
                    break;
                acc_phase ^= static_cast<uint32_t>((x_len - 1) / kSumPiece & 1) << acc;
            } else {
                if (!mbar_wait_warp(&bar_acc_full[acc], (acc_phase >> acc) & 1u, abort_word, kDevTimeoutEpilogue)) break;
                tc_fence_after_sync();
            }
            acc_phase ^= 1u << acc;
            drain_tile<kI8, kRaggedX, kGpDrainRows>(taddr, t, a, col, stage, row_scales, tile_scales, t.x_len == 0, lane, first_row,
                                                     kGpEpilogueWarps / 4 * kGpDrainRows);
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_acc_empty[acc]), 0));
            if (!in_pieces) acc ^= 1;
        }
    } else if (warp == 2 + kGpEpilogueWarps) {
        // ---------------- which tiles (both CTAs) ----------------
        // In the weight gradient all but what is summed over follows from the sizes, and waits for no other kernel.
        if (!kRaggedX && a.offsets != nullptr) {
            grid_dependency_wait();
            build_group_table(table, a, blockIdx.x == 0);
        }
        const int row_tiles = group_row_tiles<kRaggedX>(a, 0);   // wgrad: of every group
        const int num_tiles = (kRaggedX ? a.experts * row_tiles : table->tiles_before[a.experts]) * col_tiles;
        bool bad = false;
        for (int batch = 0;; ++batch) {
            const int half = batch & 1;
            if (batch >= 2 && !mbar_wait_warp(&bar_tiles_empty[half], (static_cast<uint32_t>(batch >> 1) & 1u) ^ 1u, abort_word, kDevTimeoutMma)) break;
            const int64_t tile = pair + static_cast<int64_t>(batch * kGpBatch + lane) * num_pairs;
            GroupTile g = {};   // no rows: the end
            if (lane < kGpBatch) {
                if (tile < num_tiles) {
                    if (kRaggedX) {
                        const int per_group = row_tiles * col_tiles;
                        const int e = static_cast<int>(tile) / per_group;
                        g = banded_tile<true>(a, e, 0, 0, static_cast<int>(tile) - e * per_group, row_tiles, col_tiles, 2 * kGpCols);
                    } else {
                        g = group_tile(table, a, static_cast<int>(tile), col_tiles, 2 * kGpCols);
                    }
                }
            }
            if (kRaggedX && batch == 0) grid_dependency_wait();   // only what is summed over depends on the offsets
            if (lane < kGpBatch) {
                if (kRaggedX && g.rows > 0) group_range(a, g.e, g.x0, g.x_len, bad);
                tile_ring[half * kGpBatch + lane] = g;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_tiles_full[half]);
            if (pair + static_cast<int64_t>((batch + 1) * kGpBatch - 1) * num_pairs >= num_tiles) break;   // the end marker is out
        }
        if (bad) atomicMax(a.status, static_cast<uint32_t>(kDevIndexOutOfRange));
    } else if (kRaggedX) {
        // ---------------- clears the foreign rows of last steps (both CTAs) ----------------
        int tails = 0;
        while (cursor.next<true>(t)) {
            const int first = t.x_len & 15;
            if (first == 0) continue;
            const int slot = tails & 1;
            if (!mbar_wait_warp(&bar_tail_full[slot], static_cast<uint32_t>(tails >> 1) & 1u, abort_word, kDevTimeoutMma)) break;
            ++tails;
            uint8_t* p = smem_tail + slot * kGpTailSlot + first * 128;
            for (int i = lane; i < (16 - first) * 8; i += 32)
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(p + c * kGpTailPiece + i * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_tail_ready[slot]), 0));
        }
    }

    // ---------------- teardown: neither CTA frees TMEM or exits while its peer may still touch it ----------------
    __syncwarp();
    tc_fence_before_sync();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, 512);
    }
    if (threadIdx.x == 0 && *abort_word != 0) atomicMax(a.status, *abort_word);
}

template <bool kI8, bool kPCols, bool kRaggedX, bool kLong>
static int launch_variant(const CUtensorMap& tp, const CUtensorMap& tq, const CUtensorMap& tp_small, const CUtensorMap& tq_small,
                          const GroupedArgs& a, int pairs, const DeviceInfo* dev, cudaStream_t stream) {
    auto kernel = grouped_pair_kernel<kI8, kPCols, kRaggedX, kLong>;
    constexpr int smem = PairSmem<kI8, kRaggedX>::kTotal;
    static OncePerDevice once;
    if (int rc = raise_smem_limit_once(once, dev->device, kernel, smem)) return rc;
    TCB_CUDA(launch_overlapped(kernel, dim3(2 * pairs), dim3(kRaggedX ? kGpThreads + 32 : kGpThreads), smem, stream, tp, tq, tp_small, tq_small, a));
    return TC_OK;
}

int launch_grouped_pair(const GroupedProblem& g, const GroupedPlan& plan, const DeviceInfo* dev, cudaStream_t stream) {
    const bool i8 = g.in_type == kTypeI8;
    GroupedArgs a = grouped_args(g, plan.tile_rows, plan.row_tiles, dev);
    a.idesc = grouped_idesc(g, 2 * kGpCols);
    // 128-row boxes; of Q also 32-row ones for tiles of fewer rows, or (wgrad) 16 rows of x of both for a group's last step
    CUtensorMap tp, tq, tp_small, tq_small;
    if (int rc = grouped_map_p(&tp, g, 128)) return rc;
    if (int rc = grouped_map_q(&tq, g, 128)) return rc;
    if (int rc = grouped_map_q(&tq_small, g, g.ragged_x ? 16 : 32)) return rc;
    if (g.ragged_x) {
        if (int rc = grouped_map_p(&tp_small, g, 16)) return rc;
    } else {
        tp_small = tp;
    }
    const int64_t max_pairs = dev->sm_count / 2;
    const int pairs = static_cast<int>(plan.tiles < max_pairs ? plan.tiles : max_pairs);
    if (i8) return launch_variant<true, false, false, false>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
    if ((g.ragged_x ? g.token_rows : g.other) > kSumPiece) {
        if (g.ragged_x) return launch_variant<false, true, true, true>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
        if (g.p_c_contiguous) return launch_variant<false, true, false, true>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
        return launch_variant<false, false, false, true>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
    }
    if (g.ragged_x) return launch_variant<false, true, true, false>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
    if (g.p_c_contiguous) return launch_variant<false, true, false, false>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
    return launch_variant<false, false, false, false>(tp, tq, tp_small, tq_small, a, pairs, dev, stream);
}

}  // namespace tcb
