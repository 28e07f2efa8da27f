// Grouped products for few output tiles: one lone CTA per 128 output columns x up to 128 rows, the sum over x cut into
// as many pieces as the cluster has CTAs, the pieces added through distributed shared memory. See grouped.h for the common form.
//   warp 0      TMA producer: per stage 128 bytes of x for 128 columns of P and the tile's rows of Q;
//   warp 1      TMEM owner and MMA issuer (M = 128, N = rows of the tile rounded up); for wgrad it also clears the rows
//               of the next group in the last x block before the MMAs read them;
//   warps 2..9  epilogue, two per TMEM lane quarter.
// With one or a few rows per group the work is reading P once. Two CTAs fit on an SM, so that one streams while the other
// starts or drains. Partial sums are added in rank order: the result does not change from run to run, no workspace and no
// atomics are needed.
#include "grouped.cuh"

namespace tcb {

constexpr int kGsCols = 128;
constexpr int kGsEpilogueWarps = 8;
constexpr int kGsThreads = 64 + 32 * kGsEpilogueWarps;
constexpr int kGsP = 128 * 128;                 // bytes of P per stage
constexpr int kGsRing = 108 * 1024;             // bytes of the ring where two CTAs share an SM
constexpr int kGsRingAlone = 216 * 1024;        // and where the grid leaves each its own
constexpr int kGsTail = 512;                    // barriers, tile
constexpr int kGsMaxStages = 12;
constexpr int gs_smem(int ring) { return ring + kGsTail + 1024; }
static_assert(2 * (gs_smem(kGsRing) + 1024) <= 233472 && gs_smem(kGsRingAlone) <= 232448, "shared memory of an SM");

template <bool kI8>
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    if (kI8) {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
            "}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
            : "memory");
    } else {
        umma_f16_ss(d_tmem, a_desc, b_desc, idesc, accumulate);
    }
}

__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t cluster_addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}

// Adds the partial sums of kRows rows of four columns over the cluster, in rank order.
template <bool kI8, int kRows>
__device__ __forceinline__ void sum_partials(uint32_t local_addr, uint32_t row_step, int splits, float (&v)[kRows][4]) {
    uint4 p[kRows][8];
#pragma unroll
    for (int s = 0; s < 8; ++s)
        if (s < splits) {
            const uint32_t at = map_to_cta(local_addr, static_cast<uint32_t>(s));
#pragma unroll
            for (int r = 0; r < kRows; ++r) p[r][s] = ld_cluster_v4(at + static_cast<uint32_t>(r) * row_step);
        }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        uint32_t t[4] = {p[r][0].x, p[r][0].y, p[r][0].z, p[r][0].w};
#pragma unroll
        for (int s = 1; s < 8; ++s)
            if (s < splits) {
                const uint32_t q[4] = {p[r][s].x, p[r][s].y, p[r][s].z, p[r][s].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) t[j] = kI8 ? t[j] + q[j] : __float_as_uint(__uint_as_float(t[j]) + __uint_as_float(q[j]));
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[r][j] = kI8 ? __int2float_rn(static_cast<int>(t[j])) : __uint_as_float(t[j]);
    }
}

// Four columns of one row of the output, `cols` of them inside it.
__device__ __forceinline__ void store_four(const GroupedArgs& a, int64_t at, const float (&v)[4], int cols) {
    if (a.out_type == TC_F32) {
        float* out = static_cast<float*>(a.out) + at;
        if (a.vector_out && cols >= 4) {
            *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) out[j] = v[j];
        }
    } else {
        uint16_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = to_half_bits(v[j], a.out_type);
        uint16_t* out = static_cast<uint16_t*>(a.out) + at;
        if (a.vector_out && cols >= 4) {
            *reinterpret_cast<uint2*>(out) = make_uint2(h[0] | (static_cast<uint32_t>(h[1]) << 16), h[2] | (static_cast<uint32_t>(h[3]) << 16));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) out[j] = h[j];
        }
    }
}

// The tile that is number row_tile among the row tiles of all groups, with columns from col0 on: the group it lies in is found
// by one warp, each lane summing a run of consecutive groups, and written to *out by the lane that has it. rows == 0: there
// is no such tile.
template <bool kRaggedX>
__device__ __forceinline__ void find_tile(const GroupedArgs& a, int row_tile, int col0, GroupTile* out, bool report) {
    const int lane = threadIdx.x & 31;
    const int run = (a.experts + 31) >> 5;
    const int e0 = lane * run, e1 = min(a.experts, e0 + run);
    bool bad = false;
    int first = 0, len = 0, tiles = 0;     // of the last group of the run
    int64_t mine = 0;
    for (int e = e0; e < e1; ++e) {
        group_range(a, e, first, len, bad);
        tiles = group_row_tiles<kRaggedX>(a, len);
        mine += tiles;
    }
    int64_t before = warp_inclusive_sum(mine) - mine;
    if (report && __any_sync(0xffffffffu, bad) && lane == 0) atomicMax(a.status, static_cast<uint32_t>(kDevIndexOutOfRange));
    const bool here = row_tile >= before && row_tile < before + mine;
    if (here) {
        int e = e1 - 1;
        if (run > 1) {
            for (e = e0; e < e1; ++e) {
                group_range(a, e, first, len, bad);
                tiles = group_row_tiles<kRaggedX>(a, len);
                if (row_tile < before + tiles) break;
                before += tiles;
            }
        }
        *out = make_group_tile<kRaggedX>(a, e, first, len, static_cast<int>(row_tile - before), tiles, col0);
    }
    if (!__any_sync(0xffffffffu, here) && lane == 0) out->rows = 0;
}

// The epilogue's part in a sum that comes in `before_last` + 1 pieces: waits for each, adds it to the total, and leaves the whole
// sum in the accumulator. One warp; false when a wait ran out.
static __device__ __noinline__ bool join_pieces(uint32_t acc, uint32_t total, uint64_t* bar_full, uint64_t* bar_empty, int before_last,
                                                int rows, int first, volatile uint32_t* abort_word) {
    for (int piece = 0;; ++piece) {
        if (!mbar_wait_warp(bar_full, static_cast<uint32_t>(piece) & 1u, abort_word, kDevTimeoutEpilogue)) return false;
        tc_fence_after_sync();
        const bool is_last = piece == before_last;
        add_sum_piece(acc, total, piece == 0, is_last, rows, first, 64, 32);
        if (is_last) return true;
        tc_fence_before_sync();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar_empty);
    }
}

// kLong: a CTA's part of a sum may be longer than kSumPiece (never for 8-bit operands, whose sums are exact).
template <bool kI8, bool kPCols, bool kRaggedX, bool kLong>
__global__ void __launch_bounds__(kGsThreads, 2)
grouped_split_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const GroupedArgs a,
                     int splits, int ring_bytes) {
    constexpr int kBlockX = kI8 ? 128 : 64;   // x elements per stage
    constexpr int kStepX = kBlockX / 4;       // per MMA
    constexpr int kPieceBlocks = kSumPiece / kBlockX;
    static_assert(!(kI8 && kLong));
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = align_smem_1024(smem_raw);
    const int q_bytes = a.tile_rows * 128;
    const int stage_bytes = kGsP + q_bytes;
    const int stages = min(kGsMaxStages, ring_bytes / stage_bytes);
    uint64_t* bar_full = reinterpret_cast<uint64_t*>(ring + ring_bytes);
    uint64_t* bar_empty = bar_full + kGsMaxStages;
    uint64_t* bar_acc = bar_empty + kGsMaxStages;
    uint64_t* bar_acc_empty = bar_acc + 1;   // of sums in pieces
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_acc_empty + 1);
    volatile uint32_t* abort_word = tmem_slot + 1;
    GroupTile* shared_tile = reinterpret_cast<GroupTile*>(tmem_slot + 2);
    float* scales = reinterpret_cast<float*>(ring);   // epilogue, after the ring has been read

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int rank = splits > 1 ? static_cast<int>(__shfl_sync(0xffffffffu, cluster_ctarank(), 0)) : 0;
    const int col_tiles = (a.cols + kGsCols - 1) / kGsCols;
    // the total of a long sum takes as many columns again as the accumulator
    const uint32_t tmem_cols = static_cast<uint32_t>(max(32, kLong ? 2 * a.tile_rows : a.tile_rows));

    if (threadIdx.x == 0) {
        for (int s = 0; s < kGsMaxStages; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        mbar_init(bar_acc, 1);
        mbar_init(bar_acc_empty, kGsEpilogueWarps);
        *abort_word = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, tmem_cols);
        tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmap_p);
        tma_prefetch_desc(&tmap_q);
    }
    // Without offsets the tile follows from the sizes, and the set-up is over before the kernel in front is (0.8 us of a
    // call of 4 to 6).
    const bool dense = a.offsets == nullptr;
    const int row_tile = static_cast<int>(blockIdx.x) / splits / col_tiles;
    const int col0 = (static_cast<int>(blockIdx.x) / splits - row_tile * col_tiles) * kGsCols;
    if (dense && threadIdx.x == 0) *shared_tile = make_group_tile<false>(a, 0, 0, a.token_rows, row_tile, group_row_tiles<false>(a, a.token_rows), col0);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    // The next kernel may come once TMEM is allocated, not before: where it shares an SM, it could take columns that a CTA of this
    // one still has to get, and would then wait for this kernel with them.
    grid_launch_dependents();
    grid_dependency_wait();   // the offsets may come from the kernel before this one
    if (!dense) {
        if (warp == 0) find_tile<kRaggedX>(a, row_tile, col0, shared_tile, blockIdx.x == 0);
        __syncthreads();
    }
    const uint32_t tmem_base = *tmem_slot;
    const GroupTile t = *shared_tile;
    const int all_blocks = (t.x_len + kBlockX - 1) / kBlockX;
    const int per_rank = (all_blocks + splits - 1) / splits;
    const int block0 = min(all_blocks, rank * per_rank);
    const int block1 = t.rows > 0 ? min(all_blocks, block0 + per_rank) : block0;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        const bool leader = elect_one_sync();
        int stage = 0;
        uint32_t phase = 0;
        for (int b = block0; b < block1; ++b) {
            if (!mbar_wait_warp(&bar_empty[stage], phase ^ 1u, abort_word, kDevTimeoutProducer)) break;
            if (leader) {
                uint8_t* dst_p = ring + stage * stage_bytes;
                uint8_t* dst_q = dst_p + kGsP;
                const int x = b * kBlockX;
                mbar_arrive_expect_tx(&bar_full[stage], static_cast<uint32_t>(stage_bytes));
                if (kPCols) {
                    const int y = kRaggedX ? t.x0 + x : x;
                    const int z = kRaggedX ? 0 : t.e;
                    tma_load_3d(dst_p, &tmap_p, &bar_full[stage], t.col0, y, z);
                    tma_load_3d(dst_p + 8192, &tmap_p, &bar_full[stage], t.col0 + 64, y, z);
                } else {
                    tma_load_3d(dst_p, &tmap_p, &bar_full[stage], x, t.col0, t.e);
                }
                if (kRaggedX) {
                    for (int r = 0; r < a.tile_rows; r += 64) tma_load_2d(dst_q + r * 128, &tmap_q, &bar_full[stage], t.row0 + r, t.x0 + x);
                } else {
                    tma_load_2d(dst_q, &tmap_q, &bar_full[stage], x, t.row0);
                }
            }
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA issuer: the whole warp, one elected lane executes the MMAs ----------------
        const bool leader = elect_one_sync();
        const uint32_t idesc = a.idesc | (static_cast<uint32_t>(t.width >> 3) << 17);
        const uint32_t desc_hi = smem_desc_hi_sw128(1024);
        const uint32_t p_lo0 = smem_desc_lo(smem_u32(ring), kPCols ? 8192 : 16);
        const uint32_t q_lo0 = smem_desc_lo(smem_u32(ring) + kGsP, kRaggedX ? 8192 : 16);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        uint32_t acc_phase = 0;
        int first = block0;   // of the piece
        for (int b = block0; b < block1; ++b) {
            if (kLong && b == first + kPieceBlocks) {
                first = b;
                if (leader) umma_commit(bar_acc);
                if (!mbar_wait_warp(bar_acc_empty, acc_phase, abort_word, kDevTimeoutMma)) {
                    ok = false;
                    break;
                }
                acc_phase ^= 1u;
            }
            if (!mbar_wait_warp(&bar_full[stage], phase, abort_word, kDevTimeoutMma)) {
                ok = false;
                break;
            }
            const int rest = t.x_len - b * kBlockX;
            if (kRaggedX && rest < kBlockX && (rest & 15) != 0) {
                // rows of 128 bytes in each 64-wide piece of both operands, up to the end of the last K step
                const int n = ((rest + 15) & ~15) - rest;
                for (int piece = 0; piece < stage_bytes; piece += 8192)
                    for (int i = lane; i < n * 8; i += 32)
                        *reinterpret_cast<uint4*>(ring + stage * stage_bytes + piece + (rest + (i >> 3)) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
            }
            tc_fence_after_sync();
            const uint32_t p_lo = p_lo0 + static_cast<uint32_t>(stage * stage_bytes) / 16;
            const uint32_t q_lo = q_lo0 + static_cast<uint32_t>(stage * stage_bytes) / 16;
            const int steps = min(4, (rest + kStepX - 1) / kStepX);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k < steps && leader)
                    umma_ss<kI8>(tmem_base, smem_desc_join(p_lo + k * (kPCols ? 2048u >> 4 : 2u), desc_hi),
                                 smem_desc_join(q_lo + k * (kRaggedX ? 2048u >> 4 : 2u), desc_hi), idesc, b != first || k != 0);
            }
            if (leader) umma_commit(&bar_empty[stage]);
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (ok && leader && t.rows > 0) umma_commit(bar_acc);   // not where nobody waits for it: the CTA may be gone by then
        __syncwarp();
    }

    // ---------------- epilogue ----------------
    // a warp reads the TMEM lanes of its quarter, the two of a quarter take turns at blocks of 32 rows
    const int quarter = warp & 3;
    const int part_of_rows = (warp - 2) >> 2;
    const bool drains = warp >= 2;
    const bool summed = block1 > block0;   // else this CTA's part is zero
    TileScales tile_scales = {};
    if (kI8 && drains && t.rows > 0 && splits == 1) tile_scales = load_scales<kI8>(t, a, t.col0 + quarter * 32, lane, part_of_rows * 32);
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    bool ok = drains && t.rows > 0;
    if (kLong && ok && block1 - block0 > kPieceBlocks) {
        ok = join_pieces(taddr, taddr + static_cast<uint32_t>(a.tile_rows), bar_acc, bar_acc_empty, (block1 - block0 - 1) / kPieceBlocks,
                         t.rows, part_of_rows * 32, abort_word);
    } else if (ok) {
        ok = mbar_wait_warp(bar_acc, 0, abort_word, kDevTimeoutEpilogue);
        if (ok) tc_fence_after_sync();
    }
    const int64_t out0 = (kRaggedX ? t.e * a.stride_o : 0) + static_cast<int64_t>(t.row0) * a.ldo;
    if (splits == 1) {
        if (ok) drain_tile<kI8, kRaggedX, 32>(taddr, t, a, t.col0 + quarter * 32, ring + 4096 + (warp - 2) * 2048, scales + (warp - 2) * 32,
                                          tile_scales, !summed, lane, part_of_rows * 32, 64);
    } else {
        // raw partial sums [row][column] into shared memory (every MMA of this CTA has read the ring), then rank s adds up and
        // writes its share of the rows
        uint32_t* part = reinterpret_cast<uint32_t*>(ring);
        if (ok) {
            for (int j0 = part_of_rows * 32; j0 < t.rows; j0 += 64) {
                uint32_t r[32];
                tmem_ld_x32(taddr + static_cast<uint32_t>(j0), r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (j0 + j < t.rows) part[(j0 + j) * kGsCols + quarter * 32 + lane] = summed ? r[j] : 0u;
            }
        }
        __syncwarp();
        cluster_sync_all();
        if (ok) {
            // a warp takes every eighth row of the share, two at a time, four columns a thread
            const int share = (t.rows + splits - 1) / splits;
            const int end = min(t.rows, (rank + 1) * share);
            const int my_col = t.col0 + lane * 4;
            const int cols = a.cols - my_col;
            float sp4[4] = {1.f, 1.f, 1.f, 1.f};
            if (kI8) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < cols) sp4[j] = a.scale_p[static_cast<int64_t>(t.e) * a.cols + my_col + j];
            }
            constexpr uint32_t kRow = kGsCols * 4;
            const uint32_t mine = smem_u32(part) + static_cast<uint32_t>(lane) * 16;
            for (int row = rank * share + warp - 2; row < end; row += 2 * kGsEpilogueWarps) {
                float v[2][4];
                const bool two = row + kGsEpilogueWarps < end;
                // the second row, where there is none, is read from the first one's place
                sum_partials<kI8, 2>(mine + static_cast<uint32_t>(row) * kRow, two ? kGsEpilogueWarps * kRow : 0, splits, v);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (r == 1 && !two) break;
                    if (kI8) {
                        const float sq = a.scale_q[t.row0 + row + kGsEpilogueWarps * r];
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[r][j] = v[r][j] * sq * sp4[j];
                    }
                    if (cols > 0) store_four(a, out0 + (row + kGsEpilogueWarps * r) * a.ldo + my_col, v[r], cols);
                }
            }
        }
        __syncwarp();
        cluster_sync_all();   // nobody leaves while its partial sums may still be read
    }

    // ---------------- teardown ----------------
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, tmem_cols);
    }
    if (threadIdx.x == 0 && *abort_word != 0) atomicMax(a.status, *abort_word);
}

template <bool kI8, bool kPCols, bool kRaggedX, bool kLong>
static int launch_variant(const CUtensorMap& tp, const CUtensorMap& tq, const GroupedArgs& a, const GroupedPlan& plan, const DeviceInfo* dev,
                          cudaStream_t stream) {
    auto kernel = grouped_split_kernel<kI8, kPCols, kRaggedX, kLong>;
    static OncePerDevice once;
    if (int rc = raise_smem_limit_once(once, dev->device, kernel, gs_smem(kGsRingAlone))) return rc;
    const int ring = plan.alone ? kGsRingAlone : kGsRing;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(plan.tiles * plan.splits));
    cfg.blockDim = dim3(kGsThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(gs_smem(ring));
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(plan.splits);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = plan.splits > 1 ? 2 : 1;
    TCB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tp, tq, a, plan.splits, ring));
    return TC_OK;
}

int launch_grouped_split(const GroupedProblem& g, const GroupedPlan& plan, const DeviceInfo* dev, cudaStream_t stream) {
    const bool i8 = g.in_type == kTypeI8;
    GroupedArgs a = grouped_args(g, plan.tile_rows, plan.row_tiles, dev);
    a.idesc = grouped_idesc(g, kGsCols);
    CUtensorMap tp, tq;
    // P: 128 columns by 128 bytes of x, or (columns contiguous) 64 columns by 64 x; Q: the tile's rows alike
    if (int rc = grouped_map_p(&tp, g, g.p_c_contiguous ? 64 : 128)) return rc;
    if (int rc = grouped_map_q(&tq, g, g.ragged_x ? 64 : plan.tile_rows)) return rc;
    if (i8) return launch_variant<true, false, false, false>(tp, tq, a, plan, dev, stream);
    const int64_t most_blocks = ((g.ragged_x ? g.token_rows : g.other) + 63) / 64;
    if ((most_blocks + plan.splits - 1) / plan.splits > kSumPiece / 64) {
        if (g.ragged_x) return launch_variant<false, true, true, true>(tp, tq, a, plan, dev, stream);
        if (g.p_c_contiguous) return launch_variant<false, true, false, true>(tp, tq, a, plan, dev, stream);
        return launch_variant<false, false, false, true>(tp, tq, a, plan, dev, stream);
    }
    if (g.ragged_x) return launch_variant<false, true, true, false>(tp, tq, a, plan, dev, stream);
    if (g.p_c_contiguous) return launch_variant<false, true, false, false>(tp, tq, a, plan, dev, stream);
    return launch_variant<false, false, false, false>(tp, tq, a, plan, dev, stream);
}

}  // namespace tcb
