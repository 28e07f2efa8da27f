// Entry points of the products grouped by expert and of the scaled 8-bit product (one group): argument checks and the
// choice of the kernel.
#include "grouped.h"
#include "sm100.cuh"

#include <algorithm>
#include <initializer_list>

namespace tcb {

static bool half_type(int t) { return t == TC_F16 || t == TC_BF16; }
static bool any_type(int t) { return t == TC_F32 || half_type(t); }
static int type_bytes(int t) { return t == TC_F32 ? 4 : 2; }

// Checks shared by the entry points. es: bytes of an input element.
static int check_sizes(const char* op, int64_t rows, int64_t experts, int64_t N, int64_t K) {
    TCB_REQUIRE(rows >= 0, "%s: the number of rows must not be negative (got %lld)", op, (long long)rows);
    TCB_REQUIRE(experts > 0 && N > 0 && K > 0, "%s: experts, N and K must be positive (got %lld, %lld, %lld)", op, (long long)experts,
                (long long)N, (long long)K);
    // coordinates are 32-bit and run up to a tile past the end
    constexpr int64_t kMost = (1ll << 31) - 1024;
    TCB_REQUIRE(rows < kMost && N < kMost && K < kMost, "%s: a dimension does not fit in 31 bits", op);
    if (experts > kMaxExperts) return fail(TC_ERR_UNSUPPORTED, "%s: %lld experts, at most %d are supported", op, (long long)experts, kMaxExperts);
    return TC_OK;
}

// What the joining of pieces (kSumPiece) leaves uncertain grows by 2^-24 a piece, 2^-10 of the sum of magnitudes for this many
// terms.
static int check_terms(const char* op, const char* name, int64_t terms) {
    if (terms > (1ll << 27)) return fail(TC_ERR_UNSUPPORTED, "%s: sums over %s = %lld terms, at most %lld are supported", op, name, (long long)terms, 1ll << 27);
    return TC_OK;
}

// The output against everything that a call reads. What is read twice (experts in one place, A within B) may overlap.
static int check_distinct(const char* op, const char* out_name, const Extent& out, std::initializer_list<Extent> inputs) {
    for (const Extent& in : inputs) TCB_REQUIRE(!extents_meet(out, in), "%s: %s must not overlap an operand", op, out_name);
    return TC_OK;
}

static Extent offsets_of(const void* ptr, int64_t experts, int wide) { return extent_of_vector(ptr, experts + 1, wide ? 8 : 4); }

static int check_input(const char* op, const char* name, const void* ptr, int64_t ld, int64_t cols, int es) {
    TCB_REQUIRE(ptr != nullptr, "%s: null pointer argument (%s)", op, name);
    TCB_REQUIRE(ld >= cols, "%s: leading dimension of %s smaller than the row length", op, name);
    TCB_REQUIRE(ld % (16 / es) == 0, "%s: row stride of %s must be a multiple of %d elements (16 bytes), got %lld", op, name, 16 / es, (long long)ld);
    TCB_REQUIRE(ld < (1ll << 40) / es, "%s: row stride of %s is too large", op, name);
    TCB_REQUIRE(aligned16(ptr), "%s: %s must be 16-byte aligned", op, name);
    return TC_OK;
}

static int check_stack(const char* op, const char* name, int64_t stride, int64_t cols, int64_t experts, int es) {
    TCB_REQUIRE(experts == 1 || stride >= cols, "%s: expert stride of %s smaller than a row", op, name);
    TCB_REQUIRE(stride % (16 / es) == 0, "%s: expert stride of %s must be a multiple of %d elements (16 bytes), got %lld", op, name, 16 / es, (long long)stride);
    TCB_REQUIRE(stride < (1ll << 40) / es, "%s: expert stride of %s is too large", op, name);
    return TC_OK;
}

static int check_output(const char* op, const char* name, const void* ptr, int64_t ld, int64_t cols, int type) {
    TCB_REQUIRE(ptr != nullptr, "%s: null pointer argument (%s)", op, name);
    TCB_REQUIRE(ld >= cols, "%s: leading dimension of %s smaller than the row length", op, name);
    TCB_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % type_bytes(type) == 0, "%s: %s must be aligned to its type", op, name);
    return TC_OK;
}

static int check_offsets(const char* op, const void* offsets, int wide) {
    TCB_REQUIRE(offsets != nullptr, "%s: null pointer argument (offsets)", op);
    TCB_REQUIRE(reinterpret_cast<uintptr_t>(offsets) % (wide ? 8 : 4) == 0, "%s: offsets must be aligned to their type", op);
    return TC_OK;
}

static int check_half_types(const char* op, int in_type, int out_type) {
    TCB_REQUIRE(half_type(in_type), "%s: in_type %d is not fp16 or bf16", op, in_type);
    TCB_REQUIRE(out_type == in_type || out_type == TC_F32, "%s: the result is of the input's type or fp32, got type %d", op, out_type);
    return TC_OK;
}

static int check_i8(const char* op, int64_t K, int c_type, const float* scale_a, const float* scale_b) {
    TCB_REQUIRE(any_type(c_type), "%s: c_type %d is not fp32, fp16 or bf16", op, c_type);
    if (K > 131071) return fail(TC_ERR_UNSUPPORTED, "%s: K = %lld, beyond 131071 a sum of 8-bit products can overflow 32 bits", op, (long long)K);
    TCB_REQUIRE(scale_a && scale_b, "%s: null pointer argument (scales)", op);
    TCB_REQUIRE(reinterpret_cast<uintptr_t>(scale_a) % 4 == 0 && reinterpret_cast<uintptr_t>(scale_b) % 4 == 0, "%s: scales must be 4-byte aligned", op);
    return TC_OK;
}

uint32_t grouped_idesc(const GroupedProblem& g, int m) {
    if (g.in_type == kTypeI8) return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(m >> 4) << 24);
    return make_idesc_f16_f32(m, 0, g.p_c_contiguous, g.ragged_x) | (g.in_type == TC_BF16 ? kIdescBf16Inputs : 0u);
}

static int encode_operand(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
                          int in_type) {
    if (in_type == kTypeI8) return encode_tmap_i8_sw128(map, base, rank, dims, strides, box);
    return encode_tmap_f16_sw128(map, base, rank, dims, strides, box, in_type == TC_BF16);
}

int grouped_map_p(CUtensorMap* map, const GroupedProblem& g, int box_rows) {
    // B [experts, rows, row length], or for wgrad A [token_rows, cols]
    const uint64_t es = g.in_type == kTypeI8 ? 1 : 2;
    const int64_t inner = g.p_c_contiguous ? g.cols : g.other;
    const int64_t outer = g.ragged_x ? g.token_rows : g.p_c_contiguous ? g.other : g.cols;
    const bool stack = !g.ragged_x && g.experts > 1;
    const uint64_t dims[3] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(outer), stack ? static_cast<uint64_t>(g.experts) : 1};
    const uint64_t strides[2] = {static_cast<uint64_t>(g.ldp) * es, static_cast<uint64_t>(stack ? g.stride_p : g.ldp) * es};
    const uint32_t box[3] = {static_cast<uint32_t>(128 / es), static_cast<uint32_t>(box_rows), 1};
    return encode_operand(map, g.p, 3, dims, strides, box, g.in_type);
}

int grouped_map_q(CUtensorMap* map, const GroupedProblem& g, int box_rows) {
    const uint64_t es = g.in_type == kTypeI8 ? 1 : 2;
    const uint64_t dims[2] = {static_cast<uint64_t>(g.other), static_cast<uint64_t>(g.token_rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(g.ldq) * es};
    const uint32_t box[2] = {static_cast<uint32_t>(128 / es), static_cast<uint32_t>(box_rows)};
    return encode_operand(map, g.q, 2, dims, strides, box, g.in_type);
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The kernel and tile for a problem, from its sizes alone; of the offsets the host knows nothing, so the rule takes the
// rows to be spread evenly, or nearly so. Times below in us: B200, CUDA graph replays, three sets of operands in turn.
//  * One group, and the weight gradient: pair tiles (256 columns x up to 256 rows) once there are more of them than the 74 pairs
//    and 128 rows or more to fill them: int8 2048 x 2560 x 2048 (80 tiles) 14.9 against 15.7 in the split kernel, weight
//    gradient of one [2048,2560] from 2048 rows 26.7 against 30.2; a short sum gains nothing (int8 2048 x 2432 x 512 9.3 against
//    8.8), and with 64 tiles the split kernel, of whose tiles two run on an SM, is ahead (int8 2048^3 9.4 against 11.1).
//  * Groups with weights of their own come out uneven: half a tile of each counts as wasted. The split kernel as long as its
//    tiles of 128 rows all run at once, two per SM (1600 rows, 12 x [2048,2048]: 23.7 against 29.2 in two unequal waves of pair
//    tiles; input gradient of 7 x [512,1536], 2048 rows: 7.7 against 9.0), or nearly so where groups of fewer than 128 rows
//    leave half of a pair tile empty (2500 rows, 20 x [1408,2048]: 26.0 against 29.4). Beyond that pair tiles (4096 rows, 16 x
//    [1024,2048]: 28.4 against 31.1; 2000 rows, 16 x [2048,2048]: 31.4 against 37.7; 6400 rows, 64 x [2048,1024]: 55 against
//    65), but not for fewer than 96 rows a group (1024 rows, 16 x [4096,2048]: 52.9 against 48.9).
//  * Else the split kernel. Where the weights' bytes count (few rows per group), a tile takes all rows of a group up to
//    four times the even share, so that a popular expert's weights are read once: 16 x [2048,2048] with 512 rows 24.6
//    with 128-row tiles against 29.7 with 32.
//  * Tiles are halved while they still all run at once, one per SM: int8 1024^3 3.7 with 64 rows, 4.1 with 128; for long
//    sums not below 64 rows, where cutting the sum does more (int8 300 x 1024 x 8192 8.7 with two pieces of 64-row
//    tiles, 9.9 with 32-row tiles), unless even eight pieces would leave most SMs idle (64 x 512 x 4096: 6.0 against 7.2).
//  * The sum is cut in four where that many pieces still run at once (int8 1 x 4096 x 4096 5.1, in one piece 5.9; 64 x 2048
//    x 4096 5.1 and 6.1). Two pieces save less than joining them costs unless the sum is long (128 x 4096 x 4096 7.5, in one
//    piece 6.7; 300 x 1024 x 8192 8.7 and 10.1). Clusters of eight only for a handful of tiles: a GPC holds two of them at
//    most, and a weight gradient of 512 x 512 from 4096 rows takes 13.3 in eight pieces and 8.3 in four.
static GroupedPlan grouped_plan(const GroupedProblem& g, int sm_count) {
    const int64_t groups = g.offsets == nullptr ? 1 : g.ragged_x ? g.experts : (g.experts < g.token_rows ? g.experts : g.token_rows);
    const int64_t share = ceil_div(g.token_rows, groups);               // rows of a group, spread evenly
    const int64_t rows = g.ragged_x ? g.other : share;                   // extent of an output slice
    const int64_t stages = ceil_div((g.ragged_x ? share : g.other) * (g.in_type == kTypeI8 ? 1 : 2), 128);   // of the split kernel
    auto tiles = [&](int64_t tile_rows, int64_t tile_cols) { return groups * ceil_div(rows, tile_rows) * ceil_div(g.cols, tile_cols); };
    GroupedPlan p;
    p.splits = 1;
    const bool own_weights = groups > 1 && !g.ragged_x;
    const int64_t lone2 = std::max(2 * groups, g.token_rows / 64 + groups) * ceil_div(g.cols, 128);   // twice the split kernel's tiles
    p.pair = own_weights ? share >= 96 && 100 * lone2 > (share >= 128 ? 100 : 118) * 4 * sm_count
                         : rows >= 128 && tiles(256, 256) > sm_count / 2;
    if (p.pair) {
        p.tile_rows = 256;
    } else {
        const int64_t want = own_weights ? 4 * share : rows;
        p.tile_rows = g.ragged_x ? 64 : 16;
        while (p.tile_rows < 128 && p.tile_rows < want) p.tile_rows *= 2;
        const int64_t least = g.ragged_x || stages > 16 ? 64 : 32;
        while (p.tile_rows > least && tiles(p.tile_rows / 2, 128) <= sm_count && (!own_weights || share > 128 || p.tile_rows / 2 >= share))
            p.tile_rows /= 2;
        while (p.tile_rows > (g.ragged_x ? 64 : 16) && 8 * tiles(p.tile_rows, 128) < 48) p.tile_rows /= 2;
        const int64_t n = tiles(p.tile_rows, 128);
        const int64_t room = own_weights ? sm_count / 2 : sm_count;   // uneven groups make more tiles than counted here
        if (8 * n <= 64 && stages >= 64) p.splits = 8;
        else if (4 * n <= room && stages >= 32) p.splits = 4;
        else if (2 * n <= room && stages >= 48) p.splits = 2;
    }
    // a bound on the output tiles for any offsets that do not overlap
    p.row_tiles = g.ragged_x ? groups * ceil_div(g.other, p.tile_rows)
                              : g.offsets == nullptr ? ceil_div(g.token_rows, p.tile_rows) : g.token_rows / p.tile_rows + groups;
    p.tiles = p.row_tiles * ceil_div(g.cols, p.pair ? 256 : 128);
    // The split kernel's CTAs get an SM each, and the ring of one, when they need no more: a few beyond the SMs, of which
    // some will find no tile, do not change that (9 experts x [1001,776], 1333 rows: 152 CTAs 10.8 alone, 14.3 two to an SM).
    // So it is where the bound is well above the SMs but the tiles of uneven groups probably are not (2600 rows, 13 x [640,2048]
    // 12.7 and 17.0; 1500 rows, 14 x [896,1024] 8.5 and 10.8); nearer to the SMs a second wave would cost what the ring gains
    // (1900 rows, 11 x [896,2048], for three spreads of the rows 19.8, 20.3, 12.9 alone, 17.4, 16.9, 17.4 two to an SM).
    p.alone = (tiles(p.tile_rows, 128) * p.splits <= sm_count && 10 * p.tiles * p.splits <= 11 * sm_count) ||
              (own_weights && p.tile_rows == 128 && p.splits == 1 && 10 * lone2 <= 18 * sm_count && 4 * p.tiles <= 5 * sm_count);
    return p;
}

static int launch_grouped(const GroupedProblem& g, tc_stream_t stream) {
    const DeviceInfo* dev = nullptr;
    if (int rc = current_device(&dev)) return rc;
    const GroupedPlan plan = grouped_plan(g, dev->sm_count);
    if (plan.tiles * plan.splits >= (1ll << 31))
        return fail(TC_ERR_UNSUPPORTED, "grouped product: too many output tiles (%lld experts, %lld rows, %lld columns)", (long long)g.experts,
                    (long long)g.token_rows, (long long)g.cols);
    auto s = static_cast<cudaStream_t>(stream);
    return plan.pair ? launch_grouped_pair(g, plan, dev, s) : launch_grouped_split(g, plan, dev, s);
}

#define TCB_TRY(expr)             \
    do {                          \
        if (int _rc = (expr)) return _rc; \
    } while (0)

}  // namespace tcb

extern "C" int tc_gemm_i8(const void* A, const void* B, const float* scale_a, const float* scale_b, void* C, int64_t M, int64_t N,
                          int64_t K, int64_t lda, int64_t ldb, int64_t ldc, int c_type, tc_stream_t stream) {
    using namespace tcb;
    const char* op = "gemm_i8";
    TCB_TRY(check_sizes(op, M, 1, N, K));
    if (M == 0) return TC_OK;
    TCB_TRY(check_i8(op, K, c_type, scale_a, scale_b));
    TCB_TRY(check_input(op, "A", A, lda, K, 1));
    TCB_TRY(check_input(op, "B", B, ldb, K, 1));
    TCB_TRY(check_output(op, "C", C, ldc, N, c_type));
    TCB_TRY(check_distinct(op, "C", extent_of_rows(C, M, N, ldc, type_bytes(c_type)),
                           {extent_of_rows(A, M, K, lda, 1), extent_of_rows(B, N, K, ldb, 1), extent_of_vector(scale_a, M, 4), extent_of_vector(scale_b, N, 4)}));
    return launch_grouped({B, A, scale_b, scale_a, nullptr, 0, C, M, 1, N, K, ldb, 0, lda, ldc, 0, kTypeI8, c_type, false, false}, stream);
}

extern "C" int tc_grouped_gemm_i8(const void* A, const void* B, const float* scale_a, const float* scale_b, const void* offsets,
                                  int offsets_are_int64, void* C, int64_t rows, int64_t experts, int64_t N, int64_t K, int64_t lda,
                                  int64_t ldb, int64_t stride_b, int64_t ldc, int c_type, tc_stream_t stream) {
    using namespace tcb;
    const char* op = "grouped_gemm_i8";
    TCB_TRY(check_sizes(op, rows, experts, N, K));
    TCB_TRY(check_offsets(op, offsets, offsets_are_int64));
    if (rows == 0) return TC_OK;
    TCB_TRY(check_i8(op, K, c_type, scale_a, scale_b));
    TCB_TRY(check_input(op, "A", A, lda, K, 1));
    TCB_TRY(check_input(op, "B", B, ldb, K, 1));
    TCB_TRY(check_stack(op, "B", stride_b, K, experts, 1));
    TCB_TRY(check_output(op, "C", C, ldc, N, c_type));
    TCB_TRY(check_distinct(op, "C", extent_of_rows(C, rows, N, ldc, type_bytes(c_type)),
                           {extent_of_rows(A, rows, K, lda, 1), extent_of_stack(B, experts, N, K, ldb, stride_b, 1), extent_of_vector(scale_a, rows, 4),
                            extent_of_vector(scale_b, experts * N, 4), offsets_of(offsets, experts, offsets_are_int64)}));
    return launch_grouped({B, A, scale_b, scale_a, offsets, offsets_are_int64, C, rows, experts, N, K, ldb, stride_b, lda, ldc, 0, kTypeI8, c_type,
                           false, false}, stream);
}

extern "C" int tc_grouped_gemm(const void* A, const void* B, const void* offsets, int offsets_are_int64, void* C, int64_t rows,
                               int64_t experts, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t stride_b, int64_t ldc,
                               int in_type, int c_type, tc_stream_t stream) {
    using namespace tcb;
    const char* op = "grouped_gemm";
    TCB_TRY(check_sizes(op, rows, experts, N, K));
    TCB_TRY(check_half_types(op, in_type, c_type));
    TCB_TRY(check_offsets(op, offsets, offsets_are_int64));
    if (rows == 0) return TC_OK;
    TCB_TRY(check_input(op, "A", A, lda, K, 2));
    TCB_TRY(check_input(op, "B", B, ldb, K, 2));
    TCB_TRY(check_stack(op, "B", stride_b, K, experts, 2));
    TCB_TRY(check_output(op, "C", C, ldc, N, c_type));
    TCB_TRY(check_terms(op, "K", K));
    TCB_TRY(check_distinct(op, "C", extent_of_rows(C, rows, N, ldc, type_bytes(c_type)),
                           {extent_of_rows(A, rows, K, lda, 2), extent_of_stack(B, experts, N, K, ldb, stride_b, 2), offsets_of(offsets, experts, offsets_are_int64)}));
    return launch_grouped({B, A, nullptr, nullptr, offsets, offsets_are_int64, C, rows, experts, N, K, ldb, stride_b, lda, ldc, 0, in_type, c_type,
                           false, false}, stream);
}

extern "C" int tc_grouped_gemm_dgrad(const void* dC, const void* B, const void* offsets, int offsets_are_int64, void* dA,
                                     int64_t rows, int64_t experts, int64_t N, int64_t K, int64_t lddc, int64_t ldb,
                                     int64_t stride_b, int64_t ldda, int in_type, int da_type, tc_stream_t stream) {
    using namespace tcb;
    const char* op = "grouped_gemm_dgrad";
    TCB_TRY(check_sizes(op, rows, experts, N, K));
    TCB_TRY(check_half_types(op, in_type, da_type));
    TCB_TRY(check_offsets(op, offsets, offsets_are_int64));
    if (rows == 0) return TC_OK;
    TCB_TRY(check_input(op, "dC", dC, lddc, N, 2));
    TCB_TRY(check_input(op, "B", B, ldb, K, 2));
    TCB_TRY(check_stack(op, "B", stride_b, K, experts, 2));
    TCB_TRY(check_output(op, "dA", dA, ldda, K, da_type));
    TCB_TRY(check_terms(op, "N", N));
    TCB_TRY(check_distinct(op, "dA", extent_of_rows(dA, rows, K, ldda, type_bytes(da_type)),
                           {extent_of_rows(dC, rows, N, lddc, 2), extent_of_stack(B, experts, N, K, ldb, stride_b, 2), offsets_of(offsets, experts, offsets_are_int64)}));
    return launch_grouped({B, dC, nullptr, nullptr, offsets, offsets_are_int64, dA, rows, experts, K, N, ldb, stride_b, lddc, ldda, 0, in_type, da_type,
                           true, false}, stream);
}

extern "C" int tc_grouped_gemm_wgrad(const void* dC, const void* A, const void* offsets, int offsets_are_int64, void* dB,
                                     int64_t rows, int64_t experts, int64_t N, int64_t K, int64_t lddc, int64_t lda, int64_t lddb,
                                     int64_t stride_db, int in_type, int db_type, tc_stream_t stream) {
    using namespace tcb;
    const char* op = "grouped_gemm_wgrad";
    TCB_TRY(check_sizes(op, rows, experts, N, K));
    TCB_TRY(check_half_types(op, in_type, db_type));
    TCB_TRY(check_offsets(op, offsets, offsets_are_int64));
    if (rows > 0) {
        TCB_TRY(check_input(op, "dC", dC, lddc, N, 2));
        TCB_TRY(check_input(op, "A", A, lda, K, 2));
    }
    TCB_TRY(check_output(op, "dB", dB, lddb, K, db_type));
    TCB_TRY(check_terms(op, "rows", rows));
    TCB_REQUIRE(experts == 1 || stride_db >= K, "%s: expert stride of dB smaller than a row", op);
    const Extent out = extent_of_stack(dB, experts, N, K, lddb, stride_db, type_bytes(db_type));
    TCB_REQUIRE(!slices_meet(out), "%s: the experts of dB must not overlap each other", op);
    TCB_TRY(check_distinct(op, "dB", out, {offsets_of(offsets, experts, offsets_are_int64)}));
    if (rows > 0) TCB_TRY(check_distinct(op, "dB", out, {extent_of_rows(dC, rows, N, lddc, 2), extent_of_rows(A, rows, K, lda, 2)}));
    if (rows == 0) {   // nothing to sum over, and no tensors to describe to TMA
        const size_t es = static_cast<size_t>(type_bytes(db_type));
        for (int64_t e = 0; e < experts; ++e)
            TCB_CUDA(cudaMemset2DAsync(static_cast<uint8_t*>(dB) + static_cast<size_t>(e * stride_db) * es, static_cast<size_t>(lddb) * es, 0,
                                       static_cast<size_t>(K) * es, static_cast<size_t>(N), static_cast<cudaStream_t>(stream)));
        return TC_OK;
    }
    return launch_grouped({A, dC, nullptr, nullptr, offsets, offsets_are_int64, dB, rows, experts, K, N, lda, 0, lddc, lddb, stride_db, in_type, db_type,
                           true, true}, stream);
}
