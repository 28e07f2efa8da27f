// Matrix products grouped by expert, and the scaled 8-bit product (one group): one thread per output element.
#include <cuda_bf16.h>

#include "host.h"
#include "sm100.cuh"

namespace tcb {

enum GroupedMode { kForward, kForwardI8, kDgrad, kWgrad };

struct GroupedParams {
    const void* p;          // fwd: B, dgrad: B, wgrad: A
    const void* q;          // fwd: A, dgrad: dC, wgrad: dC
    const float* scale_a;
    const float* scale_b;
    const void* offsets;    // null: one group of all rows
    int offsets_are_int64;
    void* out;
    int64_t rows, experts, N, K, ldp, stride_p, ldq, ldo, stride_o;
    int in_type, out_type;
    uint32_t* status;
};

__device__ __forceinline__ float load_half(const void* p, int64_t i, int type) {
    return type == TC_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_out(void* p, int64_t i, float v, int type) {
    if (type == TC_F32) static_cast<float*>(p)[i] = v;
    else if (type == TC_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Row range of a group, clamped into the tensor; *bad is set when an offset lies outside or the pair decreases.
__device__ __forceinline__ void group_rows(const GroupedParams& p, int e, int64_t& first, int64_t& last, bool& bad) {
    if (p.offsets == nullptr) {
        first = 0;
        last = p.rows;
        return;
    }
    const int64_t a = p.offsets_are_int64 ? static_cast<const int64_t*>(p.offsets)[e] : static_cast<const int32_t*>(p.offsets)[e];
    const int64_t b = p.offsets_are_int64 ? static_cast<const int64_t*>(p.offsets)[e + 1] : static_cast<const int32_t*>(p.offsets)[e + 1];
    bad |= a < 0 || b > p.rows || b < a;
    first = min(max(a, static_cast<int64_t>(0)), p.rows);
    last = max(first, min(max(b, static_cast<int64_t>(0)), p.rows));
}

template <int kMode>
__global__ void __launch_bounds__(256) grouped_kernel(const GroupedParams p) {
    bool bad = false;
    for (int64_t e = blockIdx.z; e < p.experts; e += gridDim.z) {
        int64_t first = 0, last = 0;
        group_rows(p, static_cast<int>(e), first, last, bad);
        const int64_t out_rows = kMode == kWgrad ? p.N : last - first;
        const int64_t out_cols = kMode == kForward || kMode == kForwardI8 ? p.N : p.K;
        for (int64_t r = blockIdx.y * 16 + threadIdx.y; r < out_rows; r += gridDim.y * 16) {
            for (int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x; c < out_cols; c += static_cast<int64_t>(gridDim.x) * 16) {
                if (kMode == kForwardI8) {
                    const int8_t* a = static_cast<const int8_t*>(p.q) + (first + r) * p.ldq;
                    const int8_t* b = static_cast<const int8_t*>(p.p) + e * p.stride_p + c * p.ldp;
                    int acc = 0;
                    for (int64_t k = 0; k < p.K; ++k) acc += static_cast<int>(a[k]) * static_cast<int>(b[k]);
                    const float v = static_cast<float>(acc) * p.scale_a[first + r] * p.scale_b[e * p.N + c];
                    store_out(p.out, (first + r) * p.ldo + c, v, p.out_type);
                } else {
                    float acc = 0.f;
                    if (kMode == kForward) {
                        for (int64_t k = 0; k < p.K; ++k)
                            acc = fmaf(load_half(p.q, (first + r) * p.ldq + k, p.in_type), load_half(p.p, e * p.stride_p + c * p.ldp + k, p.in_type), acc);
                    } else if (kMode == kDgrad) {
                        for (int64_t n = 0; n < p.N; ++n)
                            acc = fmaf(load_half(p.q, (first + r) * p.ldq + n, p.in_type), load_half(p.p, e * p.stride_p + n * p.ldp + c, p.in_type), acc);
                    } else {
                        for (int64_t t = first; t < last; ++t)
                            acc = fmaf(load_half(p.q, t * p.ldq + r, p.in_type), load_half(p.p, t * p.ldp + c, p.in_type), acc);
                    }
                    store_out(p.out, (kMode == kWgrad ? e * p.stride_o + r * p.ldo : (first + r) * p.ldo) + c, acc, p.out_type);
                }
            }
        }
    }
    if (bad) atomicMax(p.status, static_cast<uint32_t>(kDevIndexOutOfRange));
}

template <int kMode>
static int launch_grouped(GroupedParams& p, cudaStream_t stream) {
    const DeviceInfo* dev = nullptr;
    if (int rc = current_device(&dev)) return rc;
    p.status = dev->status_word;
    const int64_t out_cols = kMode == kForward || kMode == kForwardI8 ? p.N : p.K;
    const int64_t out_rows = kMode == kWgrad ? p.N : p.rows;
    const dim3 grid(static_cast<unsigned>(min((out_cols + 15) / 16, static_cast<int64_t>(1024))),
                    static_cast<unsigned>(max(static_cast<int64_t>(1), min((out_rows + 15) / 16, static_cast<int64_t>(1024)))),
                    static_cast<unsigned>(min(p.experts, static_cast<int64_t>(1024))));
    grouped_kernel<kMode><<<grid, dim3(16, 16), 0, stream>>>(p);
    TCB_CUDA(cudaGetLastError());
    return TC_OK;
}

static bool half_type(int t) { return t == TC_F16 || t == TC_BF16; }
static bool any_type(int t) { return t == TC_F32 || half_type(t); }
static int type_bytes(int t) { return t == TC_F32 ? 4 : 2; }

// Checks shared by the entry points. es: bytes of an input element.
static int check_sizes(const char* op, int64_t rows, int64_t experts, int64_t N, int64_t K) {
    TCB_REQUIRE(rows >= 0, "%s: the number of rows must not be negative (got %lld)", op, (long long)rows);
    TCB_REQUIRE(experts > 0 && N > 0 && K > 0, "%s: experts, N and K must be positive (got %lld, %lld, %lld)", op, (long long)experts,
                (long long)N, (long long)K);
    TCB_REQUIRE(rows < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31), "%s: a dimension does not fit in 31 bits", op);
    if (experts > 2048) return fail(TC_ERR_UNSUPPORTED, "%s: %lld experts, at most 2048 are supported", op, (long long)experts);
    return TC_OK;
}

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
    GroupedParams p{B, A, scale_a, scale_b, nullptr, 0, C, M, 1, N, K, ldb, 0, lda, ldc, 0, 0, c_type, nullptr};
    return launch_grouped<kForwardI8>(p, static_cast<cudaStream_t>(stream));
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
    GroupedParams p{B, A, scale_a, scale_b, offsets, offsets_are_int64, C, rows, experts, N, K, ldb, stride_b, lda, ldc, 0, 0, c_type, nullptr};
    return launch_grouped<kForwardI8>(p, static_cast<cudaStream_t>(stream));
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
    GroupedParams p{B, A, nullptr, nullptr, offsets, offsets_are_int64, C, rows, experts, N, K, ldb, stride_b, lda, ldc, 0, in_type, c_type, nullptr};
    return launch_grouped<kForward>(p, static_cast<cudaStream_t>(stream));
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
    GroupedParams p{B, dC, nullptr, nullptr, offsets, offsets_are_int64, dA, rows, experts, N, K, ldb, stride_b, lddc, ldda, 0, in_type, da_type, nullptr};
    return launch_grouped<kDgrad>(p, static_cast<cudaStream_t>(stream));
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
    TCB_REQUIRE(experts == 1 || stride_db >= K, "%s: expert stride of dB smaller than a row", op);
    GroupedParams p{A, dC, nullptr, nullptr, offsets, offsets_are_int64, dB, rows, experts, N, K, lda, 0, lddc, lddb, stride_db, in_type, db_type, nullptr};
    return launch_grouped<kWgrad>(p, static_cast<cudaStream_t>(stream));
}
