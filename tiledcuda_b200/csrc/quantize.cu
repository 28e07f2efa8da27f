// Rounding of rows to 8-bit integers with one scale per row: scale = max(amax / 127, 2^-126), q = x / scale to nearest,
// ties to even. One block per row, the row read twice.
#include "host.h"
#include "sm100.cuh"

#include <cuda_bf16.h>

namespace tcb {

constexpr int kQuantThreads = 256;

// x / scale rounded as the exact quotient would be. x * (1 / scale) is off by less than 2e-5 for quotients up to 127
// (two roundings of 2^-24 each), so only a quotient within 1e-4 of a half can round the other way; there x is compared
// with half * scale, a product of 9 and 24 significant bits that is exact in fp64.
__device__ __forceinline__ float quantize_value(float x, float inv, float scale) {
    const float t = x * inv;
    float r = rintf(t);
    if (fabsf(fabsf(t - r) - 0.5f) < 1e-4f) {
        const float low = floorf(t);
        const double border = (static_cast<double>(low) + 0.5) * static_cast<double>(scale);
        const double xd = static_cast<double>(x);
        if (xd > border) r = low + 1.f;
        else if (xd < border) r = low;
        else r = 2.f * rintf(0.5f * low + 0.25f);   // the even one of low and low + 1
    }
    return r;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale_out, int64_t cols, int64_t ldx,
                     int64_t ldq) {
    const T* row = x + static_cast<int64_t>(blockIdx.x) * ldx;
    int8_t* out = q + static_cast<int64_t>(blockIdx.x) * ldq;
    __shared__ uint32_t warp_max[kQuantThreads / 32];
    // the bit pattern of |x| orders like its value, infinities above every number and NaN above those
    uint32_t m = 0;
    for (int64_t c = threadIdx.x; c < cols; c += kQuantThreads) m = max(m, __float_as_uint(to_float(row[c])) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kQuantThreads / 32; ++w) m = max(m, warp_max[w]);
    float scale = __fdiv_rn(__uint_as_float(m), 127.f);
    if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;
    const bool finite = m < 0x7f800000u;
    const float inv = __fdiv_rn(1.f, scale);
    for (int64_t c = threadIdx.x; c < cols; c += kQuantThreads)
        out[c] = finite ? static_cast<int8_t>(quantize_value(to_float(row[c]), inv, scale)) : static_cast<int8_t>(0);
    if (threadIdx.x == 0) scale_out[blockIdx.x] = scale;
}

template <typename T>
static int launch_quantize(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t ldx, int64_t ldq, cudaStream_t stream) {
    quantize_rows_kernel<T><<<dim3(static_cast<unsigned>(rows)), kQuantThreads, 0, stream>>>(
        static_cast<const T*>(x), static_cast<int8_t*>(q), scale, cols, ldx, ldq);
    TCB_CUDA(cudaGetLastError());
    return TC_OK;
}

}  // namespace tcb

extern "C" int tc_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t ldx, int64_t ldq,
                                int x_type, tc_stream_t stream) {
    using namespace tcb;
    TCB_REQUIRE(rows >= 0 && cols > 0, "quantize_rows: rows must not be negative and cols must be positive (got %lld, %lld)",
                (long long)rows, (long long)cols);
    TCB_REQUIRE(rows < (1ll << 31) && cols < (1ll << 31), "quantize_rows: a dimension does not fit in 31 bits");
    TCB_REQUIRE(x_type == TC_F32 || x_type == TC_F16 || x_type == TC_BF16, "quantize_rows: x_type %d is not fp32, fp16 or bf16", x_type);
    TCB_REQUIRE(ldx >= cols && ldq >= cols, "quantize_rows: leading dimension smaller than the row length");
    if (rows == 0) return TC_OK;
    TCB_REQUIRE(x && q && scale, "quantize_rows: null pointer argument");
    const int es = x_type == TC_F32 ? 4 : 2;
    TCB_REQUIRE(reinterpret_cast<uintptr_t>(x) % es == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0, "quantize_rows: x and scale must be aligned to their types");
    const DeviceInfo* dev = nullptr;
    if (int rc = current_device(&dev)) return rc;
    auto s = static_cast<cudaStream_t>(stream);
    if (x_type == TC_F32) return launch_quantize<float>(x, q, scale, rows, cols, ldx, ldq, s);
    if (x_type == TC_F16) return launch_quantize<__half>(x, q, scale, rows, cols, ldx, ldq, s);
    return launch_quantize<__nv_bfloat16>(x, q, scale, rows, cols, ldx, ldq, s);
}
