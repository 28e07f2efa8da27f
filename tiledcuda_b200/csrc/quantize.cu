// Rounding of rows to 8-bit integers with one scale per row: scale = max(amax * c, 2^-126) with c = 1 / 127 in fp32,
// q = x / scale to nearest, ties to even. Bound by memory: each element is read once (2 or 4 bytes) and written once
// (1 byte). A row stays in the registers of the threads that own it between the maximum and the rounding; rows too long
// for that, or not on 16-byte boundaries, are read a second time (out of L2).
#include "host.h"
#include "sm100.cuh"

#include <cuda_bf16.h>

namespace tcb {

constexpr int kQuantThreads = 256;
constexpr int kQuantChunk = 16;   // consecutive elements of a thread: 16 bytes of q

// x / scale rounded as the exact quotient would be. r, the rounded x * (1 / scale), is off by one at most, and only where the
// quotient is within 1e-5 of a half-integer (the reciprocal's rounding times 127.5). e = x - r * scale tells: it comes out of one
// fma, exact near |e| = scale / 2, where x and r * scale cancel to 24 bits (or is a half-step above it next to r = 1, where a
// tie and a larger |e| lead to the same answer). r is right if |e| < scale / 2, and a tie goes to the even neighbour. Exact
// ties are not rare: bf16 rows hold x = amax / 2 once in a few thousand elements.
constexpr float kToInteger = 12582912.f;   // 1.5 * 2^23: added, it leaves the value rounded to an integer in the low mantissa bits

__device__ __forceinline__ float settle(float r, float e, float half) {
    const bool wrong = fabsf(e) > half || (fabsf(e) == half && (__float_as_uint(r + kToInteger) & 1u));
    return wrong ? r + copysignf(1.f, e) : r;
}

__device__ __forceinline__ int8_t quantize_one(float x, float inv, float scale) {
    const float r = fmaf(x, inv, kToInteger) - kToInteger;
    return static_cast<int8_t>(settle(r, fmaf(-r, scale, x), 0.5f * scale));
}

// Loads of 16 elements as eight or sixteen words, their largest magnitude, and their values. Magnitudes compare as bit
// patterns of |x| in fp32, infinities above every number and NaN above those.
template <typename T>
struct Chunk;
template <>
struct Chunk<float> {
    static constexpr int kWords = 16;
    static __device__ __forceinline__ uint32_t largest(const uint32_t (&w)[16]) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
        return m;
    }
    static __device__ __forceinline__ void values(const uint32_t (&w)[16], float (&v)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
    }
};
template <>
struct Chunk<__half> {
    static constexpr int kWords = 8;
    static __device__ __forceinline__ uint32_t largest(const uint32_t (&w)[8]) {
        __half2 m = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
        return __float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))) & 0x7fffffffu;
    }
    static __device__ __forceinline__ void values(const uint32_t (&w)[8], float (&v)[16]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
template <>
struct Chunk<__nv_bfloat16> {
    static constexpr int kWords = 8;
    static __device__ __forceinline__ uint32_t largest(const uint32_t (&w)[8]) {
        __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
        return __float_as_uint(__bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)))) & 0x7fffffffu;
    }
    static __device__ __forceinline__ void values(const uint32_t (&w)[8], float (&v)[16]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Scale of a row from the bit pattern of its largest magnitude. `rounds`: the row is finite; else all of q is 0.
__device__ __forceinline__ void row_scale(uint32_t largest, float& scale, float& inv, bool& rounds) {
    scale = __uint_as_float(largest) * (1.f / 127.f);
    if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;
    inv = __fdiv_rn(1.f, scale);
    rounds = largest < 0x7f800000u;
}

template <typename T>
__device__ __forceinline__ uint4 quantize_chunk(const uint32_t (&w)[Chunk<T>::kWords], float inv, float scale, bool rounds) {
    float v[kQuantChunk];
    Chunk<T>::values(w, v);
    const uint64_t inv2 = pack2(inv, inv), up = pack2(kToInteger, kToInteger), down = pack2(-kToInteger, -kToInteger);
    const uint64_t minus_scale2 = pack2(-scale, -scale);
    uint32_t b[kQuantChunk];
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < kQuantChunk; i += 2) {
        const uint64_t x2 = pack2(v[i], v[i + 1]);
        const uint64_t shifted = fma2(x2, inv2, up);
        const uint64_t e2 = fma2(add2(shifted, down), minus_scale2, x2);
        float s0, s1, e0, e1;
        unpack2(shifted, s0, s1);
        unpack2(e2, e0, e1);
        b[i] = __float_as_uint(s0);
        b[i + 1] = __float_as_uint(s1);
        far = fmax3(far, fabsf(e0), fabsf(e1));
    }
    if (far >= 0.5f * scale) {
#pragma unroll
        for (int i = 0; i < kQuantChunk; ++i) {
            const float r = __uint_as_float(b[i]) - kToInteger;
            b[i] = __float_as_uint(settle(r, fmaf(-r, scale, v[i]), 0.5f * scale) + kToInteger);
        }
    }
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = rounds ? __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410) : 0u;
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename T, int kChunks>
__device__ __forceinline__ void load_chunks(uint32_t (&w)[kChunks][Chunk<T>::kWords], const T* src, int whole, int thread, int threads, bool live) {
    constexpr int kWords = Chunk<T>::kWords;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int chunk = c * threads + thread;
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[c][i] = 0;
        if (live && chunk < whole) {
            const uint4* p = reinterpret_cast<const uint4*>(src + static_cast<int64_t>(chunk) * kQuantChunk);
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 u = __ldcs(p + i);
                w[c][4 * i] = u.x;
                w[c][4 * i + 1] = u.y;
                w[c][4 * i + 2] = u.z;
                w[c][4 * i + 3] = u.w;
            }
        }
    }
}

// Rows on 16-byte boundaries (x and q), a row in the registers of `threads` threads (a power of two up to 1024), kChunks
// chunks a thread; a block takes blockDim / threads rows at a time and loads the next ones before it rounds these. What is left
// over behind the whole chunks of a row goes element by element.
// kBlock: most threads of a block; 256 where the rows allow, which leaves a thread 80 registers and the loop free of spills.
template <typename T, int kChunks, int kBlock>
__global__ void __launch_bounds__(kBlock, kBlock == 256 ? 3 : 1)
quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale_out, int rows, int cols, int64_t ldx,
                     int64_t ldq, int threads) {
    __shared__ uint32_t warp_max[2][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int thread = static_cast<int>(threadIdx.x) & (threads - 1);
    const int per_block = static_cast<int>(blockDim.x) / threads;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
    const int whole = cols / kQuantChunk;
    grid_launch_dependents();
    grid_dependency_wait();
    uint32_t w[kChunks][Chunk<T>::kWords];
    int64_t row = static_cast<int64_t>(blockIdx.x) * per_block + static_cast<int>(threadIdx.x) / threads;
    load_chunks<T, kChunks>(w, x + row * ldx, whole, thread, threads, row < rows);
    int buffer = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_block; base < rows; base += step, row += step) {
        const bool live = row < rows;
        const T* src = x + row * ldx;
        uint32_t m = 0;
        if (live)
            for (int i = whole * kQuantChunk + thread; i < cols; i += threads) m = max(m, __float_as_uint(to_float(src[i])) & 0x7fffffffu);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) m = max(m, Chunk<T>::largest(w[c]));
        uint32_t next[kChunks][Chunk<T>::kWords];
        load_chunks<T, kChunks>(next, src + step * ldx, whole, thread, threads, row + step < rows);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
            if (d < threads) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (threads > 32) {
            if (lane == 0) warp_max[buffer][warp] = m;
            __syncthreads();
            const int warps = threads >> 5;
            m = __reduce_max_sync(0xffffffffu, lane < warps ? warp_max[buffer][(warp & ~(warps - 1)) + lane] : 0u);
            buffer ^= 1;
        }
        if (live) {
            float scale, inv;
            bool rounds;
            row_scale(m, scale, inv, rounds);
            int8_t* dst = q + row * ldq;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int chunk = c * threads + thread;
                if (chunk < whole) *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(chunk) * kQuantChunk) = quantize_chunk<T>(w[c], inv, scale, rounds);
            }
            for (int i = whole * kQuantChunk + thread; i < cols; i += threads)
                dst[i] = rounds ? quantize_one(to_float(src[i]), inv, scale) : static_cast<int8_t>(0);
            if (thread == 0) scale_out[row] = scale;
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < Chunk<T>::kWords; ++i) w[c][i] = next[c][i];
    }
}

// Any alignment and length: one block per row, element by element, the row read twice.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads)
quantize_rows_any_kernel(const T* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale_out, int64_t cols, int64_t ldx,
                         int64_t ldq) {
    grid_launch_dependents();
    grid_dependency_wait();
    const T* row = x + static_cast<int64_t>(blockIdx.x) * ldx;
    int8_t* out = q + static_cast<int64_t>(blockIdx.x) * ldq;
    __shared__ uint32_t warp_max[32];
    uint32_t m = 0;
#pragma unroll 8
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) m = max(m, __float_as_uint(to_float(row[c])) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < kThreads / 32 ? warp_max[threadIdx.x & 31] : 0u);
    float scale, inv;
    bool rounds;
    row_scale(m, scale, inv, rounds);
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < cols; c += kThreads)
        out[c] = rounds ? quantize_one(to_float(row[c]), inv, scale) : static_cast<int8_t>(0);
    if (threadIdx.x == 0) scale_out[blockIdx.x] = scale;
}

template <typename T, int kChunks>
static int launch_chunks(const T* x, int8_t* q, float* scale, int64_t rows, int64_t cols, int64_t ldx, int64_t ldq, int threads, int sm_count,
                         cudaStream_t stream) {
    const int block = threads > kQuantThreads ? threads : kQuantThreads;
    const int64_t blocks = (rows * threads + block - 1) / block;
    const int64_t resident = static_cast<int64_t>(sm_count) * (block > kQuantThreads ? 1024 / block : 3);
    const dim3 grid(static_cast<unsigned>(blocks < resident ? blocks : resident));
    if (block > kQuantThreads) {
        TCB_CUDA(launch_overlapped(quantize_rows_kernel<T, kChunks, 1024>, grid, dim3(block), 0, stream, x, q, scale, static_cast<int>(rows),
                                   static_cast<int>(cols), ldx, ldq, threads));
    } else {
        TCB_CUDA(launch_overlapped(quantize_rows_kernel<T, kChunks, 256>, grid, dim3(block), 0, stream, x, q, scale, static_cast<int>(rows),
                                   static_cast<int>(cols), ldx, ldq, threads));
    }
    return TC_OK;
}

template <typename T>
static int launch_quantize(const void* xv, void* qv, float* scale, int64_t rows, int64_t cols, int64_t ldx, int64_t ldq, int sm_count,
                           cudaStream_t stream) {
    const T* x = static_cast<const T*>(xv);
    int8_t* q = static_cast<int8_t*>(qv);
    const int64_t es = sizeof(T);
    const int64_t chunks = (cols + kQuantChunk - 1) / kQuantChunk;
    const bool granular = aligned16(x) && aligned16(q) && (ldx * es) % 16 == 0 && ldq % 16 == 0;
    constexpr int kMost = sizeof(T) == 4 ? 1 : 2;   // chunks a thread can hold twice over in 64 registers
    if (!granular || chunks > kMost * 1024) {
        // more threads a row where the rows alone do not fill the SMs: 512 x 65536 fp16 49 us, 124 with 256 threads; 2000 x 4099 28 and 11
        const dim3 grid(static_cast<unsigned>(rows));
        if (cols > 4096 && rows < 8 * sm_count) {
            TCB_CUDA(launch_overlapped(quantize_rows_any_kernel<T, 1024>, grid, dim3(1024), 0, stream, x, q, scale, cols, ldx, ldq));
        } else {
            TCB_CUDA(launch_overlapped(quantize_rows_any_kernel<T, kQuantThreads>, grid, dim3(kQuantThreads), 0, stream, x, q, scale, cols, ldx, ldq));
        }
        return TC_OK;
    }
    // Few rows: as many threads as chunks. Many rows: two chunks a thread, so that a thread has four loads in flight
    // (8192 x 8192: fp16 34.4 us, 5.9 TB/s; bf16 38.5, fp32 50.6, 6.6 TB/s. fp16 took 46.8 before the next row's loads were
    // issued ahead of the rounding).
    const int per_thread = rows >= 1024 || chunks > 1024 ? kMost : 1;
    int threads = 1;
    while (threads < 1024 && static_cast<int64_t>(threads) * per_thread < chunks) threads *= 2;
    if (per_thread == 2) return launch_chunks<T, kMost>(x, q, scale, rows, cols, ldx, ldq, threads, sm_count, stream);
    return launch_chunks<T, 1>(x, q, scale, rows, cols, ldx, ldq, threads, sm_count, stream);
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
    const Extent xs = extent_of_rows(x, rows, cols, ldx, es), qs = extent_of_rows(q, rows, cols, ldq, 1), scales = extent_of_vector(scale, rows, 4);
    TCB_REQUIRE(!extents_meet(qs, xs) && !extents_meet(scales, xs) && !extents_meet(scales, qs),
                "quantize_rows: q and scale must not overlap x or each other");
    const DeviceInfo* dev = nullptr;
    if (int rc = current_device(&dev)) return rc;
    auto s = static_cast<cudaStream_t>(stream);
    if (x_type == TC_F32) return launch_quantize<float>(x, q, scale, rows, cols, ldx, ldq, dev->sm_count, s);
    if (x_type == TC_F16) return launch_quantize<__half>(x, q, scale, rows, cols, ldx, ldq, dev->sm_count, s);
    return launch_quantize<__nv_bfloat16>(x, q, scale, rows, cols, ldx, ldq, dev->sm_count, s);
}
