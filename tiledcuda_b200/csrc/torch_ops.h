// The grouped and 8-bit products as functions of tensors (torch_bind.cc): their checks, then the call of the C ABI on the
// tensors' device and its current stream. A refusal of the arguments is a c10::Error, a CUDA call that failed a CudaFailure.
#pragma once

#include <ATen/core/Tensor.h>
#include <c10/util/Exception.h>

namespace tiledcuda {

class CudaFailure : public c10::Error {
    using c10::Error::Error;
};

void quantize_rows(const at::Tensor& x, at::Tensor& q, at::Tensor& scale);
void gemm_i8(const at::Tensor& A, const at::Tensor& B, const at::Tensor& scale_a, const at::Tensor& scale_b, at::Tensor& C);
void grouped_gemm(const at::Tensor& A, const at::Tensor& B, const at::Tensor& offsets, at::Tensor& C);
void grouped_gemm_i8(const at::Tensor& A, const at::Tensor& B, const at::Tensor& scale_a, const at::Tensor& scale_b,
                     const at::Tensor& offsets, at::Tensor& C);
void grouped_gemm_dgrad(const at::Tensor& dC, const at::Tensor& B, const at::Tensor& offsets, at::Tensor& dA);
void grouped_gemm_wgrad(const at::Tensor& dC, const at::Tensor& A, const at::Tensor& offsets, at::Tensor& dB);

}  // namespace tiledcuda
