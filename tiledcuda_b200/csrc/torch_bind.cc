// torch.ops.tiledcuda.*: the reference's operator registry (src/torch_bind.cc:8-11 registers scatter_nd
// and flash_attention_fwd) re-created over the C ABI, plus the ops the reference only has as C++
// examples (gemm, back2back_gemm) or names without code (lstm_cell). Every op writes into
// caller-allocated tensors and returns nothing, launches on the current CUDA stream and never
// synchronises. A failing status becomes a c10::Error (RuntimeError in Python); there is no CPU
// kernel registered, so a CPU tensor is a dispatcher error, not a fallback.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <algorithm>
#include <initializer_list>
#include <vector>

#include "../../include/tiledcuda_b200.h"
#include "torch_ops.h"

namespace {

void check(const char* op, int status) {
    if (status == TC_ERR_CUDA)
        throw tiledcuda::CudaFailure({__func__, __FILE__, static_cast<uint32_t>(__LINE__)},
                                     c10::str("tiledcuda::", op, " failed with status ", status, ": ", tc_last_error()));
    TORCH_CHECK(status == TC_OK, "tiledcuda::", op, " failed with status ", status, ": ", tc_last_error());
}

tc_stream_t stream_of(const at::Tensor& t) {
    return static_cast<tc_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

void need(const at::Tensor& t, const char* name, at::ScalarType dtype) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// Every tensor of a call lives on the device of the first one: the C ABI takes raw pointers and cannot tell.
void same_device(const char* op, const at::Tensor& first, std::initializer_list<const at::Tensor*> rest) {
    for (const at::Tensor* t : rest)
        TORCH_CHECK(t->device() == first.device(), op, ": all tensors must be on one device (got ", first.device(), " and ",
                    t->device(), ")");
}

// Shape rules shared by both scatter ops: indices [..., k] with k <= data.dim(), and updates holding exactly one
// slice (the trailing data.dim() - k dimensions of data) per index tuple. Returns n, the number of tuples.
int64_t scatter_shapes(const char* op, const at::Tensor& data, const at::Tensor& updates, const at::Tensor& indices) {
    TORCH_CHECK(data.is_cuda() && updates.is_cuda() && indices.is_cuda(), op, " needs CUDA tensors");
    same_device(op, data, {&updates, &indices});
    TORCH_CHECK(data.is_contiguous() && updates.is_contiguous() && indices.is_contiguous(), op, " needs contiguous tensors");
    TORCH_CHECK(updates.scalar_type() == data.scalar_type(), op, ": updates and data must have the same dtype");
    TORCH_CHECK(indices.scalar_type() == at::kLong || indices.scalar_type() == at::kInt, op, ": indices must be int32 or int64");
    TORCH_CHECK(indices.dim() >= 1 && data.dim() >= 1, op, ": indices and data must have at least one dimension");
    const int64_t k = indices.size(-1);
    TORCH_CHECK(k >= 1 && k <= data.dim(), op, ": index tuples of length ", k, " do not fit a table of rank ", data.dim());
    const int64_t n = indices.numel() / k;
    int64_t slice = 1;
    for (int64_t i = k; i < data.dim(); ++i) slice *= data.size(i);
    TORCH_CHECK(updates.numel() == n * slice, op, ": updates has ", updates.numel(), " elements, ", n, " tuples of ", slice,
                " elements need ", n * slice);
    return n;
}

// Same argument order as the reference's custom_scatter_op(data, updates, indices)
// (include/kernels/scatter_nd.hpp:39-40). data keeps its N-D shape; indices is [..., k].
void scatter_nd_op(at::Tensor& data, const at::Tensor& updates, const at::Tensor& indices) {
    const int64_t n = scatter_shapes("scatter_nd", data, updates, indices);
    const bool i64 = indices.scalar_type() == at::kLong;
    const int64_t k = indices.size(-1);
    std::vector<int64_t> dims(data.sizes().begin(), data.sizes().end());
    c10::cuda::CUDAGuard guard(data.device());
    check("scatter_nd", tc_scatter_nd(data.data_ptr(), updates.data_ptr(), indices.data_ptr(), i64 ? 1 : 0, dims.data(),
                                      static_cast<int>(dims.size()), n, static_cast<int>(k),
                                      static_cast<int>(data.element_size()), stream_of(data)));
}

// The accumulating form, which is what the reference's kernel does (src/kernels/scatter_nd.cu:44-47).
void scatter_nd_add_op(at::Tensor& data, const at::Tensor& updates, const at::Tensor& indices) {
    const int64_t n = scatter_shapes("scatter_nd_add", data, updates, indices);
    int elem_type = -1;
    switch (data.scalar_type()) {
        case at::kFloat: elem_type = 0; break;
        case at::kHalf: elem_type = 1; break;
        case at::kInt: elem_type = 2; break;
        case at::kDouble: elem_type = 3; break;
        default: TORCH_CHECK(false, "scatter_nd_add supports float32, float16, int32 and float64 tables");
    }
    const bool i64 = indices.scalar_type() == at::kLong;
    const int64_t k = indices.size(-1);
    std::vector<int64_t> dims(data.sizes().begin(), data.sizes().end());
    c10::cuda::CUDAGuard guard(data.device());
    check("scatter_nd_add", tc_scatter_nd_add(data.data_ptr(), updates.data_ptr(), indices.data_ptr(), i64 ? 1 : 0, dims.data(),
                                              static_cast<int>(dims.size()), n, static_cast<int>(k), elem_type, stream_of(data)));
}

// Same signature as custom_flash_attention_op (include/kernels/flash_attn.hpp:35-37): flattened fp16
// Q [m,k], K [n,k], V^T [p,n], O [m,p]; one head; no softmax scale.
void flash_attention_fwd_op(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, at::Tensor& O, int64_t m,
                            int64_t n, int64_t k, int64_t p) {
    need(Q, "Q", at::kHalf);
    need(K, "K", at::kHalf);
    need(V, "V", at::kHalf);
    need(O, "O", at::kHalf);
    same_device("flash_attention_fwd", Q, {&K, &V, &O});
    TORCH_CHECK(m > 0 && n > 0 && k > 0 && p > 0, "flash_attention_fwd: m, n, k, p must be positive");
    TORCH_CHECK(Q.numel() == m * k && K.numel() == n * k && V.numel() == n * p && O.numel() == m * p,
                "flash_attention_fwd: tensor sizes do not match m, n, k, p");
    c10::cuda::CUDAGuard guard(Q.device());
    check("flash_attention_fwd", tc_flash_attn_fwd_f16(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), nullptr, 1, 1, m,
                                                       n, k, p, 1.0f, 1, stream_of(Q)));
}

// Batched, scaled attention: Q [B,H,Sq,D], K [B,H,Skv,D], V [B,H,Skv,Dv] (or V^T), O [B,H,Sq,Dv].
void flash_attn_op(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, at::Tensor& O, double scale,
                   bool v_is_transposed) {
    need(Q, "Q", at::kHalf);
    need(K, "K", at::kHalf);
    need(V, "V", at::kHalf);
    need(O, "O", at::kHalf);
    same_device("flash_attn", Q, {&K, &V, &O});
    TORCH_CHECK(Q.dim() == 4 && K.dim() == 4 && V.dim() == 4 && O.dim() == 4, "flash_attn: tensors must be [B,H,S,D]");
    const int64_t b = Q.size(0), h = Q.size(1), sq = Q.size(2), d = Q.size(3), skv = K.size(2);
    const int64_t dv = v_is_transposed ? V.size(2) : V.size(3);
    TORCH_CHECK(K.size(0) == b && K.size(1) == h && K.size(3) == d, "flash_attn: K shape mismatch");
    TORCH_CHECK(V.size(0) == b && V.size(1) == h && (v_is_transposed ? V.size(3) : V.size(2)) == skv, "flash_attn: V shape mismatch");
    TORCH_CHECK(O.size(0) == b && O.size(1) == h && O.size(2) == sq && O.size(3) == dv, "flash_attn: O shape mismatch");
    c10::cuda::CUDAGuard guard(Q.device());
    check("flash_attn", tc_flash_attn_fwd_f16(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), nullptr, b, h, sq, skv, d, dv,
                                              static_cast<float>(scale), v_is_transposed ? 1 : 0, stream_of(Q)));
}

// flash_attn with a causal mask (bottom-right aligned) and / or [B,S,H,D] operands.
void flash_attn_ex_op(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, at::Tensor& O, double scale, bool causal,
                      bool seq_major) {
    need(Q, "Q", at::kHalf);
    need(K, "K", at::kHalf);
    need(V, "V", at::kHalf);
    need(O, "O", at::kHalf);
    same_device("flash_attn_ex", Q, {&K, &V, &O});
    TORCH_CHECK(Q.dim() == 4 && K.dim() == 4 && V.dim() == 4 && O.dim() == 4, "flash_attn_ex: tensors must be 4-D");
    const int sd = seq_major ? 1 : 2, hd = seq_major ? 2 : 1;
    const int64_t b = Q.size(0), h = Q.size(hd), sq = Q.size(sd), d = Q.size(3), skv = K.size(sd), dv = V.size(3);
    TORCH_CHECK(K.size(0) == b && K.size(hd) == h && K.size(3) == d, "flash_attn_ex: K shape mismatch");
    TORCH_CHECK(V.size(0) == b && V.size(hd) == h && V.size(sd) == skv, "flash_attn_ex: V shape mismatch");
    TORCH_CHECK(K.size(sd) == skv, "flash_attn_ex: K shape mismatch");
    TORCH_CHECK(O.size(0) == b && O.size(hd) == h && O.size(sd) == sq && O.size(3) == dv, "flash_attn_ex: O shape mismatch");
    c10::cuda::CUDAGuard guard(Q.device());
    check("flash_attn_ex", tc_flash_attn_fwd_ex_f16(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), nullptr, b, h, sq, skv, d,
                                                    dv, static_cast<float>(scale), 0, causal ? 1 : 0, seq_major ? 1 : 0, stream_of(Q)));
}

// C[M,N] fp32 = A[M,K] @ B[N,K]^T (B is the column-major operand of the reference's GEMM examples).
void gemm_op(const at::Tensor& A, const at::Tensor& B, at::Tensor& C) {
    need(A, "A", at::kHalf);
    need(B, "B", at::kHalf);
    need(C, "C", at::kFloat);
    same_device("gemm", A, {&B, &C});
    TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && C.dim() == 2, "gemm: tensors must be 2-D");
    TORCH_CHECK(B.size(1) == A.size(1) && C.size(0) == A.size(0) && C.size(1) == B.size(0), "gemm: shape mismatch");
    c10::cuda::CUDAGuard guard(A.device());
    check("gemm", tc_gemm_f16_f32(A.data_ptr(), B.data_ptr(), C.data_ptr(), A.size(0), B.size(0), A.size(1), A.size(1), B.size(1),
                                  C.size(1), stream_of(A)));
}

// E fp32 [.., M,P] = fp16(A @ B^T) @ D^T; A [.., M,K], B [.., N,K], D [.., P,N]; 2-D or batched 3-D.
void back2back_gemm_op(const at::Tensor& A, const at::Tensor& B, const at::Tensor& D, at::Tensor& E) {
    need(A, "A", at::kHalf);
    need(B, "B", at::kHalf);
    need(D, "D", at::kHalf);
    need(E, "E", at::kFloat);
    same_device("back2back_gemm", A, {&B, &D, &E});
    TORCH_CHECK((A.dim() == 2 || A.dim() == 3) && B.dim() == A.dim() && D.dim() == A.dim() && E.dim() == A.dim(),
                "back2back_gemm: tensors must all be 2-D or all 3-D");
    const int64_t batch = A.dim() == 3 ? A.size(0) : 1;
    const int64_t m = A.size(-2), k = A.size(-1), n = B.size(-2), p = D.size(-2);
    TORCH_CHECK(B.size(-1) == k && D.size(-1) == n && E.size(-2) == m && E.size(-1) == p, "back2back_gemm: shape mismatch");
    TORCH_CHECK(A.dim() == 2 || (B.size(0) == batch && D.size(0) == batch && E.size(0) == batch), "back2back_gemm: batch mismatch");
    c10::cuda::CUDAGuard guard(A.device());
    check("back2back_gemm", tc_b2b_gemm_f16(A.data_ptr(), B.data_ptr(), D.data_ptr(), E.data_ptr(), m, n, k, p, batch, stream_of(A)));
}

// One LSTM cell step, gate order (i, f, g, o); bias may be an undefined tensor (None).
void lstm_cell_op(const at::Tensor& W, const at::Tensor& U, const c10::optional<at::Tensor>& bias, const at::Tensor& x,
                  const at::Tensor& h_prev, const at::Tensor& c_prev, at::Tensor& h_out, at::Tensor& c_out) {
    need(W, "W", at::kHalf);
    need(U, "U", at::kHalf);
    need(x, "x", at::kHalf);
    need(h_prev, "h_prev", at::kHalf);
    need(h_out, "h_out", at::kHalf);
    need(c_prev, "c_prev", at::kFloat);
    need(c_out, "c_out", at::kFloat);
    const float* b = nullptr;
    if (bias.has_value() && bias->defined()) {
        need(*bias, "bias", at::kFloat);
        b = bias->data_ptr<float>();
    }
    same_device("lstm_cell", x, {&W, &U, &h_prev, &c_prev, &h_out, &c_out});
    TORCH_CHECK(W.dim() == 2 && U.dim() == 2 && x.dim() == 2, "lstm_cell: W, U and x must be 2-D");
    const int64_t batch = x.size(0), input = x.size(1), hidden = U.size(1);
    TORCH_CHECK(W.size(0) == 4 * hidden && W.size(1) == input && U.size(0) == 4 * hidden, "lstm_cell: weight shape mismatch");
    for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&h_prev, &c_prev, &h_out, &c_out})
        TORCH_CHECK(t->dim() == 2 && t->size(0) == batch && t->size(1) == hidden, "lstm_cell: h_prev, c_prev, h_out and c_out must be [",
                    batch, ", ", hidden, "], got ", t->sizes());
    if (b != nullptr) {
        same_device("lstm_cell", x, {&*bias});
        TORCH_CHECK(bias->numel() == 4 * hidden, "lstm_cell: bias must have 4 * hidden = ", 4 * hidden, " elements, got ", bias->numel());
    }
    TORCH_CHECK(h_out.data_ptr() != h_prev.data_ptr(), "lstm_cell: h_out must not alias h_prev");
    c10::cuda::CUDAGuard guard(x.device());
    check("lstm_cell", tc_lstm_cell_f16(W.data_ptr(), U.data_ptr(), b, x.data_ptr(), h_prev.data_ptr(), c_prev.data_ptr<float>(),
                                        h_out.data_ptr(), c_out.data_ptr<float>(), batch, input, hidden, stream_of(x)));
}

// ---- scaled 8-bit and expert-grouped products -------------------------------------------------------------------
int type_code(const at::Tensor& t) {
    return t.scalar_type() == at::kFloat ? TC_F32 : t.scalar_type() == at::kHalf ? TC_F16 : TC_BF16;
}
bool is_half(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// A CUDA tensor of this shape whose last dimension is dense; other strides are the caller's.
void need_rows(const char* op, const char* name, const at::Tensor& t, at::IntArrayRef shape, bool type_ok) {
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor");
    TORCH_CHECK(type_ok, op, ": ", name, " may not be ", t.scalar_type());
    TORCH_CHECK(t.sizes() == shape, op, ": ", name, " must be ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, op, ": ", name, " must have unit inner stride");
}

// Stride of a dimension; that of a dimension of one element is never stepped over and may be anything, so it is
// replaced by the dense one, rounded up to what the kernels' loads are granular in.
int64_t ld(const at::Tensor& t, int64_t dim, int64_t granule = 1) {
    if (t.size(dim) > 1) return t.stride(dim);
    const int64_t inner = dim + 2 == t.dim() ? t.size(dim + 1) : t.size(dim + 1) * ld(t, dim + 1, granule);
    return (std::max<int64_t>(1, inner) + granule - 1) / granule * granule;
}

int wide_offsets(const char* op, const at::Tensor& offsets, int64_t experts) {
    need_rows(op, "offsets", offsets, {experts + 1}, offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong);
    return offsets.scalar_type() == at::kLong ? 1 : 0;
}

}  // namespace

namespace tiledcuda {

void quantize_rows(const at::Tensor& x, at::Tensor& q, at::Tensor& scale) {
    const char* op = "quantize_rows";
    TORCH_CHECK(x.dim() == 2, op, ": x must be 2-D");
    need_rows(op, "x", x, x.sizes(), x.scalar_type() == at::kFloat || is_half(x));
    need_rows(op, "q", q, x.sizes(), q.scalar_type() == at::kChar);
    need_rows(op, "scale", scale, {x.size(0)}, scale.scalar_type() == at::kFloat);
    same_device(op, x, {&q, &scale});
    c10::cuda::CUDAGuard guard(x.device());
    check(op, tc_quantize_rows(x.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), x.size(0), x.size(1), ld(x, 0), ld(q, 0), type_code(x),
                               stream_of(x)));
}

void gemm_i8(const at::Tensor& A, const at::Tensor& B, const at::Tensor& scale_a, const at::Tensor& scale_b, at::Tensor& C) {
    const char* op = "gemm_i8";
    TORCH_CHECK(A.dim() == 2 && B.dim() == 2, op, ": A and B must be 2-D");
    const int64_t m = A.size(0), k = A.size(1), n = B.size(0);
    need_rows(op, "A", A, {m, k}, A.scalar_type() == at::kChar);
    need_rows(op, "B", B, {n, k}, B.scalar_type() == at::kChar);
    need_rows(op, "scale_a", scale_a, {m}, scale_a.scalar_type() == at::kFloat);
    need_rows(op, "scale_b", scale_b, {n}, scale_b.scalar_type() == at::kFloat);
    need_rows(op, "C", C, {m, n}, C.scalar_type() == at::kFloat || is_half(C));
    same_device(op, A, {&B, &scale_a, &scale_b, &C});
    c10::cuda::CUDAGuard guard(A.device());
    check(op, tc_gemm_i8(A.data_ptr(), B.data_ptr(), scale_a.data_ptr<float>(), scale_b.data_ptr<float>(), C.data_ptr(), m, n, k, ld(A, 0, 16),
                         ld(B, 0, 16), ld(C, 0), type_code(C), stream_of(A)));
}

void grouped_gemm(const at::Tensor& A, const at::Tensor& B, const at::Tensor& offsets, at::Tensor& C) {
    const char* op = "grouped_gemm";
    TORCH_CHECK(A.dim() == 2 && B.dim() == 3, op, ": A must be 2-D and B 3-D");
    const int64_t t = A.size(0), k = A.size(1), e = B.size(0), n = B.size(1);
    need_rows(op, "A", A, {t, k}, is_half(A));
    need_rows(op, "B", B, {e, n, k}, B.scalar_type() == A.scalar_type());
    need_rows(op, "C", C, {t, n}, C.scalar_type() == A.scalar_type() || C.scalar_type() == at::kFloat);
    const int wide = wide_offsets(op, offsets, e);
    same_device(op, A, {&B, &offsets, &C});
    c10::cuda::CUDAGuard guard(A.device());
    check(op, tc_grouped_gemm(A.data_ptr(), B.data_ptr(), offsets.data_ptr(), wide, C.data_ptr(), t, e, n, k, ld(A, 0, 8), ld(B, 1, 8),
                              ld(B, 0, 8), ld(C, 0), type_code(A), type_code(C), stream_of(A)));
}

void grouped_gemm_i8(const at::Tensor& A, const at::Tensor& B, const at::Tensor& scale_a, const at::Tensor& scale_b,
                        const at::Tensor& offsets, at::Tensor& C) {
    const char* op = "grouped_gemm_i8";
    TORCH_CHECK(A.dim() == 2 && B.dim() == 3, op, ": A must be 2-D and B 3-D");
    const int64_t t = A.size(0), k = A.size(1), e = B.size(0), n = B.size(1);
    need_rows(op, "A", A, {t, k}, A.scalar_type() == at::kChar);
    need_rows(op, "B", B, {e, n, k}, B.scalar_type() == at::kChar);
    need_rows(op, "scale_a", scale_a, {t}, scale_a.scalar_type() == at::kFloat);
    need_rows(op, "scale_b", scale_b, {e, n}, scale_b.scalar_type() == at::kFloat);
    TORCH_CHECK(scale_b.is_contiguous(), op, ": scale_b must be contiguous");
    need_rows(op, "C", C, {t, n}, C.scalar_type() == at::kFloat || is_half(C));
    const int wide = wide_offsets(op, offsets, e);
    same_device(op, A, {&B, &scale_a, &scale_b, &offsets, &C});
    c10::cuda::CUDAGuard guard(A.device());
    check(op, tc_grouped_gemm_i8(A.data_ptr(), B.data_ptr(), scale_a.data_ptr<float>(), scale_b.data_ptr<float>(), offsets.data_ptr(), wide,
                                 C.data_ptr(), t, e, n, k, ld(A, 0, 16), ld(B, 1, 16), ld(B, 0, 16), ld(C, 0), type_code(C), stream_of(A)));
}

void grouped_gemm_dgrad(const at::Tensor& dC, const at::Tensor& B, const at::Tensor& offsets, at::Tensor& dA) {
    const char* op = "grouped_gemm_dgrad";
    TORCH_CHECK(dC.dim() == 2 && B.dim() == 3, op, ": dC must be 2-D and B 3-D");
    const int64_t t = dC.size(0), n = dC.size(1), e = B.size(0), k = B.size(2);
    need_rows(op, "dC", dC, {t, n}, is_half(dC));
    need_rows(op, "B", B, {e, n, k}, B.scalar_type() == dC.scalar_type());
    need_rows(op, "dA", dA, {t, k}, dA.scalar_type() == dC.scalar_type() || dA.scalar_type() == at::kFloat);
    const int wide = wide_offsets(op, offsets, e);
    same_device(op, dC, {&B, &offsets, &dA});
    c10::cuda::CUDAGuard guard(dC.device());
    check(op, tc_grouped_gemm_dgrad(dC.data_ptr(), B.data_ptr(), offsets.data_ptr(), wide, dA.data_ptr(), t, e, n, k, ld(dC, 0, 8), ld(B, 1, 8),
                                    ld(B, 0, 8), ld(dA, 0), type_code(dC), type_code(dA), stream_of(dC)));
}

void grouped_gemm_wgrad(const at::Tensor& dC, const at::Tensor& A, const at::Tensor& offsets, at::Tensor& dB) {
    const char* op = "grouped_gemm_wgrad";
    TORCH_CHECK(dC.dim() == 2 && A.dim() == 2 && dB.dim() == 3, op, ": dC and A must be 2-D and dB 3-D");
    const int64_t t = dC.size(0), n = dC.size(1), e = dB.size(0), k = A.size(1);
    need_rows(op, "dC", dC, {t, n}, is_half(dC));
    need_rows(op, "A", A, {t, k}, A.scalar_type() == dC.scalar_type());
    need_rows(op, "dB", dB, {e, n, k}, dB.scalar_type() == dC.scalar_type() || dB.scalar_type() == at::kFloat);
    const int wide = wide_offsets(op, offsets, e);
    same_device(op, dC, {&A, &offsets, &dB});
    c10::cuda::CUDAGuard guard(dC.device());
    check(op, tc_grouped_gemm_wgrad(dC.data_ptr(), A.data_ptr(), offsets.data_ptr(), wide, dB.data_ptr(), t, e, n, k, ld(dC, 0, 8), ld(A, 0, 8),
                                    ld(dB, 1), ld(dB, 0), type_code(dC), type_code(dB), stream_of(dC)));
}

}  // namespace tiledcuda

TORCH_LIBRARY(tiledcuda, m) {
    m.def("scatter_nd(Tensor(a!) data, Tensor updates, Tensor indices) -> ()");
    m.def("flash_attention_fwd(Tensor Q, Tensor K, Tensor V, Tensor(a!) O, int m, int n, int k, int p) -> ()");
    m.def("flash_attn(Tensor Q, Tensor K, Tensor V, Tensor(a!) O, float scale, bool v_is_transposed) -> ()");
    m.def("flash_attn_ex(Tensor Q, Tensor K, Tensor V, Tensor(a!) O, float scale, bool causal, bool seq_major) -> ()");
    m.def("scatter_nd_add(Tensor(a!) data, Tensor updates, Tensor indices) -> ()");
    m.def("gemm(Tensor A, Tensor B, Tensor(a!) C) -> ()");
    m.def("back2back_gemm(Tensor A, Tensor B, Tensor D, Tensor(a!) E) -> ()");
    m.def("lstm_cell(Tensor W, Tensor U, Tensor? bias, Tensor x, Tensor h_prev, Tensor c_prev, Tensor(a!) h_out, "
          "Tensor(b!) c_out) -> ()");
    m.def("quantize_rows(Tensor x, Tensor(a!) q, Tensor(b!) scale) -> ()");
    m.def("gemm_i8(Tensor A, Tensor B, Tensor scale_a, Tensor scale_b, Tensor(a!) C) -> ()");
    m.def("grouped_gemm(Tensor A, Tensor B, Tensor offsets, Tensor(a!) C) -> ()");
    m.def("grouped_gemm_i8(Tensor A, Tensor B, Tensor scale_a, Tensor scale_b, Tensor offsets, Tensor(a!) C) -> ()");
    m.def("grouped_gemm_dgrad(Tensor dC, Tensor B, Tensor offsets, Tensor(a!) dA) -> ()");
    m.def("grouped_gemm_wgrad(Tensor dC, Tensor A, Tensor offsets, Tensor(a!) dB) -> ()");
}

TORCH_LIBRARY_IMPL(tiledcuda, CUDA, m) {
    m.impl("scatter_nd", &scatter_nd_op);
    m.impl("flash_attention_fwd", &flash_attention_fwd_op);
    m.impl("flash_attn", &flash_attn_op);
    m.impl("flash_attn_ex", &flash_attn_ex_op);
    m.impl("scatter_nd_add", &scatter_nd_add_op);
    m.impl("gemm", &gemm_op);
    m.impl("back2back_gemm", &back2back_gemm_op);
    m.impl("lstm_cell", &lstm_cell_op);
    m.impl("quantize_rows", &tiledcuda::quantize_rows);
    m.impl("gemm_i8", &tiledcuda::gemm_i8);
    m.impl("grouped_gemm", &tiledcuda::grouped_gemm);
    m.impl("grouped_gemm_i8", &tiledcuda::grouped_gemm_i8);
    m.impl("grouped_gemm_dgrad", &tiledcuda::grouped_gemm_dgrad);
    m.impl("grouped_gemm_wgrad", &tiledcuda::grouped_gemm_wgrad);
}

// The grouped and 8-bit products take no part in autograd (their gradients are operators of their own): parameters that
// require grad may be operands, and the call goes straight to the kernel.
TORCH_LIBRARY_IMPL(tiledcuda, Autograd, m) {
    for (const char* op : {"quantize_rows", "gemm_i8", "grouped_gemm", "grouped_gemm_i8", "grouped_gemm_dgrad", "grouped_gemm_wgrad"})
        m.impl(op, torch::CppFunction::makeFallthrough());
}
