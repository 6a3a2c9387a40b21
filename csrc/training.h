// Declarations of the operators around a training step's products (layernorm.cu, rotary.cu, clip.cu, vocab_loss.cu; autograd nodes in training.cpp).
#pragma once
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>

#include <array>

namespace q38 {

using OptTensor = c10::optional<at::Tensor>;

// A CUDA tensor without the dispatcher's way, which costs a short call as much as its kernel's launch.
inline at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, at::Device device) { return at::detail::empty_cuda(sizes, type, device, c10::nullopt); }

// Lets `kernel` take `bytes` of dynamic shared memory on the current device; the driver is asked when a kernel and device need more than before (gemm_persistent.cu).
void allow_shared_memory(const void* kernel, int bytes);

// Any x with a last dimension -> {y of x's shape, [2, rows] mean and 1 / deviation (undefined without `save`)}.
std::pair<at::Tensor, at::Tensor> layer_norm_fwd(const at::Tensor& x, const OptTensor& w, const OptTensor& b, double eps, at::ScalarType out_type, bool save);
// {dx, dw, db}, undefined where not wanted.
std::array<at::Tensor, 3> layer_norm_bwd(const at::Tensor& dy, const at::Tensor& x, const OptTensor& w, const OptTensor& b, const at::Tensor& stats, bool want_dx, bool want_dw, bool want_db);

void rotary_check(const at::Tensor& q, const OptTensor& k, const at::Tensor& pos, const at::Tensor& freq);
// q, k [batch, seq, heads, dim], either may be undefined; sign -1: the gradient.
std::pair<at::Tensor, at::Tensor> rotary_apply(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& freq, double magnitude, bool interleaved, double sign);

at::Tensor clip_grad_norm(at::TensorList grads, at::TensorList outs, double max_norm, bool scale);

// A bf16 matrix as TMA reads it: itself, or a copy in padded rows where its rows are not contiguous, on 16 bytes and a multiple of that apart.
at::Tensor vocab_rows(const at::Tensor& t);
// hidden [rows, h], weight [vocabulary, h] bf16, both as vocab_rows gives them; reduction 0 none, 1 sum, 2 mean over the rows that count.
// `shape`: of the losses without a reduction.  Returns {loss (that shape, or 0-dim), log2 of the rows' sums [rows], number of rows that count (undefined without a reduction)}.
std::array<at::Tensor, 3> vocab_loss_fwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, at::IntArrayRef shape, int64_t reduction,
                                         const at::Tensor& err);
// g: gradient of the loss ([rows] fp32 without a reduction, one element with one).  Returns {dh (bf16, or fp32 with `fp32_dh`), dW}: undefined where not wanted or, for dW,
// where it was added to `grad` (fp32 [vocabulary, h], contiguous).  `workspace`: bytes that dz of one piece may take; 256 columns are taken in any case.
std::pair<at::Tensor, at::Tensor> vocab_loss_bwd(const at::Tensor& g, const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target, const at::Tensor& lse2,
                                                 const at::Tensor& count, int64_t reduction, bool want_dh, bool fp32_dh, bool want_dw, bool fp32_dw, const at::Tensor& grad, int64_t workspace,
                                                 const at::Tensor& err);

}  // namespace q38
