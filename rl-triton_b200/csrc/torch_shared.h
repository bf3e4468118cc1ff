// torch_shared.h -- what the operator files of librlscan_torch.so share
// (defined in torch_ops.cpp).
#pragma once
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>

namespace rls_torch {

// The workspace of (device, stream), for num_elements steps or more.
at::Tensor workspace_for(const at::Device& dev, cudaStream_t s, int64_t num_elements);
cudaStream_t stream_of(const at::Tensor& t);
// Raises for a status other than RLS_OK.
void check(int st, const char* what);
// Contiguous and 16-byte aligned; f32(): and float32.
at::Tensor ready(const at::Tensor& t);
std::optional<at::Tensor> ready(const std::optional<at::Tensor>& t);
at::Tensor f32(const at::Tensor& t);
std::optional<at::Tensor> f32(const std::optional<at::Tensor>& t);

}  // namespace rls_torch
