// Python binding of the gradient norm and clipping over a list of tensors.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <functional>

#include "olb_api.h"

namespace {

// Strides that cannot address one element twice (sufficient: sorted by stride, each one clears the span below it).
bool no_self_overlap(const at::Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.emplace_back(t.stride(d), t.size(d));
  std::sort(dims.begin(), dims.end());
  int64_t span = 1;
  for (const auto& [stride, size] : dims) {
    if (stride < span) return false;
    span = stride * (size - 1) + span;
  }
  return true;
}

// The norm as a 0-dim fp32 tensor; nothing when a tensor's type is not one the kernels read (the caller has another way).
// Dense tensors are read, and scaled, where they lie, whatever the order of their axes; the others through a copy.
c10::optional<at::Tensor> grad_clip(const pybind11::list& items, bool inf_norm, bool scale, double max_norm, double eps) {
  TORCH_CHECK_VALUE(!items.empty(), "no gradients");
  std::vector<std::reference_wrapper<const at::Tensor>> grads;  // the list holds them for the length of the call
  grads.reserve(items.size());
  for (const pybind11::handle& item : items) {
    TORCH_CHECK_TYPE(THPVariable_Check(item.ptr()), "gradients must be tensors");
    grads.emplace_back(THPVariable_Unpack(item.ptr()));
  }
  const at::Device device = grads[0].get().device();
  std::vector<olb_clip_tensor> list;
  list.reserve(grads.size());
  std::vector<std::pair<at::Tensor, at::Tensor>> copies;   // a tensor that is not dense, and its copy
  for (const at::Tensor& g : grads) {
    TORCH_CHECK_VALUE(g.device() == device, "the gradients are on different devices");
    TORCH_CHECK_VALUE(g.layout() == at::kStrided, "sparse gradients are not supported");
    if (!g.is_cuda() || (g.scalar_type() != at::kBFloat16 && g.scalar_type() != at::kFloat) || g.is_conj() || g.is_neg()) return c10::nullopt;
  }
  for (const at::Tensor& g : grads)
    TORCH_CHECK_NOT_IMPLEMENTED(!g._fw_grad(0).defined(), "gradients that are forward-mode duals are not supported");
  c10::cuda::CUDAGuard guard(device);
  for (const at::Tensor& g : grads) {
    if (g.numel() == 0) continue;
    const at::Tensor* dense = &g;
    if (!g.is_non_overlapping_and_dense()) {
      TORCH_CHECK_VALUE(!scale || no_self_overlap(g), "a gradient to be scaled addresses an element more than once");
      copies.emplace_back(g, g.contiguous());
      dense = &copies.back().second;
    }
    list.push_back({dense->data_ptr(), dense->numel(), dense->scalar_type() == at::kFloat});
  }
  if (scale) {
    // the same memory twice would be scaled by two blocks at once (a copy is not: whatever it shares holds the same values)
    std::vector<std::pair<const char*, const char*>> spans;
    spans.reserve(list.size());
    for (const olb_clip_tensor& x : list) {
      const char* p = static_cast<const char*>(x.ptr);
      spans.emplace_back(p, p + x.n * (x.fp32 ? 4 : 2));
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      TORCH_CHECK_VALUE(spans[i].first >= spans[i - 1].second, "gradients to be scaled share memory");
  }
  const int n = static_cast<int>(list.size());
  const int room = olb_grad_clip_parts(list.data(), n);
  at::Tensor partial = at::empty({room}, at::TensorOptions().dtype(at::kDouble).device(device));
  at::Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device));
  const int rc = olb_grad_clip(list.data(), n, inf_norm, scale, static_cast<float>(max_norm), static_cast<float>(eps),
                               partial.data_ptr<double>(), room, norm.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, "olb_grad_clip failed with code " + std::to_string(rc));
  if (scale) {
    at::NoGradGuard no_grad;
    for (auto& [g, copy] : copies) g.copy_(copy);
    for (const at::Tensor& g : grads)
      if (g.numel() && !g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
  }
  return norm;
}

}  // namespace

void register_grad_clip(pybind11::module& m) { m.def("grad_clip", &grad_clip); }
