// ATen-level wrapper of the gradient-list kernels (grad_norm.cu): the norm of
// a list of tensors and clipping by it.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>

#include "dlvk/aten_ops.h"
#include "dlvk/kernels.h"
#include "dlvk/overlap.h"

namespace dlvk {
namespace aten {
namespace {

// Each written tensor must share no byte with another one of the call, written
// or (`read`: the inputs that are not their own outputs) read.
void check_disjoint(std::vector<Extent>& written, const std::vector<Extent>& read, const char* what) {
  if (written.empty()) return;
  const auto apart = [&](const Extent& a, const Extent& b) {
    TORCH_CHECK(!share_bytes(a, b), "dlvk.", what, ": tensors ", std::min(a.index, b.index), " and ",
                std::max(a.index, b.index), " of the call share memory, which is written");
  };
  const auto before = [](const Extent& a, const Extent& b) { return a.lo < b.lo; };
  if (!std::is_sorted(written.begin(), written.end(), before)) std::sort(written.begin(), written.end(), before);
  std::vector<uintptr_t> reach(written.size());  // the highest end so far
  uintptr_t end = 0;
  for (size_t i = 0; i < written.size(); ++i) {
    // usually nothing overlaps even as ranges
    for (size_t k = i; k > 0 && reach[k - 1] > written[i].lo; --k) apart(written[k - 1], written[i]);
    end = std::max(end, written[i].hi);
    reach[i] = end;
  }
  for (const Extent& r : read) {
    if (r.hi <= written[0].lo || r.lo >= end) continue;
    size_t k = std::lower_bound(written.begin(), written.end(), r.hi,
                                [](const Extent& w, uintptr_t v) { return w.lo < v; }) - written.begin();
    for (; k > 0 && reach[k - 1] > r.lo; --k) apart(written[k - 1], r);
  }
}

bool dense_alike(const at::Tensor& a, const at::Tensor& b) {
  if (a.is_contiguous() && b.is_contiguous()) return true;
  return a.is_non_overlapping_and_dense() && a.strides() == b.strides();
}

StridedItem strided_item(const at::Tensor& in, const at::Tensor& out, uint8_t kind, const char* what) {
  StridedItem s{};
  s.in = in.data_ptr();
  s.out = out.data_ptr();
  s.n = in.numel();
  s.kind = kind;
  int64_t size[4], si[4], so[4];
  int nd = 0;
  for (int64_t d = 0; d < in.dim(); ++d) {
    if (in.size(d) == 1) continue;
    if (nd > 0 && si[nd - 1] == in.stride(d) * in.size(d) && so[nd - 1] == out.stride(d) * out.size(d)) {
      size[nd - 1] *= in.size(d);  // continues the dimension before it
      si[nd - 1] = in.stride(d);
      so[nd - 1] = out.stride(d);
      continue;
    }
    TORCH_CHECK(nd < 4, "dlvk.", what, ": a tensor with more than four separate strides; pass a contiguous one");
    size[nd] = in.size(d);
    si[nd] = in.stride(d);
    so[nd] = out.stride(d);
    ++nd;
  }
  for (int d = 0; d < 4; ++d) s.size[d] = 1;
  for (int d = 0; d < nd; ++d) {
    s.size[4 - nd + d] = size[d];
    s.in_stride[4 - nd + d] = si[d];
    s.out_stride[4 - nd + d] = so[d];
  }
  return s;
}

at::Tensor run(const TensorRefs& grads, const TensorRefs* outs, bool scale, double max_norm, const char* what) {
  TORCH_CHECK(!grads.empty(), "dlvk.", what, ": an empty list has no device; the norm of no tensors is 0");
  TORCH_CHECK(outs == nullptr || outs->size() == grads.size(), "dlvk.", what, ": ", grads.size(), " gradients and ",
              outs ? outs->size() : 0, " outputs");
  check_cuda(*grads[0], "gradients");
  const at::Device dev = grads[0]->device();
  std::vector<DenseItem> dense;
  std::vector<StridedItem> strided;
  std::vector<Extent> written, read;
  dense.reserve(grads.size());
  if (scale) written.reserve(grads.size());
  if (scale && outs) read.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const at::Tensor& t = *grads[i];
    const at::Tensor& o = outs ? *(*outs)[i] : t;
    TORCH_CHECK(t.device() == dev && o.device() == dev, "dlvk.", what, ": tensor ", i, " is on another device than ",
                dev);
    const auto ti = t.scalar_type(), to = o.scalar_type();
    TORCH_CHECK((ti == at::kFloat || ti == at::kBFloat16) && (to == at::kFloat || to == at::kBFloat16), "dlvk.", what,
                ": tensor ", i, " is neither fp32 nor bf16");
    TORCH_CHECK(t.layout() == at::kStrided && o.layout() == at::kStrided, "dlvk.", what, ": tensor ", i,
                " is not strided");
    if (outs)
      TORCH_CHECK(t.sizes() == o.sizes(), "dlvk.", what, ": gradient ", i, " is ", t.sizes(), ", its output ",
                  o.sizes());
    if (t.numel() == 0) continue;
    const bool same = t.data_ptr() == o.data_ptr();
    if (outs && same)
      TORCH_CHECK(ti == to && t.strides() == o.strides(), "dlvk.", what, ": output ", i,
                  " starts where its gradient does but is laid out otherwise");
    const uint8_t kind = (uint8_t)((ti == at::kBFloat16 ? 1 : 0) | (to == at::kBFloat16 ? 2 : 0));
    if (dense_alike(t, o)) dense.push_back({t.data_ptr(), o.data_ptr(), t.numel(), kind});
    else strided.push_back(strided_item(t, o, kind, what));
    if (scale) {
      TORCH_CHECK(o.is_contiguous() || !may_repeat(o), "dlvk.", what, ": output ", i,
                  " repeats its elements, or may (an expanded or unfolded tensor)");
      written.push_back(extent_of(o, (int64_t)i));
      if (!same) read.push_back(extent_of(t, (int64_t)i));
    }
  }
  if (scale) check_disjoint(written, read, what);
  c10::cuda::CUDAGuard g(dev);
  const PdlScope pdl;
  at::AutoDispatchBelowADInplaceOrView below;
  auto opt = grads[0]->options();
  at::Tensor norm = at::empty({}, opt.dtype(at::kFloat));
  const int parts = grad_norm_parts(dense.data(), (int)dense.size(), strided.data(), (int)strided.size());
  at::Tensor partial = at::empty({std::max(parts, 1)}, opt.dtype(at::kDouble));
  grad_norm(dense.data(), (int)dense.size(), strided.data(), (int)strided.size(), scale, (float)max_norm,
            norm.data_ptr<float>(), partial.data_ptr<double>(), stream());
  return norm;
}

}  // namespace

at::Tensor global_norm_op(const TensorRefs& grads) { return run(grads, nullptr, false, 0.0, "global_norm"); }

at::Tensor clip_global_norm_op(const TensorRefs& grads, double max_norm, const TensorRefs* out) {
  TORCH_CHECK(max_norm > 0.0, "dlvk.clip_global_norm: max_norm must be above 0, got ", max_norm);
  return run(grads, out, true, max_norm, "clip_global_norm");
}

}  // namespace aten
}  // namespace dlvk
