// Host side of the operators of the linear-attention core and of its
// matrices' updates: argument checks that keep the kernels in bounds, output
// and workspace tensors (torch's allocator, so a captured graph owns its
// own), launches on the current stream of the operands' device.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <hip/hip_runtime.h>

#include <vector>

#include "core_ops.h"

extern "C" {
long layer_norm_part_elems(int, long, long, int);
int layer_norm_aligned(int, const void*, const void*, long, const void*,
                       const void*, long);
void launch_layer_norm_fwd(int, int, const void*, long, const void*,
                           const void*, void*, float*, float*, long, long,
                           float, hipStream_t);
void launch_layer_norm_bwd(int, int, int, const void*, const void*, long,
                           const void*, const float*, const float*, void*,
                           float*, void*, void*, long, long, hipStream_t);
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

hipStream_t stream_here() {
  return c10::hip::getCurrentHIPStream().stream();
}

int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kFloat16: return 2;
    default:
      TORCH_CHECK(false, name, " must be fp32, bf16 or fp16");
  }
}

const void* ptr(const OptTensor& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

// ---------------------------------------------------------------------------
// layer norm. x (rows, cols) with unit column stride; the row stride is free
// ---------------------------------------------------------------------------
void check_norm_operands(const Tensor& x, const OptTensor& w,
                         const OptTensor& b) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) > 0 &&
                  (x.stride(1) == 1 || x.size(1) == 1) && x.stride(0) >= 0,
              "layer_norm: x must be a GPU matrix with unit column stride");
  for (const auto* p : {&w, &b}) {
    if (!p->has_value()) continue;
    const Tensor& t = **p;
    TORCH_CHECK(t.device() == x.device() && t.dim() == 1 &&
                    t.size(0) == x.size(1) && t.is_contiguous(),
                "layer_norm: weight and bias must be (cols,) on x's device");
    TORCH_CHECK(t.scalar_type() == torch::kFloat32 ||
                    t.scalar_type() == x.scalar_type(),
                "layer_norm: weight and bias must be fp32 or of x's type");
  }
  TORCH_CHECK(!w.has_value() || !b.has_value() ||
                  w->scalar_type() == b->scalar_type(),
              "layer_norm: weight and bias must have one type");
}

std::vector<Tensor> layer_norm_fwd(Tensor x, OptTensor w, OptTensor b,
                                   double eps, bool save) {
  check_norm_operands(x, w, b);
  const int xt = type_code(x, "x");
  const int wt = w.has_value() ? type_code(*w, "weight")
                 : b.has_value() ? type_code(*b, "bias") : xt;
  const long rows = x.size(0), cols = x.size(1);
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty({rows, cols}, x.options());
  auto fopts = x.options().dtype(torch::kFloat32);
  auto stats = torch::empty({2, save ? rows : 0}, fopts);
  if (rows > 0) {
    float* mean = save ? stats.data_ptr<float>() : nullptr;
    launch_layer_norm_fwd(xt, wt, x.data_ptr(), x.stride(0), ptr(w), ptr(b),
                          y.data_ptr(), mean, save ? mean + rows : nullptr,
                          rows, cols, (float)eps, stream_here());
    check_launch("layer_norm");
  }
  return {y, stats};
}

std::vector<OptTensor> layer_norm_bwd(Tensor dy, Tensor x, OptTensor w,
                                      Tensor stats, bool need_dx,
                                      bool need_dw, bool need_db,
                                      bool param_fp32) {
  check_norm_operands(x, w, c10::nullopt);
  const long rows = x.size(0), cols = x.size(1);
  TORCH_CHECK(dy.device() == x.device() && dy.sizes() == x.sizes() &&
                  dy.scalar_type() == x.scalar_type() && dy.is_contiguous(),
              "layer_norm: the output's gradient must match the output");
  TORCH_CHECK(stats.device() == x.device() && stats.is_contiguous() &&
                  stats.scalar_type() == torch::kFloat32 &&
                  stats.numel() == 2 * rows,
              "layer_norm: saved statistics do not match x");
  const int xt = type_code(x, "x");
  const int wt = w.has_value() ? type_code(*w, "weight")
                 : param_fp32 ? 0 : xt;
  const c10::DeviceGuard guard(x.device());
  auto popts = x.options();
  if (wt == 0) popts = popts.dtype(torch::kFloat32);
  OptTensor dx, dw, db;
  if (need_dx) dx = torch::empty({rows, cols}, x.options());
  if (rows == 0) {
    if (need_dw) dw = torch::zeros({cols}, popts);
    if (need_db) db = torch::zeros({cols}, popts);
    return {dx, dw, db};
  }
  if (need_dw) dw = torch::empty({cols}, popts);
  if (need_db) db = torch::empty({cols}, popts);
  const int al = layer_norm_aligned(xt, dy.data_ptr(), x.data_ptr(),
                                    x.stride(0), ptr(w), ptr(dx), cols);
  Tensor part;
  if (need_dw || need_db)
    part = torch::empty({layer_norm_part_elems(xt, rows, cols, al)},
                        x.options().dtype(torch::kFloat32));
  launch_layer_norm_bwd(
      xt, wt, al, dy.data_ptr(), x.data_ptr(), x.stride(0), ptr(w),
      stats.data_ptr<float>(), stats.data_ptr<float>() + rows,
      const_cast<void*>(ptr(dx)),
      part.defined() ? part.data_ptr<float>() : nullptr,
      const_cast<void*>(ptr(dw)), const_cast<void*>(ptr(db)), rows, cols,
      stream_here());
  check_launch("layer_norm backward");
  return {dx, dw, db};
}

}  // namespace

void register_core_ops(pybind11::module_& m) {
  m.def("layer_norm_fwd", &layer_norm_fwd, py::arg("x"),
        py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5, py::arg("save") = false);
  m.def("layer_norm_bwd", &layer_norm_bwd, py::arg("dy"), py::arg("x"),
        py::arg("weight"), py::arg("stats"), py::arg("need_dx"),
        py::arg("need_dw"), py::arg("need_db"), py::arg("param_fp32"));
}
