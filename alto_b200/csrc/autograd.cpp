// Autograd function of the RMS norm, compiled against torch: allocation, stream, device and graph in C++ around the C ABI's
// two entry points.
//
// A step of a few thousand rows takes 6 to 20 us of kernels; as a Python function each way it took the host 93 us (forward 27,
// and behind each of autograd's two changes of thread a cold interpreter: 21 for a backward pass that takes 15 when warm),
// more than a string of tensor operations that keeps no graph.  1023 x 1537 fp32: 65 us a step (98 before), tensor operations
// 84 to 86; 8192 x 4096 bf16 with residual 90 us (117 before) for 88 of kernels.
//
// The library stays free of torch: its entry points come as addresses from the handle that alto_b200/_lib.py holds.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>

#include "altob200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

struct Entries {
  decltype(&altob200_rms_norm_forward) forward;
  decltype(&altob200_rms_norm_backward_work_bytes) work_bytes;
  decltype(&altob200_rms_norm_backward) backward;
} entry = {};

// The package's own error, as a refused call of the other operators raises it.
void check(int status, const char* where) {
  if (status == ALTOB200_OK) return;
  pybind11::gil_scoped_acquire gil;
  const auto error = pybind11::module_::import("alto_b200._lib").attr("Altob200Error");
  PyErr_SetObject(error.ptr(), error(status, where).ptr());
  throw pybind11::error_already_set();
}

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? ALTOB200_DT_BF16 : ALTOB200_DT_F32; }

// Rows whose elements are neighbours and that do not overlap: the tensor's own, or a copy's.
struct Rows {
  Tensor hold;
  int64_t ld;
  Rows(const Tensor& t, int64_t cols) : hold(t), ld(cols) {
    if (t.is_contiguous()) return;      // of one row or column too, whose strides say nothing
    if (t.dim() != 2) hold = t.reshape({-1, cols});
    if (hold.is_contiguous()) return;
    if (hold.stride(1) == 1 && hold.stride(0) >= cols) ld = hold.stride(0);
    else hold = hold.contiguous();
  }
  void* p() const { return hold.data_ptr(); }
};

class Norm : public torch::autograd::Function<Norm> {
 public:
  static variable_list forward(AutogradContext* ctx, const Variable& x, const Variable& weight, const std::optional<Tensor>& residual,
                               double eps) {
    const c10::cuda::CUDAGuard device(x.device());
    const int64_t cols = x.size(-1);
    const Rows in(x, cols);
    const Tensor w = weight.contiguous();
    // in the shape of x, not views of rows: the caller may write to them
    const Tensor out = at::empty(x.sizes(), x.options());
    altob200_rms_norm_args a = {};
    a.rows = x.numel() / cols;
    a.cols = cols;
    a.ld_x = in.ld;
    a.x = in.p();
    a.weight = w.data_ptr();
    a.out = out.data_ptr();
    a.eps = (float)eps;
    a.dtype = dtype_of(x);
    a.weight_dtype = dtype_of(weight);
    a.format = -1;
    Tensor stream;
    std::optional<Rows> added;
    if (residual.has_value()) {
      added.emplace(*residual, cols);
      stream = at::empty(x.sizes(), x.options());
      a.ld_residual = added->ld;
      a.residual = added->p();
      a.stream_out = stream.data_ptr();
    }
    check(entry.forward(&a, c10::cuda::getCurrentCUDAStream().stream()), "altob200_rms_norm_forward");
    ctx->set_materialize_grads(false);
    ctx->saved_data["eps"] = eps;
    ctx->save_for_backward({stream.defined() ? stream : x, weight});
    if (!stream.defined()) return {out};
    return {out, stream};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &stream = saved[0], &weight = saved[1], &grad = grads[0];
    const bool residual = grads.size() > 1, need_weight = ctx->needs_input_grad(1);
    const Tensor grad_stream = residual ? grads[1] : Tensor();
    Tensor grad_rows, grad_weight;
    if (!grad.defined()) {      // only the stream was used
      grad_rows = grad_stream;
      if (need_weight) grad_weight = at::zeros_like(weight);
    } else {
      const bool graph = at::GradMode::is_enabled();
      const at::AutoGradMode no_graph(false);
      const c10::cuda::CUDAGuard device(stream.device());
      const int64_t cols = stream.size(-1);
      const Rows r(stream, cols), g(grad, cols);
      const Tensor w = weight.contiguous();
      grad_rows = at::empty(stream.sizes(), stream.options());
      altob200_rms_norm_grad_args a = {};
      a.rows = stream.numel() / cols;
      a.cols = cols;
      a.ld_grad = g.ld;
      a.ld_stream = r.ld;
      a.grad_out = g.p();
      a.stream = r.p();
      a.weight = w.data_ptr();
      a.grad_in = grad_rows.data_ptr();
      a.eps = (float)ctx->saved_data["eps"].toDouble();
      a.dtype = dtype_of(stream);
      a.weight_dtype = dtype_of(weight);
      std::optional<Rows> ds;
      if (grad_stream.defined()) {
        ds.emplace(grad_stream, cols);
        a.ld_grad_stream = ds->ld;
        a.grad_stream = ds->p();
      }
      Tensor work;
      if (need_weight) {
        grad_weight = at::empty(weight.sizes(), weight.options());
        a.grad_weight = grad_weight.data_ptr();
        if (a.rows > 0) work = at::empty({entry.work_bytes(&a)}, stream.options().dtype(at::kByte));
      }
      check(entry.backward(&a, work.defined() ? work.data_ptr() : nullptr, c10::cuda::getCurrentCUDAStream().stream()),
            "altob200_rms_norm_backward");
      if (graph) {      // a second derivative is refused when it is asked for
        variable_list first;
        for (const Tensor* t : {&grad_rows, &grad_weight})
          if (t->defined()) first.push_back(t->detach().requires_grad_(true));
        const auto refuse = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate the gradient of rms_norm, which has none", (int64_t)first.size());
        const at::AutoGradMode again(true);
        first = (*refuse)(std::move(first));
        grad_rows = first[0];
        if (need_weight) grad_weight = first[1];
      }
    }
    return {grad_rows, grad_weight, residual ? grad_rows : Tensor(), Tensor()};
  }
};

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.def("bind", [](uintptr_t forward, uintptr_t work_bytes, uintptr_t backward) {
    entry = {reinterpret_cast<decltype(entry.forward)>(forward), reinterpret_cast<decltype(entry.work_bytes)>(work_bytes),
             reinterpret_cast<decltype(entry.backward)>(backward)};
  });
  // operands as alto_b200/norm.py has checked them
  m.def("rms_norm", [](const Tensor& x, const Tensor& weight, double eps) { return Norm::apply(x, weight, std::optional<Tensor>(), eps)[0]; },
        pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("rms_norm_residual",
        [](const Tensor& x, const Tensor& weight, const Tensor& residual, double eps) {
          const auto both = Norm::apply(x, weight, std::optional<Tensor>(residual), eps);
          return std::make_tuple(both[0], both[1]);
        },
        pybind11::call_guard<pybind11::gil_scoped_release>());
}
