// Autograd functions of the RMS norm and of the FP8 block linears, serving by their codes, and the walk over lists of gradients,
// compiled against torch: allocation, stream, device and graph in C++ around the C ABI's entry points.
//
// A step of a few thousand rows takes 6 to 20 us of kernels; as a Python function each way it took the host 93 us (forward 27,
// and behind each of autograd's two changes of thread a cold interpreter: 21 for a backward pass that takes 15 when warm),
// more than a string of tensor operations that keeps no graph.  1023 x 1537 fp32: 65 us a step (98 before), tensor operations
// 84 to 86; 8192 x 4096 bf16 with residual 90 us (117 before) for 88 of kernels.  A step of an FP8 block linear, 513 x 768 x 1040 fp32:
// 208 us as a Python function, 95 here (47 as a captured graph; a step of one elementwise product takes 57); 24 tokens past a
// 4096 x 4096 weight 12.3 us with the operands looked at in Python, 9.8 here.
//
// The library stays free of torch: its entry points come as addresses from the handle that alto_b200/_lib.py holds.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <initializer_list>
#include <memory>
#include <optional>
#include <string>
#include <utility>
#include <vector>

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
  decltype(&altob200_grad_norm_work_bytes) norm_work_bytes;
  decltype(&altob200_grad_norm) grad_norm;
  decltype(&altob200_clip_grads) clip_grads;
  decltype(&altob200_fp8_block_quantize) fp8_quantize;
  decltype(&altob200_fp8_block_quantize_squares) fp8_squares;
  decltype(&altob200_fp8_block_gemm) fp8_gemm;
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

// Gradients in a graph of their own: a second derivative is refused when it is asked for.
void refuse_second(std::initializer_list<Tensor*> grads, const char* of) {
  variable_list first;
  for (const Tensor* t : grads)
    if (t->defined()) first.push_back(t->detach().requires_grad_(true));
  if (first.empty()) return;
  const auto refuse = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate the gradient of ") + of + ", which has none", (int64_t)first.size());
  const at::AutoGradMode again(true);
  first = (*refuse)(std::move(first));
  size_t i = 0;
  for (Tensor* t : grads)
    if (t->defined()) *t = first[i++];
}

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
      if (graph) refuse_second({&grad_rows, &grad_weight}, "rms_norm");
    }
    return {grad_rows, grad_weight, residual ? grad_rows : Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------------------
// FP8 with one fp32 scale for each block of 128 (alto_b200/fp8_block.py has the checks and the words)
// ---------------------------------------------------------------------------------------
void* stream_here() { return c10::cuda::getCurrentCUDAStream().stream(); }
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// [rows, cols] with neighbouring columns, rows that do not overlap and begin on 16 bytes: the tensor's own, or a copy's.
Tensor fp8_rows(const Tensor& t) {
  Tensor x = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  const bool at16 = reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0;
  if (x.stride(1) == 1 && at16 && (x.size(0) <= 1 || (x.stride(0) >= x.size(1) && x.stride(0) * x.element_size() % 16 == 0))) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}
Tensor fp8_packed(const Tensor& t) {
  if (!t.is_contiguous()) return t.contiguous();
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 ? t : t.clone();
}
struct Coded {
  Tensor codes, scales;
  bool there() const { return codes.defined(); }
};
altob200_fp8_block_scale by_row(const Tensor& s) { return {(const float*)s.const_data_ptr(), 1, s.stride(0), 0, 0, 7}; }
altob200_fp8_block_scale by_square(const Tensor& s, bool transposed) {
  const int64_t r = s.stride(1), c = s.stride(2);
  return {(const float*)s.const_data_ptr(), transposed ? c : r, transposed ? r : c, s.stride(0), 7, 7};
}
// x2 in blocks of its rows and / or of its columns (of 128 rows from every expert's first).
void fp8_quantize(const Tensor& x2, int32_t fmt, const Tensor& offs, Coded* rows, Coded* cols) {
  const int64_t R = x2.size(0), C = x2.size(1);
  const auto bytes = x2.options().dtype(at::kByte), floats = x2.options().dtype(at::kFloat);
  altob200_fp8_block_quant_args a = {};
  a.x = x2.const_data_ptr();
  a.rows = R;
  a.cols = C;
  a.ld = R > 1 ? x2.stride(0) : C;
  if (offs.defined()) {
    a.offs = (const int32_t*)offs.const_data_ptr();
    a.experts = (int32_t)offs.numel();
  }
  if (rows != nullptr) {
    *rows = {at::empty({R, C}, bytes), at::empty({blocks_of(C), R}, floats)};
    a.row_codes = rows->codes.data_ptr();
    a.row_scales = (float*)rows->scales.data_ptr();
  }
  if (cols != nullptr) {
    const int64_t blocks = offs.defined() ? R / 128 + offs.numel() : blocks_of(R);
    *cols = {at::empty({C, blocks * 128}, bytes), at::empty({blocks, C}, floats)};
    a.col_codes = cols->codes.data_ptr();
    a.col_scales = (float*)cols->scales.data_ptr();
    a.ld_col = blocks * 128;
  }
  a.dtype = dtype_of(x2);
  a.format = fmt;
  if (R > 0 && (rows != nullptr || cols != nullptr)) check(entry.fp8_quantize(&a, stream_here()), "altob200_fp8_block_quantize");
}
// D = A B^T; sa without scales: a is numbers.
void fp8_gemm(const Tensor& a, const altob200_fp8_block_scale& sa, const Tensor& b, const altob200_fp8_block_scale& sb, const Tensor& out,
              int32_t fmt, int64_t M, int64_t N, int64_t K, int32_t mode, const Tensor& offs, int64_t k_rows, bool b_ready = false) {
  altob200_fp8_block_gemm_args g = {};
  g.M = M;
  g.N = N;
  g.K = K;
  g.lda = M > 1 ? a.stride(0) : K;
  g.ldd = N;
  g.k_rows = k_rows;
  g.a = a.const_data_ptr();
  g.b = b.const_data_ptr();
  g.sa = sa;
  g.sb = sb;
  if (offs.defined()) {
    g.offs = (const int32_t*)offs.const_data_ptr();
    g.experts = (int32_t)offs.numel();
  }
  g.d = out.data_ptr();
  g.mode = mode;
  g.format = fmt;
  g.a_dtype = sa.scales == nullptr ? dtype_of(a) : -1;
  g.out_dtype = dtype_of(out);
  g.b_ready = b_ready;
  check(entry.fp8_gemm(&g, stream_here()), "altob200_fp8_block_gemm");
}

// The linear, dense (weight [N, K]) or by expert (weight [E, K, N], ends of the experts' rows).  `weight` is what the graph
// knows (a wrapper, too), `data` its numbers.
class Fp8Linear : public torch::autograd::Function<Fp8Linear> {
 public:
  static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& weight, const Tensor& data, const std::optional<Tensor>& ends,
                          int64_t fmt64, bool need_x, bool need_w) {
    const c10::cuda::CUDAGuard device(x.device());
    const int32_t fmt = (int32_t)fmt64;
    const Tensor offs = ends.value_or(Tensor());
    const bool grouped = offs.defined();
    const Tensor x2 = fp8_rows(x.detach());
    Tensor w = data;
    // matrices as they lie in memory, [rows, cols]: of the weight N x K, or K x N
    bool kn = false;
    if (grouped) {
      kn = w.stride(2) == 1 || w.stride(1) != 1;
      w = fp8_packed(kn ? w : w.transpose(1, 2));
    } else {
      w = fp8_rows(w).unsqueeze(0);
    }
    const int64_t E = w.size(0), R = w.size(1), C = w.size(2), N = kn ? C : R, K = kn ? R : C, M = x2.size(0);
    const auto bytes = w.options().dtype(at::kByte);
    const bool need_plain = !kn || need_x, need_t = kn || need_x;
    const Tensor plain = need_plain ? at::empty({E, R, C}, bytes) : Tensor(), turned = need_t ? at::empty({E, C, R}, bytes) : Tensor();
    const Tensor scales = at::empty({E, blocks_of(R), blocks_of(C)}, w.options().dtype(at::kFloat));
    check(entry.fp8_squares(w.const_data_ptr(), dtype_of(w), fmt, E, R, C, w.stride(1), w.stride(0), need_plain ? plain.data_ptr() : nullptr,
                            need_t ? turned.data_ptr() : nullptr, (float*)scales.data_ptr(), stream_here()), "altob200_fp8_block_quantize_squares");
    Coded rows, cols;
    fp8_quantize(x2, fmt, offs, &rows, need_w ? &cols : nullptr);
    auto shape = x.sizes().vec();
    shape.back() = N;
    const Tensor out = at::empty(shape, x.options());
    fp8_gemm(rows.codes, by_row(rows.scales), kn ? turned : plain, by_square(scales, kn), out, fmt, M, N, K, grouped ? 1 : 0, offs, 0);
    ctx->save_for_backward({cols.codes, cols.scales, need_x ? (kn ? plain : turned) : Tensor(), need_x ? scales : Tensor(), offs});
    ctx->saved_data["dims"] = std::vector<int64_t>{M, K, N, fmt64, kn ? 1 : 0};
    ctx->saved_data["shape"] = x.sizes().vec();
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto dims = ctx->saved_data["dims"].toIntVector();
    const int64_t M = dims[0], K = dims[1], N = dims[2];
    const int32_t fmt = (int32_t)dims[3];
    const Tensor &grad = grads[0], &offs = saved[4];
    const bool graph = at::GradMode::is_enabled(), need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), grouped = offs.defined();
    Tensor dx, dw;
    {
      const at::AutoGradMode no_graph(false);
      const c10::cuda::CUDAGuard device(grad.device());
      const Tensor g2 = fp8_rows(grad);
      Coded rows, cols;
      if (need_x || need_w) fp8_quantize(g2, fmt, offs, need_x ? &rows : nullptr, need_w ? &cols : nullptr);
      if (need_x) {
        dx = at::empty(ctx->saved_data["shape"].toIntVector(), grad.options());
        fp8_gemm(rows.codes, by_row(rows.scales), saved[2], by_square(saved[3], dims[4] == 0), dx, fmt, M, K, N, grouped ? 1 : 0, offs, 0);
      }
      if (need_w && grouped) {
        dw = at::empty({offs.numel(), K, N}, grad.options());
        fp8_gemm(saved[0], by_row(saved[1]), cols.codes, by_row(cols.scales), dw, fmt, K, N, cols.codes.size(1), 2, offs, M);
      } else if (need_w) {
        dw = M > 0 ? at::empty({N, K}, grad.options()) : at::zeros({N, K}, grad.options());
        if (M > 0) fp8_gemm(cols.codes, by_row(cols.scales), saved[0], by_row(saved[1]), dw, fmt, N, K, cols.codes.size(1), 0, Tensor(), 0);
      }
    }
    if (graph) refuse_second({&dx, &dw}, "a linear in FP8 blocks");
    return {dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// x times codes of weights [E or 1, N, K]; few rows an expert are quantised by the product itself.
Tensor fp8_serve(const Tensor& x, const Tensor& w_codes, const Tensor& w_scales, const std::optional<Tensor>& ends, int64_t fmt) {
  const at::AutoGradMode no_graph(false);
  const c10::cuda::CUDAGuard device(x.device());
  const int64_t N = w_codes.size(-2), K = w_codes.size(-1);
  auto shape = x.sizes().vec();
  shape.back() = N;
  const Tensor out = at::empty(shape, x.options()), x2 = fp8_rows(x), w = fp8_packed(w_codes), offs = ends.value_or(Tensor());
  const Tensor s = w_scales.dim() == 3 ? w_scales : w_scales.unsqueeze(0);
  const int64_t M = x2.size(0);
  const int32_t mode = offs.defined() ? 1 : 0;
  // Up to eight rows go to a product that quantises them itself, each of its blocks all of a row's numbers, where a launch in front
  // is longer than that: N x K 512 x 512 in 1.9 us against 3.4, 4096 x 4096 6.7 against 7.9, 14336 x 4096 16.1 against 16.4, eight
  // experts of 4096 x 1024 12.5 against 15.0, but 2048 x 8192 9.9 against 8.9, 8192 x 8192 21.7 against 16.5, 28672 x 4096 28.6
  // against 26.8, eight experts of 4096 x 4096 31.2 against 29.8.
  const int64_t read = (offs.defined() ? std::min(M, offs.numel()) : 1) * N * K;
  if (M <= 8 && K <= 6144 && read <= (int64_t)1 << 26) {
    fp8_gemm(x2, altob200_fp8_block_scale{}, w, by_square(s, false), out, (int32_t)fmt, M, N, K, mode, offs, 0);
  } else {
    Coded rows;
    fp8_quantize(x2, (int32_t)fmt, Tensor(), &rows, nullptr);
    fp8_gemm(rows.codes, by_row(rows.scales), w, by_square(s, false), out, (int32_t)fmt, M, N, K, mode, offs, 0, true);
  }
  return out;
}

// The operands of the linears, looked at here: a few attributes of Python's cost as much as a small product takes.  False: what
// alto_b200/fp8_block.py has to look at, to say what is wrong or to take a wrapper's data.
bool fp8_number(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has(c10::DispatchKey::Python) &&
         (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat);
}
bool fp8_ends(const std::optional<Tensor>& offs, const Tensor& x, int64_t experts) {
  return offs.has_value() && offs->scalar_type() == at::kInt && offs->device() == x.device() && offs->dim() == 1 && offs->size(0) == experts &&
         offs->is_contiguous() && experts > 0;
}
std::optional<Tensor> fp8_try_serve(const Tensor& x, const Tensor& w_codes, const Tensor& w_scales, const std::optional<Tensor>& offs) {
  const int64_t dims = offs.has_value() ? 3 : 2;
  if (!fp8_number(x) || x.dim() < 1 || (dims == 3 && x.dim() != 2) || (at::GradMode::is_enabled() && (x.requires_grad() || w_scales.requires_grad())))
    return std::nullopt;
  const bool e4 = w_codes.scalar_type() == at::kFloat8_e4m3fn;
  if ((!e4 && w_codes.scalar_type() != at::kFloat8_e5m2) || w_codes.dim() != dims || w_codes.device() != x.device()) return std::nullopt;
  const int64_t N = w_codes.size(-2), K = w_codes.size(-1);
  if (N <= 0 || K <= 0 || N % 16 != 0 || K % 16 != 0 || x.size(-1) != K) return std::nullopt;
  if (w_scales.scalar_type() != at::kFloat || w_scales.dim() != dims || w_scales.device() != x.device() || w_scales.size(-2) != blocks_of(N) ||
      w_scales.size(-1) != blocks_of(K))
    return std::nullopt;
  if (dims == 3 && (w_scales.size(0) != w_codes.size(0) || !fp8_ends(offs, x, w_codes.size(0)))) return std::nullopt;
  const pybind11::gil_scoped_release no_gil;
  return fp8_serve(x, w_codes, w_scales, offs, e4 ? ALTOB200_FMT_MXFP8_E4M3 : ALTOB200_FMT_MXFP8_E5M2);
}
Tensor fp8_linear(const Tensor& x, const Tensor& weight, const Tensor& data, const std::optional<Tensor>& offs, int64_t fmt) {
  // (inside forward every input says what it said before, and the mode is off)
  const bool graph = at::GradMode::is_enabled();
  return Fp8Linear::apply(x, weight, data.detach(), offs, fmt, graph && x.requires_grad(), graph && weight.requires_grad());
}
std::optional<Tensor> fp8_try_linear(const Tensor& x, const Tensor& w, const std::optional<Tensor>& offs, int64_t fmt) {
  const int64_t dims = offs.has_value() ? 3 : 2;
  if (!fp8_number(x) || !fp8_number(w) || x.dim() < 1 || (dims == 3 && x.dim() != 2) || w.dim() != dims || w.scalar_type() != x.scalar_type() ||
      w.device() != x.device() || x.size(-1) != w.size(1))
    return std::nullopt;
  for (int64_t d = dims - 2; d < dims; ++d)
    if (w.size(d) <= 0 || w.size(d) % 16 != 0) return std::nullopt;
  if (dims == 3 && !fp8_ends(offs, x, w.size(0))) return std::nullopt;
  const pybind11::gil_scoped_release no_gil;
  return fp8_linear(x, w, w, offs, fmt);
}

// ---------------------------------------------------------------------------------------
// norm of many tensors and clipping by it (alto_b200/grad_clip.py)
// ---------------------------------------------------------------------------------------
// Where the first of the tensors is.
std::optional<c10::Device> on_device(const pybind11::list& l) {
  if (l.size() == 0 || !THPVariable_Check(PyList_GET_ITEM(l.ptr(), 0))) return std::nullopt;
  const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(l.ptr(), 0));
  return t.is_cuda() ? std::optional<c10::Device>(t.device()) : std::nullopt;
}

// Lists of tensors as the entry points take them.  A tensor whose elements are not neighbours in memory goes through a copy
// (and back, where it is written).  Thousands of tensors make up a call's host time, so the lists are walked once, without taking
// references.
struct GradList {
  std::unique_ptr<const void*[]> grads;
  std::unique_ptr<void*[]> outs;
  std::unique_ptr<int64_t[]> sizes;
  std::unique_ptr<int32_t[]> dtypes;
  std::vector<Tensor> hold;
  std::vector<std::pair<Tensor, Tensor>> back;      // (copy, where it belongs)
  std::unique_ptr<c10::TensorImpl*[]> written;
  std::vector<const void*> seen;                    // a table of the addresses that are written, at most half full
  Tensor first;
  altob200_grad_list list = {};

  size_t place(const void* p) const { return (reinterpret_cast<uintptr_t>(p) * 0x9E3779B97F4A7C15ull >> 20) & (seen.size() - 1); }
  // A tensor that is there twice would be scaled by two blocks at once: refused.
  void once(const void* p) {
    size_t at = place(p);
    while (seen[at] != nullptr) {
      if (seen[at] == p) throw pybind11::value_error("clip_grads expects tensors that do not overlap: one is in the list twice");
      at = (at + 1) & (seen.size() - 1);
    }
    seen[at] = p;
  }

  bool is_written(const void* p) const {
    size_t at = place(p);
    while (seen[at] != nullptr && seen[at] != p) at = (at + 1) & (seen.size() - 1);
    return seen[at] != nullptr;
  }

  // A gradient that another one is scaled into would be read while it is written.  False: it takes a look at each (lists that lie in
  // memory one behind the other, each type for itself, need none).
  bool apart(size_t n) const {
    uintptr_t low[4] = {UINTPTR_MAX, UINTPTR_MAX, UINTPTR_MAX, UINTPTR_MAX}, high[4] = {0, 0, 0, 0};      // read and written, of either type
    for (int type = 0; type < 2; ++type) {
      uintptr_t rl = UINTPTR_MAX, rh = 0, wl = UINTPTR_MAX, wh = 0;
      for (size_t i = 0; i < n; ++i) {
        if ((dtypes[i] == ALTOB200_DT_F32) != (type == 1)) continue;
        const uintptr_t r = reinterpret_cast<uintptr_t>(grads[i]), w = reinterpret_cast<uintptr_t>(outs[i]);
        rl = std::min(rl, r), rh = std::max(rh, r), wl = std::min(wl, w), wh = std::max(wh, w);
      }
      low[2 * type] = rl, high[2 * type] = rh, low[2 * type + 1] = wl, high[2 * type + 1] = wh;
    }
    for (int r = 0; r < 4; r += 2)
      for (int w = 1; w < 4; w += 2)
        if (low[r] <= high[w] && low[w] <= high[r]) return false;
    return true;
  }

  // The tensor of an object that the kernels can take, or null.  `keys`: those of the one before, which say the same of this one.
  static const Tensor* plain(PyObject* o, c10::DispatchKeySet& keys) {
    if (!THPVariable_Check(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    if (t.key_set() != keys) {
      if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.key_set().has(c10::DispatchKey::Python)) return nullptr;
      keys = t.key_set();
    }
    return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat ? &t : nullptr;
  }
  // False: a list that alto_b200/grad_clip.py has to look at.
  bool take(const pybind11::list& in, const pybind11::list& out, bool writes) {
    const size_t n = in.size();
    const bool others = out.size() != 0;
    if (n == 0 || (others && out.size() != n)) return false;
    grads.reset(new const void*[n]), sizes.reset(new int64_t[n]), dtypes.reset(new int32_t[n]);
    if (writes) {
      outs.reset(new void*[n]), written.reset(new c10::TensorImpl*[n]);
      size_t room = 16;
      while (room < 2 * n) room *= 2;
      seen.assign(room, nullptr);
    }
    PyObject *const *const items = PySequence_Fast_ITEMS(in.ptr()), *const *const others_items = PySequence_Fast_ITEMS(out.ptr());
    c10::Device device(c10::kCPU);
    c10::DispatchKeySet keys, out_keys;
    for (size_t i = 0; i < n; ++i) {
      const Tensor* g = plain(items[i], keys);
      if (g == nullptr) return false;
      if (i == 0) {
        first = *g;
        device = g->device();
      } else if (g->device() != device) {
        return false;
      }
      const Tensor* o = g;
      if (others) {
        o = plain(others_items[i], out_keys);
        if (o == nullptr || o->device() != device || o->scalar_type() != g->scalar_type() || o->sizes() != g->sizes()) return false;
      }
      sizes[i] = g->numel();
      dtypes[i] = dtype_of(*g);
      if (writes) {
        written[i] = o->unsafeGetTensorImpl();
        outs[i] = o->mutable_data_ptr();
        if (sizes[i] != 0) once(outs[i]);
      }
      if (g->is_contiguous() && o->is_contiguous()) {
        grads[i] = g->const_data_ptr();
        continue;
      }
      if (!g->is_non_overlapping_and_dense()) {
        hold.push_back(g->contiguous());
        grads[i] = hold.back().const_data_ptr();
      } else {
        grads[i] = g->const_data_ptr();
      }
      if (!writes || (g->is_non_overlapping_and_dense() && o->strides() == g->strides())) continue;
      at::assert_no_internal_overlap(*o);      // (before anything is scaled)
      // in the order of what is read
      back.emplace_back(at::empty_like(g->is_non_overlapping_and_dense() ? *g : hold.back()), *o);
      outs[i] = back.back().first.mutable_data_ptr();
    }
    if (others && !apart(n))
      for (size_t i = 0; i < n; ++i)
        if (sizes[i] != 0 && grads[i] != outs[i] && is_written(grads[i]) && grads[i] != THPVariable_Unpack(others_items[i]).const_data_ptr())
          throw pybind11::value_error("clip_grads expects out to hold none of grads but in its own place");
    // what autograd has kept of a tensor that changes is no longer what it was
    for (size_t i = 0; writes && i < n; ++i)
      if (!written[i]->is_inference()) written[i]->bump_version();
    list = {grads.get(), outs.get(), sizes.get(), dtypes.get(), (int64_t)n};
    return true;
  }
  void finish() {
    for (auto& b : back) b.second.copy_(b.first);
  }
};

// (total fp64, norm fp32) of the tensors together
std::optional<std::pair<Tensor, Tensor>> grad_norm(const pybind11::list& grads, bool inf) {
  const at::AutoGradMode no_graph(false);
  GradList l;
  const c10::cuda::OptionalCUDAGuard device(on_device(grads));
  if (!l.take(grads, pybind11::list(), false)) return std::nullopt;
  const auto options = l.first.options();
  const Tensor total = at::empty({}, options.dtype(at::kDouble)), norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor work = at::empty({entry.norm_work_bytes(l.list.count)}, options.dtype(at::kByte));
  check(entry.grad_norm(&l.list, inf, work.data_ptr(), (double*)total.data_ptr(), (float*)norm.data_ptr(), stream_here()), "altob200_grad_norm");
  return std::make_pair(total, norm);
}

std::optional<Tensor> clip_grads(const pybind11::list& grads, const pybind11::list& outs, double max_norm, bool inf,
                                 const std::optional<Tensor>& total) {
  const at::AutoGradMode no_graph(false);
  GradList l;
  const c10::cuda::OptionalCUDAGuard device(on_device(grads));
  if (!l.take(grads, outs, true)) return std::nullopt;
  const auto options = l.first.options();
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  Tensor work;
  if (!total.has_value()) work = at::empty({entry.norm_work_bytes(l.list.count)}, options.dtype(at::kByte));
  check(entry.clip_grads(&l.list, inf, max_norm, total.has_value() ? (const double*)total->data_ptr() : nullptr,
                         work.defined() ? work.data_ptr() : nullptr, (float*)norm.data_ptr(), stream_here()), "altob200_clip_grads");
  l.finish();
  return norm;
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.def("bind", [](uintptr_t forward, uintptr_t work_bytes, uintptr_t backward, uintptr_t norm_work_bytes, uintptr_t grad_norm,
                   uintptr_t clip_grads, uintptr_t fp8_quantize, uintptr_t fp8_squares, uintptr_t fp8_gemm) {
    entry = {reinterpret_cast<decltype(entry.forward)>(forward), reinterpret_cast<decltype(entry.work_bytes)>(work_bytes),
             reinterpret_cast<decltype(entry.backward)>(backward), reinterpret_cast<decltype(entry.norm_work_bytes)>(norm_work_bytes),
             reinterpret_cast<decltype(entry.grad_norm)>(grad_norm), reinterpret_cast<decltype(entry.clip_grads)>(clip_grads),
             reinterpret_cast<decltype(entry.fp8_quantize)>(fp8_quantize), reinterpret_cast<decltype(entry.fp8_squares)>(fp8_squares),
             reinterpret_cast<decltype(entry.fp8_gemm)>(fp8_gemm)};
  });
  m.def("fp8_linear", &fp8_linear, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("fp8_serve", &fp8_serve, pybind11::call_guard<pybind11::gil_scoped_release>());
  // None: operands that alto_b200/fp8_block.py, a list that alto_b200/grad_clip.py has to look at
  m.def("fp8_try_serve", &fp8_try_serve);
  m.def("fp8_try_linear", &fp8_try_linear);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grads", &clip_grads);
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
