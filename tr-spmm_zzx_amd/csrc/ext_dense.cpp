// The dense operators (trs_embed .. trs_matmul_i8) on torch tensors, behind trspmm/dense.py: argument checks,
// outputs and workspaces that are not given, and the call.  Here and not in Python, because a call on a few
// rows is bound by this path (1 x 4096 x 4096 codes: 10.1 us a call from Python over a kernel of 5.5).
//
// `dev` is the current device, `stream` the launch stream's handle; the caller has made that stream torch's
// current one, so what is allocated here belongs to it.  Wrong arguments raise ValueError, a status other
// than TRS_OK raises trspmm._native.TrsError.
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "trspmm.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using Given = std::optional<Tensor>;
using Type = std::optional<at::ScalarType>;

[[noreturn]] void wrong(const std::string& what) { throw py::value_error(what); }

void ok(int rc, const char* where) {
  if (rc == TRS_OK) return;
  const py::object error = py::module_::import("trspmm._native").attr("TrsError");
  PyErr_SetObject(error.ptr(), error(rc, where, trs_last_error()).ptr());
  throw py::error_already_set();
}

void* stream_of(int64_t stream) { return reinterpret_cast<void*>(stream); }

void on_device(const char* name, const Tensor& t, int64_t dev) {
  if (!t.is_cuda()) wrong(std::string(name) + " must be a CUDA tensor");
  if (t.get_device() != dev)
    wrong(std::string(name) + " is on cuda:" + std::to_string(t.get_device()) + ", not on the current device cuda:" +
          std::to_string(dev));
}

int type_of(const char* name, at::ScalarType t) {
  if (t == at::kFloat) return TRS_F32;
  if (t == at::kHalf) return TRS_F16;
  if (t == at::kBFloat16) return TRS_BF16;
  wrong(std::string(name) + " must be float32, float16 or bfloat16 (got " + c10::toString(t) + ")");
}

// A 2-D GPU matrix with unit column stride and rows that do not overlap: `t` itself, or a copy.
Tensor matrix(const char* name, const Tensor& t, int64_t dev) {
  on_device(name, t, dev);
  if (t.dim() != 2) wrong(std::string(name) + " must be a 2-D tensor");
  const bool columns = t.size(1) <= 1 || t.stride(1) == 1, rows = t.size(0) <= 1 || t.stride(0) >= t.size(1);
  return columns && rows ? t : t.contiguous();
}

// Leading dimension: a single row's stride says nothing.
int64_t ld(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

int32_t width_of(const Tensor& t) {
  if (t.size(1) > INT32_MAX) wrong("rows of more than 2^31 - 1 elements");
  return (int32_t)t.size(1);
}

const Tensor& vector(const char* name, const Tensor& t, int64_t n, int64_t dev) {
  on_device(name, t, dev);
  if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
    wrong(std::string(name) + " must be a contiguous 1-D tensor of " + std::to_string(n) + " elements");
  return t;
}

const Tensor& floats(const char* name, const Tensor& t, int64_t n, int64_t dev) {
  if (t.scalar_type() != at::kFloat) wrong(std::string(name) + " must be float32");
  return vector(name, t, n, dev);
}

Tensor fresh(at::IntArrayRef shape, at::ScalarType type, int64_t dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (at::DeviceIndex)dev)));
}

// An output's type: `dtype` or the one that it has by default, and that of the output that is given.
at::ScalarType type_out(const Given& out, const Type& dtype, at::ScalarType by_default) {
  if (out && dtype && out->scalar_type() != *dtype)
    wrong(std::string("out is ") + c10::toString(out->scalar_type()) + ", dtype asks for " + c10::toString(*dtype));
  return out ? out->scalar_type() : dtype.value_or(by_default);
}

// The given output, checked, or a new one.
Tensor output(const char* name, const Given& out, int64_t rows, int64_t width, at::ScalarType type, int64_t dev) {
  if (!out) return fresh({rows, width}, type, dev);
  on_device(name, *out, dev);
  if (out->scalar_type() != type || out->dim() != 2 || out->size(0) != rows || out->size(1) != width ||
      (width > 1 && out->stride(1) != 1) || (rows > 1 && out->stride(0) < width))
    wrong(std::string(name) + " must be a " + c10::toString(type) + " tensor [" + std::to_string(rows) + ", " +
          std::to_string(width) + "] with unit column stride");
  return *out;
}

// The given workspace, if it is large enough and on the C entries' boundary, or a new one.
Tensor workspace_of(const Given& workspace, int64_t need, int64_t dev) {
  if (workspace) {
    on_device("workspace", *workspace, dev);
    if (!workspace->is_contiguous()) wrong("workspace must be contiguous");
    if ((int64_t)workspace->nbytes() >= need && (reinterpret_cast<uintptr_t>(workspace->data_ptr()) & 7) == 0) return *workspace;
  }
  return need > 0 ? fresh({need}, at::kByte, dev) : Tensor();
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::pair<Tensor, int32_t> ids_of(const Tensor& ids, int64_t dev) {
  on_device("ids", ids, dev);
  const bool wide = ids.scalar_type() == at::kLong;
  if (ids.dim() != 1 || (!wide && ids.scalar_type() != at::kInt)) wrong("ids must be a 1-D tensor of int32 or int64");
  return {ids.size(0) > 1 && ids.stride(0) != 1 ? ids.contiguous() : ids, wide ? 64 : 32};
}

Tensor embed(const Tensor& table_in, const Tensor& ids_in, double scale, const Type& dtype, const Given& out_in, int64_t dev,
             int64_t stream) {
  const Tensor table = matrix("table", table_in, dev);
  const auto [ids, bits] = ids_of(ids_in, dev);
  const at::ScalarType type = type_out(out_in, dtype, table.scalar_type());
  const int t_type = type_of("table", table.scalar_type()), o_type = type_of("dtype", type);
  const Tensor out = output("out", out_in, ids.size(0), table.size(1), type, dev);
  ok(trs_embed(table.data_ptr(), t_type, ld(table), table.size(0), ids.data_ptr(), bits, ids.size(0), width_of(table),
               (float)scale, out.data_ptr(), o_type, ld(out), stream_of(stream)),
     "trs_embed");
  return out;
}

Tensor embed_grad(const Tensor& grad_in, const Tensor& ids_in, int64_t rows, double scale, const Type& dtype,
                  const Given& out_in, const Given& workspace, int64_t dev, int64_t stream) {
  const Tensor grad = matrix("grad", grad_in, dev);
  const auto [ids, bits] = ids_of(ids_in, dev);
  const int64_t count = grad.size(0);
  if (ids.size(0) != count)
    wrong("grad has " + std::to_string(count) + " rows for " + std::to_string(ids.size(0)) + " ids");
  if (rows < 0) wrong("rows must not be negative");
  const at::ScalarType type = type_out(out_in, dtype, at::kFloat);
  const int g_type = type_of("grad", grad.scalar_type()), o_type = type_of("dtype", type);
  const int32_t width = width_of(grad);
  const int64_t need = trs_embed_grad_workspace_bytes(count, rows, width);
  const Tensor ws = workspace_of(workspace, need, dev);
  const Tensor out = output("out", out_in, rows, width, type, dev);
  ok(trs_embed_grad(grad.data_ptr(), g_type, ld(grad), ids.data_ptr(), bits, count, rows, width, (float)scale,
                    out.data_ptr(), o_type, ld(out), data(ws), need, stream_of(stream)),
     "trs_embed_grad");
  return out;
}

// x, the residual and its output as both norms take them.
struct NormOperands {
  Tensor x, residual, r;
  int x_type, r_type = 0, w_type;
  int64_t rows;
  int32_t width;
  NormOperands(const Tensor& x_in, const Tensor& weight, const Given& residual_in, const Given& r_out, int64_t dev)
      : x(matrix("x", x_in, dev)) {
    rows = x.size(0);
    width = width_of(x);
    vector("weight", weight, width, dev);
    x_type = type_of("x", x.scalar_type());
    w_type = type_of("weight", weight.scalar_type());
    if (!residual_in) {
      if (r_out) wrong("r_out needs a residual");
      return;
    }
    residual = matrix("residual", *residual_in, dev);
    if (residual.sizes() != x.sizes()) wrong("residual must have x's shape");
    r_type = type_of("residual", residual.scalar_type());
    r = output("r_out", r_out, rows, width, residual.scalar_type(), dev);
  }
  int64_t ldr() const { return residual.defined() ? ld(residual) : 0; }
  int64_t ldro() const { return r.defined() ? ld(r) : 0; }
  Given r_given() const { return r.defined() ? Given(r) : Given(); }
};

std::tuple<Tensor, Given> rms_norm(const Tensor& x, const Tensor& weight, const Given& residual, double eps, const Type& dtype,
                                   const Given& out_in, const Given& r_out, int64_t dev, int64_t stream) {
  const NormOperands n(x, weight, residual, r_out, dev);
  const at::ScalarType type = type_out(out_in, dtype, n.x.scalar_type());
  const int y_type = type_of("dtype", type);
  const Tensor out = output("out", out_in, n.rows, n.width, type, dev);
  ok(trs_rms_norm(n.x.data_ptr(), n.x_type, ld(n.x), data(n.residual), n.r_type, n.ldr(), weight.data_ptr(), n.w_type,
                  (float)eps, n.rows, n.width, out.data_ptr(), y_type, ld(out), data(n.r), n.ldro(), stream_of(stream)),
     "trs_rms_norm");
  return {out, n.r_given()};
}

std::tuple<Tensor, Tensor, Given> rms_norm_i8(const Tensor& x, const Tensor& weight, const Given& residual, double eps,
                                              const Given& out_in, const Given& scale_in, const Given& r_out, int64_t dev,
                                              int64_t stream) {
  const NormOperands n(x, weight, residual, r_out, dev);
  const Tensor out = output("out", out_in, n.rows, n.width, at::kChar, dev);
  const Tensor scale = scale_in ? floats("scale", *scale_in, n.rows, dev) : fresh({n.rows}, at::kFloat, dev);
  if (n.width == 0) scale.zero_();   // the C entry has nothing to do then, but an empty row is a row of zeros
  ok(trs_rms_norm_i8(n.x.data_ptr(), n.x_type, ld(n.x), data(n.residual), n.r_type, n.ldr(), weight.data_ptr(), n.w_type,
                     (float)eps, n.rows, n.width, static_cast<int8_t*>(out.data_ptr()), ld(out),
                     static_cast<float*>(scale.data_ptr()), data(n.r), n.ldro(), stream_of(stream)),
     "trs_rms_norm_i8");
  return {out, scale, n.r_given()};
}

std::tuple<Tensor, Tensor> rms_norm_grad(const Tensor& grad_in, const Tensor& r_in, const Tensor& weight, const Given& more_in,
                                         double eps, const Given& out_in, const Given& dweight_in, const Given& workspace,
                                         int64_t dev, int64_t stream) {
  const Tensor grad = matrix("grad", grad_in, dev), r = matrix("r", r_in, dev);
  if (grad.sizes() != r.sizes()) wrong("grad must have r's shape");
  const int64_t rows = r.size(0);
  const int32_t width = width_of(r);
  vector("weight", weight, width, dev);
  const int g_type = type_of("grad", grad.scalar_type()), r_type = type_of("r", r.scalar_type()),
            w_type = type_of("weight", weight.scalar_type());
  Tensor more;
  if (more_in) {
    more = matrix("grad_r", *more_in, dev);
    if (more.sizes() != r.sizes() || more.scalar_type() != r.scalar_type()) wrong("grad_r must have r's shape and type");
  }
  const int64_t need = trs_rms_norm_grad_workspace_bytes(rows, width);
  const Tensor ws = workspace_of(workspace, need, dev);
  const Tensor out = output("out", out_in, rows, width, r.scalar_type(), dev);
  const Tensor dweight = dweight_in ? floats("dweight", *dweight_in, width, dev) : fresh({width}, at::kFloat, dev);
  ok(trs_rms_norm_grad(grad.data_ptr(), g_type, ld(grad), r.data_ptr(), r_type, ld(r), weight.data_ptr(), w_type, data(more),
                       more.defined() ? ld(more) : 0, (float)eps, rows, width, out.data_ptr(), ld(out),
                       static_cast<float*>(dweight.data_ptr()), data(ws), need, stream_of(stream)),
     "trs_rms_norm_grad");
  return {out, dweight};
}

Tensor matmul_i8(const Tensor& a_in, const Tensor& a_scale, const Tensor& w_in, const Tensor& w_scale, const Given& bias,
                 const Type& dtype, const Given& out_in, int64_t dev, int64_t stream) {
  if (a_in.scalar_type() != at::kChar) wrong("a must be int8");
  if (w_in.scalar_type() != at::kChar) wrong("w must be int8");
  const Tensor a = matrix("a", a_in, dev), w = matrix("w", w_in, dev);
  const int64_t m = a.size(0), n = w.size(0);
  if (w.size(1) != a.size(1))
    wrong("a has " + std::to_string(a.size(1)) + " columns and w " + std::to_string(w.size(1)));
  if (n > INT32_MAX) wrong("more than 2^31 - 1 output channels");
  floats("a_scale", a_scale, m, dev);
  floats("w_scale", w_scale, n, dev);
  if (bias) floats("bias", *bias, n, dev);
  const at::ScalarType type = type_out(out_in, dtype, at::kHalf);
  const int o_type = type_of("dtype", type);
  const Tensor out = output("out", out_in, m, n, type, dev);
  ok(trs_matmul_i8(static_cast<const int8_t*>(a.data_ptr()), ld(a), static_cast<const float*>(a_scale.data_ptr()),
                   static_cast<const int8_t*>(w.data_ptr()), ld(w), static_cast<const float*>(w_scale.data_ptr()),
                   bias ? static_cast<const float*>(bias->data_ptr()) : nullptr, m, (int32_t)n, width_of(a), out.data_ptr(),
                   o_type, ld(out), stream_of(stream)),
     "trs_matmul_i8");
  return out;
}

}  // namespace

void bind_dense(pybind11::module_& m) {
  m.def("embed", &embed);
  m.def("embed_grad", &embed_grad);
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_i8", &rms_norm_i8);
  m.def("rms_norm_grad", &rms_norm_grad);
  m.def("matmul_i8", &matmul_i8);
}
