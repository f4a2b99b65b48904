// The dense operators (trs_embed .. trs_adamw) on torch tensors, behind trspmm/dense.py: argument checks,
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

// Autograd refuses a backward pass through what it saved of them before.
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Of a call that has gone well: the outputs that were given.
void changed(std::initializer_list<const Given*> outputs) {
  for (const Given* t : outputs)
    if (*t) changed(**t);
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
  changed({&out_in});
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
  changed({&out_in});
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
  changed({&out_in, &r_out});
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
  changed({&out_in, &scale_in, &r_out});
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
  changed({&out_in, &dweight_in});
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
  changed({&out_in});
  return out;
}

// ---------------------------------------------------------------------------------------------
// 4-bit codes: uint8 [rows, 16 * blocks], and a scale for each block, float8_e8m0fnu [rows, blocks] (or its bytes).

constexpr int64_t kBlock = 32, kBlockBytes = 16;
int64_t blocks_of(int64_t width) { return (width + kBlock - 1) / kBlock; }

bool is_scale(at::ScalarType t) { return t == at::kFloat8_e8m0fnu || t == at::kByte; }

// Codes [rows, 16 * blocks] whose rows start on 16-byte boundaries: `t` itself, or a copy.
Tensor codes_of(const char* name, const Tensor& t, int64_t dev) {
  on_device(name, t, dev);
  if (t.scalar_type() != at::kByte || t.dim() != 2 || t.size(1) % kBlockBytes != 0)
    wrong(std::string(name) + " must be a 2-D tensor of uint8 with 16 columns for each block");
  const Tensor m = matrix(name, t, dev);
  const bool there = m.numel() == 0 || ((reinterpret_cast<uintptr_t>(m.data_ptr()) | (m.size(0) > 1 ? (uintptr_t)m.stride(0) : 0)) & 15) == 0;
  return there ? m : m.clone(at::MemoryFormat::Contiguous);
}

Tensor scales_of(const char* name, const Tensor& t, int64_t rows, int64_t blocks, int64_t dev) {
  on_device(name, t, dev);
  if (!is_scale(t.scalar_type()) || t.dim() != 2 || t.size(0) != rows || t.size(1) != blocks)
    wrong(std::string(name) + " must be a float8_e8m0fnu or uint8 tensor [" + std::to_string(rows) + ", " + std::to_string(blocks) + "]");
  return matrix(name, t, dev);
}

// Outputs of a quantisation: those that are given, checked, or new ones.
struct CodesOut {
  Tensor codes, scale;
  CodesOut(const Given& out, const Given& scale_in, int64_t rows, int64_t width, int64_t dev) {
    const int64_t blocks = blocks_of(width);
    codes = output("out", out, rows, blocks * kBlockBytes, at::kByte, dev);
    if (codes.numel() > 0 && ((reinterpret_cast<uintptr_t>(codes.data_ptr()) | (rows > 1 ? (uintptr_t)codes.stride(0) : 0)) & 15) != 0)
      wrong("rows of out must start on 16-byte boundaries");
    if (scale_in && !is_scale(scale_in->scalar_type())) wrong("scale must be float8_e8m0fnu or uint8");
    scale = output("scale", scale_in, rows, blocks, scale_in ? scale_in->scalar_type() : at::kFloat8_e8m0fnu, dev);
  }
  uint8_t* codes_at() const { return static_cast<uint8_t*>(codes.data_ptr()); }
  uint8_t* scale_at() const { return static_cast<uint8_t*>(scale.data_ptr()); }
};

const uint8_t* bytes(const Tensor& t) { return static_cast<const uint8_t*>(t.data_ptr()); }

std::tuple<Tensor, Tensor> quant_mx4(const Tensor& x_in, const Given& out, const Given& scale, int64_t dev, int64_t stream) {
  const Tensor x = matrix("x", x_in, dev);
  const int x_type = type_of("x", x.scalar_type());
  const CodesOut o(out, scale, x.size(0), x.size(1), dev);
  ok(trs_quant_mx4(x.data_ptr(), x_type, ld(x), x.size(0), width_of(x), o.codes_at(), ld(o.codes), o.scale_at(), ld(o.scale),
                   stream_of(stream)),
     "trs_quant_mx4");
  changed({&out, &scale});
  return {o.codes, o.scale};
}

Tensor dequant_mx4(const Tensor& codes_in, const Tensor& scale_in, int64_t width, const Type& dtype, const Given& out_in,
                   int64_t dev, int64_t stream) {
  const Tensor codes = codes_of("codes", codes_in, dev);
  const int64_t rows = codes.size(0), blocks = codes.size(1) / kBlockBytes;
  if (width < 0 || blocks_of(width) != blocks)
    wrong("a width of " + std::to_string(width) + " has " + std::to_string(blocks_of(width)) + " blocks, codes have " + std::to_string(blocks));
  if (width > INT32_MAX) wrong("rows of more than 2^31 - 1 elements");
  const Tensor scale = scales_of("scale", scale_in, rows, blocks, dev);
  const at::ScalarType type = type_out(out_in, dtype, at::kHalf);
  const int o_type = type_of("dtype", type);
  const Tensor out = output("out", out_in, rows, width, type, dev);
  ok(trs_dequant_mx4(bytes(codes), ld(codes), bytes(scale), ld(scale), rows, (int32_t)width, out.data_ptr(), o_type, ld(out),
                     stream_of(stream)),
     "trs_dequant_mx4");
  changed({&out_in});
  return out;
}

std::tuple<Tensor, Tensor, Given> rms_norm_mx4(const Tensor& x, const Tensor& weight, const Given& residual, double eps,
                                               const Given& out, const Given& scale, const Given& r_out, int64_t dev,
                                               int64_t stream) {
  const NormOperands n(x, weight, residual, r_out, dev);
  const CodesOut o(out, scale, n.rows, n.width, dev);
  ok(trs_rms_norm_mx4(n.x.data_ptr(), n.x_type, ld(n.x), data(n.residual), n.r_type, n.ldr(), weight.data_ptr(), n.w_type,
                      (float)eps, n.rows, n.width, o.codes_at(), ld(o.codes), o.scale_at(), ld(o.scale), data(n.r), n.ldro(),
                      stream_of(stream)),
     "trs_rms_norm_mx4");
  changed({&out, &scale, &r_out});
  return {o.codes, o.scale, n.r_given()};
}

Tensor matmul_mx4(const Tensor& a_in, const Tensor& a_scale_in, const Tensor& w_in, const Tensor& w_scale_in, const Given& bias,
                  const Type& dtype, const Given& out_in, int64_t dev, int64_t stream) {
  const Tensor a = codes_of("a", a_in, dev), w = codes_of("w", w_in, dev);
  const int64_t m = a.size(0), n = w.size(0), blocks = a.size(1) / kBlockBytes;
  if (w.size(1) != a.size(1))
    wrong("a has " + std::to_string(blocks) + " blocks in a row and w " + std::to_string(w.size(1) / kBlockBytes));
  if (n > INT32_MAX || blocks > INT32_MAX) wrong("more than 2^31 - 1 output channels or blocks");
  const Tensor a_scale = scales_of("a_scale", a_scale_in, m, blocks, dev), w_scale = scales_of("w_scale", w_scale_in, n, blocks, dev);
  if (bias) floats("bias", *bias, n, dev);
  const at::ScalarType type = type_out(out_in, dtype, at::kHalf);
  const int o_type = type_of("dtype", type);
  const Tensor out = output("out", out_in, m, n, type, dev);
  ok(trs_matmul_mx4(bytes(a), ld(a), bytes(a_scale), ld(a_scale), bytes(w), ld(w), bytes(w_scale), ld(w_scale),
                    bias ? static_cast<const float*>(bias->data_ptr()) : nullptr, m, (int32_t)n, (int32_t)blocks, out.data_ptr(),
                    o_type, ld(out), stream_of(stream)),
     "trs_matmul_mx4");
  changed({&out_in});
  return out;
}

// ---------------------------------------------------------------------------------------------
// A number of the host's or a tensor of one element on the GPU.
template <class T>
const T* one_of(const char* name, const py::object& x, at::ScalarType type, int64_t dev) {
  const Tensor t = x.cast<Tensor>();
  on_device(name, t, dev);
  if (t.scalar_type() != type || t.numel() != 1)
    wrong(std::string(name) + " must be a number or a " + c10::toString(type) + " tensor of one element");
  return static_cast<const T*>(t.data_ptr());
}

template <class T>
T number(const char* name, const char* what, const py::object& x) {
  try {
    return x.cast<T>();
  } catch (const py::cast_error&) {
    wrong(std::string(name) + " must be " + what);
  }
  return T();
}

bool is_tensor(const py::object& x) { return THPVariable_Check(x.ptr()); }

// A sequence's items without a cast of each: a list of some hundred tensors is walked in every step.
class Items {
 public:
  Items(const char* name, const py::handle& x) : fast_(py::reinterpret_steal<py::object>(PySequence_Fast(x.ptr(), name))) {
    if (!fast_) throw py::error_already_set();
  }
  size_t size() const { return (size_t)PySequence_Fast_GET_SIZE(fast_.ptr()); }
  PyObject* operator[](size_t i) const { return PySequence_Fast_GET_ITEM(fast_.ptr(), (Py_ssize_t)i); }

 private:
  py::object fast_;
};

std::string at_index(const char* name, size_t i) { return std::string(name) + "[" + std::to_string(i) + "]"; }

const Tensor& tensor_at(const char* name, size_t i, PyObject* x, int64_t dev) {
  if (!THPVariable_Check(x)) wrong(at_index(name, i) + " must be a tensor");
  const Tensor& t = THPVariable_Unpack(x);
  if (!t.is_cuda() || t.get_device() != dev) on_device(at_index(name, i).c_str(), t, dev);
  return t;
}

// A tensor that the step writes: contiguous, of n elements.
void* flat(const char* name, size_t i, const Tensor& t, int64_t n) {
  if (!t.is_contiguous()) wrong(at_index(name, i) + " must be contiguous");
  if (t.numel() != n) wrong(at_index(name, i) + " must have " + std::to_string(n) + " elements (it has " + std::to_string(t.numel()) + ")");
  return t.data_ptr();
}

void adamw(const py::object& params_in, const py::object& grads_in, const py::object& states_in, const py::object& step,
           const py::object& lr, std::pair<double, double> betas, double eps, const py::object& decay, const py::object& copies_in,
           const py::object& grad_scale, const Given& skip, int64_t seed, int64_t dev, int64_t stream) {
  const Items params("params must be a sequence of tensors", params_in), grads("grads must be a sequence of tensors", grads_in),
      states("states must be a sequence", states_in);
  const size_t count = params.size();
  if (grads.size() != count || states.size() != count)
    wrong(std::to_string(count) + " params, " + std::to_string(grads.size()) + " grads and " + std::to_string(states.size()) + " states");
  trs_adamw_options o;
  trs_adamw_options_default(&o);
  if (is_tensor(lr)) o.lr_device = one_of<float>("lr", lr, at::kFloat, dev);
  else o.lr = number<double>("lr", "a number or a tensor", lr);
  if (is_tensor(step)) o.step_device = one_of<int64_t>("step", step, at::kLong, dev);
  else o.step = number<int64_t>("step", "an integer or a tensor", step);
  if (is_tensor(grad_scale)) o.grad_scale_device = one_of<float>("grad_scale", grad_scale, at::kFloat, dev);
  else o.grad_scale = number<double>("grad_scale", "a number or a tensor", grad_scale);
  if (skip) o.skip = one_of<float>("skip", py::cast(*skip), at::kFloat, dev);
  o.beta1 = betas.first, o.beta2 = betas.second, o.eps = eps;
  if (seed < 0 || seed > (int64_t)UINT32_MAX) wrong("seed must be in 0 .. 2^32 - 1");
  o.seed = (uint32_t)seed;
  const bool each = PySequence_Check(decay.ptr());
  const char* const numbers = "a number, or one for each of the params";
  const double decay_all = each ? 0.0 : number<double>("weight_decay", numbers, decay);
  const std::vector<double> decays = each ? number<std::vector<double>>("weight_decay", numbers, decay) : std::vector<double>();
  if (each && decays.size() != count) wrong("weight_decay must be a number, or one for each of the params");
  std::optional<Items> copies;
  if (!copies_in.is_none()) copies.emplace("copies must be a sequence of tensors", copies_in);
  if (copies && copies->size() != count) wrong("copies must have one entry for each of the params (None: no copy)");
  std::vector<trs_adamw_tensor> list(count);
  std::vector<Tensor> made;   // contiguous copies of gradients
  for (size_t i = 0; i < count; ++i) {
    trs_adamw_tensor& t = list[i];
    t = trs_adamw_tensor{};
    const Tensor& p = tensor_at("params", i, params[i], dev);
    const int64_t n = p.numel();
    t.count = n;
    t.weight_decay = (float)(each ? decays[i] : decay_all);
    t.param = flat("params", i, p, n);
    t.param_type = type_of("params", p.scalar_type());
    const Tensor& g = tensor_at("grads", i, grads[i], dev);
    t.grad_type = type_of("grads", g.scalar_type());
    if (g.sizes() != p.sizes()) wrong(at_index("grads", i) + " must have its parameter's shape");
    if (g.is_contiguous()) {
      t.grad = g.data_ptr();
    } else {
      made.push_back(g.contiguous());
      t.grad = made.back().data_ptr();
    }
    const Items state("a state is (m, v) or (m, v, m_scale, v_scale)", states[i]);
    const size_t parts = state.size();
    if (parts != 2 && (parts != 4 || (state[2] == Py_None) != (state[3] == Py_None))) wrong("a state is (m, v) or (m, v, m_scale, v_scale)");
    const Tensor &m = tensor_at("m of states", i, state[0], dev), &v = tensor_at("v of states", i, state[1], dev);
    const bool small = parts == 4 && state[2] != Py_None;
    const at::ScalarType type = small ? at::kFloat8_e4m3fn : at::kFloat;
    if (m.scalar_type() != type || v.scalar_type() != type)
      wrong("m and v must be float32, or float8_e4m3fn with scales (" + at_index("states", i) + ")");
    t.m = flat("m of states", i, m, n);
    t.v = flat("v of states", i, v, n);
    if (small) {
      const Tensor &ms = tensor_at("m_scale of states", i, state[2], dev), &vs = tensor_at("v_scale of states", i, state[3], dev);
      if (!is_scale(ms.scalar_type()) || !is_scale(vs.scalar_type())) wrong("scales of states must be float8_e8m0fnu or uint8");
      t.m_scale = static_cast<uint8_t*>(flat("m_scale of states", i, ms, blocks_of(n)));
      t.v_scale = static_cast<uint8_t*>(flat("v_scale of states", i, vs, blocks_of(n)));
    }
    if (copies && (*copies)[i] != Py_None) {
      const Tensor& c = tensor_at("copies", i, (*copies)[i], dev);
      t.copy = flat("copies", i, c, n);
      t.copy_type = type_of("copies", c.scalar_type());
    }
  }
  ok(trs_adamw(list.data(), (int64_t)count, &o, stream_of(stream)), "trs_adamw");
  // States are no operands of a loss: the counters of 148 tensors' states took 6 to 11 us beside the call's 32 to 37.
  for (size_t i = 0; i < count; ++i) {
    changed(THPVariable_Unpack(params[i]));
    if (copies && (*copies)[i] != Py_None) changed(THPVariable_Unpack((*copies)[i]));
  }
}

}  // namespace

void bind_dense(pybind11::module_& m) {
  m.def("embed", &embed);
  m.def("embed_grad", &embed_grad);
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_i8", &rms_norm_i8);
  m.def("rms_norm_grad", &rms_norm_grad);
  m.def("matmul_i8", &matmul_i8);
  m.def("quant_mx4", &quant_mx4);
  m.def("dequant_mx4", &dequant_mx4);
  m.def("rms_norm_mx4", &rms_norm_mx4);
  m.def("matmul_mx4", &matmul_mx4);
  m.def("adamw", &adamw);
}
