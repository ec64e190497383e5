// Python binding of the gated feed-forward and 8-bit entries: argument checks, output and workspace
// tensors and the C ABI call in one native function.  These operators take microseconds on the GPU for a
// decoding step, less than the same steps cost in Python (a block's forward call: 16 us there, 9 here).
// torch supplies tensors, its allocator and its current stream; everything computed is behind the C ABI.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/utils/pybind.h>

#include <tuple>

#include "../../include/fastnn_b200_kernels.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = c10::optional<Tensor>;

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

void check_rc(int rc, const char* name) {
  if (rc == 0) return;
  const py::object error = py::module_::import("fastnn_b200.cuda_backend").attr("CudaError");
  PyErr_SetString(error.ptr(), (std::string("CUDA ") + name + " failed").c_str());
  throw py::error_already_set();
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (int64_t v : s) t += std::to_string(v) + ",";
  return t + ")";
}

int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return FASTNN_B200_F32;
  if (t == at::kHalf) return FASTNN_B200_F16;
  if (t == at::kBFloat16) return FASTNN_B200_BF16;
  return -1;
}

int float_code(const Tensor& x) {
  const int code = dtype_code(x.scalar_type());
  if (code < 0 || !x.is_cuda() || x.dim() < 1)
    refuse("x: expected a float32, float16 or bfloat16 CUDA tensor");
  return code;
}

void check_act(int act) {
  if (act != FASTNN_B200_ACT_NONE && act != FASTNN_B200_ACT_RELU && act != FASTNN_B200_ACT_GELU &&
      act != FASTNN_B200_ACT_SILU)
    refuse("act must be ACT_NONE, ACT_RELU, ACT_GELU or ACT_SILU");
}

// Sizes cross the C ABI as int.
int to_int(int64_t v) {
  if (v > 0x7fffffff) refuse("sizes above 2^31 - 1 are not supported");
  return static_cast<int>(v);
}

// The library's context on the tensor's device, which must be the current one.
void enter(const Tensor& t) {
  static bool ready[64];
  const int dev = t.get_device();
  if (c10::cuda::current_device() != dev) refuse("tensor is not on the current CUDA device");
  if (dev < 64 && ready[dev]) return;
  check_rc(fastnn_cuda_init(dev), "initialisation");
  if (dev < 64) ready[dev] = true;
}

void check_like(const Tensor& t, const char* name, at::ScalarType type, const Tensor& like, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.device() != like.device() || !t.is_contiguous())
    refuse(std::string(name) + ": expected a contiguous tensor of the operands' type on their device");
  if (t.sizes() != shape)
    refuse(std::string(name) + ": expected shape " + shape_text(shape) + ", got " + shape_text(t.sizes()));
}

// Row stride of a tensor [.., cols] whose rows are contiguous, evenly spaced and apart.
int64_t row_stride(const Tensor& t, int64_t cols, const char* name) {
  if (t.is_contiguous()) return cols;
  const int64_t d = t.dim();
  if (t.stride(d - 1) == 1 || cols == 1) {
    if (t.numel() <= cols) return cols;
    // the leading dimensions, from the last, must step like one: sizes of 1 aside
    int64_t ld = 0, next = 0;
    bool even = true;
    for (int64_t i = d - 2; i >= 0; --i) {
      if (t.size(i) == 1) continue;
      if (ld == 0) ld = next = t.stride(i);
      if (t.stride(i) != next) even = false;
      next *= t.size(i);
    }
    if (even && ld >= cols) return ld;
  }
  refuse(std::string(name) + ": rows must be contiguous, evenly spaced and not overlap");
}

inline uintptr_t address(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
Tensor bytes_like(const Tensor& t, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, t.options().dtype(at::kByte).memory_format(c10::nullopt));
}
std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
  std::vector<int64_t> s = t.sizes().vec();
  s.back() = last;
  return s;
}
Tensor output(const OptTensor& out, at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  if (!out.has_value()) return at::empty(shape, like.options().dtype(type));
  check_like(*out, "out", type, like, shape);
  return *out;
}

struct Block {
  int code, rows, d, f;
  int64_t ld;
};
Block check_block(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int act) {
  Block b;
  b.code = float_code(x);
  check_act(act);
  if (wg.dim() != 2 || wg.numel() == 0) refuse("w_gate must be [d_ff, d_model], neither of them 0");
  const int64_t f = wg.size(0), d = wg.size(1);
  if (x.size(-1) != d) refuse("Expected input features " + std::to_string(d));
  const at::ScalarType t = x.scalar_type();
  const int64_t up[2] = {f, d}, down[2] = {d, f};
  check_like(wg, "w_gate", t, x, up);
  check_like(wu, "w_up", t, x, up);
  check_like(wd, "w_down", t, x, down);
  b.ld = row_stride(x, d, "x");
  b.f = to_int(f);
  b.d = to_int(d);
  b.rows = to_int(x.numel() / d);
  enter(x);
  return b;
}

py::object gated_ffn_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int act,
                             bool return_pre, const OptTensor& out) {
  const Block b = check_block(x, wg, wu, wd, act);
  const uintptr_t bits = address(x) | address(wg) | address(wu) | address(wd) | static_cast<uintptr_t>(b.ld * x.element_size());
  const Tensor y = output(out, x.sizes(), x.scalar_type(), x);
  Tensor gate, up;
  if (return_pre) {
    gate = at::empty(with_last(x, b.f), x.options());
    up = at::empty_like(gate);
  }
  const size_t n = fastnn_b200_gated_ffn_workspace(b.code, b.rows, b.d, b.f, 0, (bits & 15) != 0);
  const Tensor ws = bytes_like(x, n);
  check_rc(fastnn_b200_gated_ffn_forward(b.code, x.data_ptr(), b.ld, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(),
                                         y.data_ptr(), return_pre ? gate.data_ptr() : nullptr,
                                         return_pre ? up.data_ptr() : nullptr, b.rows, b.d, b.f, act, ws.data_ptr(), n,
                                         stream_of(x)),
           "gated_ffn_forward");
  if (return_pre) return py::cast(std::make_tuple(y, gate, up));
  return py::cast(y);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_ffn_backward(const Tensor& dy, const Tensor& x, const Tensor& gate,
                                                              const Tensor& up, const Tensor& wg, const Tensor& wu,
                                                              const Tensor& wd, int act) {
  const Block b = check_block(x, wg, wu, wd, act);
  if (dy.scalar_type() != x.scalar_type() || dy.device() != x.device() || dy.sizes() != x.sizes())
    refuse("dy: expected a tensor like x");
  const int64_t ld_dy = row_stride(dy, b.d, "dy");
  const std::vector<int64_t> saved = with_last(x, b.f);
  check_like(gate, "gate", x.scalar_type(), x, saved);
  check_like(up, "up", x.scalar_type(), x, saved);
  uintptr_t bits = static_cast<uintptr_t>((b.ld | ld_dy) * x.element_size());
  for (const Tensor* t : {&dy, &x, &gate, &up, &wg, &wu, &wd}) bits |= address(*t);
  const Tensor dx = at::empty(x.sizes(), x.options());
  const Tensor dwg = at::empty_like(wg), dwu = at::empty_like(wu), dwd = at::empty_like(wd);
  const size_t n = fastnn_b200_gated_ffn_workspace(b.code, b.rows, b.d, b.f, 1, (bits & 15) != 0);
  const Tensor ws = bytes_like(x, n);
  check_rc(fastnn_b200_gated_ffn_backward(b.code, dy.data_ptr(), ld_dy, x.data_ptr(), b.ld, gate.data_ptr(),
                                          up.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dx.data_ptr(),
                                          dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr(), b.rows, b.d, b.f, act,
                                          ws.data_ptr(), n, stream_of(x)),
           "gated_ffn_backward");
  return std::make_tuple(dx, dwg, dwu, dwd);
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  const int code = float_code(x);
  const int64_t cols = x.size(-1);
  if (cols < 1) refuse("x: rows need at least one column");
  const int64_t ld = row_stride(x, cols, "x");
  const int rows = to_int(x.numel() / cols);
  enter(x);
  const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
  const Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  check_rc(fastnn_b200_quantize_rows(code, x.data_ptr(), ld, static_cast<signed char*>(q.data_ptr()),
                                     static_cast<float*>(scale.data_ptr()), rows, to_int(cols), stream_of(x)),
           "quantize_rows");
  return std::make_tuple(q, scale);
}

// The checks that the two 8-bit products share; the second weight is undefined for the plain one.
Tensor int8_product(const Tensor& xq, const Tensor& xs, const Tensor& w, const Tensor& ws, const Tensor& w2,
                    const Tensor& ws2, const OptTensor& bias, int act, at::ScalarType type, const OptTensor& out) {
  if (xq.scalar_type() != at::kChar || !xq.is_cuda() || xq.dim() < 1 || !xq.is_contiguous())
    refuse("xq: expected a contiguous int8 CUDA tensor");
  check_act(act);
  const int code = dtype_code(type);
  if (code < 0) refuse("out_dtype must be float32, float16 or bfloat16");
  if (w.dim() != 2 || w.numel() == 0) refuse("weights must be [out_features, in_features], neither of them 0");
  const int64_t n = w.size(0), k = w.size(1);
  if (xq.size(-1) != k) refuse("Expected input features " + std::to_string(k));
  if (k > 131071) refuse("in_features above 131071 could overflow the 32-bit sums");
  const bool gated = w2.defined();
  const int64_t wshape[2] = {n, k}, cols[1] = {n};
  check_like(xs, "x_scale", at::kFloat, xq, xq.sizes().slice(0, xq.dim() - 1));
  check_like(w, "weight", at::kChar, xq, wshape);
  check_like(ws, "weight scale", at::kFloat, xq, cols);
  if (gated) {
    check_like(w2, "up weight", at::kChar, xq, wshape);
    check_like(ws2, "up scale", at::kFloat, xq, cols);
  }
  if (bias.has_value()) check_like(*bias, "bias", at::kFloat, xq, cols);
  const int rows = to_int(xq.numel() / k), ni = to_int(n), ki = static_cast<int>(k);
  enter(xq);
  const Tensor y = output(out, with_last(xq, n), type, xq);
  const uintptr_t bits = address(xq) | address(w) | (gated ? address(w2) : 0);
  size_t bytes = 0;
  Tensor space;
  if ((bits | static_cast<uintptr_t>(k)) & 15) {           // rows of a multiple of 16 bytes need none
    bytes = fastnn_b200_int8_workspace(rows, ki, ni, gated, (bits & 15) != 0);
    space = bytes_like(xq, bytes);
  }
  void* at_space = bytes > 0 ? space.data_ptr() : nullptr;
  auto q = [](const Tensor& t) { return static_cast<const signed char*>(t.data_ptr()); };
  auto f = [](const Tensor& t) { return static_cast<const float*>(t.data_ptr()); };
  if (gated)
    check_rc(fastnn_b200_int8_gated_forward(q(xq), f(xs), q(w), f(ws), q(w2), f(ws2), y.data_ptr(), code, rows, ki, ni,
                                            act, at_space, bytes, stream_of(xq)),
             "int8_gated_forward");
  else
    check_rc(fastnn_b200_int8_linear_forward(q(xq), f(xs), q(w), f(ws), bias.has_value() ? f(*bias) : nullptr,
                                             y.data_ptr(), code, rows, ki, ni, act, at_space, bytes, stream_of(xq)),
             "int8_linear_forward");
  return y;
}

at::ScalarType scalar_type(const py::object& dtype) {
  if (!THPDtype_Check(dtype.ptr())) refuse("out_dtype must be float32, float16 or bfloat16");
  return reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  m.def("gated_ffn_forward", &gated_ffn_forward);
  m.def("gated_ffn_backward", &gated_ffn_backward);
  m.def("quantize_rows", &quantize_rows);
  m.def("int8_linear_forward",
        [](const Tensor& xq, const Tensor& xs, const Tensor& w, const Tensor& ws, const OptTensor& bias, int act,
           const py::object& dtype, const OptTensor& out) {
          return int8_product(xq, xs, w, ws, Tensor(), Tensor(), bias, act, scalar_type(dtype), out);
        });
  m.def("int8_gated_forward",
        [](const Tensor& xq, const Tensor& xs, const Tensor& wg, const Tensor& gs, const Tensor& wu, const Tensor& us,
           int act, const py::object& dtype, const OptTensor& out) {
          return int8_product(xq, xs, wg, gs, wu, us, c10::nullopt, act, scalar_type(dtype), out);
        });
}
