// torch_binding.cpp -- the Python entry points of the router and of the 4-bit operators
// (fmoe_b200/router.py, fmoe_b200/fp4.py): argument checks, outputs and workspaces from torch's
// allocator, the current stream, then the C ABI of include/fmoe.h.
//
// These calls are short: a token's routing takes 3.5 us on the device. Through ctypes the host
// side alone took 12 us (26 us for the expert layer); compiled it takes 5.5 (16).
//
// Errors are those of the other bindings: ValueError for a wrong device, layout, shape or value,
// TypeError for a wrong dtype, RuntimeError for a CUDA failure, DeviceError for a device error
// word.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "fmoe.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

[[noreturn]] void value_error(const std::string& msg) { throw py::value_error(msg); }
[[noreturn]] void type_error(const std::string& msg) { throw py::type_error(msg); }

[[noreturn]] void raise(const char* where, int rc) {
  const std::string msg = std::string(where) + ": " + fmoe_last_error();
  if (rc == FMOE_ERR_VALUE || rc == FMOE_ERR_WORKSPACE) value_error(msg);
  if (rc == FMOE_ERR_TYPE) type_error(msg);
  throw std::runtime_error(msg);
}

Tensor tensor_of(py::handle h, const std::string& name) {
  if (!THPVariable_Check(h.ptr())) value_error(name + " must be a torch.Tensor");
  return THPVariable_Unpack(h.ptr());
}

OptTensor optional_of(py::handle h, const std::string& name) {
  if (h.is_none()) return std::nullopt;
  return tensor_of(h, name);
}

std::string shape_text(c10::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + ")";
}

// A contiguous CUDA tensor of this shape and type, on `dev`.
void expect(const Tensor& t, const std::string& name, c10::IntArrayRef shape, at::ScalarType dtype,
            c10::Device dev) {
  if (!t.is_cuda()) value_error(name + " must be a CUDA tensor");
  if (!t.is_contiguous()) value_error(name + " must be contiguous");
  if (t.sizes() != shape)
    value_error(name + " shape mismatch: expected " + shape_text(shape) + ", got " +
                shape_text(t.sizes()));
  if (t.scalar_type() != dtype)
    type_error(name + " dtype mismatch: expected " + std::string(c10::toString(dtype)) + ", got " +
               c10::toString(t.scalar_type()));
  if (t.device() != dev)
    value_error(name + " must be on " + dev.str() + ", got " + t.device().str());
}

int dtype_code(at::ScalarType t, const std::string& name) {
  if (t == at::kFloat) return FMOE_F32;
  if (t == at::kBFloat16) return FMOE_BF16;
  if (t == at::kHalf) return FMOE_F16;
  type_error(name + " dtype mismatch: expected float32, bfloat16 or float16, got " +
             c10::toString(t));
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// (at::empty without its dispatch, 0.4 us a tensor)
Tensor empty(c10::IntArrayRef shape, at::ScalarType dtype, c10::Device dev) {
  return at::detail::empty_cuda(shape, dtype, dev, std::nullopt);
}

// A dual tensor's tangent would be lost: no operator here has a forward-mode derivative.
void refuse_tangent(const Tensor& t, const std::string& name) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    value_error(name + " carries a forward-mode tangent, which this operator does not pass on");
}

// ------------------------------------------------------------------------------- router
Tensor logits_of(py::handle h) {
  if (!THPVariable_Check(h.ptr()) || THPVariable_Unpack(h.ptr()).dim() != 2)
    value_error("logits must be 2D");
  Tensor x = THPVariable_Unpack(h.ptr());
  refuse_tangent(x, "logits");
  if (!x.is_cuda()) value_error("logits must be a CUDA tensor");
  // rows may be padded; anything else (transposed, broadcast) is laid out first
  const int64_t T = x.size(0), E = x.size(1);
  if ((x.stride(1) != 1 && E > 1) || (x.stride(0) < E && T > 1)) x = x.contiguous();
  return x;
}

fmoe_router router_of(const Tensor& x, int64_t top_k, int score, int64_t n_group,
                      int64_t topk_group, int group_score, bool renormalize, double scale) {
  auto narrow = [](int64_t v) {  // sizes that no int holds stay out of range
    return (int32_t)std::min<int64_t>(std::max<int64_t>(v, -1), 1 << 20);
  };
  fmoe_router r = {};
  r.num_tokens = x.size(0);
  r.num_experts = narrow(x.size(1));
  r.logits_stride = x.size(0) > 1 ? x.stride(0) : x.size(1);
  r.top_k = narrow(top_k);
  r.n_group = narrow(n_group);
  r.topk_group = narrow(topk_group);
  r.score = score;
  r.group_score = group_score;
  r.renormalize = renormalize;
  r.logits_dtype = dtype_code(x.scalar_type(), "logits");
  r.bias_dtype = FMOE_F32;
  r.scale = (float)scale;
  return r;
}

std::tuple<Tensor, Tensor> route_experts(py::handle logits, int64_t top_k, int score,
                                         py::handle bias_h, int64_t n_group, int64_t topk_group,
                                         int group_score, bool renormalize, double scale) {
  const Tensor x = logits_of(logits);
  fmoe_router r =
      router_of(x, top_k, score, n_group, topk_group, group_score, renormalize, scale);
  const c10::Device dev = x.device();
  const OptTensor bias = optional_of(bias_h, "bias");
  if (bias) {
    if (bias->scalar_type() != at::kFloat && bias->scalar_type() != at::kBFloat16)
      type_error(std::string("bias dtype mismatch: expected float32 or bfloat16, got ") +
                 c10::toString(bias->scalar_type()));
    expect(*bias, "bias", {x.size(1)}, bias->scalar_type(), dev);
    r.bias_dtype = bias->scalar_type() == at::kFloat ? FMOE_F32 : FMOE_BF16;
  }
  const int64_t k = std::max<int64_t>(std::min<int64_t>(top_k, 1024), 0);
  c10::cuda::CUDAGuard guard(dev);
  Tensor idx = empty({x.size(0), k}, at::kInt, dev), w = empty({x.size(0), k}, at::kFloat, dev);
  const fmoe_route_out out = {idx.data_ptr<int32_t>(), w.data_ptr<float>()};
  const int rc = fmoe_route_experts(&r, x.data_ptr(), bias ? bias->data_ptr() : nullptr, &out,
                                    stream_of(dev));
  if (rc != FMOE_OK) raise("route_experts", rc);
  return {idx, w};
}

Tensor route_experts_backward(py::handle grad_h, py::handle logits, py::handle idx_h, int score,
                              bool renormalize, double scale) {
  const Tensor x = logits_of(logits);
  if (!THPVariable_Check(idx_h.ptr()) || THPVariable_Unpack(idx_h.ptr()).dim() != 2)
    value_error("topk_idx must be 2D");
  const Tensor idx = THPVariable_Unpack(idx_h.ptr());
  const int64_t T = x.size(0), K = idx.size(1);
  const c10::Device dev = x.device();
  const fmoe_router r =
      router_of(x, K, score, 1, 1, FMOE_GROUP_TOP2, renormalize, scale);
  expect(idx, "topk_idx", {T, K}, at::kInt, dev);
  const Tensor grad = tensor_of(grad_h, "grad_w").contiguous();  // it may arrive broadcast
  refuse_tangent(grad, "grad_w");
  expect(grad, "grad_w", {T, K}, at::kFloat, dev);
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = empty({T, x.size(1)}, x.scalar_type(), dev);
  const int rc = fmoe_route_experts_backward(&r, grad.data_ptr<float>(), x.data_ptr(),
                                             idx.data_ptr<int32_t>(), out.data_ptr(),
                                             stream_of(dev));
  if (rc != FMOE_OK) raise("route_experts_backward", rc);
  return out;
}

// ------------------------------------------------------------------------------- 4 bits
int block_of(int format) { return format == FMOE_MXFP4 ? 32 : 16; }

std::vector<int64_t> scale_shape(c10::IntArrayRef lead, int64_t rows, int64_t cols, int format) {
  std::vector<int64_t> s(lead.begin(), lead.end());
  const int64_t tile = 4 * block_of(format);
  s.push_back((rows + 127) / 128);
  s.push_back((cols + tile - 1) / tile);
  s.push_back(512);
  return s;
}

const float* global_scale(const OptTensor& g, int64_t count, c10::Device dev,
                          const std::string& name, int format) {
  if (!g) return nullptr;
  if (format == FMOE_MXFP4) value_error(name + ": mxfp4 has no global scale");
  if (g->device() != dev) value_error(name + " must be a tensor on " + dev.str());
  if (g->numel() != count || !g->is_contiguous())
    value_error(name + " must have one contiguous element per matrix");
  if (g->scalar_type() != at::kFloat)
    type_error(name + " dtype mismatch: expected Float, got " + c10::toString(g->scalar_type()));
  return g->data_ptr<float>();
}

// Checked argument block of an Fp4Tensor's parts.
struct Matrix {
  Tensor codes, scales;
  OptTensor global;
  fmoe_fp4_matrix m;
};
Matrix matrix_of(py::handle codes, py::handle scales, py::handle global, int format, int dims,
                 const std::string& name) {
  Matrix r;
  r.codes = tensor_of(codes, name + ".codes");
  r.scales = tensor_of(scales, name + ".scales");
  r.global = optional_of(global, name + ".global_scale");
  const int64_t n = r.codes.dim();
  if (!(dims == n || (dims == 0 && (n == 2 || n == 3))))
    value_error(name + ".codes must be " + (dims ? std::to_string(dims) + "D" : "2D or 3D"));
  const c10::Device dev = r.codes.device();
  if (!r.codes.is_cuda()) value_error(name + ".codes must be a CUDA tensor");
  expect(r.codes, name + ".codes", r.codes.sizes(), at::kByte, dev);
  const auto lead = r.codes.sizes().slice(0, n - 2);
  const int64_t rows = r.codes.size(-2), cols = 2 * r.codes.size(-1);
  expect(r.scales, name + ".scales", scale_shape(lead, rows, cols, format), at::kByte, dev);
  const int64_t batch = lead.empty() ? 1 : lead[0];
  r.m = {};
  r.m.codes = r.codes.data_ptr();
  r.m.scales = r.scales.data_ptr();
  r.m.global_scale = global_scale(r.global, batch, dev, name + ".global_scale", format);
  r.m.rows = rows;
  r.m.cols = cols;
  r.m.batch = (int32_t)std::min<int64_t>(batch, 1 << 20);
  r.m.format = format;
  return r;
}

Tensor out_of(py::handle h, c10::IntArrayRef shape, at::ScalarType dtype, c10::Device dev) {
  dtype_code(dtype, "output");
  if (h.is_none()) return empty(shape, dtype, dev);
  const Tensor out = tensor_of(h, "out");
  expect(out, "out", shape, dtype, dev);
  return out;
}

at::ScalarType scalar_type(py::handle dtype) {
  if (!THPDtype_Check(dtype.ptr())) type_error("output dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
}

// codes and scales of x, into given tensors or new ones
std::tuple<Tensor, Tensor> quantize_fp4(py::handle x_h, int format, py::handle global_h,
                                        py::handle codes_h, py::handle scales_h) {
  if (!THPVariable_Check(x_h.ptr())) value_error("x must be 2D or 3D");
  Tensor x = THPVariable_Unpack(x_h.ptr());
  if (x.dim() != 2 && x.dim() != 3) value_error("x must be 2D or 3D");
  if (!x.is_cuda()) value_error("x must be a CUDA tensor");
  const int dtype = dtype_code(x.scalar_type(), "x");
  const int64_t rows = x.size(-2), cols = x.size(-1);
  if (cols % 32 || cols == 0)
    value_error("x must have a multiple of 32 columns, got " + std::to_string(cols));
  if (x.stride(-1) != 1) x = x.contiguous();
  const c10::Device dev = x.device();
  const auto lead = x.sizes().slice(0, x.dim() - 2);
  c10::cuda::CUDAGuard guard(dev);
  Tensor codes, scales;
  if (codes_h.is_none()) {
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() /= 2;
    codes = empty(shape, at::kByte, dev);
    scales = empty(scale_shape(lead, rows, cols, format), at::kByte, dev);
  } else {
    codes = tensor_of(codes_h, "out.codes");
    scales = tensor_of(scales_h, "out.scales");
    if (codes.device() != dev || codes.dim() != x.dim() || codes.size(-1) * 2 != cols ||
        codes.size(-2) != rows || (x.dim() == 3 && codes.size(0) != x.size(0)))
      value_error("out must have the format, shape and device of the result");
  }
  const py::object a = py::reinterpret_steal<py::object>(THPVariable_Wrap(codes));
  const py::object b = py::reinterpret_steal<py::object>(THPVariable_Wrap(scales));
  Matrix q = matrix_of(a, b, global_h, format, (int)x.dim(), "out");
  if (x.dim() == 3 && x.size(0) == 0) return {codes, scales};
  const int rc = fmoe_fp4_quantize(&q.m, x.data_ptr(), dtype, x.stride(-2),
                                   x.dim() == 3 ? x.stride(0) : 0, stream_of(dev));
  if (rc != FMOE_OK) raise("quantize_fp4", rc);
  return {codes, scales};
}

Tensor dequantize_fp4(py::handle codes, py::handle scales, py::handle global, int format,
                      py::handle dtype_h, py::handle out_h) {
  const Matrix q = matrix_of(codes, scales, global, format, 0, "q");
  const c10::Device dev = q.codes.device();
  const at::ScalarType dtype = scalar_type(dtype_h);
  std::vector<int64_t> shape(q.codes.sizes().begin(), q.codes.sizes().end());
  shape.back() *= 2;
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = out_of(out_h, shape, dtype, dev);
  if (out.numel() == 0) return out;
  const int rc =
      fmoe_fp4_dequantize(&q.m, out.data_ptr(), dtype_code(dtype, "output"), stream_of(dev));
  if (rc != FMOE_OK) raise("dequantize_fp4", rc);
  return out;
}

void raise_device_error(c10::Device dev, const char* when) {
  int32_t bits = 0;
  const int rc = fmoe_poll_device_error(&bits);
  if (rc != FMOE_OK) raise("poll_device_error", rc);
  if (bits == 0) return;
  char hex[16];
  std::snprintf(hex, sizeof(hex), "0x%x", (unsigned)bits);
  const py::object type = py::module_::import("fmoe_b200").attr("DeviceError");
  PyErr_SetString(type.ptr(), (std::string(when) + ": the fused MoE kernels on " + dev.str() +
                               " reported device error " + hex +
                               " (a bounded wait expired); that call's output is invalid")
                                  .c_str());
  throw py::error_already_set();
}

// Waits for the current stream, where the caller wants to hear of this call's own errors.
void check_call(c10::Device dev) {
  {
    py::gil_scoped_release release;
    c10::cuda::getCurrentCUDAStream(dev.index()).synchronize();
  }
  raise_device_error(dev, "this call");
}

Tensor matmul_fp4(py::handle a_codes, py::handle a_scales, py::handle a_global, int a_format,
                  py::handle b_codes, py::handle b_scales, py::handle b_global, int b_format,
                  py::handle dtype_h, py::handle out_h, bool check) {
  const Matrix a = matrix_of(a_codes, a_scales, a_global, a_format, 2, "a");
  const Matrix b = matrix_of(b_codes, b_scales, b_global, b_format, 2, "b");
  const c10::Device dev = a.codes.device();
  if (b.codes.device() != dev) value_error("a and b must be on the same device");
  const at::ScalarType dtype = scalar_type(dtype_h);
  c10::cuda::CUDAGuard guard(dev);
  raise_device_error(dev, "an earlier call on this device");
  Tensor out = out_of(out_h, {a.m.rows, b.m.rows}, dtype, dev);
  const int rc =
      fmoe_fp4_matmul(&a.m, &b.m, out.data_ptr(), dtype_code(dtype, "output"), stream_of(dev));
  if (rc != FMOE_OK) raise("matmul_fp4", rc);
  if (check) check_call(dev);
  return out;
}

// The layer has no derivative: a graph that ends here without a word would train nothing.
void refuse_gradient(const Tensor& t, const std::string& name) {
  refuse_tangent(t, name);
  if (c10::GradMode::is_enabled() && t.requires_grad())
    value_error(name + " requires a gradient, and forward_fp4 has no gradient: detach it, or call "
                       "under torch.no_grad()");
}

Tensor forward_fp4(py::handle x_h, py::handle idx_h, py::handle w_h, py::handle c13, py::handle s13,
                   py::handle g13, int f13, py::handle c2, py::handle s2, py::handle g2, int f2,
                   int64_t offset, py::handle input_scale, py::handle intermediate_scale,
                   py::handle out_h, py::handle workspace_h, bool check) {
  if (f13 != f2) value_error("w13 and w2 must have the same format");
  if (!THPVariable_Check(x_h.ptr()) || THPVariable_Unpack(x_h.ptr()).dim() != 2)
    value_error("hidden_states must be 2D");
  if (!THPVariable_Check(idx_h.ptr()) || THPVariable_Unpack(idx_h.ptr()).dim() != 2)
    value_error("topk_idx must be 2D");
  const Tensor x = THPVariable_Unpack(x_h.ptr()), idx = THPVariable_Unpack(idx_h.ptr());
  const Tensor w = tensor_of(w_h, "topk_w");
  refuse_gradient(x, "hidden_states");
  refuse_gradient(w, "topk_w");
  const int dtype = dtype_code(x.scalar_type(), "hidden_states");
  const Matrix w13 = matrix_of(c13, s13, g13, f13, 3, "w13"), w2 = matrix_of(c2, s2, g2, f2, 3, "w2");
  const c10::Device dev = w13.codes.device();
  const int64_t T = idx.size(0), K = idx.size(1);
  const int64_t E = w13.codes.size(0), H = w13.m.cols, I = w13.m.rows / 2;
  if (w13.m.rows % 2 || w2.codes.size(0) != E || w2.m.rows != H || w2.m.cols != I)
    value_error("w13 must be [E, 2I, H] and w2 [E, H, I] in 4 bits, got codes " +
                shape_text(w13.codes.sizes()) + " and " + shape_text(w2.codes.sizes()));
  if (w2.codes.device() != dev) value_error("w13 and w2 must be on the same device");
  expect(x, "hidden_states", {T, H}, x.scalar_type(), dev);
  expect(idx, "topk_idx", {T, K}, at::kInt, dev);
  expect(w, "topk_w", {T, K}, at::kFloat, dev);
  const OptTensor gx = optional_of(input_scale, "input_scale");
  const OptTensor gc = optional_of(intermediate_scale, "intermediate_scale");
  if (offset < 0 || offset > INT32_MAX)  // (of ids that are int32)
    value_error("local_expert_offset must be in [0, 2^31), got " + std::to_string(offset));
  auto narrow = [](int64_t v) { return (int32_t)std::min<int64_t>(v, 1 << 30); };
  fmoe_fp4_problem p = {};
  p.num_tokens = T;
  p.hidden_size = narrow(H);
  p.intermediate_size = narrow(I);
  p.num_local_experts = narrow(E);
  p.top_k = narrow(K);
  p.local_expert_offset = (int32_t)offset;
  p.format = f13;
  p.dtype = dtype;
  fmoe_fp4_tensors t = {};
  t.input_scale = global_scale(gx, 1, dev, "input_scale", f13);
  t.intermediate_scale = global_scale(gc, 1, dev, "intermediate_scale", f13);
  size_t bytes = 0;
  int rc = fmoe_fp4_workspace_size(&p, &bytes);
  if (rc != FMOE_OK) raise("forward_fp4", rc);
  c10::cuda::CUDAGuard guard(dev);
  raise_device_error(dev, "an earlier call on this device");
  Tensor out = out_of(out_h, {T, H}, at::kBFloat16, dev);
  if (T == 0) return out;
  Tensor workspace;
  if (workspace_h.is_none()) {
    // from the allocator, which orders it with this stream and keeps it for a capturing graph
    workspace = empty({(int64_t)bytes}, at::kByte, dev);
  } else {
    workspace = tensor_of(workspace_h, "workspace");
    if (workspace.device() != dev || !workspace.is_contiguous())
      value_error("workspace must be contiguous on " + dev.str());
  }
  // the C call asks for 16-byte alignment; some tokens' part of a routing may have 4
  auto aligned = [](const Tensor& v) {
    return reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 ? v.clone() : v;
  };
  const Tensor idx16 = aligned(idx), w16 = aligned(w);
  t.hidden_states = x.data_ptr();
  t.topk_idx = idx16.data_ptr<int32_t>();
  t.topk_w = w16.data_ptr<float>();
  t.w13 = w13.m.codes;
  t.w13_scales = w13.m.scales;
  t.w13_global = w13.m.global_scale;
  t.w2 = w2.m.codes;
  t.w2_scales = w2.m.scales;
  t.w2_global = w2.m.global_scale;
  t.output = out.data_ptr();
  rc = fmoe_fp4_forward(&p, &t, workspace.data_ptr(), workspace.nbytes(), stream_of(dev));
  if (rc != FMOE_OK) raise("forward_fp4", rc);
  if (check) check_call(dev);
  return out;
}

}  // namespace

PYBIND11_MODULE(fmoe_torch, m) {
  m.def("route_experts", &route_experts);
  m.def("route_experts_backward", &route_experts_backward);
  m.def("quantize_fp4", &quantize_fp4);
  m.def("dequantize_fp4", &dequantize_fp4);
  m.def("matmul_fp4", &matmul_fp4);
  m.def("forward_fp4", &forward_fp4);
}
