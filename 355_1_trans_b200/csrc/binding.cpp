// binding.cpp -- Python entry points of the operators in ops.cu, without the
// cost of filling ctypes structs attribute by attribute.  A decode step's
// kernels run for 3 to 15 us each, so the host's share of a call decides how
// fast a loop of them runs: a one-token linear took 18 us of host time through
// ctypes and takes 6 to 7 through here.
//
// Each function checks its tensors, fills the C-ABI struct of
// include/bsgemm_b200.h, allocates outputs and workspace from torch's caching
// allocator and launches on the current stream; the allocator learns that the
// caller's tensors are in use there, those that are copied first too.  A wrong tensor raises ValueError; a status
// of the library raises the class given to set_error, with the status.
// 355_1_trans_b200/ops.py documents the arguments and passes them by position.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/bsgemm_b200.h"

namespace {

using at::Tensor;

PyObject* g_error = nullptr;   // BsgemmError(status, name)

// ---- arguments --------------------------------------------------------------
const Tensor& tensor(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
// None or a tensor
Tensor optional(PyObject* o, const char* what) { return o == Py_None ? Tensor() : tensor(o, what); }

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
int small(PyObject* o) {
  const long long v = integer(o);
  TORCH_CHECK_VALUE(v >= INT_MIN && v <= INT_MAX, "integer argument out of range");
  return static_cast<int>(v);
}
int extent(int64_t v) {
  TORCH_CHECK_VALUE(v <= INT_MAX, "a dimension or stride is past the library's 32-bit limit");
  return static_cast<int>(v);
}

bool real(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }
int real_code(at::ScalarType t) { return t == at::kFloat ? BSG_IN_FP32 : BSG_IN_BF16; }   // == BSG_OUT_*
bool fp8(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kByte; }
bool fp4x2(at::ScalarType t) { return t == at::kByte || t == at::kFloat4_e2m1fn_x2; }
bool e8m0(at::ScalarType t) { return t == at::kByte || t == at::kFloat8_e8m0fnu; }

int64_t scales_size(int64_t rows, int64_t kg) { return (rows + 127) / 128 * ((kg + 3) / 4) * 512; }

// A caller's tensor that a copy on the current stream reads: the allocator must not
// hand its memory on before that copy has run.
const Tensor& read_here(const Tensor& t) {
  if (t.is_cuda())
    c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), c10::cuda::getCurrentCUDAStream(t.get_device()));
  return t;
}

// A 2-D tensor with unit inner stride and rows that do not overlap, and its row stride.
struct Rows {
  Tensor t;
  int64_t ld;
};
// The row stride of such a tensor, -1 where t is another.
int64_t row_stride(const Tensor& t) {
  const int64_t cols = t.size(1);
  if (t.is_contiguous()) return cols;
  const int64_t ld = t.size(0) == 1 ? cols : t.stride(0);
  return ld < cols || (t.stride(1) != 1 && cols > 1) ? -1 : ld;
}
Rows rows_of(const Tensor& t) {
  const int64_t ld = row_stride(t);
  if (ld < 0) return {read_here(t).contiguous(), t.size(1)};
  return {t, ld};
}

Tensor make(const Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::empty(shape, like.options().dtype(dtype));
}

// What the kernels read in 16-byte chunks, at 16-byte offsets and strides: a view at
// any other is copied.
bool off16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0; }
Tensor aligned(const Tensor& t) { return off16(t) ? read_here(t).clone(at::MemoryFormat::Contiguous) : t; }
Rows aligned_rows(const Tensor& t) {
  const int64_t rows = t.size(0), cols = t.size(1), ld = row_stride(t), chunk = 16 / t.element_size();
  if (ld >= 0 && !off16(t) && (rows <= 1 || ld % chunk == 0)) return {t, ld};
  const int64_t to = (cols + chunk - 1) / chunk * chunk;
  Tensor copy = make(t, {rows, to}, t.scalar_type()).narrow(1, 0, cols);
  copy.copy_(read_here(t));
  return {copy, to};
}

// An output [rows, cols] of a real type: a new one, or the caller's checked.
Rows real_out(const Tensor& out, int64_t rows, int64_t cols, at::ScalarType dtype, const Tensor& like) {
  if (!out.defined()) return {make(like, {rows, cols}, dtype), cols};
  TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == rows && out.size(1) == cols && out.scalar_type() == dtype &&
                        out.device() == like.device() && (cols <= 1 || out.stride(1) == 1),
                    "out must be a tensor of shape (", rows, ", ", cols, ") and dtype ", dtype,
                    " with unit inner stride on the inputs' GPU");
  return {out, rows > 1 ? out.stride(0) : cols};
}

// (elements, native scales) of an MX output [rows, cols].
struct Mx {
  Tensor q, sf;
};
Mx mx_out(PyObject* out, int64_t rows, int64_t cols, int fmt, const Tensor& like) {
  TORCH_CHECK_VALUE(cols % 128 == 0, "an MX output needs a multiple of 128 columns");
  const bool f8 = fmt == BSG_OUT_MXFP8;
  const int64_t width = f8 ? cols : cols / 2, size = scales_size(rows, cols / 32);
  if (out == Py_None)
    return {make(like, {rows, width}, f8 ? at::kFloat8_e4m3fn : at::kByte), make(like, {size}, at::kByte)};
  TORCH_CHECK_VALUE(PyTuple_Check(out) && PyTuple_GET_SIZE(out) == 2, "out of an MX format is (elements, scales)");
  Mx m{tensor(PyTuple_GET_ITEM(out, 0), "out[0]"), tensor(PyTuple_GET_ITEM(out, 1), "out[1]")};
  for (const Tensor& t : {m.q, m.sf})
    TORCH_CHECK_VALUE(t.device() == like.device() && t.is_contiguous(),
                      "out must hold contiguous tensors on the inputs' GPU");
  TORCH_CHECK_VALUE(m.q.dim() == 2 && m.q.size(0) == rows && m.q.size(1) == width &&
                        (f8 ? fp8(m.q.scalar_type()) : fp4x2(m.q.scalar_type())) && e8m0(m.sf.scalar_type()) &&
                        m.sf.numel() >= size,
                    "out must be (elements (", rows, ", ", width, "), ", size, " scale bytes)");
  return m;
}

// None: a new workspace of `need` bytes; else the caller's.
Tensor workspace_of(PyObject* given, size_t need, const Tensor& like) {
  if (given == Py_None) return make(like, {static_cast<int64_t>(need)}, at::kByte);
  const Tensor& w = tensor(given, "workspace");
  TORCH_CHECK_VALUE(w.device() == like.device() && w.is_contiguous() && w.nbytes() >= need, "workspace needs ", need,
                    " contiguous bytes on the inputs' GPU");
  return w;
}

// ---- launch -----------------------------------------------------------------
// Runs call(stream) and records the caller's tensors on that stream.
template <typename F>
bool launch(const char* name, const Tensor& like, std::initializer_list<const Tensor*> tensors, F call) {
  const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(like.get_device());
  const int status = call(reinterpret_cast<bsg_stream_t>(stream.stream()));
  if (status != BSG_OK) {
    PyObject* e = PyObject_CallFunction(g_error, "is", status, name);
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
    return false;
  }
  for (const Tensor* t : tensors)
    if (t->defined() && t->is_cuda()) c10::cuda::CUDACachingAllocator::recordStream(t->storage().data_ptr(), stream);
  return true;
}

PyObject* pair_of(const Tensor& a, const Tensor& b) {
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
  return t;
}
PyObject* wrap_or_none(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// Checks A [m, k], B [n, k] and their scales and fills their part of a.
void operands(bsgemm_args& a, const Tensor& A, const Tensor& B, const Tensor& As, const Tensor& Bs, bool fp4,
              bool native, int b_format, int kernel) {
  TORCH_CHECK_VALUE(A.dim() == 2 && B.dim() == 2, "A and B must be 2-D");
  TORCH_CHECK_VALUE(A.is_cuda() && B.device() == A.device() && As.device() == A.device() && Bs.device() == A.device(),
                    "all inputs must be on the same GPU");
  TORCH_CHECK_VALUE(fp4 ? fp4x2(A.scalar_type()) && fp4x2(B.scalar_type()) : fp8(A.scalar_type()) && fp8(B.scalar_type()),
                    "A/B must hold ", fp4 ? "packed E2M1" : "E4M3FN", " bytes");
  TORCH_CHECK_VALUE(e8m0(As.scalar_type()) && e8m0(Bs.scalar_type()), "scales must be E8M0 bytes");
  const int64_t m = A.size(0), n = B.size(0), kb = A.size(1), k = fp4 ? 2 * kb : kb, kg = k / 32;
  TORCH_CHECK_VALUE(B.size(1) == kb, "A and B disagree on K");
  TORCH_CHECK_VALUE(A.stride(1) == 1 && B.stride(1) == 1, "A and B must have unit stride in the last dimension");
  bsgemm_args_init(&a);
  const Tensor* const scales[2] = {&As, &Bs};
  const int64_t rows[2] = {m, n};
  for (int i = 0; i < 2; ++i) {
    const Tensor& t = *scales[i];
    if (native) {
      TORCH_CHECK_VALUE(t.is_contiguous() && t.numel() >= scales_size(rows[i], kg), "native scales of ", rows[i],
                        " rows need ", scales_size(rows[i], kg), " contiguous bytes");
    } else {
      TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows[i] && t.size(1) == kg && (kg <= 1 || t.stride(1) == 1),
                        "scale must be [", rows[i], ", ", kg, "] with unit inner stride");
    }
  }
  a.sfa_format = a.sfb_format = native ? BSG_SF_NATIVE : BSG_SF_ROWMAJOR;
  if (!native) {
    a.stride_sfa = extent(m > 1 ? As.stride(0) : kg);
    a.stride_sfb = extent(n > 1 ? Bs.stride(0) : kg);
  }
  a.ptr_a = A.data_ptr();
  a.ptr_b = B.data_ptr();
  a.ptr_sfa = As.data_ptr();
  a.ptr_sfb = Bs.data_ptr();
  a.m = extent(m);
  a.n = extent(n);
  a.k = extent(k);
  a.stride_a = extent(m > 1 ? A.stride(0) : kb);
  a.stride_b = extent(n > 1 ? B.stride(0) : kb);
  a.b_format = b_format;
  a.kernel = kernel;
}

// ---- entry points -------------------------------------------------------------
// epilogue_gemm(gated, fp4, A, B, A_scale, B_scale, bias, activation, residual, out_format, out, native, b_format,
//               split_k, workspace, grid_blocks, kernel)
PyObject* epilogue_gemm(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 17, "epilogue_gemm takes 17 arguments");
  const bool gated = integer(v[0]) != 0, fp4 = integer(v[1]) != 0;
  const Tensor &A = tensor(v[2], "A"), &B = tensor(v[3], "B"), &As = tensor(v[4], "A_scale"), &Bs = tensor(v[5], "B_scale");
  Tensor bias = optional(v[6], "bias");
  Rows residual{optional(v[8], "residual"), 0};
  const int fmt = small(v[9]);
  bsgemm_args a;
  operands(a, A, B, As, Bs, fp4, integer(v[11]) != 0, small(v[12]), small(v[16]));
  a.split_k = small(v[13]);
  a.grid_blocks = small(v[15]);
  TORCH_CHECK_VALUE(!gated || a.n % 64 == 0, "B must hold whole blocks of 32 gate and 32 up rows (pack_gated)");
  const int n_out = gated ? a.n / 2 : a.n;
  const c10::cuda::CUDAGuard guard(A.device());
  bsgemm_epilogue e{};
  e.activation = small(v[7]);
  Rows c;
  Mx mx;
  if (fmt >= BSG_OUT_MXFP8) {
    mx = mx_out(v[10], a.m, n_out, fmt, A);
    c = {mx.q, mx.q.size(1)};
    e.ptr_sfc = mx.sf.data_ptr();
  } else {
    c = real_out(optional(v[10], "out"), a.m, n_out, fmt == BSG_OUT_FP32 ? at::kFloat : at::kBFloat16, A);
  }
  a.out_dtype = fmt;
  a.ptr_c = c.t.data_ptr();
  a.stride_c = extent(c.ld);
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == a.n && real(bias.scalar_type()) &&
                          bias.device() == A.device() && bias.is_contiguous(),
                      "bias must be a contiguous bf16 or fp32 tensor of ", a.n, " elements");
    bias = aligned(bias);
    e.bias = bias.data_ptr();
    e.bias_dtype = real_code(bias.scalar_type());
  }
  if (residual.t.defined()) {
    TORCH_CHECK_VALUE(residual.t.dim() == 2 && residual.t.size(0) == a.m && residual.t.size(1) == a.n &&
                          real(residual.t.scalar_type()) && residual.t.device() == A.device(),
                      "residual must be a bf16 or fp32 tensor of shape (", a.m, ", ", a.n, ")");
    residual = aligned_rows(residual.t);
    e.residual = residual.t.data_ptr();
    e.residual_dtype = real_code(residual.t.scalar_type());
    e.stride_residual = residual.ld;
  }
  Tensor ws;
  if (v[14] != Py_False && a.m > 0) {
    const size_t need = bsgemm_epilogue_workspace_size(fp4 ? BSG_FAMILY_MXFP4 : BSG_FAMILY_MXFP8, &a);
    if (need) {
      ws = workspace_of(v[14], need, A);
      a.workspace = ws.data_ptr();
      a.workspace_bytes = ws.nbytes();
    }
  }
  using Entry = int (*)(const bsgemm_args*, const bsgemm_epilogue*, bsg_stream_t);
  const Entry entry = gated ? (fp4 ? bsgemm_a4w4_mxfp4_gated : bsgemm_a8w8_mxfp8_gated)
                            : (fp4 ? bsgemm_a4w4_mxfp4_linear : bsgemm_a8w8_mxfp8_linear);
  const char* name = gated ? (fp4 ? "bsgemm_a4w4_mxfp4_gated" : "bsgemm_a8w8_mxfp8_gated")
                           : (fp4 ? "bsgemm_a4w4_mxfp4_linear" : "bsgemm_a8w8_mxfp8_linear");
  // (outputs and workspace made here belong to this stream already: recording them changes nothing)
  if (!launch(name, A, {&A, &B, &As, &Bs, &bias, &residual.t, &c.t, &mx.sf, &ws},
              [&](bsg_stream_t s) { return entry(&a, &e, s); }))
    return nullptr;
  return fmt >= BSG_OUT_MXFP8 ? pair_of(mx.q, mx.sf) : THPVariable_Wrap(c.t);
  END_HANDLE_TH_ERRORS
}

// gated_backward(fp4, grad, A, B, A_scale, B_scale, activation, native, need_input, need_weight, workspace,
//                grid_blocks, kernel)
PyObject* gated_backward(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 13, "gated_backward takes 13 arguments");
  const bool fp4 = integer(v[0]) != 0, want_a = integer(v[8]) != 0, want_w = integer(v[9]) != 0;
  const Tensor &grad = tensor(v[1], "grad"), &A = tensor(v[2], "A"), &B = tensor(v[3], "B");
  const Tensor &As = tensor(v[4], "A_scale"), &Bs = tensor(v[5], "B_scale");
  bsgemm_args a;
  operands(a, A, B, As, Bs, fp4, integer(v[7]) != 0, BSG_B_RAW, small(v[12]));
  a.grid_blocks = small(v[11]);
  TORCH_CHECK_VALUE(a.n % 64 == 0, "B must hold whole blocks of 32 gate and 32 up rows (pack_gated)");
  const int f = a.n / 2;
  TORCH_CHECK_VALUE(grad.dim() == 2 && grad.size(0) == a.m && grad.size(1) == f && grad.scalar_type() == at::kBFloat16 &&
                        grad.device() == A.device(),
                    "grad must be a bf16 tensor of shape (", a.m, ", ", f, ") on the inputs' GPU");
  const c10::cuda::CUDAGuard guard(A.device());
  const Rows h = aligned_rows(grad);
  bsgemm_gated_grad g{};
  g.activation = small(v[6]);
  g.grad_h = h.t.data_ptr();
  g.stride_grad_h = h.ld;
  Tensor da, dg, du;
  if (want_a) {
    da = make(A, {a.m, a.k}, at::kBFloat16);
    // (a tensor of no rows has no address; the call wants one for "this gradient, please")
    g.grad_a = a.m > 0 ? da.data_ptr() : B.data_ptr();
    g.stride_grad_a = a.k;
  }
  if (want_w) {
    dg = make(A, {f, a.k}, at::kBFloat16);
    du = make(A, {f, a.k}, at::kBFloat16);
    g.grad_gate = dg.data_ptr();
    g.grad_up = du.data_ptr();
    g.stride_grad_w = a.k;
  }
  const Tensor ws = workspace_of(
      v[10], bsgemm_gated_backward_workspace_size(fp4 ? BSG_FAMILY_MXFP4 : BSG_FAMILY_MXFP8, &a), A);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = ws.nbytes();
  const auto entry = fp4 ? bsgemm_a4w4_mxfp4_gated_backward : bsgemm_a8w8_mxfp8_gated_backward;
  if (!launch(fp4 ? "bsgemm_a4w4_mxfp4_gated_backward" : "bsgemm_a8w8_mxfp8_gated_backward", A,
              {&h.t, &A, &B, &As, &Bs, &ws}, [&](bsg_stream_t s) { return entry(&a, &g, s); }))
    return nullptr;
  PyObject* t = PyTuple_New(3);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, wrap_or_none(da));
  PyTuple_SET_ITEM(t, 1, wrap_or_none(dg));
  PyTuple_SET_ITEM(t, 2, wrap_or_none(du));
  return t;
  END_HANDLE_TH_ERRORS
}

// Checks x and the parameters of a layer norm; the parameters' type.
at::ScalarType norm_input(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  TORCH_CHECK_VALUE(x.dim() == 2 && real(x.scalar_type()) && x.is_cuda() && x.size(1) >= 1,
                    "x must be a 2-D bf16 or fp32 CUDA tensor");
  at::ScalarType t = x.scalar_type();
  const Tensor* first = nullptr;
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == x.size(1) && real(p->scalar_type()) && p->device() == x.device() &&
                          p->is_contiguous(),
                      "weight and bias must be contiguous bf16 or fp32 tensors of ", x.size(1), " elements");
    TORCH_CHECK_VALUE(!first || first->scalar_type() == p->scalar_type(), "weight and bias must have one type");
    first = p;
    t = p->scalar_type();
  }
  return t;
}

// layer_norm(x, weight, bias, eps, out_format or -1 for x's type, rowmajor scales, out, return_stats)
PyObject* layer_norm(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 8, "layer_norm takes 8 arguments");
  const Tensor& x = tensor(v[0], "x");
  Tensor weight = optional(v[1], "weight"), bias = optional(v[2], "bias");
  const at::ScalarType ptype = norm_input(x, weight, bias);
  int fmt = small(v[4]);
  if (fmt < 0) fmt = real_code(x.scalar_type());
  const bool rowmajor = integer(v[5]) != 0, stats = integer(v[7]) != 0, mx_fmt = fmt >= BSG_OUT_MXFP8;
  const c10::cuda::CUDAGuard guard(x.device());
  // (the library writes MX elements from whole 16-byte chunks only)
  const Rows r = mx_fmt ? aligned_rows(x) : rows_of(x);
  if (mx_fmt)
    for (Tensor* p : {&weight, &bias})
      if (p->defined()) *p = aligned(*p);
  const int64_t rows = x.size(0), cols = x.size(1);
  bsgemm_layer_norm_args a{};
  const double eps = PyFloat_AsDouble(v[3]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  a.eps = static_cast<float>(eps);
  Rows y;
  Mx mx;
  if (mx_fmt) {
    TORCH_CHECK_VALUE(!rowmajor || v[6] == Py_None, "out takes native scales");
    if (rowmajor) {
      TORCH_CHECK_VALUE(cols % 128 == 0, "an MX output needs a multiple of 128 columns");
      mx = {fmt == BSG_OUT_MXFP8 ? make(x, {rows, cols}, at::kFloat8_e4m3fn) : make(x, {rows, cols / 2}, at::kByte),
            make(x, {rows, cols / 32}, at::kByte)};
      a.sf_format = BSG_SF_ROWMAJOR;
      a.ld_sf = cols / 32;
    } else {
      mx = mx_out(v[6], rows, cols, fmt, x);
      a.sf_format = BSG_SF_NATIVE;
    }
    y = {mx.q, mx.q.size(1)};
    a.sf = mx.sf.data_ptr();
  } else {
    y = real_out(optional(v[6], "out"), rows, cols, fmt == BSG_OUT_FP32 ? at::kFloat : at::kBFloat16, x);
  }
  Tensor mean, rstd;
  if (stats) {
    mean = make(x, {rows}, at::kFloat);
    rstd = make(x, {rows}, at::kFloat);
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
  }
  a.x = r.t.data_ptr();
  a.y = y.t.data_ptr();
  a.weight = weight.defined() ? weight.data_ptr() : nullptr;
  a.bias = bias.defined() ? bias.data_ptr() : nullptr;
  a.ldx = r.ld;
  a.ldy = y.ld;
  a.rows = extent(rows);
  a.cols = extent(cols);
  a.dtype = real_code(x.scalar_type());
  a.param_dtype = real_code(ptype);
  a.out_format = fmt;
  if (!launch("bsgemm_layer_norm", x, {&r.t, &weight, &bias, &y.t, &mx.sf},
              [&](bsg_stream_t s) { return bsgemm_layer_norm(&a, s); }))
    return nullptr;
  if (!stats) return mx_fmt ? pair_of(mx.q, mx.sf) : THPVariable_Wrap(y.t);
  PyObject* t = PyTuple_New(mx_fmt ? 4 : 3);
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(y.t));
  if (mx_fmt) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(mx.sf));
  PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(mean));
  PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(rstd));
  return t;
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(dy, x, weight, mean, rstd, need_weight_grad, out, workspace)
PyObject* layer_norm_backward(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 8, "layer_norm_backward takes 8 arguments");
  const Tensor &dy = tensor(v[0], "dy"), &x = tensor(v[1], "x"), &mean = tensor(v[3], "mean"), &rstd = tensor(v[4], "rstd");
  const Tensor weight = optional(v[2], "weight");
  const at::ScalarType ptype = norm_input(x, weight, Tensor());
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
                    "dy must be like x");
  const int64_t rows = x.size(0), cols = x.size(1);
  for (const Tensor* s : {&mean, &rstd})
    TORCH_CHECK_VALUE(s->dim() == 1 && s->size(0) == rows && s->scalar_type() == at::kFloat &&
                          s->device() == x.device() && s->is_contiguous(),
                      "mean and rstd must be contiguous fp32 tensors of ", rows, " elements");
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows rx = rows_of(x), rdy = rows_of(dy);
  const Rows dx = real_out(optional(v[6], "out"), rows, cols, x.scalar_type(), x);
  bsgemm_layer_norm_grad_args a{};
  Tensor dw, db;
  if (integer(v[5]) != 0) {
    dw = make(x, {cols}, ptype);
    db = make(x, {cols}, ptype);
    a.dweight = dw.data_ptr();
    a.dbias = db.data_ptr();
  }
  const Tensor ws = workspace_of(v[7], bsgemm_layer_norm_backward_workspace_size(extent(rows), extent(cols)), x);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = ws.nbytes();
  a.dy = rdy.t.data_ptr();
  a.x = rx.t.data_ptr();
  a.weight = weight.defined() ? weight.data_ptr() : nullptr;
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.dx = dx.t.data_ptr();
  a.lddy = rdy.ld;
  a.ldx = rx.ld;
  a.lddx = dx.ld;
  a.rows = static_cast<int>(rows);
  a.cols = static_cast<int>(cols);
  a.dtype = real_code(x.scalar_type());
  a.param_dtype = real_code(ptype);
  if (!launch("bsgemm_layer_norm_backward", x, {&rdy.t, &rx.t, &weight, &mean, &rstd, &dx.t, &ws},
              [&](bsg_stream_t s) { return bsgemm_layer_norm_backward(&a, s); }))
    return nullptr;
  PyObject* t = PyTuple_New(3);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(dx.t));
  PyTuple_SET_ITEM(t, 1, wrap_or_none(dw));
  PyTuple_SET_ITEM(t, 2, wrap_or_none(db));
  return t;
  END_HANDLE_TH_ERRORS
}

// dequantize(q, sf, fp4, native, fp32 output)
PyObject* dequantize(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 5, "dequantize takes 5 arguments");
  const Tensor &q = tensor(v[0], "q"), &sf = tensor(v[1], "sf");
  const bool fp4 = integer(v[2]) != 0, native = integer(v[3]) != 0, f32 = integer(v[4]) != 0;
  TORCH_CHECK_VALUE(q.dim() == 2 && q.is_cuda() && (fp4 ? fp4x2(q.scalar_type()) : fp8(q.scalar_type())),
                    "q must be a 2-D CUDA tensor of ", fp4 ? "packed E2M1" : "E4M3FN", " bytes");
  TORCH_CHECK_VALUE(e8m0(sf.scalar_type()) && sf.device() == q.device(), "sf must hold E8M0 bytes on q's GPU");
  const int64_t rows = q.size(0), cols = fp4 ? 2 * q.size(1) : q.size(1);
  const c10::cuda::CUDAGuard guard(q.device());
  Rows s{sf, 0};
  if (native) {
    TORCH_CHECK_VALUE(sf.is_contiguous() && sf.numel() >= scales_size(rows, cols / 32), "native scales need ",
                      scales_size(rows, cols / 32), " contiguous bytes");
  } else {
    TORCH_CHECK_VALUE(sf.dim() == 2 && sf.size(0) == rows && sf.size(1) == cols / 32, "sf must be [", rows, ", ",
                      cols / 32, "]");
    s = rows_of(sf);
  }
  const Rows r = rows_of(q);
  const Tensor y = make(q, {rows, cols}, f32 ? at::kFloat : at::kBFloat16);
  if (!launch("bsgemm_dequantize", q, {&r.t, &s.t}, [&](bsg_stream_t st) {
        return bsgemm_dequantize(r.t.data_ptr(), r.ld, s.t.data_ptr(), native ? BSG_SF_NATIVE : BSG_SF_ROWMAJOR, s.ld,
                                 fp4 ? BSG_QUANT_MXFP4 : BSG_QUANT_MXFP8, extent(rows), extent(cols), y.data_ptr(),
                                 f32 ? BSG_OUT_FP32 : BSG_OUT_BF16, cols, st);
      }))
    return nullptr;
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(g_error, cls);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(epilogue_gemm), FAST(gated_backward),     FAST(layer_norm),
                         FAST(layer_norm_backward), FAST(dequantize), {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bsgemm_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__bsgemm_ops() { return PyModule_Create(&module); }
