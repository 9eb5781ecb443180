// binding.cpp -- Python entry points of the operators in ops.cu and attention.cu, without the
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
// 355_1_trans_b200/ops.py and attention.py document the arguments and pass them by position.
#include <cmath>
#include <string>

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

// (through the dispatcher, so that modes see it and deterministic ones fill it; straight from the CUDA allocator a tensor
// takes 0.9 us of host time for 1.15)
Tensor make(const Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::empty(shape, like.options().dtype(dtype));
}

// n elements of a 1-D tensor from the first on, sharing its memory; for small results that
// would cost more to allocate than to compute.
Tensor part(const Tensor& whole, int64_t first, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  t.unsafeGetTensorImpl()->set_storage_offset(first);
  return t;
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

// ---- attention ------------------------------------------------------------------
// [n, heads, width] with unit inner stride, and its other two strides.
struct Heads {
  Tensor t;
  int64_t stride = 0, head_stride = 0;
  void* data() const { return t.defined() ? t.data_ptr() : nullptr; }
};
void check_heads(const Tensor& t, const char* what, const Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == 3 && t.is_cuda() && t.device() == like.device(), what, " must be a 3-D CUDA tensor [n, heads, dim]",
                    t.is_cuda() && like.is_cuda() ? " on the inputs' GPU" : "");
}
Heads strides_of(const Tensor& t) {
  const int64_t width = t.size(2), hs = t.size(1) == 1 ? width : t.stride(1);
  return {t, t.size(0) == 1 ? hs * t.size(1) : t.stride(0), hs};
}
// Copied where its inner stride is not one; with `chunks` also where the kernels could
// not read it in 16-byte chunks (an expanded dimension among these).
Heads heads_of(const Tensor& t, bool chunks) {
  const Heads h = strides_of(t);
  const int64_t e = 16 / t.element_size();
  const bool unit = t.size(2) <= 1 || t.stride(2) == 1;
  const bool whole = !off16(t) && h.stride % e == 0 && h.head_stride % e == 0 && h.stride >= e && h.head_stride >= e;
  if (t.numel() == 0 || (unit && (!chunks || whole))) return h;
  return strides_of(read_here(t).clone(at::MemoryFormat::Contiguous));
}
Heads heads_out(PyObject* out, const char* what, int64_t n, int64_t heads, int64_t width, at::ScalarType dtype, const Tensor& like) {
  if (out == Py_None) return strides_of(make(like, {n, heads, width}, dtype));
  const Tensor& t = tensor(out, what);
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == n && t.size(1) == heads && t.size(2) == width && t.scalar_type() == dtype &&
                        t.device() == like.device() && (width <= 1 || t.stride(2) == 1),
                    what, " must be a tensor of shape (", n, ", ", heads, ", ", width, ") and dtype ", dtype,
                    " with unit inner stride on the inputs' GPU");
  return strides_of(t);
}
// A 1-D int32 tensor, contiguous (copied where it is not).
Tensor ints(const Tensor& t, const char* what, int64_t n, const Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == 1 && (n < 0 || t.size(0) == n) && t.scalar_type() == at::kInt && t.device() == like.device(), what,
                    " must be a 1-D int32 tensor", n < 0 ? std::string() : " of " + std::to_string(n) + " elements", " on the inputs' GPU");
  return t.is_contiguous() ? t : read_here(t).contiguous();
}
// A table [rows, columns] int32 with unit inner stride.
int64_t table_stride(const Tensor& t, int64_t rows, const Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.scalar_type() == at::kInt && t.device() == like.device() &&
                        (t.size(1) <= 1 || t.stride(1) == 1),
                    "block_table must be an int32 tensor [", rows, ", columns] with unit inner stride on the inputs' GPU");
  return rows > 1 ? t.stride(0) : t.size(1);
}
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return static_cast<float>(v);
}
// None: dim^-1/2
float scale_of(PyObject* o, int64_t dim) { return o == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim))) : number(o); }

struct Cache {
  Tensor part[4];
  bsgemm_kv_cache c{};
};
// The four parts of a cache from v[0 .. 3].
Cache cache_of(PyObject* const* v) {
  Cache r;
  const char* names[4] = {"cache.k", "cache.k_scale", "cache.v", "cache.v_scale"};
  for (int i = 0; i < 4; ++i) {
    r.part[i] = tensor(v[i], names[i]);
    TORCH_CHECK_VALUE(r.part[i].scalar_type() == at::kByte && r.part[i].is_cuda() && r.part[i].is_contiguous() &&
                          r.part[i].device() == r.part[0].device(),
                      names[i], " must be a contiguous uint8 CUDA tensor (new_kv_cache)");
  }
  const Tensor& k = r.part[0];
  TORCH_CHECK_VALUE(k.dim() == 4, "cache.k must be [pages, heads, page, dim / 2]");
  const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), half = k.size(3), groups = half / 16, quads = page / 4;
  TORCH_CHECK_VALUE(r.part[1].sizes() == at::IntArrayRef({pages, heads, page, groups}) &&
                        r.part[2].sizes() == at::IntArrayRef({pages, heads, quads, half, 4}) &&
                        r.part[3].sizes() == at::IntArrayRef({pages, heads, quads, groups, 4}),
                    "the cache's parts do not belong together (new_kv_cache)");
  r.c.k = k.data_ptr();
  r.c.k_scale = r.part[1].data_ptr();
  r.c.v = r.part[2].data_ptr();
  r.c.v_scale = r.part[3].data_ptr();
  r.c.pages = pages;
  r.c.page = extent(page);
  r.c.heads = extent(heads);
  r.c.dim = extent(2 * half);
  return r;
}

// rotary(q, k, positions, frequencies, factor, interleaved, inverse, q_out, k_out)
PyObject* rotary(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 9, "rotary takes 9 arguments");
  const Tensor &q = tensor(v[0], "q"), &positions = tensor(v[2], "positions"), &frequencies = tensor(v[3], "frequencies");
  const Tensor k = optional(v[1], "k");
  check_heads(q, "q", q);
  TORCH_CHECK_VALUE(real(q.scalar_type()), "q must be bf16 or fp32");
  const int64_t n = q.size(0), dim = q.size(2);
  if (k.defined()) {
    check_heads(k, "k", q);
    TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.size(0) == n && k.size(2) == dim, "k must be like q but for its heads");
  }
  TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == n && positions.device() == q.device() &&
                        (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
                    "positions must be int32 or int64 [", n, "] on the inputs' GPU");
  TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.scalar_type() == at::kDouble && frequencies.device() == q.device() &&
                        frequencies.size(0) >= 1 && 2 * frequencies.size(0) <= dim,
                    "the plan's frequencies must be a 1-D float64 tensor of at most dim / 2 elements on the inputs' GPU");
  const c10::cuda::CUDAGuard guard(q.device());
  const Heads hq = heads_of(q, false), hk = k.defined() ? heads_of(k, false) : Heads{};
  const Tensor at_ = positions.is_contiguous() ? positions : read_here(positions).contiguous();
  const Tensor f = frequencies.is_contiguous() ? frequencies : read_here(frequencies).contiguous();
  const Heads oq = heads_out(v[7], "out[0]", n, q.size(1), dim, q.scalar_type(), q);
  const Heads ok = k.defined() ? heads_out(v[8], "out[1]", n, k.size(1), dim, q.scalar_type(), q) : Heads{};
  bsgemm_rotary_args a{};
  a.q = hq.data();
  a.k = hk.data();
  a.q_out = oq.data();
  a.k_out = ok.data();
  a.positions = at_.data_ptr();
  a.frequencies = f.data_ptr<double>();
  a.q_stride = hq.stride;
  a.q_head_stride = hq.head_stride;
  a.k_stride = hk.stride;
  a.k_head_stride = hk.head_stride;
  a.q_out_stride = oq.stride;
  a.q_out_head_stride = oq.head_stride;
  a.k_out_stride = ok.stride;
  a.k_out_head_stride = ok.head_stride;
  a.tokens = extent(n);
  a.q_heads = extent(q.size(1));
  a.k_heads = k.defined() ? extent(k.size(1)) : 0;
  a.dim = extent(dim);
  a.rot = extent(2 * f.size(0));
  a.dtype = real_code(q.scalar_type());
  a.positions_64 = positions.scalar_type() == at::kLong;
  a.factor = number(v[4]);
  a.interleaved = integer(v[5]) != 0;
  a.inverse = integer(v[6]) != 0;
  if (!launch("bsgemm_rotary", q, {&hq.t, &hk.t, &at_, &f, &oq.t, &ok.t}, [&](bsg_stream_t s) { return bsgemm_rotary(&a, s); }))
    return nullptr;
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(oq.t));
  PyTuple_SET_ITEM(t, 1, wrap_or_none(ok.t));
  return t;
  END_HANDLE_TH_ERRORS
}

// paged_slots(cached, fresh, block_table, free_pages, page, tokens, first_free)
PyObject* paged_slots(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 7, "paged_slots takes 7 arguments");
  const Tensor& given = tensor(v[0], "cached");
  TORCH_CHECK_VALUE(given.is_cuda(), "cached must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(given.device());
  const Tensor cached = ints(given, "cached", -1, given);
  const int64_t requests = cached.size(0);
  const Tensor fresh = ints(tensor(v[1], "new"), "new", requests, given);
  const Tensor& table = tensor(v[2], "block_table");
  const Tensor free_pages = ints(tensor(v[3], "free_pages"), "free_pages", -1, given);
  Tensor first = optional(v[6], "first_free");
  if (first.defined()) first = ints(first, "first_free", 1, given);
  bsgemm_paged_slots_args a{};
  a.table_stride = table_stride(table, requests, given);
  a.page = small(v[4]);
  a.tokens = small(v[5]);
  TORCH_CHECK_VALUE(a.page >= 1 && a.tokens >= 0, "page_size must be at least 1 and tokens at least 0");
  const Tensor slots = make(given, {a.tokens}, at::kLong), whole = make(given, {a.tokens + 2 * requests + 2}, at::kInt);
  const Tensor positions = part(whole, 0, a.tokens), offsets = part(whole, a.tokens, requests + 1);
  const Tensor lengths = part(whole, a.tokens + requests + 1, requests), taken = part(whole, a.tokens + 2 * requests + 1, 1);
  a.cached = cached.data_ptr<int>();
  a.fresh = fresh.data_ptr<int>();
  a.block_table = table.data_ptr<int>();
  a.free_pages = free_pages.data_ptr<int>();
  a.first_free = first.defined() ? first.data_ptr<int>() : nullptr;
  a.slots = reinterpret_cast<long long*>(slots.data_ptr<int64_t>());
  a.positions = positions.data_ptr<int>();
  a.offsets = offsets.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.pages_taken = taken.data_ptr<int>();
  a.requests = extent(requests);
  a.columns = extent(table.size(1));
  a.free_count = extent(free_pages.size(0));
  if (!launch("bsgemm_paged_slots", given, {&cached, &fresh, &table, &free_pages, &first},
              [&](bsg_stream_t s) { return bsgemm_paged_slots(&a, s); }))
    return nullptr;
  PyObject* t = PyTuple_New(5);
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor* o : {&slots, &positions, &offsets, &lengths, &taken}) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(*o));
  return t;
  END_HANDLE_TH_ERRORS
}

Tensor slots_of(PyObject* o, int64_t n, const Tensor& like) {
  const Tensor& t = tensor(o, "slots");
  TORCH_CHECK_VALUE(t.dim() == 1 && (n < 0 || t.size(0) == n) && t.scalar_type() == at::kLong && t.device() == like.device(),
                    "slots must be a 1-D int64 tensor, one a token, on the cache's GPU");
  return t.is_contiguous() ? t : read_here(t).contiguous();
}
bsgemm_cache_rows cache_rows(const Heads& k, const Heads& v, const Tensor& slots) {
  bsgemm_cache_rows r{};
  r.k = k.data();
  r.v = v.data();
  r.slots = reinterpret_cast<const long long*>(slots.data_ptr<int64_t>());
  r.k_stride = k.stride;
  r.k_head_stride = k.head_stride;
  r.v_stride = v.stride;
  r.v_head_stride = v.head_stride;
  r.tokens = extent(slots.size(0));
  r.dtype = real_code(k.t.scalar_type());
  return r;
}

// cache_append(cache's four parts, k, v, slots)
PyObject* cache_append(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 7, "cache_append takes 7 arguments");
  const Cache c = cache_of(v);
  const Tensor& like = c.part[0];
  const Tensor &k = tensor(v[4], "k"), &x = tensor(v[5], "v");
  check_heads(k, "k", like);
  check_heads(x, "v", like);
  TORCH_CHECK_VALUE(k.size(1) == c.c.heads && k.size(2) == c.c.dim && x.sizes() == k.sizes() && real(k.scalar_type()) &&
                        x.scalar_type() == k.scalar_type(),
                    "k and v must be bf16 or fp32 [tokens, ", c.c.heads, ", ", c.c.dim, "]");
  const c10::cuda::CUDAGuard guard(like.device());
  const Tensor slots = slots_of(v[6], k.size(0), like);
  const Heads hk = heads_of(k, true), hv = heads_of(x, true);
  const bsgemm_cache_rows r = cache_rows(hk, hv, slots);
  if (!launch("bsgemm_cache_append", like, {&c.part[0], &c.part[1], &c.part[2], &c.part[3], &hk.t, &hv.t, &slots},
              [&](bsg_stream_t s) { return bsgemm_cache_append(&c.c, &r, s); }))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// cache_read(cache's four parts, slots)
PyObject* cache_read(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 5, "cache_read takes 5 arguments");
  const Cache c = cache_of(v);
  const Tensor& like = c.part[0];
  const c10::cuda::CUDAGuard guard(like.device());
  const Tensor slots = slots_of(v[4], -1, like);
  const int64_t n = slots.size(0);
  const Heads k = strides_of(make(like, {n, c.c.heads, c.c.dim}, at::kBFloat16));
  const Heads x = strides_of(make(like, {n, c.c.heads, c.c.dim}, at::kBFloat16));
  const bsgemm_cache_rows r = cache_rows(k, x, slots);
  if (!launch("bsgemm_cache_read", like, {&c.part[0], &c.part[1], &c.part[2], &c.part[3], &slots},
              [&](bsg_stream_t s) { return bsgemm_cache_read(&c.c, &r, s); }))
    return nullptr;
  return pair_of(k.t, x.t);
  END_HANDLE_TH_ERRORS
}

// cache_attention(q, cache's four parts, block_table, lengths, scale, out, workspace)
PyObject* cache_attention(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 10, "cache_attention takes 10 arguments");
  const Tensor& q = tensor(v[0], "q");
  const Cache c = cache_of(v + 1);
  const Tensor& table = tensor(v[5], "block_table");
  check_heads(q, "q", c.part[0]);
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 && q.size(2) == c.c.dim && c.c.heads > 0 && q.size(1) > 0 && q.size(1) % c.c.heads == 0,
                    "q must be bf16 [requests, a multiple of ", c.c.heads, " heads, ", c.c.dim, "]");
  const int64_t requests = q.size(0);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor lengths = ints(tensor(v[6], "lengths"), "lengths", requests, q);
  bsgemm_cache_attention_args a{};
  a.table_stride = table_stride(table, requests, q);
  const Heads hq = heads_of(q, true);
  const Heads out = heads_out(v[8], "out", requests, q.size(1), c.c.dim, at::kBFloat16, q);
  a.scale = scale_of(v[7], c.c.dim);
  a.q = hq.data();
  a.out = out.data();
  a.block_table = table.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.q_stride = hq.stride;
  a.q_head_stride = hq.head_stride;
  a.out_stride = out.stride;
  a.out_head_stride = out.head_stride;
  a.requests = extent(requests);
  a.q_heads = extent(q.size(1));
  a.columns = extent(table.size(1));
  const Tensor ws = workspace_of(v[9], bsgemm_cache_attention_workspace_size(&c.c, a.q_heads), q);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = ws.nbytes();
  if (!launch("bsgemm_cache_attention", q,
              {&hq.t, &c.part[0], &c.part[1], &c.part[2], &c.part[3], &table, &lengths, &out.t, &ws},
              [&](bsg_stream_t s) { return bsgemm_cache_attention(&c.c, &a, s); }))
    return nullptr;
  return THPVariable_Wrap(out.t);
  END_HANDLE_TH_ERRORS
}

// prompt_attention(q, k, v, offsets, offsets_k, causal, scale, out, return_lse)
PyObject* prompt_attention(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 9, "prompt_attention takes 9 arguments");
  const Tensor &q = tensor(v[0], "q"), &k = tensor(v[1], "k"), &x = tensor(v[2], "v");
  check_heads(q, "q", q);
  check_heads(k, "k", q);
  check_heads(x, "v", q);
  const int64_t n = q.size(0), heads = q.size(1), dim = q.size(2);
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && x.scalar_type() == at::kBFloat16,
                    "q, k and v must be bf16");
  TORCH_CHECK_VALUE(k.size(2) == dim && x.sizes() == k.sizes() && k.size(1) > 0 && heads > 0 && heads % k.size(1) == 0,
                    "k and v must be [tokens, heads, ", dim, "], q's heads a multiple of theirs");
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor offsets = ints(tensor(v[3], "offsets"), "offsets", -1, q);
  TORCH_CHECK_VALUE(offsets.size(0) >= 1, "offsets must hold at least one element");
  Tensor offsets_k = optional(v[4], "offsets_k");
  if (offsets_k.defined()) offsets_k = ints(offsets_k, "offsets_k", offsets.size(0), q);
  TORCH_CHECK_VALUE(offsets_k.defined() || k.size(0) == n, "k and v must have q's ", n, " rows unless offsets_k is given");
  const Heads hq = heads_of(q, true), hk = heads_of(k, true), hv = heads_of(x, true);
  const Heads out = heads_out(v[7], "out", n, heads, dim, at::kBFloat16, q);
  Tensor lse;
  if (integer(v[8]) != 0) lse = make(q, {n, heads}, at::kFloat);
  bsgemm_prompt_attention_args a{};
  a.q = hq.data();
  a.k = hk.data();
  a.v = hv.data();
  a.out = out.data();
  a.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
  a.offsets = offsets.data_ptr<int>();
  a.offsets_k = offsets_k.defined() ? offsets_k.data_ptr<int>() : nullptr;
  a.q_stride = hq.stride;
  a.q_head_stride = hq.head_stride;
  a.k_stride = hk.stride;
  a.k_head_stride = hk.head_stride;
  a.v_stride = hv.stride;
  a.v_head_stride = hv.head_stride;
  a.out_stride = out.stride;
  a.out_head_stride = out.head_stride;
  a.tokens = extent(n);
  a.tokens_k = extent(k.size(0));
  a.sequences = extent(offsets.size(0) - 1);
  a.q_heads = extent(heads);
  a.heads = extent(k.size(1));
  a.dim = extent(dim);
  a.causal = integer(v[5]) != 0;
  a.scale = scale_of(v[6], dim);
  // (new results leave no row as the allocator had it)
  const int fill_out = v[7] == Py_None, fill_lse = lse.defined();
  if (!launch("bsgemm_prompt_attention", q, {&hq.t, &hk.t, &hv.t, &offsets, &offsets_k, &out.t},
              [&](bsg_stream_t s) { return bsgemm_prompt_attention_fill(&a, fill_out, fill_lse, s); }))
    return nullptr;
  return lse.defined() ? pair_of(out.t, lse) : THPVariable_Wrap(out.t);
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(g_error, cls);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(epilogue_gemm), FAST(gated_backward),     FAST(layer_norm),
                         FAST(layer_norm_backward), FAST(dequantize), FAST(rotary), FAST(paged_slots),
                         FAST(cache_append), FAST(cache_read), FAST(cache_attention), FAST(prompt_attention),
                         {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bsgemm_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__bsgemm_ops() { return PyModule_Create(&module); }
