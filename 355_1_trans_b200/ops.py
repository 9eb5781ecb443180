"""Operators around the block-scaled GEMMs: linear layers with bias, activation
and residual in the GEMM's epilogue, the gated feed-forward product and its
gradient, layer norm and its gradient, dequantise.

Together they are a transformer's feed-forward block with nothing but MX
elements between its kernels::

    q, sf = layer_norm(x, w, b, out_format="mxfp8")
    h, hs = gated_a8w8_mxfp8(q, W13, sf, W13_scale, activation="silu", out_format="mxfp8")
    x = linear_a8w8_mxfp8(h, W2, hs, W2_scale, residual=x)

As elsewhere in the package the functions check their tensors, fill a C-ABI
argument struct and launch on the current stream; there is no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import (FAMILY_MXFP4, FAMILY_MXFP8, KERNELS, LAYOUTS, SF_NATIVE, SF_ROWMAJOR, Args, BsgemmError, _B_FORMATS,
               _FP4, _FP8, _SCALE_U8, _tuned, lib, pack_scales)

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
MX_FORMATS = {"mxfp8": 2, "mxfp4": 3}                          # BSG_OUT_*
_OUT_DTYPES = {torch.bfloat16: 0, torch.float32: 1}            # BSG_OUT_* and BSG_IN_*
_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


class Epilogue(ctypes.Structure):
    """bsgemm_epilogue"""
    _fields_ = [("bias", _P), ("residual", _P), ("ptr_sfc", _P), ("stride_residual", _L), ("bias_dtype", _I),
                ("residual_dtype", _I), ("activation", _I), ("reserved", _I)]


class GatedGrad(ctypes.Structure):
    """bsgemm_gated_grad"""
    _fields_ = [("grad_h", _P), ("grad_a", _P), ("grad_gate", _P), ("grad_up", _P), ("stride_grad_h", _L),
                ("stride_grad_a", _L), ("stride_grad_w", _L), ("activation", _I), ("reserved", _I)]


class LayerNormArgs(ctypes.Structure):
    """bsgemm_layer_norm_args"""
    _fields_ = [("x", _P), ("weight", _P), ("bias", _P), ("y", _P), ("mean", _P), ("rstd", _P), ("sf", _P),
                ("ldx", _L), ("ldy", _L), ("ld_sf", _L), ("rows", _I), ("cols", _I), ("dtype", _I),
                ("param_dtype", _I), ("out_format", _I), ("sf_format", _I), ("eps", ctypes.c_float), ("reserved", _I)]


class LayerNormGradArgs(ctypes.Structure):
    """bsgemm_layer_norm_grad_args"""
    _fields_ = [("dy", _P), ("x", _P), ("weight", _P), ("mean", _P), ("rstd", _P), ("dx", _P), ("dweight", _P),
                ("dbias", _P), ("workspace", _P), ("workspace_bytes", ctypes.c_size_t), ("lddy", _L), ("ldx", _L),
                ("lddx", _L), ("rows", _I), ("cols", _I), ("dtype", _I), ("param_dtype", _I)]


# torch.cuda.Stream objects by (device, handle): record_stream wants the object,
# and looking the current one up costs ten times its handle.  A decode step's
# kernels run for a few microseconds, so what these functions cost on the host
# decides how fast a loop of them runs.
_streams: dict = {}


def _call(name, device, tensors, *args):
    """Launch on `device`'s current stream; the allocator learns that the
    caller's tensors are in use there (those made here belong to that stream)."""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(name, device, tensors, *args)
    handle = torch._C._cuda_getCurrentRawStream(index)
    status = getattr(lib(), name)(*args, handle)
    if status:
        raise BsgemmError(status, name)
    stream = _streams.get((index, handle))
    if stream is None:
        stream = _streams[index, handle] = torch.cuda.current_stream(device)
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def _scales_size(rows, kg):
    """native_scales_size without the call."""
    return (rows + 127) // 128 * ((kg + 3) // 4) * 512


def _rows(t):
    """(tensor, row stride) of a 2-D tensor with unit inner stride and rows that do not overlap."""
    rows, cols = t.shape
    if t.is_contiguous():
        return t, cols
    ld, inner = t.stride()
    if rows == 1:
        ld = cols
    if ld < cols or (inner != 1 and cols > 1):
        return t.contiguous(), cols
    return t, ld


def _mx_out(out, m, n, fmt, like):
    """(elements, native scales) of an MX output [m, n]."""
    if n % 128:
        raise ValueError(f"an {fmt} output needs a multiple of 128 columns")
    shape, dtype = ((m, n), torch.float8_e4m3fn) if fmt == "mxfp8" else ((m, n // 2), torch.uint8)
    size = _scales_size(m, n // 32)
    if out is None:
        return like.new_empty(shape, dtype=dtype), like.new_empty(size, dtype=torch.uint8)
    q, sf = out
    for t in (q, sf):
        if t.device != like.device or not t.is_contiguous():
            raise ValueError("out must hold contiguous tensors on the inputs' GPU")
    if tuple(q.shape) != shape or q.dtype not in (dtype, torch.uint8) or sf.dtype not in _SCALE_U8 or sf.numel() < size:
        raise ValueError(f"out must be ({fmt} elements {shape}, {size} scale bytes)")
    return q, sf


def _plain_out(out, shape, dtype, like):
    """(C, its row stride)"""
    if out is None:
        return like.new_empty(shape, dtype=dtype), shape[1]
    if tuple(out.shape) != shape or out.dtype != dtype or out.device != like.device or (
            out.shape[1] > 1 and out.stride(1) != 1):
        raise ValueError(f"out must be a tensor of shape {shape} and dtype {dtype} with unit inner stride")
    return out, out.stride(0) if shape[0] > 1 else shape[1]


def _workspace(workspace, need, like):
    """(tensor, whether it is the caller's)"""
    if workspace is None:
        return like.new_empty(need, dtype=torch.uint8), False
    if workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace needs {need} bytes")
    return workspace, True


def _operands(args, A, B, A_scale, B_scale, fp4, scale_format, b_format, kernel):
    """Checks A [m, k] and B [n, k] with their scales and fills their part of args; (m, n, k)."""
    if A.dim() != 2 or B.dim() != 2:
        raise ValueError("A and B must be 2-D")
    device = A.device
    if not A.is_cuda or B.device != device or A_scale.device != device or B_scale.device != device:
        raise ValueError("all inputs must be on the same GPU")
    ok_types = _FP4 if fp4 else _FP8
    if A.dtype not in ok_types or B.dtype not in ok_types:
        raise ValueError("A/B must hold %s bytes" % ("packed E2M1" if fp4 else "E4M3FN"))
    if A_scale.dtype not in _SCALE_U8 or B_scale.dtype not in _SCALE_U8:
        raise ValueError("scales must be E8M0 bytes")
    if kernel not in KERNELS:
        raise ValueError(f"kernel must be one of {sorted(KERNELS)}")
    if b_format not in _B_FORMATS:
        raise ValueError(f"b_format must be one of {sorted(_B_FORMATS)}")
    m, kb = A.shape
    n, kb_b = B.shape
    k = 2 * kb if fp4 else kb
    if kb_b != kb:
        raise ValueError("A and B disagree on K")
    lda, inner_a = A.stride()
    ldb, inner_b = B.stride()
    if inner_a != 1 or inner_b != 1:
        raise ValueError("A and B must have unit stride in the last dimension")
    kg = k // 32
    if scale_format == "native":
        for t, rows in ((A_scale, m), (B_scale, n)):
            if not t.is_contiguous() or t.numel() < _scales_size(rows, kg):
                raise ValueError(f"native scales of {rows} rows need {_scales_size(rows, kg)} contiguous bytes")
        args.sfa_format = args.sfb_format = SF_NATIVE
    elif scale_format == "rowmajor":
        for t, rows in ((A_scale, m), (B_scale, n)):
            if tuple(t.shape) != (rows, kg) or (kg > 1 and t.stride(1) != 1):
                raise ValueError(f"scale must be [{rows}, {kg}] with unit inner stride")
        args.sfa_format = args.sfb_format = SF_ROWMAJOR
        args.stride_sfa = A_scale.stride(0) if m > 1 else kg
        args.stride_sfb = B_scale.stride(0) if n > 1 else kg
    else:
        raise ValueError("scale_format must be 'native' or 'rowmajor'")
    args.ptr_a, args.ptr_b = A.data_ptr(), B.data_ptr()
    args.ptr_sfa, args.ptr_sfb = A_scale.data_ptr(), B_scale.data_ptr()
    args.m, args.n, args.k, args.batch = m, n, k, 1
    args.stride_a = lda if m > 1 else kb
    args.stride_b = ldb if n > 1 else kb
    args.layout = LAYOUTS["tn"]
    args.b_format = _B_FORMATS[b_format]
    args.kernel = KERNELS[kernel]
    return m, n, k


def _epilogue_gemm(name, A, B, A_scale, B_scale, *, fp4, gated, bias, activation, residual, out_dtype, out_format, out,
                   scale_format, b_format, split_k, workspace, grid_blocks, kernel):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)}")
    if out_format is None and out_dtype not in _OUT_DTYPES:
        raise ValueError("out_dtype must be bfloat16 or float32")
    if out_format is not None and out_format not in MX_FORMATS:
        raise ValueError(f"out_format must be one of {sorted(MX_FORMATS)}")
    args, epi = Args(), Epilogue()
    m, n, k = _operands(args, A, B, A_scale, B_scale, fp4, scale_format, b_format, kernel)
    if gated and n % 64:
        raise ValueError("B must hold whole blocks of 32 gate and 32 up rows (pack_gated)")
    n_out = n // 2 if gated else n
    sf = None
    if out_format is None:
        c, args.stride_c = _plain_out(out, (m, n_out), out_dtype, A)
        result = c
        args.out_dtype = _OUT_DTYPES[out_dtype]
    else:
        result = c, sf = _mx_out(out, m, n_out, out_format, A)
        args.stride_c = c.shape[1]
        args.out_dtype = MX_FORMATS[out_format]
        epi.ptr_sfc = sf.data_ptr()
    args.ptr_c = c.data_ptr()
    epi.activation = ACTIVATIONS[activation]
    if bias is not None:
        if bias.shape != (n,) or bias.dtype not in _OUT_DTYPES or bias.device != A.device or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous bf16 or fp32 tensor of {n} elements")
        epi.bias, epi.bias_dtype = bias.data_ptr(), _OUT_DTYPES[bias.dtype]
    if residual is not None:
        if residual.shape != (m, n) or residual.dtype not in _OUT_DTYPES or residual.device != A.device:
            raise ValueError(f"residual must be a bf16 or fp32 tensor of shape {(m, n)}")
        residual, ld = _rows(residual)
        epi.residual, epi.residual_dtype, epi.stride_residual = residual.data_ptr(), _OUT_DTYPES[residual.dtype], ld
    kernel, split_k = _tuned("mxfp4" if fp4 else "mxfp8", m, n, k, kernel, split_k)
    args.kernel, args.split_k, args.grid_blocks = KERNELS[kernel], split_k, grid_blocks
    tensors = [A, B, A_scale, B_scale, bias, residual]
    if out is not None:
        tensors += (c, sf)
    if workspace is not False and m > 0:
        need = lib().bsgemm_epilogue_workspace_size(FAMILY_MXFP4 if fp4 else FAMILY_MXFP8, ctypes.byref(args))
        if need:
            workspace, given = _workspace(workspace, need, A)
            args.workspace = workspace.data_ptr()
            args.workspace_bytes = workspace.numel() * workspace.element_size()
            if given:
                tensors.append(workspace)
    _call(name, A.device, tensors, ctypes.byref(args), ctypes.byref(epi))
    return result


def linear_a8w8_mxfp8(A, B, A_scale, B_scale, *, bias=None, activation=None, residual=None, out_dtype=torch.bfloat16,
                      out_format: str | None = None, out=None, scale_format: str = "native", b_format: str = "raw",
                      split_k: int = 0, workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """activation(A B^T + bias) + residual, all in the MXFP8 GEMM's epilogue.

    A [M, K] and B [N, K] E4M3 with native (pack_scales, quantize) or row-major
    E8M0 scales; B raw or shuffle_weight(16,16) bytes (b_format "shuffle16").
    bias [N] and residual [M, N] bf16 or fp32; activation None, "relu", "gelu"
    (erf), "gelu_tanh" or "silu".  Returns C [M, N] of out_dtype, or with
    out_format "mxfp8" / "mxfp4" (N % 128 == 0) the elements and native scales
    that the next GEMM reads.  out: C, or (elements, scales); it may be the
    residual itself.  workspace None: allocated when K is split; False: none
    (decode-shaped calls then split K inside CTA clusters).  kernel, split_k
    and grid_blocks as in gemm_a8w8_mxfp8."""
    return _epilogue_gemm("bsgemm_a8w8_mxfp8_linear", A, B, A_scale, B_scale, fp4=False, gated=False, bias=bias,
                          activation=activation, residual=residual, out_dtype=out_dtype, out_format=out_format, out=out,
                          scale_format=scale_format, b_format=b_format, split_k=split_k, workspace=workspace,
                          grid_blocks=grid_blocks, kernel=kernel)


def linear_a4w4_mxfp4(A, B, A_scale, B_scale, *, bias=None, activation=None, residual=None, out_dtype=torch.bfloat16,
                      out_format: str | None = None, out=None, scale_format: str = "native", b_format: str = "raw",
                      split_k: int = 0, workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """linear_a8w8_mxfp8 on packed E2M1 operands: A [M, K/2], B [N, K/2] bytes, even k in the low nibble."""
    return _epilogue_gemm("bsgemm_a4w4_mxfp4_linear", A, B, A_scale, B_scale, fp4=True, gated=False, bias=bias,
                          activation=activation, residual=residual, out_dtype=out_dtype, out_format=out_format, out=out,
                          scale_format=scale_format, b_format=b_format, split_k=split_k, workspace=workspace,
                          grid_blocks=grid_blocks, kernel=kernel)


def gated_a8w8_mxfp8(A, B, A_scale, B_scale, *, activation="silu", out_dtype=torch.bfloat16,
                     out_format: str | None = None, out=None, scale_format: str = "native", split_k: int = 0,
                     workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """Gated feed-forward product activation(A Wg^T) * (A Wu^T) in one MXFP8 GEMM.

    A [M, K]; B [2F, K] both weights interleaved in blocks of 32 rows, with its
    scales (pack_gated).  Returns [M, F] of out_dtype, or with out_format
    "mxfp8" / "mxfp4" (F % 128 == 0) elements and native scales.  The other
    arguments as in linear_a8w8_mxfp8."""
    return _epilogue_gemm("bsgemm_a8w8_mxfp8_gated", A, B, A_scale, B_scale, fp4=False, gated=True, bias=None,
                          activation=activation, residual=None, out_dtype=out_dtype, out_format=out_format, out=out,
                          scale_format=scale_format, b_format="raw", split_k=split_k, workspace=workspace,
                          grid_blocks=grid_blocks, kernel=kernel)


def gated_a4w4_mxfp4(A, B, A_scale, B_scale, *, activation="silu", out_dtype=torch.bfloat16,
                     out_format: str | None = None, out=None, scale_format: str = "native", split_k: int = 0,
                     workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """gated_a8w8_mxfp8 on packed E2M1 operands: A [M, K/2], B [2F, K/2] bytes."""
    return _epilogue_gemm("bsgemm_a4w4_mxfp4_gated", A, B, A_scale, B_scale, fp4=True, gated=True, bias=None,
                          activation=activation, residual=None, out_dtype=out_dtype, out_format=out_format, out=out,
                          scale_format=scale_format, b_format="raw", split_k=split_k, workspace=workspace,
                          grid_blocks=grid_blocks, kernel=kernel)


def pack_gated(gate, up, gate_scale, up_scale):
    """(B, B_scale) of the gated product from its two weights, once at load time.

    gate, up: [F, K] E4M3 or [F, K/2] packed E2M1 bytes, F % 32 == 0, with
    row-major E8M0 scales [F, K/32].  B [2F, ...] holds 32 gate rows, then the
    32 up rows of the same columns, and so on; B_scale is in native atoms."""
    if gate.dim() != 2 or gate.shape != up.shape or gate.dtype != up.dtype or gate.shape[0] % 32:
        raise ValueError("gate and up must be 2-D, alike, with a multiple of 32 rows")
    if gate_scale.shape != up_scale.shape or gate_scale.dim() != 2 or gate_scale.shape[0] != gate.shape[0]:
        raise ValueError("gate_scale and up_scale must be [F, K/32]")
    if gate_scale.dtype not in _SCALE_U8 or up_scale.dtype not in _SCALE_U8:
        raise ValueError("scales must be E8M0 bytes")
    if not gate.is_cuda or any(t.device != gate.device for t in (up, gate_scale, up_scale)):
        raise ValueError("all inputs must be on the same GPU")

    def interleave(a, b):
        a, b = (t.contiguous().view(torch.uint8).reshape(-1, 32, t.shape[1]) for t in (a, b))
        return torch.stack((a, b), dim=1).reshape(-1, a.shape[2])

    return interleave(gate, up).view(gate.dtype), pack_scales(interleave(gate_scale, up_scale))


def _gated_backward(name, grad, A, B, A_scale, B_scale, *, fp4, activation, scale_format, need_input_grad,
                    need_weight_grad, workspace, grid_blocks, kernel):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)}")
    if not need_input_grad and not need_weight_grad:
        raise ValueError("need_input_grad or need_weight_grad must be set")
    args, g = Args(), GatedGrad()
    m, n, k = _operands(args, A, B, A_scale, B_scale, fp4, scale_format, "raw", kernel)
    if n % 64:
        raise ValueError("B must hold whole blocks of 32 gate and 32 up rows (pack_gated)")
    device, f = A.device, n // 2
    if grad.shape != (m, f) or grad.dtype != torch.bfloat16 or grad.device != device:
        raise ValueError(f"grad must be a bf16 tensor of shape {(m, f)} on the inputs' GPU")
    grad, g.stride_grad_h = _rows(grad)
    g.grad_h = grad.data_ptr()
    g.activation = ACTIVATIONS[activation]
    grad_a = grad_gate = grad_up = None
    if need_input_grad:
        grad_a = grad.new_empty((m, k))
        # (a tensor of no rows has no address; the call wants one for "this gradient, please")
        g.grad_a, g.stride_grad_a = grad_a.data_ptr() or B.data_ptr(), k
    if need_weight_grad:
        grad_gate, grad_up = grad.new_empty((f, k)), grad.new_empty((f, k))
        g.grad_gate, g.grad_up, g.stride_grad_w = grad_gate.data_ptr(), grad_up.data_ptr(), k
    args.grid_blocks = grid_blocks
    need = lib().bsgemm_gated_backward_workspace_size(FAMILY_MXFP4 if fp4 else FAMILY_MXFP8, ctypes.byref(args))
    workspace, given = _workspace(workspace, need, A)
    args.workspace = workspace.data_ptr()
    args.workspace_bytes = workspace.numel() * workspace.element_size()
    _call(name, device, (grad, A, B, A_scale, B_scale, workspace if given else None), ctypes.byref(args), ctypes.byref(g))
    return grad_a, grad_gate, grad_up


def gated_a8w8_mxfp8_backward(grad, A, B, A_scale, B_scale, *, activation="silu", scale_format: str = "native",
                              need_input_grad: bool = True, need_weight_grad: bool = True, workspace=None,
                              grid_blocks: int = 0, kernel: str = "auto"):
    """Gradients of gated_a8w8_mxfp8 with respect to the values that its operands stand for.

    grad [M, F] bf16 and the forward pass's operands.  Returns (dA [M, K],
    dWg [F, K], dWu [F, K]) in bf16, None for those not needed.  Both
    projections are computed again (nothing is kept from the forward pass);
    their gradients are rounded to bf16 before the two products that follow.
    workspace: bsgemm_gated_backward_workspace_size bytes, allocated when
    omitted."""
    return _gated_backward("bsgemm_a8w8_mxfp8_gated_backward", grad, A, B, A_scale, B_scale, fp4=False,
                           activation=activation, scale_format=scale_format, need_input_grad=need_input_grad,
                           need_weight_grad=need_weight_grad, workspace=workspace, grid_blocks=grid_blocks, kernel=kernel)


def gated_a4w4_mxfp4_backward(grad, A, B, A_scale, B_scale, *, activation="silu", scale_format: str = "native",
                              need_input_grad: bool = True, need_weight_grad: bool = True, workspace=None,
                              grid_blocks: int = 0, kernel: str = "auto"):
    """gated_a8w8_mxfp8_backward on packed E2M1 operands."""
    return _gated_backward("bsgemm_a4w4_mxfp4_gated_backward", grad, A, B, A_scale, B_scale, fp4=True,
                           activation=activation, scale_format=scale_format, need_input_grad=need_input_grad,
                           need_weight_grad=need_weight_grad, workspace=workspace, grid_blocks=grid_blocks, kernel=kernel)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

def _norm_input(x, weight, bias):
    """Checks x and the parameters; the parameters' type."""
    if x.dim() != 2 or x.dtype not in _OUT_DTYPES or not x.is_cuda or x.shape[1] < 1:
        raise ValueError("x must be a 2-D bf16 or fp32 CUDA tensor")
    dtype = None
    for p in (weight, bias):
        if p is None:
            continue
        if p.shape != x.shape[1:] or p.dtype not in _OUT_DTYPES or p.device != x.device or not p.is_contiguous():
            raise ValueError(f"weight and bias must be contiguous bf16 or fp32 tensors of {x.shape[1]} elements")
        if dtype is not None and p.dtype != dtype:
            raise ValueError("weight and bias must have one type")
        dtype = p.dtype
    return dtype or x.dtype


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, *, out_dtype=None, out_format: str | None = None,
               scale_format: str = "native", out=None, return_stats: bool = False):
    """Layer norm of each row of x [rows, cols] (bf16 or fp32, any row stride).

    weight and bias [cols] bf16 or fp32, or None.  Returns y of out_dtype
    (default x's), or with out_format "mxfp8" / "mxfp4" (cols % 128 == 0) the
    elements and E8M0 scales ("native" atoms or "rowmajor") that the GEMMs read:
    the same as quantize(layer_norm(x)) but rounded once, in one pass.  out: y
    (it may be x), or (elements, native scales).  return_stats: returns (y,
    mean, rstd), fp32 [rows], what layer_norm_backward needs."""
    param_dtype = _norm_input(x, weight, bias)
    if out_format is not None and out_format not in MX_FORMATS:
        raise ValueError(f"out_format must be one of {sorted(MX_FORMATS)}")
    if scale_format not in ("native", "rowmajor"):
        raise ValueError("scale_format must be 'native' or 'rowmajor'")
    x, ldx = _rows(x)
    if out_format is not None and (x.data_ptr() % 16 or ldx * x.element_size() % 16):
        x, ldx = x.clone(memory_format=torch.contiguous_format), x.shape[1]
    rows, cols = x.shape
    sf = mean = rstd = None
    sf_format = ld_sf = 0
    if out_format is None:
        out_dtype = out_dtype or x.dtype
        if out_dtype not in _OUT_DTYPES:
            raise ValueError("out_dtype must be bfloat16 or float32")
        y, ldy = _plain_out(out, (rows, cols), out_dtype, x)
        result, fmt = (y,), _OUT_DTYPES[out_dtype]
    else:
        if scale_format == "rowmajor" and out is not None:
            raise ValueError("out takes native scales")
        y, sf = _mx_out(out, rows, cols, out_format, x)
        if scale_format == "rowmajor":
            sf = x.new_empty((rows, cols // 32), dtype=torch.uint8)
            sf_format, ld_sf = SF_ROWMAJOR, cols // 32
        result, fmt, ldy = (y, sf), MX_FORMATS[out_format], y.shape[1]
    if return_stats:
        mean, rstd = x.new_empty((2, rows), dtype=torch.float32).unbind(0)
        result += (mean, rstd)
    a = LayerNormArgs(x.data_ptr(), weight.data_ptr() if weight is not None else None,
                      bias.data_ptr() if bias is not None else None, y.data_ptr(),
                      mean.data_ptr() if return_stats else None, rstd.data_ptr() if return_stats else None,
                      sf.data_ptr() if sf is not None else None, ldx, ldy, ld_sf, rows, cols, _OUT_DTYPES[x.dtype],
                      _OUT_DTYPES[param_dtype], fmt, sf_format, eps, 0)
    tensors = (x, weight, bias) if out is None else (x, weight, bias, y, sf)
    _call("bsgemm_layer_norm", x.device, tensors, ctypes.byref(a))
    return result if len(result) > 1 else y


def layer_norm_backward(dy, x, weight, mean, rstd, *, need_weight_grad: bool = True, out=None, workspace=None):
    """(dx, dweight, dbias) of layer_norm from dy and x (one type, [rows, cols]) and
    the mean and rstd that it returned.  dweight and dbias have the weight's
    type (x's when weight is None) and are None without need_weight_grad; their
    sums over rows are fp32 in an order that does not depend on timing.  out:
    dx, may be dy or x.  workspace:
    bsgemm_layer_norm_backward_workspace_size(rows, cols) bytes, allocated when
    omitted."""
    param_dtype = _norm_input(x, weight, None)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must be like x")
    rows, cols = x.shape
    for s in (mean, rstd):
        if s.shape != x.shape[:1] or s.dtype != torch.float32 or s.device != x.device or not s.is_contiguous():
            raise ValueError(f"mean and rstd must be contiguous fp32 tensors of {rows} elements")
    x, ldx = _rows(x)
    dy, lddy = _rows(dy)
    dx, lddx = _plain_out(out, (rows, cols), x.dtype, x)
    dweight = dbias = None
    if need_weight_grad:
        dweight, dbias = x.new_empty((2, cols), dtype=param_dtype).unbind(0)
    need = lib().bsgemm_layer_norm_backward_workspace_size(rows, cols)
    workspace, given = _workspace(workspace, need, x)
    a = LayerNormGradArgs(dy.data_ptr(), x.data_ptr(), weight.data_ptr() if weight is not None else None, mean.data_ptr(),
                          rstd.data_ptr(), dx.data_ptr(), dweight.data_ptr() if need_weight_grad else None,
                          dbias.data_ptr() if need_weight_grad else None, workspace.data_ptr(),
                          workspace.numel() * workspace.element_size(), lddy, ldx, lddx, rows, cols, _OUT_DTYPES[x.dtype],
                          _OUT_DTYPES[param_dtype])
    _call("bsgemm_layer_norm_backward", x.device,
          (dy, x, weight, mean, rstd, dx if out is not None else None, workspace if given else None), ctypes.byref(a))
    return dx, dweight, dbias


# ---------------------------------------------------------------------------
# dequantise
# ---------------------------------------------------------------------------

def dequantize(q, sf, fmt: str = "mxfp8", *, scale_format: str = "native", out_dtype=torch.bfloat16):
    """The values [rows, cols] that MX elements and their scales stand for, the
    inverse of quantize for fmt "mxfp8" and "mxfp4"; exact in bf16 down to its
    subnormals."""
    if fmt not in MX_FORMATS:
        raise ValueError(f"fmt must be one of {sorted(MX_FORMATS)}")
    if out_dtype not in _OUT_DTYPES:
        raise ValueError("out_dtype must be bfloat16 or float32")
    if q.dim() != 2 or not q.is_cuda or q.dtype not in (_FP8 if fmt == "mxfp8" else _FP4):
        raise ValueError("q must be a 2-D CUDA tensor of %s bytes" % ("E4M3FN" if fmt == "mxfp8" else "packed E2M1"))
    if sf.dtype not in _SCALE_U8 or sf.device != q.device:
        raise ValueError("sf must hold E8M0 bytes on q's GPU")
    rows, cols = q.shape[0], q.shape[1] * (2 if fmt == "mxfp4" else 1)
    ld_sf = 0
    if scale_format == "native":
        if not sf.is_contiguous() or sf.numel() < _scales_size(rows, cols // 32):
            raise ValueError(f"native scales need {_scales_size(rows, cols // 32)} contiguous bytes")
    elif scale_format == "rowmajor":
        if tuple(sf.shape) != (rows, cols // 32):
            raise ValueError(f"sf must be [{rows}, {cols // 32}]")
        sf, ld_sf = _rows(sf)
    else:
        raise ValueError("scale_format must be 'native' or 'rowmajor'")
    q, ldq = _rows(q)
    y = q.new_empty((rows, cols), dtype=out_dtype)
    _call("bsgemm_dequantize", q.device, (q, sf), q.data_ptr(), ldq, sf.data_ptr(),
          SF_NATIVE if scale_format == "native" else SF_ROWMAJOR, ld_sf, 0 if fmt == "mxfp8" else 1, rows, cols,
          y.data_ptr(), _OUT_DTYPES[out_dtype], cols)
    return y
