"""Operators around the block-scaled GEMMs: linear layers with bias, activation
and residual in the GEMM's epilogue, the gated feed-forward product and its
gradient, layer norm and its gradient, dequantise.

Together they are a transformer's feed-forward block with nothing but MX
elements between its kernels::

    q, sf = layer_norm(x, w, b, out_format="mxfp8")
    h, hs = gated_a8w8_mxfp8(q, W13, sf, W13_scale, activation="silu", out_format="mxfp8")
    x = linear_a8w8_mxfp8(h, W2, hs, W2_scale, residual=x)

The functions launch on the current stream and raise ValueError for a wrong
tensor, BsgemmError for a status of the library; there is no fallback.  They are
no autograd functions: a tensor that requires grad goes in and a result without
a graph comes out; gradients are calls of their own.  Their
checks, allocations and argument structs are in ``csrc/binding.cpp``
(``_build/_bsgemm_ops.so``), because a decode step's kernels are shorter than the
same work in Python.
"""
from __future__ import annotations

import ctypes
import importlib.util
from functools import lru_cache

import torch

from . import (KERNELS, LIB_PATH, BsgemmError, _B_FORMATS, _SCALE_U8, _record, _tuned, lib, pack_scales, tuning)

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


@lru_cache(None)
def native():
    """The operators' compiled entry points."""
    path = LIB_PATH.parent / "_bsgemm_ops.so"
    if not path.exists():
        raise RuntimeError(f"{path} is missing: build it with `python 355_1_trans_b200/build.py` "
                           "(there is no fallback implementation)")
    lib()
    spec = importlib.util.spec_from_file_location("_bsgemm_ops", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.set_error(BsgemmError)
    return module


def _activation(name):
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)}")
    return code


def _out_code(out_dtype, out_format):
    code = _OUT_DTYPES.get(out_dtype) if out_format is None else MX_FORMATS.get(out_format)
    if code is None:
        raise ValueError("out_dtype must be bfloat16 or float32, out_format None or one of %s" % sorted(MX_FORMATS))
    return code


def _scale_code(scale_format):
    if scale_format == "native":
        return 1
    if scale_format == "rowmajor":
        return 0
    raise ValueError("scale_format must be 'native' or 'rowmajor'")


def _kernel_code(kernel):
    code = KERNELS.get(kernel)
    if code is None:
        raise ValueError(f"kernel must be one of {sorted(KERNELS)}")
    return code


def _epilogue_gemm(gated, fp4, A, B, A_scale, B_scale, bias, activation, residual, out_dtype, out_format, out,
                   scale_format, b_format, split_k, workspace, grid_blocks, kernel):
    code = _activation(activation)
    fmt = _out_code(out_dtype, out_format)
    b_code = _B_FORMATS.get(b_format)
    if b_code is None:
        raise ValueError(f"b_format must be one of {sorted(_B_FORMATS)}")
    if kernel == "auto" and split_k == 0 and tuning.active() is not None and A.dim() == 2 and B.dim() == 2:
        kernel, split_k = _tuned("mxfp4" if fp4 else "mxfp8", A.shape[0], B.shape[0], A.shape[1] * (2 if fp4 else 1),
                                 kernel, split_k)
    return native().epilogue_gemm(gated, fp4, A, B, A_scale, B_scale, bias, code, residual, fmt, out,
                                  _scale_code(scale_format), b_code, split_k, workspace, grid_blocks,
                                  _kernel_code(kernel))


def linear_a8w8_mxfp8(A, B, A_scale, B_scale, *, bias=None, activation=None, residual=None, out_dtype=torch.bfloat16,
                      out_format: str | None = None, out=None, scale_format: str = "native", b_format: str = "raw",
                      split_k: int = 0, workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """activation(A B^T + bias) + residual, all in the MXFP8 GEMM's epilogue.

    A [M, K] and B [N, K] E4M3 with native (pack_scales, quantize) or row-major
    E8M0 scales; B raw or shuffle_weight(16,16) bytes (b_format "shuffle16").
    bias [N] and residual [M, N] bf16 or fp32, at any offset and stride (copied
    first where that is off 16 bytes); activation None, "relu", "gelu" (erf),
    "gelu_tanh" or "silu".  Returns C [M, N] of out_dtype, or with
    out_format "mxfp8" / "mxfp4" (N % 128 == 0) the elements and native scales
    that the next GEMM reads.  out: C, or (elements, scales); it may be the
    residual itself.  workspace None: allocated when K is split; False: none
    (decode-shaped calls then split K inside CTA clusters).  kernel, split_k
    and grid_blocks as in gemm_a8w8_mxfp8."""
    return _epilogue_gemm(False, False, A, B, A_scale, B_scale, bias, activation, residual, out_dtype, out_format, out,
                          scale_format, b_format, split_k, workspace, grid_blocks, kernel)


def linear_a4w4_mxfp4(A, B, A_scale, B_scale, *, bias=None, activation=None, residual=None, out_dtype=torch.bfloat16,
                      out_format: str | None = None, out=None, scale_format: str = "native", b_format: str = "raw",
                      split_k: int = 0, workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """linear_a8w8_mxfp8 on packed E2M1 operands: A [M, K/2], B [N, K/2] bytes, even k in the low nibble."""
    return _epilogue_gemm(False, True, A, B, A_scale, B_scale, bias, activation, residual, out_dtype, out_format, out,
                          scale_format, b_format, split_k, workspace, grid_blocks, kernel)


def gated_a8w8_mxfp8(A, B, A_scale, B_scale, *, activation="silu", out_dtype=torch.bfloat16,
                     out_format: str | None = None, out=None, scale_format: str = "native", split_k: int = 0,
                     workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """Gated feed-forward product activation(A Wg^T) * (A Wu^T) in one MXFP8 GEMM.

    A [M, K]; B [2F, K] both weights interleaved in blocks of 32 rows, with its
    scales (pack_gated).  Returns [M, F] of out_dtype, or with out_format
    "mxfp8" / "mxfp4" (F % 128 == 0) elements and native scales.  The other
    arguments as in linear_a8w8_mxfp8."""
    return _epilogue_gemm(True, False, A, B, A_scale, B_scale, None, activation, None, out_dtype, out_format, out,
                          scale_format, "raw", split_k, workspace, grid_blocks, kernel)


def gated_a4w4_mxfp4(A, B, A_scale, B_scale, *, activation="silu", out_dtype=torch.bfloat16,
                     out_format: str | None = None, out=None, scale_format: str = "native", split_k: int = 0,
                     workspace=None, grid_blocks: int = 0, kernel: str = "auto"):
    """gated_a8w8_mxfp8 on packed E2M1 operands: A [M, K/2], B [2F, K/2] bytes."""
    return _epilogue_gemm(True, True, A, B, A_scale, B_scale, None, activation, None, out_dtype, out_format, out,
                          scale_format, "raw", split_k, workspace, grid_blocks, kernel)


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

    _record((gate, up, gate_scale, up_scale), gate.device)
    return interleave(gate, up).view(gate.dtype), pack_scales(interleave(gate_scale, up_scale))


def _gated_backward(fp4, grad, A, B, A_scale, B_scale, activation, scale_format, need_input_grad, need_weight_grad,
                    workspace, grid_blocks, kernel):
    if not need_input_grad and not need_weight_grad:
        raise ValueError("need_input_grad or need_weight_grad must be set")
    return native().gated_backward(fp4, grad, A, B, A_scale, B_scale, _activation(activation), _scale_code(scale_format),
                                   bool(need_input_grad), bool(need_weight_grad), workspace, grid_blocks,
                                   _kernel_code(kernel))


def gated_a8w8_mxfp8_backward(grad, A, B, A_scale, B_scale, *, activation="silu", scale_format: str = "native",
                              need_input_grad: bool = True, need_weight_grad: bool = True, workspace=None,
                              grid_blocks: int = 0, kernel: str = "auto"):
    """Gradients of gated_a8w8_mxfp8 with respect to the values that its operands stand for.

    grad [M, F] bf16, any offset and stride, and the forward pass's operands.  Returns (dA [M, K],
    dWg [F, K], dWu [F, K]) in bf16, None for those not needed.  Both
    projections are computed again (nothing is kept from the forward pass);
    their gradients are rounded to bf16 before the two products that follow.
    workspace: bsgemm_gated_backward_workspace_size bytes, allocated when
    omitted."""
    return _gated_backward(False, grad, A, B, A_scale, B_scale, activation, scale_format, need_input_grad, need_weight_grad,
                           workspace, grid_blocks, kernel)


def gated_a4w4_mxfp4_backward(grad, A, B, A_scale, B_scale, *, activation="silu", scale_format: str = "native",
                              need_input_grad: bool = True, need_weight_grad: bool = True, workspace=None,
                              grid_blocks: int = 0, kernel: str = "auto"):
    """gated_a8w8_mxfp8_backward on packed E2M1 operands."""
    return _gated_backward(True, grad, A, B, A_scale, B_scale, activation, scale_format, need_input_grad, need_weight_grad,
                           workspace, grid_blocks, kernel)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, *, out_dtype=None, out_format: str | None = None,
               scale_format: str = "native", out=None, return_stats: bool = False):
    """Layer norm of each row of x [rows, cols] (bf16 or fp32, any row stride).

    weight and bias [cols] bf16 or fp32, or None.  Returns y of out_dtype
    (default x's), or with out_format "mxfp8" / "mxfp4" (cols % 128 == 0) the
    elements and E8M0 scales ("native" atoms or "rowmajor") that the GEMMs read:
    the same as quantize(layer_norm(x)) but rounded once, in one pass.  out: y
    (it may be x), or (elements, native scales).  return_stats: returns (y,
    mean, rstd), fp32 [rows], what layer_norm_backward needs."""
    if out_dtype is None and out_format is None:
        fmt = -1
    else:
        fmt = _out_code(out_dtype, out_format)
    return native().layer_norm(x, weight, bias, eps, fmt, not _scale_code(scale_format), out, return_stats)


def layer_norm_backward(dy, x, weight, mean, rstd, *, need_weight_grad: bool = True, out=None, workspace=None):
    """(dx, dweight, dbias) of layer_norm from dy and x (one type, [rows, cols]) and
    the mean and rstd that it returned.  dweight and dbias have the weight's
    type (x's when weight is None) and are None without need_weight_grad; their
    sums over rows are fp32 in an order that does not depend on timing.  out:
    dx, may be dy or x.  workspace:
    bsgemm_layer_norm_backward_workspace_size(rows, cols) bytes, allocated when
    omitted."""
    return native().layer_norm_backward(dy, x, weight, mean, rstd, bool(need_weight_grad), out, workspace)


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
    return native().dequantize(q, sf, fmt == "mxfp4", _scale_code(scale_format), out_dtype is torch.float32)
