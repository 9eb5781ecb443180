"""Operators around the GEMMs without a GPU: what their entry points refuse
before any CUDA call, and the argument structs."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def ops(bs):
    import importlib
    return importlib.import_module("355_1_trans_b200.ops")


@pytest.mark.parametrize("struct", ["Epilogue", "GatedGrad", "LayerNormArgs", "LayerNormGradArgs"])
def test_structs_match_the_header(ops, struct):
    """Field names and order as in include/bsgemm_b200.h."""
    cls = getattr(ops, struct)
    name = cls.__doc__.strip()
    text = (ROOT / "include" / "bsgemm_b200.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = re.findall(r"(\w+)\s*;", body)
    assert fields == [f for f, _ in cls._fields_]


def gemm_args(bs, m=64, n=256, k=256):
    a = bs.Args()
    bs.lib().bsgemm_args_init(ctypes.byref(a))
    a.ptr_a, a.ptr_b, a.ptr_c, a.ptr_sfa, a.ptr_sfb = (i << 30 for i in range(1, 6))
    a.m, a.n, a.k = m, n, k
    a.stride_a = a.stride_b = k
    a.stride_c = n
    a.sfa_format = a.sfb_format = bs.SF_NATIVE
    return a


def change(obj, **kw):
    for key, value in kw.items():
        setattr(obj, key, value)


@pytest.mark.parametrize("entry", ["bsgemm_a8w8_mxfp8_linear", "bsgemm_a8w8_mxfp8_gated"])
def test_epilogue_refusals(bs, ops, entry):
    fn = getattr(bs.lib(), entry)
    gated = entry.endswith("gated")

    def status(epi=None, **kw):
        a, e = gemm_args(bs), ops.Epilogue()
        if gated:
            a.stride_c = 128
        change(a, **kw)
        change(e, **(epi or {}))
        return fn(ctypes.byref(a), ctypes.byref(e), None)

    a, e = gemm_args(bs), ops.Epilogue()
    assert fn(None, ctypes.byref(e), None) == bs.ERR_INVALID_VALUE
    assert fn(ctypes.byref(a), None, None) == bs.ERR_INVALID_VALUE
    for field in ("ptr_a", "ptr_b", "ptr_c", "ptr_sfa", "ptr_sfb"):
        assert status(**{field: None}) == bs.ERR_INVALID_VALUE, field
    for kw in ({"m": -1}, {"n": 0}, {"k": 0}, {"k": 192}, {"batch": 2}, {"split_k": -1}, {"kernel": 9}, {"out_dtype": 4},
               {"out_dtype": -1}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    for kw in ({"layout": bs.LAYOUTS["nn"]}, {"kernel": bs.KERNELS["wide"]}, {"b_format": bs.B_KPANEL128},
               {"sfa_format": bs.SF_KMAJOR_T}):
        assert status(**kw) == bs.ERR_UNSUPPORTED, kw
    for kw in ({"ptr_a": (1 << 30) + 8}, {"ptr_b": (2 << 30) + 4}, {"ptr_c": (3 << 30) + 2}, {"stride_a": 248},
               {"stride_a": 264}, {"stride_b": 240}, {"stride_c": 100}, {"ptr_sfa": (4 << 30) + 4}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw
    assert status({"activation": 5}) == bs.ERR_INVALID_VALUE
    assert status({"activation": -1}) == bs.ERR_INVALID_VALUE
    assert status(ptr_c=1 << 30) == bs.ERR_INVALID_VALUE            # C over A
    assert status(ptr_c=(2 << 30) + 1024) == bs.ERR_INVALID_VALUE   # C inside B
    assert status(out_dtype=2) == bs.ERR_INVALID_VALUE              # MX output without scales
    assert status({"ptr_sfc": 3 << 30}, out_dtype=2) == bs.ERR_INVALID_VALUE   # scales over C
    if gated:
        assert status(n=224) == bs.ERR_INVALID_VALUE
        assert status({"bias": 6 << 30}) == bs.ERR_UNSUPPORTED
        assert status({"residual": 6 << 30, "stride_residual": 256}) == bs.ERR_UNSUPPORTED
        assert status(b_format=bs.B_SHUFFLE16) == bs.ERR_UNSUPPORTED
        assert status({"ptr_sfc": 7 << 30}, out_dtype=2, n=192) == bs.ERR_INVALID_VALUE   # 96 columns of MX elements
    else:
        assert status(n=260, stride_c=264) == bs.ERR_ALIGNMENT
        assert status({"bias": (6 << 30) + 2}) == bs.ERR_ALIGNMENT
        assert status({"bias": 6 << 30, "bias_dtype": 2}) == bs.ERR_INVALID_VALUE
        assert status({"bias": 3 << 30}) == bs.ERR_INVALID_VALUE
        assert status({"residual": 6 << 30, "stride_residual": 255}) == bs.ERR_ALIGNMENT
        assert status({"residual": 6 << 30, "stride_residual": 260}) == bs.ERR_ALIGNMENT
        assert status({"residual": 6 << 30, "stride_residual": 256, "residual_dtype": 7}) == bs.ERR_INVALID_VALUE
        # a shifted residual under C, and C's own buffer as another type
        assert status({"residual": (3 << 30) + 16, "stride_residual": 256}) == bs.ERR_INVALID_VALUE
        assert status({"residual": 3 << 30, "stride_residual": 256, "residual_dtype": 1}) == bs.ERR_INVALID_VALUE
    assert status(m=0, ptr_a=None, ptr_sfa=None, ptr_c=None) == bs.OK   # no rows: nothing to do


def test_gated_backward_refusals(bs, ops):
    fn = bs.lib().bsgemm_a8w8_mxfp8_gated_backward

    def status(grad=None, **kw):
        a, g = gemm_args(bs), ops.GatedGrad()
        a.workspace, a.workspace_bytes = 12 << 30, 1 << 30
        change(g, grad_h=6 << 30, grad_a=7 << 30, grad_gate=8 << 30, grad_up=9 << 30, stride_grad_h=128,
               stride_grad_a=256, stride_grad_w=256)
        change(a, **kw)
        change(g, **(grad or {}))
        return fn(ctypes.byref(a), ctypes.byref(g), None)

    assert fn(None, None, None) == bs.ERR_INVALID_VALUE
    assert status(ptr_b=None) == bs.ERR_INVALID_VALUE
    assert status(n=224) == bs.ERR_INVALID_VALUE
    assert status({"grad_h": None}) == bs.ERR_INVALID_VALUE
    assert status({"grad_up": None}) == bs.ERR_INVALID_VALUE
    assert status({"grad_a": None, "grad_gate": None, "grad_up": None}) == bs.ERR_INVALID_VALUE
    assert status({"activation": 9}) == bs.ERR_INVALID_VALUE
    assert status(kernel=bs.KERNELS["swap"]) == bs.ERR_UNSUPPORTED
    assert status(split_k=2) == bs.ERR_UNSUPPORTED
    for grad in ({"stride_grad_h": 120}, {"stride_grad_h": 132}, {"stride_grad_a": 248}, {"stride_grad_w": 252},
                 {"grad_a": (7 << 30) + 8}, {"grad_h": (6 << 30) + 2}):
        assert status(grad) == bs.ERR_ALIGNMENT, grad
    assert status({"grad_up": 8 << 30}) == bs.ERR_INVALID_VALUE        # two outputs in one place
    assert status({"grad_a": 1 << 30}) == bs.ERR_INVALID_VALUE         # over A
    assert status({"grad_a": 6 << 30}) == bs.ERR_INVALID_VALUE         # over its gradient
    assert status({"grad_gate": 12 << 30}) == bs.ERR_INVALID_VALUE     # inside the workspace
    a = gemm_args(bs)
    rows = bs.lib().bsgemm_gated_backward_workspace_size(bs.FAMILY_MXFP8, ctypes.byref(a))
    assert rows == 2 * (64 * 256 + 64 * 256 + 256 * 256)
    a.sfa_format = bs.SF_ROWMAJOR
    assert bs.lib().bsgemm_gated_backward_workspace_size(bs.FAMILY_MXFP8, ctypes.byref(a)) == rows + 1024
    assert bs.lib().bsgemm_gated_backward_workspace_size(bs.FAMILY_FP8_BLOCK, ctypes.byref(a)) == 0


def test_layer_norm_refusals(bs, ops):
    def forward(**kw):
        a = ops.LayerNormArgs(x=1 << 30, y=2 << 30, weight=3 << 30, bias=4 << 30, ldx=256, ldy=256, rows=4, cols=256,
                              eps=1e-5)
        change(a, **kw)
        return bs.lib().bsgemm_layer_norm(ctypes.byref(a), None)

    assert bs.lib().bsgemm_layer_norm(None, None) == bs.ERR_INVALID_VALUE
    for kw in ({"x": None}, {"y": None}, {"rows": -1}, {"cols": 0}, {"dtype": 2}, {"param_dtype": -1}, {"out_format": 4},
               {"ldx": 255}, {"ldy": 0}, {"eps": -1.0}, {"eps": float("nan")}, {"mean": 5 << 30}, {"out_format": 2},
               {"out_format": 2, "sf": 6 << 30, "cols": 96}, {"out_format": 2, "sf": 6 << 30, "sf_format": 2},
               {"out_format": 2, "sf": 6 << 30, "sf_format": 1, "ld_sf": 7}, {"y": (1 << 30) + 512}):
        assert forward(**kw) == bs.ERR_INVALID_VALUE, kw
    assert forward(cols=20000, ldx=20000, ldy=20000) == bs.ERR_UNSUPPORTED
    for kw in ({"x": (1 << 30) + 1}, {"y": (2 << 30) + 1}, {"weight": (3 << 30) + 1}, {"mean": (5 << 30) + 2, "rstd": 6 << 30},
               {"out_format": 2, "sf": 6 << 30, "x": (1 << 30) + 2}, {"out_format": 2, "sf": 6 << 30, "ldy": 264},
               {"out_format": 2, "sf": (6 << 30) + 8}):
        assert forward(**kw) == bs.ERR_ALIGNMENT, kw
    assert forward(rows=0, x=None, y=None) == bs.OK

    def backward(**kw):
        a = ops.LayerNormGradArgs(dy=1 << 30, x=2 << 30, weight=3 << 30, mean=4 << 30, rstd=5 << 30, dx=6 << 30,
                                  dweight=7 << 30, dbias=8 << 30, workspace=9 << 30, workspace_bytes=1 << 30, lddy=256,
                                  ldx=256, lddx=256, rows=4, cols=256)
        change(a, **kw)
        return bs.lib().bsgemm_layer_norm_backward(ctypes.byref(a), None)

    assert bs.lib().bsgemm_layer_norm_backward(None, None) == bs.ERR_INVALID_VALUE
    for kw in ({"x": None}, {"dy": None}, {"dx": None}, {"mean": None}, {"rstd": None}, {"rows": -1}, {"cols": 0},
               {"lddx": 255}, {"dtype": 3}, {"dx": (1 << 30) + 512}, {"dx": 2 << 30, "lddx": 264}):
        assert backward(**kw) == bs.ERR_INVALID_VALUE, kw
    assert backward(cols=16385, ldx=16385, lddy=16385, lddx=16385) == bs.ERR_UNSUPPORTED
    for kw in ({"dweight": (7 << 30) + 1}, {"dx": (6 << 30) + 1}, {"mean": (4 << 30) + 2}):
        assert backward(**kw) == bs.ERR_ALIGNMENT, kw


def test_dequantize_refusals(bs):
    fn = bs.lib().bsgemm_dequantize
    good = [1 << 30, 256, 2 << 30, bs.SF_NATIVE, 0, 0, 4, 256, 3 << 30, 0, 256, None]

    def status(**at):
        a = list(good)
        for i, v in at.items():
            a[int(i[1:])] = v
        return fn(*a)

    for at in ({"_0": None}, {"_2": None}, {"_8": None}, {"_3": 2}, {"_5": 2}, {"_6": -1}, {"_7": 0}, {"_7": 160},
               {"_9": 2}, {"_3": 1, "_4": 7}, {"_8": 1 << 30}):
        assert status(**at) == bs.ERR_INVALID_VALUE, at
    for at in ({"_0": (1 << 30) + 8}, {"_1": 248}, {"_8": (3 << 30) + 2}, {"_10": 260}):
        assert status(**at) == bs.ERR_ALIGNMENT, at
    assert status(_6=0, _0=None, _2=None, _8=None) == bs.OK


def test_python_refusals(bs):
    """Tensors of the wrong place, type or shape raise ValueError before the library is called."""
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    q, sf = torch.zeros((4, 256), dtype=torch.uint8), torch.zeros((4, 8), dtype=torch.uint8)
    for call in (lambda: bs.layer_norm(x), lambda: bs.layer_norm_backward(x, x, None, x, x),
                 lambda: bs.linear_a8w8_mxfp8(q, q, sf, sf), lambda: bs.gated_a8w8_mxfp8(q, q, sf, sf),
                 lambda: bs.gated_a4w4_mxfp4_backward(x, q, q, sf, sf), lambda: bs.dequantize(q, sf),
                 lambda: bs.dequantize(q, sf, "fp8_block"), lambda: bs.pack_gated(q, q, sf, sf),
                 lambda: bs.linear_a8w8_mxfp8(q, q, sf, sf, activation="tanh"),
                 lambda: bs.linear_a8w8_mxfp8(q, q, sf, sf, out_dtype=torch.float16),
                 lambda: bs.gated_a8w8_mxfp8(q, q, sf, sf, out_format="fp8_block"),
                 lambda: bs.gated_a8w8_mxfp8_backward(x, q, q, sf, sf, need_input_grad=False, need_weight_grad=False)):
        with pytest.raises(ValueError):
            call()


def test_overlap_refusals(bs, ops):
    """An output over an input, a parameter, a scale or another output is refused."""
    lib = bs.lib()

    def linear(epi=None, **kw):
        a, e = gemm_args(bs), ops.Epilogue()
        change(a, **kw)
        change(e, **(epi or {}))
        return lib.bsgemm_a8w8_mxfp8_linear(ctypes.byref(a), ctypes.byref(e), None)

    mx = {"out_dtype": 2}
    for epi, kw in (({}, {"ptr_c": 4 << 30}), ({}, {"ptr_c": (5 << 30) + 1024}), ({"ptr_sfc": 4 << 30}, mx),
                    ({"ptr_sfc": (3 << 30) + 512}, mx), ({"ptr_sfc": 2 << 30}, mx),
                    ({"ptr_sfc": 6 << 30, "bias": 6 << 30}, mx),
                    ({"ptr_sfc": 6 << 30, "residual": 6 << 30, "stride_residual": 256}, mx)):
        assert linear(epi, **kw) == bs.ERR_INVALID_VALUE, (epi, kw)

    def gated_backward(**grad):
        a, g = gemm_args(bs), ops.GatedGrad()
        a.workspace, a.workspace_bytes = 12 << 30, 1 << 30
        change(g, grad_h=6 << 30, grad_a=7 << 30, grad_gate=8 << 30, grad_up=9 << 30, stride_grad_h=128,
               stride_grad_a=256, stride_grad_w=256)
        change(a, **grad.pop("args", {}))
        change(g, **grad)
        return lib.bsgemm_a8w8_mxfp8_gated_backward(ctypes.byref(a), ctypes.byref(g), None)

    for kw in ({"grad_a": 4 << 30}, {"grad_up": 5 << 30}, {"args": {"workspace": 1 << 30}},
               {"args": {"workspace": 5 << 30}}, {"args": {"workspace": 6 << 30}}):
        assert gated_backward(**kw) == bs.ERR_INVALID_VALUE, kw

    def norm(**kw):
        a = ops.LayerNormArgs(x=1 << 30, y=2 << 30, weight=3 << 30, bias=4 << 30, ldx=256, ldy=256, rows=4, cols=256,
                              eps=1e-5)
        change(a, **kw)
        return lib.bsgemm_layer_norm(ctypes.byref(a), None)

    for kw in ({"y": 3 << 30}, {"y": (4 << 30) - 16}, {"out_format": 2, "sf": 2 << 30}, {"out_format": 2, "sf": 1 << 30},
               {"out_format": 2, "sf": (3 << 30) + 256}, {"mean": 2 << 30, "rstd": 6 << 30},
               {"mean": 5 << 30, "rstd": (5 << 30) + 8}, {"mean": 5 << 30, "rstd": 1 << 30}):
        assert norm(**kw) == bs.ERR_INVALID_VALUE, kw

    def backward(**kw):
        a = ops.LayerNormGradArgs(dy=1 << 30, x=2 << 30, weight=3 << 30, mean=4 << 30, rstd=5 << 30, dx=6 << 30,
                                  dweight=7 << 30, dbias=8 << 30, workspace=9 << 30, workspace_bytes=1 << 30, lddy=256,
                                  ldx=256, lddx=256, rows=4, cols=256)
        change(a, **kw)
        return lib.bsgemm_layer_norm_backward(ctypes.byref(a), None)

    for kw in ({"dx": 3 << 30}, {"dx": 4 << 30}, {"dx": (5 << 30) - 2000}, {"dweight": 6 << 30}, {"dbias": (7 << 30) + 2}):
        assert backward(**kw) == bs.ERR_INVALID_VALUE, kw
    assert lib.bsgemm_dequantize(1 << 30, 256, 2 << 30, bs.SF_NATIVE, 0, 0, 4, 256, 2 << 30, 0, 256,
                                 None) == bs.ERR_INVALID_VALUE
