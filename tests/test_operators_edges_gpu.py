"""Operators around the GEMMs on the GPU, where their numbers and their operands
get awkward: the tails of the activations, short contractions, operands at any
offset and stride."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def zeros(bs, rows, k, cuda):
    """An MXFP8 operand of zeros with its native scales: A B^T is then exactly 0."""
    return torch.zeros((rows, k), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn), bs.pack_scales(
        torch.full((rows, k // 32), 127, dtype=torch.uint8, device=cuda))


def activation_of(bs, cuda, x, name, m, kernel):
    """activation(x) of fp32 numbers x [n], as the bias of a product that is 0, in fp32."""
    a, asf = zeros(bs, m, 256, cuda)
    b, bsf = zeros(bs, x.numel(), 256, cuda)
    got = bs.linear_a8w8_mxfp8(a, b, asf, bsf, bias=x, activation=name, out_dtype=torch.float32, kernel=kernel)
    assert torch.equal(got, got[:1].expand_as(got))
    return got[0].double().cpu()


KERNELS = [(1, "swap"), (64, "swap"), (100, "1cta"), (300, "pair")]


@pytest.mark.parametrize("m,kernel", KERNELS)
def test_gelu_keeps_its_digits(bs, cuda, m, kernel):
    """gelu to a relative error, in the tail too.

    Tolerance, relative to the value: the reciprocal's argument and result are within
    2^-23 together and move the polynomial by at most 2.7 times that; its Horner steps
    add 4 * 2^-24, the fit 1.7e-7, the exponential 2^-22, the last products 3 * 2^-24:
    2^-19.  The exponential's argument 0.72 x^2 carries two roundings and its constant's
    half: x^2 2^-23."""
    x = torch.cat((torch.linspace(-12.9, 6.0, 8000), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 50.0, 3e38, -1e3, -3e38])))
    x = torch.nn.functional.pad(x, (0, 8 - x.numel() % 8)).to(cuda)
    v = x.double().cpu()
    ref = v * torch.special.erfc(-v / 2 ** 0.5) / 2
    got = activation_of(bs, cuda, x, "gelu", m, kernel)
    err = (got - ref).abs()
    tol = (2.0 ** -19 + v * v * 2.0 ** -23) * ref.abs() + 2.0 ** -149
    tol[v.abs() > 13] = 2.0 ** -22 * ref[v.abs() > 13].abs() + 1e-37
    assert bool((err <= tol).all()), (float(v[(err - tol).argmax()]), float((err / ref.abs()).nan_to_num().max()))


@pytest.mark.parametrize("m,kernel", KERNELS)
def test_silu_tail(bs, cuda, m, kernel):
    """silu to a relative error until exp(-x) passes 2^126; from there on it may be 0.

    Tolerance: exponential 2^-22, reciprocal 2^-23, sum and product 2^-24 each, the
    argument's two roundings 2^-23 |x|: (2^-20 + 2^-23 |x|) of the value."""
    x = torch.cat((torch.linspace(-87.3, 20.0, 8000), torch.linspace(-110.0, -87.3, 512))).to(cuda)
    v = x.double().cpu()
    ref = v * torch.sigmoid(v)
    err = (activation_of(bs, cuda, x, "silu", m, kernel) - ref).abs()
    tol = (2.0 ** -20 + 2.0 ** -23 * v.abs()) * ref.abs()
    tol[v <= -87.3] = 1.1e-36
    assert bool((err <= tol).all()), (float(v[(err - tol).argmax()]), float((err / ref.abs()).max()))


@pytest.mark.parametrize("fp4,k", [(False, 32), (False, 64), (False, 96), (False, 160), (True, 128), (True, 64), (True, 320)])
def test_short_contractions_are_refused(bs, cuda, fp4, k):
    """A K that is no whole stage is an error of the call, and its size queries answer 0."""
    import ctypes

    def operand(rows):
        q = torch.zeros((rows, k // 2 if fp4 else k), dtype=torch.uint8, device=cuda)
        return q, torch.full((rows, k // 32), 127, dtype=torch.uint8, device=cuda)

    f = 64
    linear, gated, backward = ((bs.linear_a4w4_mxfp4, bs.gated_a4w4_mxfp4, bs.gated_a4w4_mxfp4_backward) if fp4 else
                               (bs.linear_a8w8_mxfp8, bs.gated_a8w8_mxfp8, bs.gated_a8w8_mxfp8_backward))
    for m in (1, 64, 300):
        (a, asf), (b, bsf) = operand(m), operand(2 * f)
        grad = torch.zeros((m, f), dtype=torch.bfloat16, device=cuda)
        for native in (True, False):
            scales = [bs.pack_scales(s) for s in (asf, bsf)] if native else [asf, bsf]
            how = {"scale_format": "native" if native else "rowmajor"}
            for kernel in ("auto", "1cta", "pair"):
                for call in (lambda: linear(a, b, *scales, kernel=kernel, **how),
                             lambda: linear(a, b, *scales, kernel=kernel, split_k=4, **how),
                             lambda: linear(a, b, *scales, kernel=kernel, workspace=False, **how),
                             lambda: gated(a, b, *scales, kernel=kernel, **how),
                             lambda: backward(grad, a, b, *scales, kernel=kernel, **how)):
                    with pytest.raises(bs.BsgemmError):
                        call()
        args = bs.Args()
        bs.lib().bsgemm_args_init(ctypes.byref(args))
        args.m, args.n, args.k = m, 2 * f, k
        family = bs.FAMILY_MXFP4 if fp4 else bs.FAMILY_MXFP8
        assert bs.lib().bsgemm_epilogue_workspace_size(family, ctypes.byref(args)) == 0
        assert bs.lib().bsgemm_gated_backward_workspace_size(family, ctypes.byref(args)) == 0
        bs.lib().bsgemm_workspace_size(family, ctypes.byref(args))   # answers
    assert bs.check_device_error() == 0


def normal(orc, shape, seed, cuda, dtype=torch.bfloat16):
    return torch.from_numpy(orc.normal(shape, seed=seed)).to(cuda).to(dtype)


def views(t):
    """t [rows, cols] at offsets and strides that are no 16 bytes, some transposed or broadcast in memory."""
    rows, cols = t.shape
    for offset, pad in ((1, 0), (0, 1), (3, 5), (8, 4)):
        flat = torch.empty(offset + rows * (cols + pad), dtype=t.dtype, device=t.device)
        v = flat[offset:].view(rows, cols + pad)[:, :cols]
        v.copy_(t)
        yield v
    yield t.t().contiguous().t()


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,n", [(1, 136), (40, 264), (300, 520)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bias_and_residual_at_any_offset(bs, orc, cuda, fp4, m, n, dtype):
    """Views of bias and residual off 16 bytes give the bits of aligned ones."""
    fmt, k = ("mxfp4" if fp4 else "mxfp8"), 512
    f = bs.linear_a4w4_mxfp4 if fp4 else bs.linear_a8w8_mxfp8
    (a, asf), (b, bsf) = bs.quantize(normal(orc, (m, k), 1, cuda), fmt), bs.quantize(normal(orc, (n, k), 2, cuda), fmt)
    bias, residual = normal(orc, (n,), 3, cuda, dtype), normal(orc, (m, n), 4, cuda, dtype)
    want = f(a, b, asf, bsf, bias=bias, residual=residual, activation="silu")
    for v in views(residual):
        assert torch.equal(f(a, b, asf, bsf, bias=bias, residual=v, activation="silu"), want)
    for offset in (1, 2, 7):
        flat = torch.empty(n + offset, dtype=dtype, device=cuda)
        flat[offset:] = bias
        assert torch.equal(f(a, b, asf, bsf, bias=flat[offset:], residual=residual, activation="silu"), want)


@pytest.mark.parametrize("m,n", [(1, 100), (30, 100), (130, 36), (300, 516)])
def test_bf16_residual_of_odd_width(bs, orc, cuda, m, n):
    """An fp32 output of columns that are no multiple of 8 takes a contiguous bf16 residual."""
    k = 256
    (a, asf), (b, bsf) = (bs.quantize(normal(orc, (r, k), i, cuda), "mxfp8") for i, r in ((1, m), (2, n)))
    residual = normal(orc, (m, n), 3, cuda)
    got = bs.linear_a8w8_mxfp8(a, b, asf, bsf, residual=residual, out_dtype=torch.float32)
    want = bs.linear_a8w8_mxfp8(a, b, asf, bsf, residual=residual.float(), out_dtype=torch.float32)
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,f", [(1, 32), (70, 96), (300, 256)])
def test_gradient_at_any_offset(bs, orc, cuda, m, f):
    """Views of dL/dh off 16 bytes give the gradients of an aligned one."""
    k = 256
    (a, asf), (b, bsf) = (bs.quantize(normal(orc, (r, k), i, cuda), "mxfp8") for i, r in ((1, m), (2, 2 * f)))
    h = normal(orc, (m, f), 3, cuda)
    want = bs.gated_a8w8_mxfp8_backward(h, a, b, asf, bsf)
    for v in views(h):
        got = bs.gated_a8w8_mxfp8_backward(v, a, b, asf, bsf)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 128), (70, 384), (9, 1536)])
def test_norm_rows_at_any_offset(bs, orc, cuda, rows, cols, dtype):
    """MX outputs of rows off 16 bytes: the bits of aligned ones."""
    x, w = normal(orc, (rows, cols), 1, cuda, dtype), normal(orc, (cols,), 2, cuda, dtype)
    want = bs.layer_norm(x, w, out_format="mxfp8")
    for v in views(x):
        got = bs.layer_norm(v, w, out_format="mxfp8")
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("scale_format", ["native", "rowmajor"])
@pytest.mark.parametrize("rows,cols", [(701, 384), (5000, 1152), (16385, 2048)])
def test_norm_of_many_rows_to_mx(bs, orc, cuda, rows, cols, fmt, scale_format):
    """A prompt's rows: bit for bit what quantize makes of the fp32 output."""
    x = normal(orc, (997, cols), 1, cuda).repeat(rows // 997 + 1, 1)[:rows] * torch.linspace(0.1, 9.0, rows, device=cuda)[:, None]
    x = x.bfloat16()
    w, b = normal(orc, (cols,), 2, cuda), normal(orc, (cols,), 3, cuda)
    q, sf = bs.layer_norm(x, w, b, out_format=fmt, scale_format=scale_format)
    want_q, want_sf = bs.quantize(bs.layer_norm(x, w, b, out_dtype=torch.float32), fmt, scale_format=scale_format)
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(sf, want_sf)
