"""Operators around the GEMMs on the GPU against their formulas in 64 bits:
linear layers (bias, activation, residual, MX output), the gated feed-forward
product and its gradient, layer norm and its gradient, dequantise.

Tolerances, from the arithmetic:
  U16 = 2^-8, U32 = 2^-24: one rounding to bf16 / fp32;
  ACC = 1e-6: the tensor cores' fp32 accumulation, relative to sum |a b|
      (the accumulation floor of the GEMM tests);
  FN  = 2^-20: an activation and the few fp32 operations around it, relative
      to the values that go into them (CUDA's expf and erff are within 2 ulp,
      the quotient within 2; no activation here has a slope above 1.13)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U16, U32, ACC, FN = 2.0 ** -8, 2.0 ** -24, 1e-6, 2.0 ** -20
SUM = 44    # roundings of a row's sum: up to 32 elements in turn in a thread, then two trees of 32
SLOPE = 1.13


# ---- operands and formulas ------------------------------------------------------

def values(q, sf, fp4):
    """fp64 values of MX elements [rows, kbytes] with row-major E8M0 bytes."""
    if fp4:
        table = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
        v = np.stack((table[q & 15], table[q >> 4]), axis=-1).reshape(q.shape[0], -1)
    else:
        v = torch.from_numpy(q.copy()).view(torch.float8_e4m3fn).double().numpy()
    return v * np.repeat(np.ldexp(1.0, sf.astype(np.int64) - 127), 32, axis=1)


class Operand:
    """A quantised matrix: fp64 values, device elements, native and row-major scales."""

    def __init__(self, bs, orc, cuda, rows, k, fp4, seed, std=1.0):
        x = orc.normal((rows, k), seed=seed) * std
        self.q, self.sf = orc.quant_mxfp4(x) if fp4 else orc.quant_mxfp8(x)
        self.v = torch.from_numpy(values(self.q, self.sf, fp4))
        self.d = torch.from_numpy(self.q).to(cuda)
        if not fp4:
            self.d = self.d.view(torch.float8_e4m3fn)
        self.rowmajor = torch.from_numpy(self.sf).to(cuda)
        self.native = bs.pack_scales(self.rowmajor)


def act(x, name):
    if name == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if name == "gelu":
        return x * torch.special.erfc(-x / math.sqrt(2)) / 2
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    if name == "silu":
        return x * torch.sigmoid(x)
    return x


def act_slope(x, name):
    """act'(x) by autograd of the formula in 64 bits; relu's at 0 is 0 (MXFP4 products do hit 0)."""
    if name == "relu":
        return (x > 0).double()
    x = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(act(x, name).sum(), x)
    return g


def rounding(ref, dtype):
    return (U16 if dtype == torch.bfloat16 else U32) * ref.abs()


def assert_within(got, ref, tol, what=""):
    got = got.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance, worst {float((err - tol).max()):.3e}"


def rel_norm(got, ref):
    return float((got.double().cpu() - ref).norm() / ref.norm())


def linear_ref(a, b, bias, name, residual):
    pre = a.v @ b.v.T
    mag = a.v.abs() @ b.v.abs().T
    if bias is not None:
        pre = pre + bias.double().cpu()
    y = act(pre, name)
    tol = SLOPE * ACC * mag + FN * (pre.abs() + mag * 2 ** -10)
    if residual is not None:
        y = y + residual.double().cpu()
        tol = tol + FN * residual.double().cpu().abs()
    return y, tol


def linear(bs, fp4):
    return bs.linear_a4w4_mxfp4 if fp4 else bs.linear_a8w8_mxfp8


def gated(bs, fp4):
    return bs.gated_a4w4_mxfp4 if fp4 else bs.gated_a8w8_mxfp8


def gated_backward(bs, fp4):
    return bs.gated_a4w4_mxfp4_backward if fp4 else bs.gated_a8w8_mxfp8_backward


def normal(orc, shape, seed, cuda, dtype=torch.bfloat16):
    return torch.from_numpy(orc.normal(shape, seed=seed)).to(cuda).to(dtype)


# ---- linear -----------------------------------------------------------------------

SHAPES = [  # m, n, k, kernel, split: every kernel, ragged rows and columns, one K block, split K both ways
    (1, 136, 256, "auto", 0), (1, 1000, 4096, "swap", 0), (16, 384, 2048, "swap", 4), (17, 520, 256, "swap", 1),
    (33, 264, 1024, "swap", 3), (64, 200, 512, "swap", 1), (64, 136, 512, "1cta", 1), (65, 392, 768, "auto", 0),
    (130, 72, 512, "1cta", 2), (257, 328, 512, "1cta", 1), (200, 520, 256, "pair", 1), (600, 776, 768, "pair", 1),
]


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,n,k,kernel,split", SHAPES)
def test_linear(bs, orc, cuda, fp4, m, n, k, kernel, split):
    a, b = Operand(bs, orc, cuda, m, k, fp4, 1), Operand(bs, orc, cuda, n, k, fp4, 2, k ** -0.5)
    names = [None, "relu", "gelu", "gelu_tanh", "silu"]
    for i, dtype in enumerate((torch.bfloat16, torch.float32)):
        name = names[(m + n + 2 * i + fp4) % 5]
        bias = normal(orc, (n,), 3, cuda, (torch.float32, torch.bfloat16)[i])
        residual = normal(orc, (m, n), 4, cuda, dtype)
        for use_bias, use_res in ((True, True), (False, False)):
            args = dict(bias=bias if use_bias else None, residual=residual if use_res else None, activation=name)
            got = linear(bs, fp4)(a.d, b.d, a.native, b.native, out_dtype=dtype, kernel=kernel, split_k=split, **args)
            ref, tol = linear_ref(a, b, args["bias"], name, args["residual"])
            assert_within(got, ref, tol + rounding(ref, dtype), f"{name} {dtype} {use_bias} {use_res}")
    assert bs.check_device_error() == 0


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,kernel,split", [(1, "swap", 1), (20, "swap", 4), (50, "swap", 3), (64, "1cta", 2),
                                            (130, "1cta", 1), (300, "pair", 1), (129, "auto", 0)])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_linear_mx_output(bs, orc, cuda, fp4, m, kernel, split, fmt):
    """MX output = quantize of the fp32 output, bit for bit, and its scales pad their atoms with 2^0."""
    n, k = 384, 1024
    a, b = Operand(bs, orc, cuda, m, k, fp4, 5), Operand(bs, orc, cuda, n, k, fp4, 6, k ** -0.5)
    bias = normal(orc, (n,), 7, cuda)
    args = dict(bias=bias, activation="gelu", kernel=kernel, split_k=split)
    for workspace in (None, False):
        if workspace is False and kernel == "1cta" and split > 1:
            continue    # only the decode kernel splits without a workspace
        f32 = linear(bs, fp4)(a.d, b.d, a.native, b.native, out_dtype=torch.float32, workspace=workspace, **args)
        q, sf = linear(bs, fp4)(a.d, b.d, a.native, b.native, out_format=fmt, workspace=workspace, **args)
        want_q, want_sf = bs.quantize(f32, fmt)
        assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
        assert torch.equal(sf, want_sf)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,kernel", [(7, "auto"), (130, "1cta"), (300, "pair")])
def test_linear_layouts(bs, orc, cuda, fp4, m, kernel):
    """Row-major scales, shuffled weights, strided A, C and residual give the bits of the plain call."""
    n, k = 272, 512
    a, b = Operand(bs, orc, cuda, m, k, fp4, 8), Operand(bs, orc, cuda, n, k, fp4, 9)
    residual = normal(orc, (m, n), 10, cuda)
    f = linear(bs, fp4)
    want = f(a.d, b.d, a.native, b.native, residual=residual, activation="silu", kernel=kernel)
    assert torch.equal(want, f(a.d, b.d, a.rowmajor, b.rowmajor, residual=residual, activation="silu", kernel=kernel,
                               scale_format="rowmajor"))
    shuffled = bs.pack_b(b.d.view(torch.uint8), "shuffle16", unpack=True).view(b.d.dtype)
    assert torch.equal(want, f(a.d, shuffled, a.native, b.native, residual=residual, activation="silu", kernel=kernel,
                               b_format="shuffle16"))
    wide_a = torch.zeros((m, a.d.shape[1] + 32), dtype=torch.uint8, device=cuda)
    wide_a[:, 16:-16] = a.d.view(torch.uint8)
    wide_r = torch.full((m, n + 16), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide_r[:, 8:8 + n] = residual
    wide_c = torch.full((m, n + 24), 7.0, dtype=torch.bfloat16, device=cuda)
    got = f(wide_a[:, 16:-16].view(a.d.dtype), b.d, a.native, b.native, residual=wide_r[:, 8:8 + n], activation="silu",
            kernel=kernel, out=wide_c[:, 8:8 + n])
    assert torch.equal(want, got)
    assert bool((wide_c[:, :8] == 7).all()) and bool((wide_c[:, 8 + n:] == 7).all())   # nothing beside C is written
    # a broadcast residual, and C over its own residual
    row = residual[:1].expand(m, n)
    assert torch.equal(f(a.d, b.d, a.native, b.native, residual=row, kernel=kernel),
                       f(a.d, b.d, a.native, b.native, residual=row.contiguous(), kernel=kernel))
    inplace = residual.clone()
    f(a.d, b.d, a.native, b.native, residual=inplace, activation="silu", kernel=kernel, out=inplace)
    assert torch.equal(want, inplace)


def test_linear_not_finite(bs, orc, cuda):
    """A NaN scale or element reaches its row alone; inf and the lowest value in bias and residual stay in their places."""
    m, n, k = 40, 256, 256
    for kernel in ("swap", "1cta", "pair"):
        a, b = Operand(bs, orc, cuda, m, k, False, 11), Operand(bs, orc, cuda, n, k, False, 12)
        clean = bs.linear_a8w8_mxfp8(a.d, b.d, a.native, b.native, activation="relu", kernel=kernel)
        a.d.view(torch.uint8)[3, 5] = 0x7F
        a.rowmajor[9, 2] = 255
        bias = torch.zeros(n, device=cuda)
        bias[17], bias[40] = float("inf"), torch.finfo(torch.float32).min
        residual = torch.zeros((m, n), device=cuda)
        residual[20, 30] = float("nan")
        got = bs.linear_a8w8_mxfp8(a.d, b.d, bs.pack_scales(a.rowmajor), b.native, bias=bias, residual=residual,
                                   activation="relu", kernel=kernel)
        assert bool(got[3].isnan().all()) and bool(got[9].isnan().all()) and bool(got[20, 30].isnan())
        rows = [r for r in range(m) if r not in (3, 9, 20)]
        assert bool((got[rows, 17] == float("inf")).all()) and bool((got[rows, 40] == 0).all())
        cols = [c for c in range(n) if c not in (17, 40)]
        assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


def test_linear_long_offsets(bs, orc, cuda):
    """C and the residual past 2^31 elements."""
    m, n, k = 140_000, 16384, 128
    assert m * n > 2 ** 31
    a, b = Operand(bs, orc, cuda, 256, k, False, 13), Operand(bs, orc, cuda, n, k, False, 14)
    A = a.d.view(torch.uint8).repeat(m // 256 + 1, 1)[:m].view(torch.float8_e4m3fn)
    sf = bs.pack_scales(a.rowmajor.repeat(m // 256 + 1, 1)[:m])
    for kernel in ("pair", "1cta"):
        want, _ = bs.linear_a8w8_mxfp8(a.d, b.d, a.native, b.native, activation="silu", out_format="mxfp8", kernel=kernel)
        want = want.view(torch.uint8)
        q, _ = bs.linear_a8w8_mxfp8(A, b.d, sf, b.native, activation="silu", out_format="mxfp8", kernel=kernel)
        q = q.view(torch.uint8)
        last = m // 256 * 256
        assert torch.equal(q[last:], want[:m - last]) and torch.equal(q[last - 256:last], want)
        del q
    residual = torch.zeros((m, n), dtype=torch.bfloat16, device=cuda)
    residual[-1] = 3.0
    got = bs.linear_a8w8_mxfp8(A, b.d, sf, b.native, residual=residual, out=residual, kernel="pair")
    few = bs.linear_a8w8_mxfp8(a.d, b.d, a.native, b.native, out_dtype=torch.float32, kernel="pair")
    row = (m - 1) % 256
    assert torch.equal(got[-1], (few[row] + 3).bfloat16()) and torch.equal(got[-2], few[row - 1].bfloat16())


# ---- gated product ------------------------------------------------------------------

class Gated:
    def __init__(self, bs, orc, cuda, m, f, k, fp4, seed):
        self.a = Operand(bs, orc, cuda, m, k, fp4, seed)
        self.g = Operand(bs, orc, cuda, f, k, fp4, seed + 1, k ** -0.5)
        self.u = Operand(bs, orc, cuda, f, k, fp4, seed + 2, k ** -0.5)
        self.b, self.b_native = bs.pack_gated(self.g.d, self.u.d, self.g.rowmajor, self.u.rowmajor)
        self.call = (self.a.d, self.b, self.a.native, self.b_native)

    def ref(self, name):
        g, u = self.a.v @ self.g.v.T, self.a.v @ self.u.v.T
        mg, mu = self.a.v.abs() @ self.g.v.abs().T, self.a.v.abs() @ self.u.v.abs().T
        tol = u.abs() * (SLOPE * ACC * mg + FN * g.abs()) + act(g, name).abs() * ACC * mu + FN * (act(g, name) * u).abs()
        return act(g, name) * u, tol + 4 * ACC * ACC * mg * mu


GATED_SHAPES = [(1, 32, 256, "auto", 0), (1, 1024, 4096, "swap", 0), (9, 96, 512, "swap", 1), (16, 160, 2048, "swap", 2),
                (31, 224, 1024, "swap", 3), (64, 416, 1024, "swap", 4), (64, 96, 512, "1cta", 1), (65, 352, 768, "auto", 0),
                (130, 32, 512, "1cta", 2), (260, 288, 512, "1cta", 1), (200, 160, 256, "pair", 1), (600, 608, 768, "pair", 1)]


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,f,k,kernel,split", GATED_SHAPES)
def test_gated(bs, orc, cuda, fp4, m, f, k, kernel, split):
    p = Gated(bs, orc, cuda, m, f, k, fp4, 20)
    names = ["silu", "gelu", "gelu_tanh", "relu", None]
    for i, dtype in enumerate((torch.bfloat16, torch.float32)):
        name = names[(m + f // 32 + i + 2 * fp4) % 5]
        ref, tol = p.ref(name)
        for workspace in (None, False):
            if workspace is False and kernel == "1cta" and split > 1:
                continue
            got = gated(bs, fp4)(*p.call, activation=name, out_dtype=dtype, kernel=kernel, split_k=split,
                                 workspace=workspace)
            assert_within(got, ref, tol + rounding(ref, dtype), f"{name} {dtype} {workspace}")
    assert bs.check_device_error() == 0


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,kernel,split", [(1, "swap", 1), (16, "swap", 2), (20, "swap", 4), (50, "swap", 3),
                                            (64, "1cta", 2), (130, "1cta", 1), (300, "pair", 1)])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_gated_mx_output(bs, orc, cuda, fp4, m, kernel, split, fmt):
    p = Gated(bs, orc, cuda, m, 256, 1024, fp4, 30)
    for workspace in (None, False):
        if workspace is False and kernel == "1cta" and split > 1:
            continue
        args = dict(kernel=kernel, split_k=split, workspace=workspace)
        want_q, want_sf = bs.quantize(gated(bs, fp4)(*p.call, out_dtype=torch.float32, **args), fmt)
        q, sf = gated(bs, fp4)(*p.call, out_format=fmt, **args)
        assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
        assert torch.equal(sf, want_sf)


def test_gated_persistent_decode(bs, orc, cuda):
    """More tiles than CTAs, so a CTA's exchange slots and accumulators go round."""
    p = Gated(bs, orc, cuda, 24, 1024, 256, False, 33)
    want = bs.gated_a8w8_mxfp8(*p.call, kernel="swap", split_k=1, out_dtype=torch.float32)
    for blocks in (1, 3):
        got = bs.gated_a8w8_mxfp8(*p.call, kernel="swap", split_k=1, out_dtype=torch.float32, grid_blocks=blocks)
        assert torch.equal(want, got)
    one = bs.gated_a8w8_mxfp8(*p.call, kernel="swap", split_k=2, out_dtype=torch.float32, workspace=False)
    two = bs.gated_a8w8_mxfp8(*p.call, kernel="swap", split_k=2, out_dtype=torch.float32, workspace=False, grid_blocks=4)
    assert torch.equal(one, two)
    assert bs.check_device_error() == 0


GRAD_SHAPES = [(1, 32, 256, "auto"), (5, 160, 512, "1cta"), (64, 96, 256, "pair"), (129, 224, 768, "1cta"),
               (300, 544, 512, "pair"), (700, 352, 256, "auto")]


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("m,f,k,kernel", GRAD_SHAPES)
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh", "relu", None])
def test_gated_backward(bs, orc, cuda, fp4, m, f, k, kernel, name):
    """Against the formula: the projections' gradients dg, du are rounded to bf16
    (U16 each, worst case over the sum), then each output once.  Also in the
    mean: two independent roundings of 2^-8 / sqrt(3) at most are under 3.3e-3."""
    p = Gated(bs, orc, cuda, m, f, k, fp4, 40)
    h = normal(orc, (m, f), 44, cuda)
    hv = h.double().cpu()
    g, u = p.a.v @ p.g.v.T, p.a.v @ p.u.v.T
    mg, mu = p.a.v.abs() @ p.g.v.abs().T, p.a.v.abs() @ p.u.v.abs().T
    slope = act_slope(g, name)
    dg, du = hv * u * slope, hv * act(g, name)
    # error of dg and du before their rounding: second derivatives are below 1.2 (relu: none off 0)
    edg = hv.abs() * (mu * ACC * slope.abs() + u.abs() * (1.2 * ACC * mg + FN)) + FN * dg.abs()
    if name == "relu":
        edg = edg + torch.where(g.abs() <= ACC * mg, (hv * u).abs(), torch.zeros_like(g))
    edu = hv.abs() * (SLOPE * ACC * mg + FN * g.abs())
    edg, edu = edg + U16 * dg.abs(), edu + U16 * du.abs()
    refs = (dg @ p.g.v + du @ p.u.v, dg.T @ p.a.v, du.T @ p.a.v)
    tols = ((edg + ACC * dg.abs()) @ p.g.v.abs() + (edu + ACC * du.abs()) @ p.u.v.abs(),
            (edg + ACC * dg.abs()).T @ p.a.v.abs(), (edu + ACC * du.abs()).T @ p.a.v.abs())
    got = gated_backward(bs, fp4)(h, *p.call, activation=name, kernel=kernel)
    for x, ref, tol, what in zip(got, refs, tols, ("dA", "dWg", "dWu")):
        assert x.dtype == torch.bfloat16
        assert_within(x, ref, tol * (1 + U16) + U16 * ref.abs(), what)
        assert rel_norm(x, ref) < 3.3e-3, what
    # one side alone gives the same bits
    only_a = gated_backward(bs, fp4)(h, *p.call, activation=name, kernel=kernel, need_weight_grad=False)
    only_w = gated_backward(bs, fp4)(h, *p.call, activation=name, kernel=kernel, need_input_grad=False)
    assert torch.equal(only_a[0], got[0]) and only_a[1] is None and only_a[2] is None
    assert only_w[0] is None and torch.equal(only_w[1], got[1]) and torch.equal(only_w[2], got[2])
    assert bs.check_device_error() == 0


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_gated_backward_differences(bs, orc, cuda, name):
    """<gradient, direction> against central differences of sum(h * act(g) u) in 64 bits.
    The kernel's error along a direction V is at most |err| |V| <= 3.3e-3 |grad| |V|."""
    m, f, k = 48, 64, 256
    p = Gated(bs, orc, cuda, m, f, k, False, 50)
    h = normal(orc, (m, f), 54, cuda)
    hv = h.double().cpu()
    got = [x.double().cpu() for x in bs.gated_a8w8_mxfp8_backward(h, *p.call, activation=name)]
    at = [p.a.v, p.g.v, p.u.v]

    def loss(a, wg, wu):
        return (hv * act(a @ wg.T, name) * (a @ wu.T)).sum()

    for i in range(3):
        v = torch.from_numpy(orc.normal(tuple(at[i].shape), seed=60 + i)).double()
        step = 1e-5
        hi, lo = ([x + s * step * v if j == i else x for j, x in enumerate(at)] for s in (1, -1))
        numeric = (loss(*hi) - loss(*lo)) / (2 * step)
        assert abs(float((got[i] * v).sum() - numeric)) <= 3.3e-3 * float(got[i].norm() * v.norm()) + 1e-6 * abs(float(numeric))


def test_gated_backward_layouts(bs, orc, cuda):
    """Row-major scales, a strided grad and a capped grid give the bits of the plain call; a given workspace is enough."""
    m, f, k = 150, 160, 384
    p = Gated(bs, orc, cuda, m, f, k, False, 70)
    h = normal(orc, (m, f), 74, cuda)
    want = bs.gated_a8w8_mxfp8_backward(h, *p.call)
    wide = torch.full((m, f + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, 8:8 + f] = h
    rows = bs.unpack_scales(p.b_native, 2 * f, k // 32)
    calls = [lambda: bs.gated_a8w8_mxfp8_backward(wide[:, 8:8 + f], *p.call),
             lambda: bs.gated_a8w8_mxfp8_backward(h, p.a.d, p.b, p.a.rowmajor, rows, scale_format="rowmajor"),
             lambda: bs.gated_a8w8_mxfp8_backward(h, *p.call, grid_blocks=2)]
    for call in calls:
        for x, y in zip(want, call()):
            assert torch.equal(x, y)
    # a grad that is one row for all tokens (stride 0)
    one = h[:1].expand(m, f)
    for x, y in zip(bs.gated_a8w8_mxfp8_backward(one, *p.call), bs.gated_a8w8_mxfp8_backward(one.contiguous(), *p.call)):
        assert torch.equal(x, y)


# ---- layer norm ------------------------------------------------------------------------

def norm_data(orc, rows, cols, seed, cuda, dtype):
    x = orc.normal((rows, cols), seed=seed) * np.linspace(0.1, 3.0, cols) + 1.5
    x[rows // 2] *= 1e-3
    return torch.from_numpy(x).to(cuda).to(dtype)


def norm_ref(x, w, b, eps):
    """(y, z, mean, rstd, tolerance of z): the mean's error is a sum's, SUM
    roundings of sum |x| / n; the variance's reaches z as half of SUM + a few."""
    x = x.double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    z = (x - mean) * rstd
    tol = U32 * (SUM * x.abs().mean(1, keepdim=True) * rstd + x.abs() * rstd + SUM * (z.abs() + 0.01))
    w = w.double().cpu() if w is not None else torch.ones(x.shape[1], dtype=torch.float64)
    b = b.double().cpu() if b is not None else torch.zeros(x.shape[1], dtype=torch.float64)
    return z * w + b, z, mean, rstd, tol, w, b


NORM_SHAPES = [(1, 1), (3, 7), (5, 33), (2, 256), (9, 264), (17, 1000), (4, 1024), (3, 1025), (5, 1537), (2, 2048),
               (6, 4096), (3, 7168), (2, 8191), (2, 10008), (2, 16384), (300, 72), (1, 7168)]


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm(bs, orc, cuda, rows, cols, dtype):
    x = norm_data(orc, rows, cols, rows * 7 + cols, cuda, dtype)
    for pdtype, out_dtype, eps in ((torch.float32, torch.float32, 1e-5), (torch.bfloat16, torch.bfloat16, 1e-6)):
        w = 1 + 0.2 * normal(orc, (cols,), 2, cuda, torch.float32)
        w, b = w.to(pdtype), normal(orc, (cols,), 3, cuda, pdtype)
        for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
            y, mean, rstd = bs.layer_norm(x, weight, bias, eps, out_dtype=out_dtype, return_stats=True)
            ref, z, m_ref, r_ref, tol, wv, bv = norm_ref(x, weight, bias, eps)
            assert_within(y, ref, tol * wv.abs() + 2 * U32 * (ref.abs() + bv.abs()) + rounding(ref, out_dtype))
            assert_within(mean, m_ref[:, 0], SUM * U32 * x.double().cpu().abs().mean(1))
            assert_within(rstd, r_ref[:, 0], r_ref[:, 0] * U32 * (SUM + 2 * SUM * (x.double().cpu().abs().mean(1) * r_ref[:, 0])))


@pytest.mark.parametrize("rows,cols", [(1, 128), (7, 1024), (130, 384), (128, 1152), (3, 7168), (2, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_layer_norm_mx_output(bs, orc, cuda, rows, cols, dtype, fmt):
    """= quantize of the fp32 output, bit for bit, in both scale layouts."""
    x = norm_data(orc, rows, cols, 5, cuda, dtype)
    w, b = 1 + 0.2 * normal(orc, (cols,), 6, cuda, torch.float32), normal(orc, (cols,), 7, cuda, torch.float32)
    f32 = bs.layer_norm(x, w, b, out_dtype=torch.float32)
    for scale_format in ("native", "rowmajor"):
        want_q, want_sf = bs.quantize(f32, fmt, scale_format=scale_format)
        q, sf = bs.layer_norm(x, w, b, out_format=fmt, scale_format=scale_format)
        assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
        assert torch.equal(sf, want_sf)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_layouts(bs, orc, cuda, dtype):
    """Strided, shifted, transposed, broadcast and aliased rows give the bits of the plain call."""
    for rows, cols in ((9, 1000), (6, 1536)):
        x = norm_data(orc, rows, cols, 8, cuda, dtype)
        w, b = normal(orc, (cols,), 9, cuda, dtype), normal(orc, (cols,), 10, cuda, dtype)
        want = bs.layer_norm(x, w, b)
        ref, z, _, _, tol, wv, bv = norm_ref(x, w, b, 1e-5)
        tol = tol * wv.abs() + 2 * U32 * (ref.abs() + bv.abs()) + rounding(ref, dtype)
        wide = torch.full((rows, cols + 16), float("nan"), dtype=dtype, device=cuda)
        wide[:, 8:8 + cols] = x
        assert torch.equal(bs.layer_norm(wide[:, 8:8 + cols], w, b), want)
        wide[:, 3:3 + cols] = x    # rows off the 16-byte grid take the other path: another order of the sums
        assert_within(bs.layer_norm(wide[:, 3:3 + cols], w, b), ref, tol)
        assert torch.equal(bs.layer_norm(x.t().contiguous().t(), w, b), want)
        row = x[:1].expand(rows, cols)
        assert torch.equal(bs.layer_norm(row, w, b), want[:1].expand(rows, cols))
        out = torch.full((rows, cols + 8), 5.0, dtype=dtype, device=cuda)
        bs.layer_norm(x, w, b, out=out[:, :cols])
        assert torch.equal(out[:, :cols], want) and bool((out[:, cols:] == 5).all())
        same = x.clone()
        bs.layer_norm(same, w, b, out=same)
        assert torch.equal(same, want)


def test_layer_norm_not_finite(bs, orc, cuda):
    """NaN and inf stay in their rows; a constant row is its bias (eps > 0); fp32 huge rows as the formula has them."""
    for cols in (520, 2048):
        x = norm_data(orc, 6, cols, 11, cuda, torch.float32)
        w, b = normal(orc, (cols,), 12, cuda, torch.float32), normal(orc, (cols,), 13, cuda, torch.float32)
        want = bs.layer_norm(x, w, b)
        x[1, 5], x[2, 7], x[4] = float("nan"), float("-inf"), 3.25
        y = bs.layer_norm(x, w, b)
        assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
        assert torch.equal(y[4], b)
        assert torch.equal(y[[0, 3, 5]], want[[0, 3, 5]])


def test_layer_norm_long_offsets(bs, orc, cuda):
    rows, cols = 140_000, 16384
    assert rows * cols > 2 ** 31
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=cuda)
    x[-3:] = norm_data(orc, 3, cols, 14, cuda, torch.bfloat16)
    want, mean, rstd = bs.layer_norm(x[-3:].clone(), return_stats=True)
    y, m, r = bs.layer_norm(x, return_stats=True)
    assert torch.equal(y[-3:], want) and torch.equal(m[-3:], mean) and torch.equal(r[-3:], rstd)
    dx, _, _ = bs.layer_norm_backward(y, x, None, m, r, out=y, need_weight_grad=False)
    few, _, _ = bs.layer_norm_backward(want, x[-3:].clone(), None, mean, rstd, need_weight_grad=False)
    assert torch.equal(dx[-3:], few)


@pytest.mark.parametrize("rows,cols", NORM_SHAPES + [(1000, 128), (700, 1100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_backward(bs, orc, cuda, rows, cols, dtype):
    """Against the formula.  z's error ez as in the forward pass (the kernel
    is given its mean and rstd); t = dy w; the two means are sums of n terms:
    SUM roundings of their terms' absolute mean."""
    x = norm_data(orc, rows, cols, 3 * rows + cols, cuda, dtype)
    w = (1 + 0.2 * normal(orc, (cols,), 2, cuda, torch.float32)).to(dtype)
    dy = normal(orc, (rows, cols), 3, cuda, dtype)
    _, z, mean, rstd, ez, wv, _ = norm_ref(x, w, None, 1e-5)
    # the statistics a forward pass would have kept
    stats = mean[:, 0].float().to(cuda), rstd[:, 0].float().to(cuda)
    d = dy.double().cpu()
    t = d * wv
    m1, m2 = t.mean(1, keepdim=True), (t * z).mean(1, keepdim=True)
    dx = rstd * (t - m1 - z * m2)
    e1 = SUM * U32 * t.abs().mean(1, keepdim=True)
    e2 = SUM * U32 * (t * z).abs().mean(1, keepdim=True) + (t.abs() * ez).mean(1, keepdim=True)
    tol = rstd * (6 * U32 * (t.abs() + m1.abs() + (z * m2).abs()) + e1 + z.abs() * e2 + ez * (m2.abs() + e2))
    weights = (d * z).sum(0), d.sum(0)
    # roundings of a column's sum: a CTA's rows in turn, 8 warps, an eighth of at most 592 CTAs, 8 slices
    serial = rows / 148 + 1 + 8 + 74 + 8
    wtol = (serial * U32 * (d * z).abs().sum(0) + (d.abs() * ez).sum(0), serial * U32 * d.abs().sum(0))
    got = bs.layer_norm_backward(dy, x, w, *stats)
    assert_within(got[0], dx, tol + rounding(dx, dtype), "dx")
    for g, ref, e, what in zip(got[1:], weights, wtol, ("dweight", "dbias")):
        assert g.dtype == dtype
        assert_within(g, ref, e + rounding(ref, dtype), what)
    again = bs.layer_norm_backward(dy, x, w, *stats)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    dx_only = bs.layer_norm_backward(dy, x, w, *stats, need_weight_grad=False)
    assert torch.equal(dx_only[0], got[0]) and dx_only[1] is None and dx_only[2] is None


def test_layer_norm_backward_differences(bs, orc, cuda):
    """The forward's own statistics, and central differences of sum(dy * y) in 64 bits along a direction."""
    rows, cols, eps = 5, 200, 1e-5
    x = norm_data(orc, rows, cols, 15, cuda, torch.float32)
    w, b = 1 + 0.2 * normal(orc, (cols,), 16, cuda, torch.float32), normal(orc, (cols,), 17, cuda, torch.float32)
    dy = normal(orc, (rows, cols), 18, cuda, torch.float32)
    _, mean, rstd = bs.layer_norm(x, w, b, eps, return_stats=True)
    got = [g.double().cpu() for g in bs.layer_norm_backward(dy, x, w, mean, rstd)]
    at = [t.double().cpu() for t in (x, w, b)]

    def loss(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return (dy.double().cpu() * (d / (d.square().mean(1, keepdim=True) + eps).sqrt() * w + b)).sum()

    for i in range(3):
        v = torch.from_numpy(orc.normal(tuple(at[i].shape), seed=70 + i)).double()
        if i == 0:
            v[rows // 2] *= 1e-3   # that row is small: a step must be too
        step = 1e-5
        hi, lo = ([t + s * step * v if j == i else t for j, t in enumerate(at)] for s in (1, -1))
        numeric = float((loss(*hi) - loss(*lo)) / (2 * step))
        assert abs(float((got[i] * v).sum()) - numeric) <= 1e-5 * float(got[i].norm() * v.norm())


def test_layer_norm_backward_layouts(bs, orc, cuda):
    for rows, cols, dtype in ((40, 1000, torch.bfloat16), (11, 1544, torch.float32)):
        x, dy = norm_data(orc, rows, cols, 19, cuda, dtype), normal(orc, (rows, cols), 20, cuda, dtype)
        w = normal(orc, (cols,), 21, cuda, torch.float32)
        _, mean, rstd = bs.layer_norm(x, w, None, return_stats=True)
        want = bs.layer_norm_backward(dy, x, w, mean, rstd)
        assert want[1].dtype == torch.float32
        wide = torch.full((rows, cols + 16), float("nan"), dtype=dtype, device=cuda)
        wide[:, 8:8 + cols] = dy
        one = dy[:1].expand(rows, cols)
        pairs = [(bs.layer_norm_backward(wide[:, 8:8 + cols], x, w, mean, rstd), want),
                 (bs.layer_norm_backward(dy.clone(), x, w, mean, rstd, out=x.clone()), want),
                 (bs.layer_norm_backward(one, x, w, mean, rstd), bs.layer_norm_backward(one.contiguous(), x, w, mean, rstd))]
        for got, ref in pairs:
            for a, b in zip(got, ref):
                assert torch.equal(a, b)
        for alias in (0, 1):    # dx over dy, dx over x
            a, b = dy.clone(), x.clone()
            got = bs.layer_norm_backward(a, b, w, mean, rstd, out=b if alias else a)
            for g, r in zip(got, want):
                assert torch.equal(g, r)


# ---- dequantise, empty inputs, streams, the block ---------------------------------------

@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("rows,cols", [(1, 128), (130, 384), (7, 32), (3, 7168)])
def test_dequantize(bs, orc, cuda, fmt, rows, cols):
    fp4 = fmt == "mxfp4"
    x = orc.normal((rows, cols), seed=22).astype(np.float32)
    q, sf = orc.quant_mxfp4(x) if fp4 else orc.quant_mxfp8(x)
    sf[0, 0], sf[-1, -1] = 1, 240
    ref = torch.from_numpy(values(q, sf, fp4))
    qd, sd = torch.from_numpy(q).to(cuda), torch.from_numpy(sf).to(cuda)
    qd = qd if fp4 else qd.view(torch.float8_e4m3fn)
    for dtype in (torch.bfloat16, torch.float32):
        got = bs.dequantize(qd, sd, fmt, scale_format="rowmajor", out_dtype=dtype)
        assert got.dtype == dtype
        # 2^-126 times an element that is a subnormal multiple of 2^-9: bf16's own subnormals end at 2^-133
        tiny = torch.full_like(ref, 2.0 ** -134 if dtype == torch.bfloat16 else 0.0)
        assert_within(got, ref, torch.where(ref.abs() < 2.0 ** -126, tiny, torch.zeros_like(ref)))
        if cols % 128 == 0:
            assert torch.equal(got, bs.dequantize(qd, bs.pack_scales(sd), fmt, out_dtype=dtype))
    sd[0, 0] = 255
    assert bool(bs.dequantize(qd, sd, fmt, scale_format="rowmajor")[0, :32].isnan().all())


def test_no_rows(bs, orc, cuda):
    """Zero tokens: outputs of no rows, gradients of the weights zero."""
    k, f = 256, 64
    p = Gated(bs, orc, cuda, 1, f, k, False, 80)
    none = p.a.d[:0]
    assert bs.linear_a8w8_mxfp8(none, p.b, p.a.native[:0], p.b_native).shape == (0, 2 * f)
    assert bs.gated_a8w8_mxfp8(none, p.b, p.a.native[:0], p.b_native).shape == (0, f)
    h = torch.empty((0, f), dtype=torch.bfloat16, device=cuda)
    da, dg, du = bs.gated_a8w8_mxfp8_backward(h, none, p.b, p.a.native[:0], p.b_native)
    assert da.shape == (0, k) and bool((dg == 0).all()) and bool((du == 0).all())
    x = torch.empty((0, 100), device=cuda)
    y, mean, rstd = bs.layer_norm(x, return_stats=True)
    assert y.shape == (0, 100) and mean.shape == (0,)
    dx, dw, db = bs.layer_norm_backward(x, x, torch.ones(100, device=cuda), mean, rstd)
    assert dx.shape == (0, 100) and bool((dw == 0).all()) and bool((db == 0).all())
    assert bs.dequantize(none, p.a.native[:0], "mxfp8").shape == (0, k)


def test_other_stream(bs, orc, cuda):
    """On a stream of their own, behind that stream's work, and with their inputs freed at once."""
    m, f, k = 70, 256, 512
    p = Gated(bs, orc, cuda, m, f, k, False, 90)
    x = norm_data(orc, m, k, 91, cuda, torch.bfloat16)
    w = torch.ones(k, dtype=torch.bfloat16, device=cuda)
    q, sf = bs.layer_norm(x, w, None, out_format="mxfp8")
    want = bs.gated_a8w8_mxfp8(q, p.b, sf, p.b_native)
    grads = bs.gated_a8w8_mxfp8_backward(want, q, p.b, sf, p.b_native)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        for _ in range(50):
            late = late + 0.02 * x.float().abs().mean() * 0   # keeps the stream busy
        late = late.to(torch.bfloat16) + x
        q2, sf2 = bs.layer_norm(late, w, None, out_format="mxfp8")
        del late
        got = bs.gated_a8w8_mxfp8(q2, p.b, sf2, p.b_native)
        got_grads = bs.gated_a8w8_mxfp8_backward(got, q2, p.b, sf2, p.b_native)
        del q2, sf2
    side.synchronize()
    assert torch.equal(got, want)
    for a, b in zip(got_grads, grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m", [1, 33, 300])
def test_feed_forward_block(bs, orc, cuda, fmt, m):
    """norm -> gated -> linear + residual through MX elements only, each step
    against the formula on the elements that the step before it gave."""
    fp4 = fmt == "mxfp4"
    d, f = 512, 512
    x = norm_data(orc, m, d, 92, cuda, torch.bfloat16)
    w, b = 1 + 0.1 * normal(orc, (d,), 93, cuda), normal(orc, (d,), 94, cuda)
    p = Gated(bs, orc, cuda, 1, f, d, fp4, 95)
    w2 = Operand(bs, orc, cuda, d, f, fp4, 98, f ** -0.5)
    q, sf = bs.layer_norm(x, w, b, out_format=fmt)
    h, hs = gated(bs, fp4)(q, p.b, sf, p.b_native, out_format=fmt)
    y = linear(bs, fp4)(h, w2.d, hs, w2.native, residual=x)
    p.a.v = bs.dequantize(q, sf, fmt, out_dtype=torch.float32).double().cpu()
    ref, _ = p.ref("silu")
    hv = bs.dequantize(h, hs, fmt, out_dtype=torch.float32).double().cpu()
    # an element is within half a spacing: 2^-4 of E4M3's value, 1/5 of E2M1's, or half the smallest step under the scale
    amax = ref.abs().reshape(m, -1, 32).amax(-1, keepdim=True)
    half = (amax / 6 * 2 * 0.25 if fp4 else amax / 448 * 2 * 2.0 ** -10).expand(m, f // 32, 32).reshape(m, f)
    assert_within(hv, ref, (0.25 if fp4 else 2.0 ** -4) * ref.abs() * 1.001 + half * 1.001)
    a2 = type("A", (), {})()
    a2.v = hv
    ref, tol = linear_ref(a2, w2, None, None, x)
    assert_within(y, ref, tol + rounding(ref, torch.bfloat16))


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh", "relu", None])
def test_gated_backward_large(bs, orc, cuda, name):
    """Gate values of about 2^68, whose square is past fp32: every slope is 0 or 1
    there, and the gradients are as close as at any other size."""
    m, f, k = 70, 96, 256
    a, g, u = (Operand(bs, orc, cuda, rows, k, False, seed) for rows, seed in ((m, 110), (f, 111), (f, 112)))
    for x, by in ((a, 34), (g, 34), (u, -34)):
        x.rowmajor = (x.rowmajor.int() + by).to(torch.uint8)
        x.native, x.v = bs.pack_scales(x.rowmajor), x.v * 2.0 ** by
    b, b_native = bs.pack_gated(g.d, u.d, g.rowmajor, u.rowmajor)
    h = normal(orc, (m, f), 113, cuda)
    hv, pre, up = h.double().cpu(), a.v @ g.v.T, a.v @ u.v.T
    dg, du = hv * up * act_slope(pre, name), hv * act(pre, name)
    got = bs.gated_a8w8_mxfp8_backward(h, a.d, b, a.native, b_native, activation=name)
    for x, ref, what in zip(got, (dg @ g.v + du @ u.v, dg.T @ a.v, du.T @ a.v), ("dA", "dWg", "dWu")):
        assert bool(x.isfinite().all()), what
        assert rel_norm(x, ref) < 3.3e-3, what
    y = bs.gated_a8w8_mxfp8(a.d, b, a.native, b_native, activation=name)
    assert rel_norm(y, act(pre, name) * up) < 2.3e-3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_mx_parameters_off_alignment(bs, orc, cuda, dtype):
    """Parameters that are views at any offset give the bits of aligned ones, MX outputs too."""
    for rows, cols in ((3, 384), (5, 1536)):
        x = norm_data(orc, rows, cols, 120, cuda, torch.bfloat16)
        flat = normal(orc, (2 * cols + 3,), 121, cuda, dtype)
        w, b = flat[1:1 + cols], flat[2 + cols:2 + 2 * cols]
        for fmt in ("mxfp8", "mxfp4"):
            got = bs.layer_norm(x, w, b, out_format=fmt)
            want = bs.layer_norm(x, w.clone(), b.clone(), out_format=fmt)
            assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("kernel", ["swap", "1cta", "pair"])
@pytest.mark.parametrize("m,n", [(1, 4), (18, 140), (50, 148), (64, 20)])
def test_linear_ragged_fp32(bs, orc, cuda, fp4, kernel, m, n):
    """fp32 outputs of any multiple of 4 columns, with both residual types, inside a
    larger tensor whose other elements stay as they are."""
    k = 512
    a, b = Operand(bs, orc, cuda, m, k, fp4, 130), Operand(bs, orc, cuda, n, k, fp4, 131, k ** -0.5)
    bias = normal(orc, (n,), 132, cuda, torch.float32)
    for dtype in (torch.float32, torch.bfloat16):
        wide = normal(orc, (m, (n + 7) // 8 * 8), 133, cuda, dtype)
        residual = wide[:, :n]
        out = torch.full((m, n + 8), 7.0, device=cuda)
        linear(bs, fp4)(a.d, b.d, a.native, b.native, bias=bias, activation="gelu", residual=residual, kernel=kernel,
                        out_dtype=torch.float32, out=out[:, :n])
        ref, tol = linear_ref(a, b, bias, "gelu", residual)
        assert_within(out[:, :n], ref, tol + rounding(ref, torch.float32))
        assert bool((out[:, n:] == 7).all())
    assert bs.check_device_error() == 0


@pytest.mark.parametrize("m,f,k", [(40, 64, 256), (128, 1024, 2048), (333, 512, 4096)])
@pytest.mark.parametrize("scale_format", ["native", "rowmajor"])
def test_gated_backward_behind_its_inputs(bs, orc, cuda, m, f, k, scale_format):
    """Calls in a row over one set of buffers, each behind the kernel that writes its
    operand, give what they give one at a time."""
    p = Gated(bs, orc, cuda, 1, f, k, False, 140)
    b_scale = p.b_native if scale_format == "native" else bs.unpack_scales(p.b_native, 2 * f, k // 32)
    xs, hs = [normal(orc, (m, k), 143 + i, cuda) for i in range(4)], [normal(orc, (m, f), 150 + i, cuda) for i in range(4)]
    q, sf = bs.layer_norm(xs[0], out_format="mxfp8", scale_format=scale_format)
    workspace = torch.empty(4 * m * f + 2 * m * k + 4 * f * k + 65536 + 8 * (m + 128 + 2 * f) * (k // 32),
                            dtype=torch.uint8, device=cuda)

    def call(i, one_at_a_time):
        if scale_format == "native":
            bs.layer_norm(xs[i], out_format="mxfp8", out=(q, sf))
        else:
            for to, made in zip((q, sf), bs.layer_norm(xs[i], out_format="mxfp8", scale_format=scale_format)):
                to.copy_(made)
        if one_at_a_time:
            torch.cuda.synchronize()
        return bs.gated_a8w8_mxfp8_backward(hs[i], q, p.b, sf, b_scale, scale_format=scale_format, workspace=workspace)

    want = []
    for i in range(4):
        want.append(call(i, True))
        torch.cuda.synchronize()
    for _ in range(5):
        got = [call(i, False) for i in range(4)]
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))
