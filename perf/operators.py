"""Workloads of the operators around the block-scaled GEMMs: layer norm and its
gradient, a linear layer with bias, activation and residual, and the gated
feed-forward product with its gradient.

A pass of each is run either in its plain form (elementary torch operations in
fp32, rounded once at the end) or, with ``own`` set, by this library's kernels.
Both take the same stored operands: MXFP8 / MXFP4 elements with their E8M0
scales as 512-byte atoms, gate and up weights interleaved in blocks of 32 rows.
"""
import importlib
import math

import torch

own = False

GROUP = 32           # elements per E8M0 scale
MOST_FLOPS = 2.2e12  # of one pass; the largest listed case has 2.17e12
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2.0, "fp32": 4.0, "mxfp8": 1.0 + 1.0 / GROUP, "mxfp4": 0.5 + 1.0 / GROUP}
QMAX = {"mxfp8": 448.0, "mxfp4": 6.0}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # the norm before a projection for one decoded token, quantised for the MXFP8 product behind it
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 7168, "dtype": "bf16", "out": "mxfp8"},
        # the same norm over the prompts of a serving batch, kept in bf16
        {"name": "norm prompt", "op": "norm", "rows": 16384, "cols": 7168, "dtype": "bf16", "out": "bf16"},
        # its gradient in a training step of 8192 tokens
        {"name": "norm grad", "op": "norm_grad", "rows": 8192, "cols": 7168, "dtype": "bf16"},
        # a small odd model in fp32: no row starts on a 16-byte boundary but one in four
        {"name": "norm grad odd", "op": "norm_grad", "rows": 1023, "cols": 1537, "dtype": "fp32"},
        # an expert's down projection for one token, MXFP4 weights
        {"name": "linear one token", "op": "linear", "fmt": "mxfp4", "m": 1, "n": 7168, "k": 2048, "act": "none",
         "bias": True, "residual": True, "out": "bf16"},
        # the first product of a feed-forward block for a decode batch of 100, quantised for the second
        {"name": "linear batch", "op": "linear", "fmt": "mxfp8", "m": 100, "n": 4096, "k": 7168, "act": "gelu",
         "bias": True, "residual": False, "out": "mxfp8"},
        # the down projection of a dense block over a prompt of 8192 tokens, added to the residual stream
        {"name": "linear prompt", "op": "linear", "fmt": "mxfp8", "m": 8192, "n": 7168, "k": 18432, "act": "none",
         "bias": True, "residual": True, "out": "bf16"},
        # a ragged prompt, MXFP4, with logits or a loss behind it in fp32
        {"name": "linear ragged", "op": "linear", "fmt": "mxfp4", "m": 1000, "n": 8192, "k": 7168, "act": "silu",
         "bias": True, "residual": False, "out": "fp32"},
        # an expert's gate and up projections for a decode batch of 16
        {"name": "gated batch", "op": "gated", "fmt": "mxfp8", "m": 16, "f": 2048, "k": 7168, "act": "silu", "out": "mxfp8"},
        # a dense block's gate and up projections over a prompt of 4096 tokens
        {"name": "gated prompt", "op": "gated", "fmt": "mxfp8", "m": 4096, "f": 18432, "k": 7168, "act": "silu", "out": "bf16"},
        # the gradient for the few tokens that a router sent to one expert, MXFP4 weights
        {"name": "gated grad ragged", "op": "gated_grad", "fmt": "mxfp4", "m": 333, "f": 2048, "k": 7168, "act": "gelu"},
        # the gradient for a training step of 8192 tokens
        {"name": "gated grad", "op": "gated_grad", "fmt": "mxfp8", "m": 8192, "f": 2048, "k": 7168, "act": "silu"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    v = min(hi, max(lo, int(v) // step * step))
    return v + step if v == 3072 else v


def draw(rng):
    op = rng.choice(("norm", "norm_grad", "linear", "linear", "gated", "gated_grad"))
    if op in ("norm", "norm_grad"):
        c = {"op": op, "rows": _log_int(rng, 1, 16384), "cols": _log_int(rng, 32, 12288), "dtype": rng.choice(("bf16", "fp32"))}
        if op == "norm":
            c["out"] = rng.choice(("bf16", "fp32", "mxfp8", "mxfp4"))
            if c["out"] in QMAX:
                c["cols"] = max(128, c["cols"] // 128 * 128)
            if c["cols"] == 3072:
                c["cols"] += 128
        return c
    fmt = rng.choice(("mxfp8", "mxfp4"))
    c = {"op": op, "fmt": fmt, "m": _log_int(rng, 1, 8192), "k": _log_int(rng, 256, 18432, 256), "act": rng.choice(ACTIVATIONS)}
    if op == "linear":
        c["out"] = rng.choice(("bf16", "fp32", "mxfp8", "mxfp4"))
        if c["out"] == "fp32":    # what is kept in fp32 are short contractions: heads and routers over a hidden size
            c["k"] = min(c["k"], 7168)
        c["n"] = _log_int(rng, 128, 18432, 128 if c["out"] in QMAX else 8)
        c["bias"], c["residual"] = rng.random() < 0.7, rng.random() < 0.5
    else:
        if op == "gated":
            c["out"] = rng.choice(("bf16", "bf16", "mxfp8", "mxfp4"))
        c["f"] = _log_int(rng, 128, 18432, 128 if c.get("out") in QMAX else 32)
    while work(c)["flops"] > MOST_FLOPS:
        c["m"] = max(1, c["m"] // 2)
    return c


def work(case):
    """Bytes and operations that a pass cannot do without: each input read once,
    each output written once; the gradient of the gated product needs both
    projections again and two products of the same size."""
    op = case["op"]
    if op in ("norm", "norm_grad"):
        r, c, e = case["rows"], case["cols"], BYTES[case["dtype"]]
        if op == "norm":
            return {"bytes": r * c * (e + BYTES[case["out"]]) + 2 * c * e, "flops": 8 * r * c}
        return {"bytes": 3 * r * c * e + 8 * r + 3 * c * e, "flops": 14 * r * c}
    m, k, e = case["m"], case["k"], BYTES[case["fmt"]]
    if op == "linear":
        n = case["n"]
        extra = (2 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0)
        return {"bytes": (m + n) * k * e + m * n * BYTES[case["out"]] + extra, "flops": 2.0 * m * n * k}
    n = 2 * case["f"]
    if op == "gated":
        return {"bytes": (m + n) * k * e + m * case["f"] * BYTES[case["out"]], "flops": 2.0 * m * n * k}
    return {"bytes": (m + n) * k * (e + 2) + m * case["f"] * 2, "flops": 6.0 * m * n * k}


# ---- stored formats -----------------------------------------------------------

def _quantise(x, fmt):
    """fp32 [rows, cols] -> (elements, E8M0 bytes [rows, cols / 32]): scale
    2^ceil(log2(amax / qmax)), elements rounded to nearest even."""
    rows, cols = x.shape
    g = x.reshape(rows, cols // GROUP, GROUP)
    mant, e = torch.frexp(g.abs().amax(-1).double() / QMAX[fmt])
    e = torch.where(mant == 0.5, e - 1, e)
    e = torch.where(mant == 0, torch.zeros_like(e), e).clamp(-127, 127)
    v = torch.ldexp(g, -e.unsqueeze(-1)).reshape(rows, cols)
    if fmt == "mxfp8":
        q = v.to(torch.float8_e4m3fn)
    else:
        a = v.abs()
        code = torch.zeros_like(a, dtype=torch.uint8)
        for i in range(7):     # a tie goes to the even code
            mid = (E2M1[i] + E2M1[i + 1]) / 2
            code += (a >= mid) if i % 2 else (a > mid)
        code |= torch.signbit(v).to(torch.uint8) << 3
        q = code[:, 0::2] | (code[:, 1::2] << 4)
    return q, (e + 127).to(torch.uint8)


def _atoms(sf):
    """E8M0 bytes [rows, groups] -> 512-byte atoms of 128 rows x 4 groups."""
    rows, kg = sf.shape
    full = torch.full(((rows + 127) // 128 * 128, (kg + 3) // 4 * 4), 127, dtype=torch.uint8, device=sf.device)
    full[:rows, :kg] = sf
    return full.reshape(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().reshape(-1)


def _from_atoms(atoms, rows, kg):
    a = atoms.reshape((rows + 127) // 128, (kg + 3) // 4, 32, 4, 4).permute(0, 3, 2, 1, 4)
    return a.reshape(-1, (kg + 3) // 4 * 4)[:rows, :kg]


def _values(q, sf, fmt):
    """The fp32 values that elements with E8M0 bytes [rows, groups] stand for."""
    if fmt == "mxfp8":
        v = q.float()
    else:
        table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=q.device)
        v = table[torch.stack((q & 15, q >> 4), dim=-1).reshape(q.shape[0], -1).int()]
    rows, cols = v.shape
    s = torch.ldexp(torch.ones_like(sf, dtype=torch.float32), sf.int() - 127)
    return (v.reshape(rows, cols // GROUP, GROUP) * s.unsqueeze(-1)).reshape(rows, cols)


def _round(y, out):
    """The one rounding at the end: to bf16 / fp32, or to the values that MX elements stand for."""
    if out in DTYPES:
        return y.to(DTYPES[out])
    q, sf = _quantise(y, out)
    return _values(q, sf, out).to(torch.bfloat16)


# ---- inputs -------------------------------------------------------------------

def _operand(rows, cols, fmt, std, g, interleave=False):
    q, sf = [], []
    for r0 in range(0, rows, 4096):
        x = torch.randn((min(4096, rows - r0), cols), device="cuda", generator=g) * std
        a, b = _quantise(x, fmt)
        q.append(a), sf.append(b)
    return torch.cat(q), _atoms(torch.cat(sf))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] in ("norm", "norm_grad"):
        r, c, t = case["rows"], case["cols"], DTYPES[case["dtype"]]
        # a residual stream: channels of unequal size, some far larger, and a mean that is not zero
        x = normal(r, c) * (0.5 + normal(c).abs()) * torch.where(torch.rand(c, device="cuda", generator=g) < 0.01, 20.0, 1.0) + 0.3
        s.update(x=x.to(t), weight=(1 + 0.1 * normal(c)).to(t), bias=(0.1 * normal(c)).to(t), eps=1e-5)
        if case["op"] == "norm_grad":
            s["dy"] = normal(r, c).to(t)
            xf = s["x"].float()
            s["mean"] = xf.mean(-1)
            s["rstd"] = ((xf - s["mean"][:, None]).square().mean(-1) + s["eps"]).rsqrt()
        return s
    m, k, fmt = case["m"], case["k"], case["fmt"]
    s["a"], s["a_scale"] = _operand(m, k, fmt, 1.0, g)
    n = case["n"] if case["op"] == "linear" else 2 * case["f"]
    # gate and up rows are drawn alike, so their interleaved form is drawn directly
    s["b"], s["b_scale"] = _operand(n, k, fmt, k ** -0.5, g)
    if case["op"] == "linear":
        s["bias_t"] = (0.1 * normal(n)).bfloat16() if case["bias"] else None
        s["residual_t"] = normal(m, n).bfloat16() if case["residual"] else None
    elif case["op"] == "gated_grad":
        s["grad"] = normal(m, case["f"]).bfloat16()
    return s


# ---- the operators --------------------------------------------------------------

def _act(x, name):
    if name == "relu":
        return x.clamp_min(0)
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return x


def _act_grad(x, name):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    if name == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    return torch.ones_like(x)


def _plain(s):
    op = s["op"]
    if op == "norm":
        x = s["x"].float()
        d = x - x.mean(-1, keepdim=True)
        y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float() + s["bias"].float()
        return _round(y, s["out"])
    if op == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
        wdy = dy * s["weight"].float()
        dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xhat * (wdy * xhat).mean(-1, keepdim=True))
        t = s["x"].dtype
        return dx.to(t), (dy * xhat).sum(0).to(t), dy.sum(0).to(t)
    m, k, fmt = s["m"], s["k"], s["fmt"]
    a = _values(s["a"], _from_atoms(s["a_scale"], m, k // GROUP), fmt)
    n = s["b"].shape[0]
    b = _values(s["b"], _from_atoms(s["b_scale"], n, k // GROUP), fmt)
    if op == "linear":
        y = a @ b.t()
        if s["bias_t"] is not None:
            y = y + s["bias_t"].float()
        y = _act(y, s["act"])
        if s["residual_t"] is not None:
            y = y + s["residual_t"].float()
        return _round(y, s["out"])
    halves = b.reshape(-1, 2, 32, k)
    wg, wu = halves[:, 0].reshape(-1, k), halves[:, 1].reshape(-1, k)
    gate, up = a @ wg.t(), a @ wu.t()
    if op == "gated":
        return _round(_act(gate, s["act"]) * up, s["out"])
    grad = s["grad"].float()
    dgate, dup = grad * up * _act_grad(gate, s["act"]), grad * _act(gate, s["act"])
    da = dgate @ wg + dup @ wu
    return da.bfloat16(), (dgate.t() @ a).bfloat16(), (dup.t() @ a).bfloat16()


def _own(s):
    bs = importlib.import_module("355_1_trans_b200")
    op = s["op"]
    if op == "norm":
        if s["out"] in QMAX:
            q, sf = bs.layer_norm(s["x"], s["weight"], s["bias"], s["eps"], out_format=s["out"])
            return bs.dequantize(q, sf, s["out"])
        return bs.layer_norm(s["x"], s["weight"], s["bias"], s["eps"], out_dtype=DTYPES[s["out"]])
    if op == "norm_grad":
        return bs.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
    fp4 = s["fmt"] == "mxfp4"
    operands = (s["a"], s["b"], s["a_scale"], s["b_scale"])
    if op == "gated_grad":
        f = bs.gated_a4w4_mxfp4_backward if fp4 else bs.gated_a8w8_mxfp8_backward
        return f(s["grad"], *operands, activation=s["act"])
    how = {"out_format": s["out"]} if s["out"] in QMAX else {"out_dtype": DTYPES[s["out"]]}
    if op == "linear":
        f = bs.linear_a4w4_mxfp4 if fp4 else bs.linear_a8w8_mxfp8
        y = f(*operands, bias=s["bias_t"], activation=s["act"], residual=s["residual_t"], **how)
    else:
        f = bs.gated_a4w4_mxfp4 if fp4 else bs.gated_a8w8_mxfp8
        y = f(*operands, activation=s["act"], **how)
    return bs.dequantize(*y, s["out"]) if s["out"] in QMAX else y


def run(s):
    """One pass through the case's operator."""
    return _own(s) if own else _plain(s)


# ---- the definition in 64 bits ----------------------------------------------------

def _f64(q, atoms, fmt):
    """Stored elements and scale atoms -> fp64 values, from the formats' bit fields."""
    rows = q.shape[0]
    if fmt == "mxfp8":
        byte = q.view(torch.uint8).long()
        sign, e, f = byte >> 7, (byte >> 3) & 15, byte & 7
        v = torch.where(e == 0, f.double() / 8 * 2.0 ** -6, torch.ldexp(1 + f.double() / 8, e - 7))
    else:
        code = torch.empty((rows, 2 * q.shape[1]), dtype=torch.long, device=q.device)
        code[:, 0::2], code[:, 1::2] = (q & 15).long(), (q >> 4).long()
        sign, e, f = code >> 3, (code >> 1) & 3, code & 1
        v = torch.where(e == 0, f.double() / 2, torch.ldexp(1 + f.double() / 2, e - 1))
    v = torch.where(sign == 1, -v, v)
    r = torch.arange(rows, device=q.device)[:, None]
    g = torch.arange(v.shape[1] // GROUP, device=q.device)[None, :]
    columns = -(-g.shape[1] // 4)
    at = ((r // 128) * columns + g // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + g % 4
    return v * torch.exp2(atoms[at].double() - 127).repeat_interleave(GROUP, 1)


def _rows_f64(s, which, rows):
    """The fp64 values of some rows of an operand, at most 4096 at a time."""
    k = s["k"]
    out = torch.empty((len(rows), k), dtype=torch.float64, device="cuda")
    full = s[which].shape[0]
    for r0 in range(0, full, 4096):
        here = (rows >= r0) & (rows < r0 + 4096)
        part = s[which][r0:r0 + 4096]
        atoms = s[which + "_scale"][r0 // 128 * (-(-k // 128)) * 512:]
        out[here] = _f64(part, atoms, s["fmt"])[rows[here] - r0]
    return out


def exact(case, seed):
    """What run returns, from the definition in fp64; for an MXFP8 output the
    values before they are rounded to its elements.  MXFP4 elements are a sixth
    of a value apart, so there the unrounded values would say nothing."""
    if case.get("out") == "mxfp4":
        return None
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        return (x - mean) / (var + s["eps"]).sqrt() * s["weight"].double() + s["bias"].double()
    if op == "norm_grad":
        x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        c = x.shape[1]
        rstd = s["rstd"].double()[:, None]
        z = (x - s["mean"].double()[:, None]) * rstd
        t = dy * w
        dx = (c * t - t.sum(1, keepdim=True) - z * (t * z).sum(1, keepdim=True)) * rstd / c
        return dx, torch.einsum("rc,rc->c", dy, z), torch.einsum("rc->c", dy)
    a = _rows_f64(s, "a", torch.arange(case["m"], device="cuda"))
    sqrt2 = math.sqrt(2.0)

    def f(v):
        return {"none": lambda: v, "relu": lambda: torch.where(v > 0, v, torch.zeros_like(v)),
                "gelu": lambda: v * torch.special.erfc(-v / sqrt2) / 2,
                "gelu_tanh": lambda: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
                "silu": lambda: v * torch.sigmoid(v)}[case["act"]]()

    def df(v):
        if case["act"] == "none":
            return torch.ones_like(v)
        if case["act"] == "relu":
            return (v > 0).double()
        if case["act"] == "gelu":
            return torch.special.erfc(-v / sqrt2) / 2 + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        c, d = (2 * math.sqrt(2 / math.pi), 0.044715) if case["act"] == "gelu_tanh" else (1.0, 0.0)
        p = torch.sigmoid(c * (v + d * v ** 3))
        return p + v * p * (1 - p) * c * (1 + 3 * d * v * v)

    if op == "linear":
        b = _rows_f64(s, "b", torch.arange(case["n"], device="cuda"))
        y = a @ b.T
        if s["bias_t"] is not None:
            y += s["bias_t"].double()
        y = f(y)
        if s["residual_t"] is not None:
            y += s["residual_t"].double()
        return y
    i = torch.arange(case["f"], device="cuda")
    wg = _rows_f64(s, "b", i // 32 * 64 + i % 32)
    wu = _rows_f64(s, "b", i // 32 * 64 + 32 + i % 32)
    gate, up = a @ wg.T, a @ wu.T
    if op == "gated":
        return f(gate) * up
    h = s["grad"].double()
    p, q = h * up * df(gate), h * f(gate)
    return p @ wg + q @ wu, p.T @ a, q.T @ a
