"""examples/feed_forward_block.py: its training step against autograd in 64 bits
on the values that its quantised operands stand for."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "examples" / "feed_forward_block.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("feed_forward_block", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("tokens", [1, 70])
def test_training_step(bs, cuda, example, fmt, tokens):
    hidden, ffn = 512, 256
    block = example.make(hidden, ffn, fmt)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn((tokens, hidden), device=cuda, generator=g).bfloat16()
    dy = torch.randn((tokens, hidden), device=cuda, generator=g).bfloat16()
    y, grads = block.step(x, lambda _: dy)
    assert torch.equal(y, block(x))
    # the elements between the steps, as the step itself made them
    q, sf, mean, rstd = bs.layer_norm(x, block.norm_weight, block.norm_bias, out_format=fmt, return_stats=True)
    h, hs = block.gated(q, block.w13, sf, block.w13_scale, out_format=fmt)

    def value(e, s):
        return bs.dequantize(e, s, fmt, out_dtype=torch.float32).double()

    w13 = value(block.w13, block.w13_scale).reshape(-1, 2, 32, hidden)
    gate, up = (w13[:, i].reshape(-1, hidden) for i in (0, 1))
    down, zq, hq = value(block.w2, block.w2_scale), value(q, sf), value(h, hs)
    d = dy.double()
    dh = d @ down
    a, b = zq @ gate.T, zq @ up.T
    s = torch.sigmoid(a)
    da, db = dh * b * s * (1 + a * (1 - s)), dh * a * s
    dz = da @ gate + db @ up
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    r = 1 / ((xd - m).square().mean(1, keepdim=True) + 1e-5).sqrt()
    z = (xd - m) * r
    t = dz * block.norm_weight.double()
    want = {"x": d + r * (t - t.mean(1, keepdim=True) - z * (t * z).mean(1, keepdim=True)),
            "norm_weight": (dz * z).sum(0), "norm_bias": dz.sum(0), "gate": da.T @ zq, "up": db.T @ zq, "down": d.T @ hq}
    # roundings to bf16 of relative size 2^-8 / sqrt 3 at most each, independent: dh, dg and du, dz, the output, and for x a sum
    bound = {"x": 5, "norm_weight": 4, "norm_bias": 4, "gate": 3, "up": 3, "down": 1}
    for name, ref in want.items():
        rel = float((grads[name].double() - ref).norm() / ref.norm())
        assert rel <= 2.0 ** -8 / math.sqrt(3) * math.sqrt(bound[name]), (name, rel)
    assert bs.check_device_error() == 0
