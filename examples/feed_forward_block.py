"""A transformer's feed-forward block on the library's operators:

    y = x + (act(z Wg^T) * (z Wu^T)) W2^T,   z = layer_norm(x)

Serving: three launches (layer norm -> gated product -> linear with residual)
with nothing but MX elements and their scales between them.  Training: the
gradients of x, the norm's parameters and the three weights, taken through the
quantisation as if it were the identity.

    python examples/feed_forward_block.py [--hidden 7168] [--ffn 2048] [--fmt mxfp8] [--tokens 1,16,1024,8192]
"""
import argparse
import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
bs = importlib.import_module("355_1_trans_b200")


class FeedForward:
    """Weights are quantised and laid out once, as a serving program would keep them."""

    def __init__(self, gate, up, down, norm_weight, norm_bias, fmt="mxfp8", activation="silu"):
        self.fmt, self.activation = fmt, activation
        fp4 = fmt == "mxfp4"
        self.gated = bs.gated_a4w4_mxfp4 if fp4 else bs.gated_a8w8_mxfp8
        self.gated_backward = bs.gated_a4w4_mxfp4_backward if fp4 else bs.gated_a8w8_mxfp8_backward
        self.linear = bs.linear_a4w4_mxfp4 if fp4 else bs.linear_a8w8_mxfp8
        (g, gs), (u, us) = (bs.quantize(w, fmt, scale_format="rowmajor") for w in (gate, up))
        self.w13, self.w13_scale = bs.pack_gated(g, u, gs, us)
        self.w2, self.w2_scale = bs.quantize(down, fmt)
        self.norm_weight, self.norm_bias = norm_weight, norm_bias

    def __call__(self, x):
        q, sf = bs.layer_norm(x, self.norm_weight, self.norm_bias, out_format=self.fmt)
        h, hs = self.gated(q, self.w13, sf, self.w13_scale, activation=self.activation, out_format=self.fmt)
        return self.linear(h, self.w2, hs, self.w2_scale, residual=x)

    def step(self, x, grad_of):
        """Forward and backward: y, then {name: gradient} for dL/dy = grad_of(y)."""
        q, sf, mean, rstd = bs.layer_norm(x, self.norm_weight, self.norm_bias, out_format=self.fmt, return_stats=True)
        h, hs = self.gated(q, self.w13, sf, self.w13_scale, activation=self.activation, out_format=self.fmt)
        y = self.linear(h, self.w2, hs, self.w2_scale, residual=x)
        dy = grad_of(y)
        dh = dy @ bs.dequantize(self.w2, self.w2_scale, self.fmt)
        dz, dgate, dup = self.gated_backward(dh, q, self.w13, sf, self.w13_scale, activation=self.activation)
        dx, dnorm_weight, dnorm_bias = bs.layer_norm_backward(dz, x, self.norm_weight, mean, rstd)
        return y, {"x": dx.add_(dy), "norm_weight": dnorm_weight, "norm_bias": dnorm_bias, "gate": dgate, "up": dup,
                   "down": dy.t() @ bs.dequantize(h, hs, self.fmt)}


def make(hidden, ffn, fmt, device="cuda", seed=0):
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(shape, device=device, generator=g) * std).bfloat16()

    return FeedForward(normal(ffn, hidden, std=hidden ** -0.5), normal(ffn, hidden, std=hidden ** -0.5),
                       normal(hidden, ffn, std=ffn ** -0.5), 1 + normal(hidden, std=0.1), normal(hidden, std=0.1), fmt)


def timed(f, repeats=20):
    for _ in range(3):
        f()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    begin.record()
    for _ in range(repeats):
        f()
    end.record()
    torch.cuda.synchronize()
    return begin.elapsed_time(end) / repeats * 1e3


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--hidden", type=int, default=7168)
    p.add_argument("--ffn", type=int, default=2048)
    p.add_argument("--fmt", choices=("mxfp8", "mxfp4"), default="mxfp8")
    p.add_argument("--tokens", default="1,16,1024,8192")
    a = p.parse_args()
    block = make(a.hidden, a.ffn, a.fmt)
    for tokens in map(int, a.tokens.split(",")):
        x = torch.randn((tokens, a.hidden), device="cuda").bfloat16()
        serve = timed(lambda: block(x))
        train = timed(lambda: block.step(x, torch.ones_like))
        print(f"{tokens} tokens, hidden {a.hidden}, ffn {a.ffn}, {a.fmt}: forward {serve:.1f} us, training step {train:.1f} us")
    if bs.check_device_error():
        raise RuntimeError("a device-side wait ran out")


if __name__ == "__main__":
    main()
