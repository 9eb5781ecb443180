"""Operators in a row over one set of buffers, each behind the kernel that writes
what it reads and some over their own inputs: the kernels start while the one
before still runs, and give the bits that they give one at a time."""
import pytest
import torch

pytestmark = pytest.mark.gpu

REPEATS = 5


def normal(orc, shape, seed, cuda, dtype=torch.bfloat16):
    return torch.from_numpy(orc.normal(shape, seed=seed)).to(cuda).to(dtype)


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def steps(step, count, one_at_a_time):
    out = []
    for i in range(count):
        if one_at_a_time:
            torch.cuda.synchronize()
        out.append(step(i, torch.cuda.synchronize if one_at_a_time else lambda: None))
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 1536), (40, 512), (64, 7168), (300, 1000), (700, 2048), (1000, 4104)])
def test_linear_then_norm_on_one_buffer(bs, orc, cuda, m, n, dtype):
    """x = layer_norm(x + A B^T), both in place."""
    k = 256
    q, sf = bs.quantize(normal(orc, (m, k), 1, cuda), "mxfp8")
    w, wsf = bs.quantize(normal(orc, (n, k), 2, cuda), "mxfp8")
    weight, bias = normal(orc, (n,), 3, cuda, dtype), normal(orc, (n,), 4, cuda, dtype)
    first = normal(orc, (m, n), 5, cuda, dtype)

    def chain(one_at_a_time):
        x = first.clone()

        def step(i, between):
            bs.linear_a8w8_mxfp8(q, w, sf, wsf, residual=x, out=x, out_dtype=dtype)
            between()
            bs.layer_norm(x, weight, bias, out=x)

        steps(step, 6, one_at_a_time)
        return x

    want = chain(True)
    assert bool(want.isfinite().all())
    for _ in range(REPEATS):
        assert same(chain(False), want)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("rows,cols", [(1, 7168), (129, 512), (2000, 2048)])
def test_dequantize_behind_its_writer(bs, orc, cuda, rows, cols, fmt):
    xs = [normal(orc, (rows, cols), 10 + i, cuda) for i in range(4)]
    q, sf = bs.quantize(xs[0], fmt)

    def step(i, between):
        bs.layer_norm(xs[i], out_format=fmt, out=(q, sf))
        between()
        return bs.dequantize(q, sf, fmt)

    want = steps(step, 4, True)
    for _ in range(REPEATS):
        assert all(map(same, steps(step, 4, False), want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(3, 264), (500, 1000), (900, 1537), (700, 4096), (300, 16384)])
@pytest.mark.parametrize("over", ["dy", "x"])
def test_norm_gradient_in_place(bs, orc, cuda, rows, cols, dtype, over):
    """dx over dy or over x, behind the kernel that writes that buffer."""
    x0, dy0 = normal(orc, (rows, cols), 20, cuda, dtype), normal(orc, (rows, cols), 21, cuda, dtype)
    weight = normal(orc, (cols,), 22, cuda, dtype)
    _, mean, rstd = bs.layer_norm(x0, weight, return_stats=True)
    x, dy = x0.clone(), dy0.clone()
    plain = bs.layer_norm_backward(dy0, x0, weight, mean, rstd)

    def step(i, between):
        x.copy_(x0)
        between()
        dy.copy_(dy0)
        between()
        got = bs.layer_norm_backward(dy, x, weight, mean, rstd, out=dy if over == "dy" else x)
        return [t.clone() for t in got]

    for one_at_a_time in (True,) + (False,) * REPEATS:
        for got in steps(step, 3, one_at_a_time):
            assert all(map(same, got, plain))


COPIED = ["layer_norm columns", "layer_norm offset", "layer_norm parameters", "layer_norm_backward", "linear residual",
          "gated_backward grad", "dequantize", "pack_gated"]


@pytest.mark.parametrize("what", COPIED)
def test_copied_inputs_freed_on_another_stream(bs, orc, cuda, what):
    """A caller's tensor that has to be copied first is still its own while the copy waits
    on a busy stream, however soon the caller drops it."""
    m, n, k, f = 96, 512, 256, 128
    q, sf = bs.quantize(normal(orc, (m, k), 30, cuda), "mxfp8")
    w, wsf = bs.quantize(normal(orc, (n, k), 31, cuda), "mxfp8")
    b, bsf = bs.quantize(normal(orc, (2 * f, k), 32, cuda), "mxfp8")
    weight = normal(orc, (n,), 33, cuda)
    rows = normal(orc, (m, n), 34, cuda)
    _, mean, rstd = bs.layer_norm(rows, return_stats=True)
    gate, gate_sf = bs.quantize(normal(orc, (f, k), 35, cuda), "mxfp8", scale_format="rowmajor")

    def flat(t, offset):   # t at an element offset in a buffer of its own
        buffer = torch.empty(t.numel() + offset, dtype=t.dtype, device=cuda)
        buffer[offset:] = t.reshape(-1)
        return buffer

    columns = lambda t: t.t().contiguous()
    make, use = {
        "layer_norm columns": (lambda: columns(rows), lambda t: bs.layer_norm(t.t())),
        "layer_norm offset": (lambda: flat(rows, 1), lambda t: bs.layer_norm(t[1:].view(m, n), out_format="mxfp8")),
        "layer_norm parameters": (lambda: flat(weight, 1), lambda t: bs.layer_norm(rows, t[1:], out_format="mxfp8")),
        "layer_norm_backward": (lambda: columns(rows), lambda t: bs.layer_norm_backward(t.t(), rows, None, mean, rstd)),
        "linear residual": (lambda: columns(rows), lambda t: bs.linear_a8w8_mxfp8(q, w, sf, wsf, residual=t.t())),
        "gated_backward grad": (lambda: columns(rows[:, :f]),
                                lambda t: bs.gated_a8w8_mxfp8_backward(t.t(), q, b, sf, bsf)),
        "dequantize": (lambda: columns(q.view(torch.uint8)), lambda t: bs.dequantize(t.t(), sf)),
        "pack_gated": (lambda: columns(gate.view(torch.uint8)), lambda t: bs.pack_gated(t.t(), gate.view(torch.uint8), gate_sf, gate_sf)),
    }[what]
    list_of = lambda r: [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None]
    want = list_of(use(make()))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        use(make())   # loads its kernels and its stream's memory, which would outlast the wait below
    for _ in range(3):
        t = make()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)   # about 10 ms
            got = list_of(use(t))
        shape, dtype, at = t.shape, t.dtype, t.data_ptr()
        del t
        over = torch.full(shape, 7, dtype=dtype, device=cuda)   # the first stream goes on at once
        if not side.query():   # the copy has not run yet
            assert over.data_ptr() != at
        torch.cuda.synchronize()
        assert all(map(same, got, want))
        del over, got
