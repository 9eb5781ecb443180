"""The attention operators together, as a serving loop uses them: prompts, decoded
tokens, requests that come and go; captured into graphs, on several streams at
once, with inputs that are freed early."""
import math

import pytest
import torch

from test_attention_gpu import BF16, check_cache_attention, check_prompt, check_rotary, gen, normal, packed, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(cuda):
    yield
    torch.cuda.synchronize()


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Block:
    """layer norm -> MXFP8 projection -> rotary in place -> cache -> attention -> MXFP8 projection + residual"""

    def __init__(self, bs, g, hq, h, dim, page, pages, requests, columns):
        self.bs, self.hq, self.h, self.dim, self.page, self.hidden = bs, hq, h, dim, page, 256
        weight = lambda n, k: bs.quantize((normal(g, n, k) * k ** -0.5).to(BF16), "mxfp8")
        self.w_in, self.w_in_scale = weight((hq + 2 * h) * dim, self.hidden)
        self.w_out, self.w_out_scale = weight(self.hidden, hq * dim)
        self.plan = bs.rotary_plan(dim, scaling="yarn", factor=4.0)
        self.cache = bs.new_kv_cache(pages, page, h, dim)
        self.table = torch.full((requests, columns), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, device="cuda", generator=g).int()
        self.first_free = i32(0)

    def project(self, x):
        q, sf = self.bs.layer_norm(x, out_format="mxfp8")
        joint = self.bs.linear_a8w8_mxfp8(q, self.w_in, sf, self.w_in_scale)
        return joint.unflatten(1, (-1, self.dim)).split([self.hq, self.h, self.h], 1)

    def __call__(self, x, cached, new, prompts):
        bs = self.bs
        p = bs.paged_slots(cached, new, self.table, self.free, self.page, x.shape[0], first_free=self.first_free)
        self.first_free += p.pages_taken
        q, k, v = self.project(x)
        bs.rotary(q, k, p.positions, self.plan, out=(q, k))
        bs.cache_append(self.cache, k, v, p.slots)
        o = bs.prompt_attention(q, k, v, p.offsets) if prompts else bs.cache_attention(q, self.cache, self.table, p.lengths)
        e, sf = bs.quantize(o.flatten(1), "mxfp8")
        return bs.linear_a8w8_mxfp8(e, self.w_out, sf, self.w_out_scale, residual=x), (p, q, k, v, o)


@pytest.mark.parametrize("hq,h,dim,page", [(8, 2, 64, 16), (4, 4, 128, 32)])
def test_serving(bs, hq, h, dim, page):
    """Three prompts, single tokens for all, one request ends and its place and pages go to another, single tokens again."""
    g = gen(hq + dim)
    lengths = [5, 3 * page, 70]
    block = Block(bs, g, hq, h, dim, page, 40, 3, 12)
    seen = [[], [], []]      # per request: (k, v) as they were appended

    def step(new, prompts):
        cached = i32(*(sum(x.shape[0] for x, _ in s) for s in seen))
        x = normal(g, sum(new), block.hidden).to(BF16)
        y, (p, q, k, v, o) = block(x, cached, i32(*new), prompts)
        assert y.shape == x.shape and y.isfinite().all()
        at = 0
        for r, n in enumerate(new):
            assert p.positions[at:at + n].tolist() == list(range(int(cached[r]), int(cached[r]) + n))
            if n:
                seen[r].append((k[at:at + n].clone(), v[at:at + n].clone()))
            at += n
        assert p.lengths.tolist() == [sum(x.shape[0] for x, _ in s) for s in seen]
        # the cache holds each request's rows, as quantize makes them, on pages that are nobody else's
        owned = []
        for r, s in enumerate(seen):
            if not s:
                continue
            n = int(p.lengths[r])
            pages = block.table[r, :-(-n // page)]
            owned += pages.tolist()
            i = torch.arange(n, device="cuda")
            held = bs.cache_read(block.cache, pages[i // page].long() * page + i % page)
            for got, rows in zip(held, (torch.cat([a for a, _ in s]), torch.cat([b for _, b in s]))):
                e, sf = bs.quantize(rows.flatten(1), "mxfp4", scale_format="rowmajor")
                assert torch.equal(got.flatten(1), bs.dequantize(e, sf, "mxfp4", scale_format="rowmajor"))
        assert len(set(owned)) == len(owned) and min(owned) >= 0
        # the turned rows, and what attention makes of them, by the formulas
        a, b, _ = block.project(x)
        check_rotary(q, a, p.positions, block.plan)
        check_rotary(k, b, p.positions, block.plan)
        if prompts:
            check_prompt(q, k, v, p.offsets, p.offsets, o, None)
        else:
            check_cache_attention(bs, q, block.cache, block.table, p.lengths, out=o)
        # one more projection of the attention's result
        e, sf = bs.quantize(o.flatten(1), "mxfp8")
        assert torch.equal(y, bs.linear_a8w8_mxfp8(e, block.w_out, sf, block.w_out_scale, residual=x))

    step(lengths, True)
    for _ in range(page + 2):
        step([1, 1, 1], False)
    # request 1 ends; its pages go to the end of the free list, its place to a prompt of 20 tokens
    gone = block.table[1][block.table[1] >= 0]
    taken = int(block.first_free)
    block.free, block.first_free = torch.cat((block.free[taken:], gone)), i32(0)
    block.table[1] = -1
    seen[1] = []
    step([0, 20, 0], True)
    for _ in range(2):
        step([1, 1, 1], False)
    assert bs.check_device_error() == 0


def test_prompts_in_pieces(bs):
    """Prompts that go on from a cached beginning, in a padded batch: the cache's rows are read back as the keys."""
    g = gen(37)
    page, h, dim = 16, 2, 64
    cache, plan = bs.new_kv_cache(40, page, h, dim), bs.rotary_plan(dim)
    table = torch.full((3, 12), -1, dtype=torch.int32, device="cuda")
    free, first = torch.randperm(40, device="cuda", generator=g).int(), i32(0)
    cached = i32(0, 0, 0)
    for new in ([50, 0, 33], [7, 64, 1], [0, 70, 40]):
        rows = sum(new) + 9
        q, k, v = (normal(g, rows, n, dim).to(BF16) for n in (4 * h, h, h))
        p = bs.paged_slots(cached, i32(*new), table, free, page, rows, first_free=first)
        first += p.pages_taken
        q, k = bs.rotary(q, k, p.positions, plan)
        bs.cache_append(cache, k, v, p.slots)
        at = torch.cat([table[r, torch.arange(n, device="cuda") // page].long() * page + torch.arange(n, device="cuda") % page
                        for r, n in enumerate(p.lengths.tolist())])
        keys, values = bs.cache_read(cache, at)
        ends = torch.cat((i32(0), p.lengths.cumsum(0).int()))
        out = torch.full_like(q, 3.0)
        bs.prompt_attention(q, keys, values, p.offsets, offsets_k=ends, out=out)
        check_prompt(q, keys, values, p.offsets, ends, out, None)
        assert (p.slots[-9:] == -1).all() and (out[-9:] == 3).all()
        # the last token of each request by the other operator, over the same cache
        last = [int(p.offsets[r + 1]) - 1 for r in range(3)]
        check_cache_attention(bs, q[last], cache, table, p.lengths)
        cached = p.lengths


def test_serving_from_a_graph(bs):
    """A decode step captured once and replayed gives the bits of the calls without it."""
    g = gen(31)
    make = lambda: Block(bs, gen(32), 8, 2, 64, 16, 64, 5, 10)
    a, b = make(), make()
    lengths = [1, 15, 16, 40, 0]
    x = normal(g, sum(lengths), 256).to(BF16)
    cached, new = i32(0, 0, 0, 0, 0), i32(*lengths)
    for block in (a, b):
        block(x, cached, new, True)
    assert torch.equal(a.table, b.table)
    steps = normal(g, 20, 5, 256).to(BF16)
    want, lens = [], i32(*lengths)
    for s in steps:
        want.append(a(s, lens, i32(1, 1, 1, 1, 1), False)[0])
        lens = lens + 1
    static, lens, ones = torch.zeros_like(steps[0]), i32(*lengths), i32(1, 1, 1, 1, 1)
    keep = [t.clone() for t in (b.table, b.first_free, lens, *b.cache)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b(static, lens, ones, False)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = b(static, lens, ones, False)
        lens += 1
    for t, k in zip((b.table, b.first_free, lens, *b.cache), keep):
        t.copy_(k)
    for s, w in zip(steps, want):
        static.copy_(s)
        graph.replay()
        assert torch.equal(y, w)
    assert torch.equal(a.table, b.table) and all(torch.equal(p, q) for p, q in zip(a.cache, b.cache))


def test_prompts_from_a_graph(bs):
    """A captured call takes other offsets than those it was captured with."""
    g = gen(33)
    q, k, v, o, _ = packed(g, [300, 41, 159], 8, 2, 128)
    out = torch.zeros_like(q)
    bs.prompt_attention(q, k, v, o, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bs.prompt_attention(q, k, v, o, out=out)
    for offsets in ([0, 300, 341, 500], [0, 1, 2, 500], [0, 0, 500, 500], [0, 250, 499, 500]):
        o.copy_(i32(*offsets))
        graph.replay()
        assert torch.equal(out, bs.prompt_attention(q, k, v, o))
        check_prompt(q, k, v, o, o, out, None)


def test_two_graphs_and_two_streams_at_once(bs):
    """Calls that run side by side (their workspaces are their own) give what each gives alone."""
    g = gen(34)
    jobs = []
    for i, (lengths, heads) in enumerate((([9000, 100, 3000], 2), ([5000] * 4, 4))):
        cache, table, n = paged(bs, g, lengths, 64, heads, 128)
        q = normal(g, len(lengths), heads * 8, 128).to(BF16)
        a = packed(g, [900, 200], 8, 2, 64 * (i + 1))[:4]
        jobs.append(((q, cache, table, n), a))
    alone = [(bs.cache_attention(*c), bs.prompt_attention(*a)) for c, a in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    results = [[] for _ in jobs]
    for _ in range(10):
        for s, (c, a), r in zip(streams, jobs, results):
            with torch.cuda.stream(s):
                r.append((bs.cache_attention(*c), bs.prompt_attention(*a)))
    torch.cuda.synchronize()
    for r, want in zip(results, alone):
        assert all(torch.equal(x, w) for pair in r for x, w in zip(pair, want))
    graphs, outs = [], []
    for c, a in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((bs.cache_attention(*c), bs.prompt_attention(*a)))
        graphs.append(graph)
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, alone):
        assert all(torch.equal(x, w) for x, w in zip(got, want))


def test_inputs_made_on_another_stream_and_freed(bs):
    """Copies that the calls make of odd tensors, and results, are the current stream's own."""
    g = gen(35)
    q, k, v, o, _ = packed(g, [700, 300], 8, 2, 64)
    want = bs.prompt_attention(q, k, v, o)
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            got = bs.prompt_attention(odd(q), odd(k), odd(v), o)
            torch.full_like(q, math.nan), torch.full_like(k, math.nan)     # take what the call has freed
            assert torch.equal(got, want)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 8, 11, 16, 24])
def test_cache_attention_of_many_requests(bs, dim, group):
    """More (request, head) pairs than the GPU holds CTAs at once: all lengths about a page and a step's tokens."""
    g = gen(dim + group)
    lengths = [(7 * i) % 150 for i in range(330)]
    cache, table, n = paged(bs, g, lengths, 32, 2, dim)
    q = normal(g, 330, 2 * group, dim).to(BF16) * 2
    got = bs.cache_attention(q, cache, table, n)
    some = torch.cat((torch.arange(0, 330, 13), torch.arange(300, 330)))
    check_cache_attention(bs, q[some], cache, table[some], n[some], out=got[some])
    # one request alone has the same answer within the same bound
    for r in (1, 64, 299):
        check_cache_attention(bs, q[r:r + 1], cache, table[r:r + 1], n[r:r + 1])


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_cache_rows_in_runs(bs, dim, page):
    """Runs of slots that begin and end anywhere in a group of four, break within one, go backwards, or skip."""
    g = gen(dim)
    patterns = []
    for begin in range(4):
        for n in (1, 2, 3, 4, 5, 6, 7, 9, 16, 33):
            patterns.append(list(range(begin, begin + n)))
    patterns += [list(range(20, 0, -1)), [0, 1, 2, 7, 8, 9, 10, 3], [4, 5, -1, 7, 8, 9, 10, 11], [-1, 0, 1, 2, 3, -1, -1, 6],
                 list(range(page - 3, page + 5)), [1, 0, 3, 2, 5, 4, 7, 6], [-1] * 5]
    for slots in patterns:
        cache = bs.KvCache(*(torch.randint(100, 120, t.shape, device="cuda", generator=g, dtype=torch.uint8)
                             for t in bs.new_kv_cache(3, page, 3, dim)))
        every = torch.arange(3 * page, device="cuda")
        before = bs.cache_read(cache, every)
        k, v = normal(g, len(slots), 3, dim).to(BF16), normal(g, len(slots), 3, dim).to(BF16)
        at = torch.tensor(slots, device="cuda")
        bs.cache_append(cache, k, v, at)
        for got, x, old, part in zip(bs.cache_read(cache, every), (k, v), before, bs.cache_read(cache, at)):
            want = old.clone()
            e, sf = bs.quantize(x.flatten(1), "mxfp4", scale_format="rowmajor")
            rows = bs.dequantize(e, sf, "mxfp4", scale_format="rowmajor").view(x.shape)
            want[at[at >= 0]] = rows[at >= 0]
            assert torch.equal(got, want), slots
            rows[at < 0] = 0
            assert torch.equal(part, rows), slots


def test_rotary_gradient_by_differences(bs):
    """The inverse is the transpose: <rotary(x) , y> = <x, inverse(y)>, and differences of the first agree."""
    g = gen(36)
    plan = bs.rotary_plan(32, scaling="linear", factor=2.0)
    positions = torch.randint(0, 5000, (40,), device="cuda", generator=g)
    x, y, dx = (normal(g, 40, 3, 48) for _ in range(3))
    turn = lambda t, **kw: bs.rotary(t, None, positions, plan, interleaved=True, **kw)[0].double()
    grad = turn(y, inverse=True)
    # each result off by at most 16 * 2^-24 of a pair's magnitudes (see check_rotary), 5760 products in a sum of fp64;
    # the difference quotient of a linear map has no other error, divided by the step of 1
    size = 16 * 2.0 ** -24 * 2 * float((x.double().abs().amax() + dx.double().abs().amax()) * y.double().abs().sum())
    assert abs(float((turn(x) * y).sum() - (x * grad).sum())) <= 2 * size
    quotient = ((turn(x + dx) - turn(x)) * y).sum()
    # (x + dx is rounded: half a step of it, through a turn that keeps sizes)
    assert abs(float(quotient - (dx * grad).sum())) <= 4 * size + 2.0 ** -23 * float(
        (x + dx).double().abs().amax() * y.double().abs().sum())


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_cache_rows_that_are_not_finite(bs, dtype):
    """Infinities, NaN, zeros, the smallest and the largest numbers: bit for bit what quantize makes of them."""
    g = gen(38)
    info = torch.finfo(dtype)
    odd = [math.inf, -math.inf, math.nan, 0.0, -0.0, info.tiny, info.smallest_normal / 4, info.max, -info.max, 6.0, 5.0, 0.25]
    x = normal(g, 4 * len(odd), 1, 128).to(dtype)
    for i, value in enumerate(odd):
        x[4 * i, 0, 7] = value
        x[4 * i + 1, 0, 32:64] = value
        x[4 * i + 2, 0, 64::2] = value
        x[4 * i + 3] *= 1e-30
        x[4 * i + 3, 0, 100] = value
    slots = torch.arange(x.shape[0], device="cuda")
    cache = bs.new_kv_cache(4, 16, 1, 128)
    bs.cache_append(cache, x, x.flip(0), slots)
    e, sf = bs.quantize(x.flatten(1), "mxfp4", scale_format="rowmajor")
    want = bs.dequantize(e, sf, "mxfp4", scale_format="rowmajor")
    k, v = bs.cache_read(cache, slots)
    assert torch.equal(k.flatten(1).view(torch.int16), want.view(torch.int16))
    assert torch.equal(v.flatten(1).flip(0).view(torch.int16), want.view(torch.int16))


def test_calls_at_the_edges(bs):
    """Caches without pages, tables without columns, far more sequences than tokens, one side of a rotary in place."""
    g = gen(39)
    empty = bs.new_kv_cache(0, 16, 2, 64)
    k = normal(g, 3, 2, 64).to(BF16)
    slots = torch.tensor([0, -1, 5], device="cuda")
    q = normal(g, 2, 4, 64).to(BF16)
    bs.cache_append(empty, k, k, slots)
    assert not any(t.any() for t in bs.cache_read(empty, slots))
    assert not bs.cache_attention(q, empty, i32(0, 3, -1, 1 << 30).view(2, 2), i32(20, 5)).any()
    cache = bs.new_kv_cache(2, 16, 2, 64)
    assert not bs.cache_attention(q, cache, i32(0, 1)[:0].view(2, 0), i32(20, 5)).any()
    assert bs.cache_attention(q[:0], cache, i32()[:0].view(0, 3), i32()).shape == (0, 4, 64)
    bs.cache_append(cache, k[:0], k[:0], slots[:0])
    assert bs.cache_read(cache, slots[:0])[0].shape == (0, 2, 64)
    # 4000 sequences for 11 tokens
    ends = torch.zeros(4001, dtype=torch.int32, device="cuda")
    ends[7:] += 4
    ends[1000:] += 1
    ends[3999:] += 6
    q, k, v, _, _ = packed(g, [11], 6, 3, 64)
    out, lse = bs.prompt_attention(q, k, v, ends, return_lse=True)
    short = i32(0, 4, 5, 11)
    check_prompt(q, k, v, short, short, out, lse)
    # each token a sequence
    ones = torch.arange(12, dtype=torch.int32, device="cuda")
    assert torch.equal(bs.prompt_attention(q, k, v, ones).view(11, 3, 2, 64), v[:, :, None].expand(11, 3, 2, 64))
    plan = bs.rotary_plan(64)
    want = bs.rotary(q, None, ones[:11], plan)[0]
    x = q.clone()
    got = bs.rotary(x, None, ones[:11], plan, out=(x, None))
    assert torch.equal(x, want) and got[1] is None
