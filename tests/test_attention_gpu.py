"""The attention operators on a GPU against their formulas in 64 bits.

Tolerances are sums of the roundings that the formulas leave: half a step of
the type (bf16 2^-8, fp32 2^-24, relative) for each rounded value, and the
fp32 accumulations' worst cases.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, FP32: 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _device(cuda):
    yield
    torch.cuda.synchronize()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


# ---- rotary -------------------------------------------------------------------------

def rotary_formula(x, positions, frequencies, factor, interleaved, inverse):
    """fp64 results, and the sum of magnitudes that each is made of."""
    rot = 2 * len(frequencies)
    t = positions.double()[:, None, None] * frequencies * (-1 if inverse else 1)
    c, s = t.cos() * factor, t.sin() * factor
    y, mag = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    u, v = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    mag[..., a] = mag[..., b] = (u.abs() + v.abs()) * abs(factor)
    return y, mag


def check_rotary(got, x, positions, plan, **kw):
    want, mag = rotary_formula(x, positions, plan.frequencies, plan.factor, kw.get("interleaved", False), kw.get("inverse", False))
    # the fraction of a turn to fp32 (pi 2^-25 rad), cosine and sine to two steps of 1 (2 * 2^-24), their
    # factor, two products and a sum (half a step each): below 8 * 2^-24 of |a| + |b|; then the result's own
    tol = 8 * 2.0 ** -24 * mag + HALF[x.dtype] * (want.abs() + 8 * 2.0 ** -24 * mag)
    assert ((got.double() - want).abs() <= tol).all()
    rot = 2 * len(plan.frequencies)
    assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot", [(1, 32, 8, 128, 128), (7, 1, 1, 64, 64), (130, 9, 3, 96, 32), (5, 4, 2, 80, 80),
                                                  (3, 2, 1, 18, 6), (2, 70, 3, 256, 256), (4, 3, 1, 512, 512), (33, 5, 5, 2, 2),
                                                  (3, 2, 2, 130, 66)])
def test_rotary(bs, dtype, interleaved, tokens, hq, hk, dim, rot):
    g = gen(tokens + dim)
    q, k = normal(g, tokens, hq, dim).to(dtype), normal(g, tokens, hk, dim).to(dtype)
    plan = bs.rotary_plan(rot, scaling="yarn", factor=8.0) if rot > 2 else bs.rotary_plan(rot)
    pos = torch.randint(0, 1 << 20, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    for inverse in (False, True):
        oq, ok = bs.rotary(q, k, pos, plan, interleaved=interleaved, inverse=inverse)
        check_rotary(oq, q, pos, plan, interleaved=interleaved, inverse=inverse)
        check_rotary(ok, k, pos, plan, interleaved=interleaved, inverse=inverse)
    if tokens > 1:   # the same through int64, a strided position list
        wide = torch.stack((pos, pos), 1).long()[:, 1]
        again = bs.rotary(q, k, wide, plan, interleaved=interleaved, inverse=True)
        assert torch.equal(again[0], oq) and torch.equal(again[1], ok)


def test_rotary_positions(bs):
    """Negative ones, zero, and beyond 32 bits."""
    q = normal(gen(1), 6, 2, 64)
    plan = bs.rotary_plan(64)
    pos = torch.tensor([0, -1, -70000, 1, 1 << 31, (1 << 33) + 5], device="cuda")
    oq, ok = bs.rotary(q, None, pos, plan)
    assert ok is None and torch.equal(oq[0], q[0])
    # fp64 angles of 2^33 turns end near 2^-20 rad: the formula's and the kernel's differ by that much
    check_rotary(oq[:4], q[:4], pos[:4], plan)
    want, mag = rotary_formula(q, pos, plan.frequencies, 1.0, False, False)
    assert ((oq.double() - want).abs() <= mag * (2.0 ** 34 * 2.0 ** -52 * 4 + 2.0 ** -20)).all()


def test_rotary_in_place_on_a_joint_projection(bs):
    g = gen(3)
    for dtype in (BF16, FP32):
        x = normal(g, 37, 12 * 64).to(dtype)
        q, k, v = (x[:, a * 64:b * 64].unflatten(1, (-1, 64)) for a, b in ((0, 8), (8, 10), (10, 12)))
        before = x.clone()
        pos, plan = torch.arange(37, device="cuda", dtype=torch.int32), bs.rotary_plan(64)
        want = bs.rotary(q, k, pos, plan)
        got = bs.rotary(q, k, pos, plan, out=(q, k))
        assert got[0].data_ptr() == q.data_ptr()
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        assert torch.equal(x[:, 640:], before[:, 640:])
        with pytest.raises(bs.BsgemmError):
            bs.rotary(q, q, pos, plan, out=(q, q))


def test_rotary_strides(bs):
    """Odd offsets, transposed heads, expanded keys, an output with gaps."""
    g = gen(4)
    plan = bs.rotary_plan(32)
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 11
    q = normal(g, 9 * 4 * 64 + 1)[1:].view(9, 4, 64)
    check_rotary(bs.rotary(q, None, pos, plan)[0], q, pos, plan)
    q = normal(g, 4, 9, 64).to(BF16).transpose(0, 1)
    check_rotary(bs.rotary(q, None, pos, plan)[0], q, pos, plan)
    q = normal(g, 9, 64, 4).to(BF16).transpose(1, 2)
    check_rotary(bs.rotary(q, None, pos, plan)[0], q, pos, plan)
    k = normal(g, 9, 1, 64).expand(9, 3, 64)
    out = torch.full((9, 3, 80), 7.0, device="cuda")
    check_rotary(bs.rotary(k, None, pos, plan, out=(out[..., :64], None))[0], k, pos, plan)
    assert (out[..., 64:] == 7).all()


def test_rotary_gradient(bs):
    """The inverse rotation of dL/dy is dL/dx, as differences of the rotation have it."""
    g = gen(5)
    plan = bs.rotary_plan(64, scaling="yarn", factor=4.0)
    pos = torch.tensor([3, 900, 70001], device="cuda", dtype=torch.int32)
    x, dy, dx = normal(g, 3, 2, 64), normal(g, 3, 2, 64), normal(g, 3, 2, 64)
    grad = bs.rotary(dy, None, pos, plan, inverse=True)[0]
    # linear: any step will do; sums of 384 products of results that are off by 8 * 2^-24 (|a| + |b|) factor, both sides
    step = bs.rotary(x + dx, None, pos, plan)[0].double() - bs.rotary(x, None, pos, plan)[0].double()
    left, right = (step * dy).sum(), (grad.double() * dx).sum()
    mag = 2 * plan.factor * ((x.abs() + dx.abs()).sum(-1) * dy.abs().amax(-1)).sum() * 2
    assert abs(left - right) <= 16 * 2.0 ** -24 * mag


def test_rotary_empty(bs):
    plan = bs.rotary_plan(64)
    q = torch.empty(0, 4, 64, device="cuda", dtype=BF16)
    assert bs.rotary(q, None, torch.empty(0, device="cuda", dtype=torch.int32), plan)[0].shape == (0, 4, 64)


# ---- slots --------------------------------------------------------------------------

def slots_formula(cached, new, table, free, page, tokens, first=0):
    slots, positions, offsets, taken = [], [], [0], 0
    table = [row[:] for row in table]
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        for t in range(c, c + n):
            col = t // page
            if t % page == 0:
                f = first + taken
                taken += 1
                if col < len(table[r]):
                    table[r][col] = free[f] if f < len(free) else -1
            p = table[r][col] if col < len(table[r]) else -1
            slots.append(p * page + t % page if p >= 0 else -1)
            positions.append(t)
        offsets.append(offsets[-1] + n)
    slots, positions = slots[:tokens], positions[:tokens]
    pad = tokens - len(slots)
    return slots + [-1] * pad, positions + [0] * pad, offsets, [max(c, 0) + max(n, 0) for c, n in zip(cached, new)], [taken], table


def check_slots(bs, cached, new, page, columns, spare=0, extra_free=8, first=None, free_count=None):
    rng = torch.Generator().manual_seed(sum(new) + page)
    owned = [-(-max(c, 0) // page) for c in cached]
    ids = torch.randperm(sum(owned) + sum(max(n, 0) for n in new) + 40, generator=rng).int().tolist()
    table = [[-1] * columns for _ in cached]
    for row, n in zip(table, owned):
        row[:n] = [ids.pop() for _ in range(min(n, columns))]
    free = ids if free_count is None else ids[:free_count]
    tokens = sum(max(n, 0) for n in new) + spare
    want = slots_formula(cached, new, table, free, page, tokens, first or 0)
    t = torch.tensor(table, dtype=torch.int32, device="cuda").reshape(len(cached), columns)
    i32 = dict(dtype=torch.int32, device="cuda")
    start = None if first is None else torch.tensor([first], **i32)
    got = bs.paged_slots(torch.tensor(cached, **i32), torch.tensor(new, **i32), t, torch.tensor(free, **i32), page, tokens,
                         first_free=start)
    for a, b in zip((*got, t), want):
        assert a.tolist() == b


@pytest.mark.parametrize("page", [1, 16, 64, 100])
def test_paged_slots(bs, page):
    cols = 600 // page + 3
    check_slots(bs, [0], [1], page, cols)
    check_slots(bs, [0, 5, 64, 63, 200, 16], [3, 0, 1, 1, 300, 0], page, cols, spare=5)
    check_slots(bs, [0, 0, 17], [0, 0, 0], page, cols, spare=3)
    check_slots(bs, [-4, 30, 0], [7, -2, 2], page, cols)                     # negative counts are none
    check_slots(bs, [10, 20], [40, 50], page, cols, first=7)
    check_slots(bs, [10, 20, 3], [90, 50, 400], page, cols, free_count=2)    # the list ends
    check_slots(bs, [0, 150], [500, 3], page, 2 if page > 1 else 100)        # the table's row ends


def test_paged_slots_many(bs):
    """Requests over several rounds of a CTA's scan, tokens over many CTAs, and a request longer than one."""
    rng = torch.Generator().manual_seed(9)
    cached = torch.randint(0, 300, (2500,), generator=rng).tolist()
    new = torch.randint(0, 4, (2500,), generator=rng).tolist()
    new[1200] = 5000
    check_slots(bs, cached, new, 16, 360, spare=1100)
    check_slots(bs, [3] * 257, [1] * 257, 16, 2)
    check_slots(bs, [0] * 1024, [1] * 1024, 16, 2)


def test_paged_slots_without_requests(bs):
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    p = bs.paged_slots(i, i, torch.empty(0, 4, dtype=torch.int32, device="cuda"), i, 16, 3)
    assert p.slots.tolist() == [-1] * 3 and p.offsets.tolist() == [0] and p.pages_taken.tolist() == [0]
    p = bs.paged_slots(i, i, torch.empty(0, 4, dtype=torch.int32, device="cuda"), i, 16, 0)
    assert p.slots.numel() == 0 and p.offsets.tolist() == [0]


def test_paged_slots_far(bs):
    """Slots past 2^31, lengths that would pass it, tokens that are cut."""
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.full((1, 2), -1, **i32)
    p = bs.paged_slots(torch.tensor([0], **i32), torch.tensor([3], **i32), table, torch.tensor([2 ** 31 - 2], **i32), 256, 3)
    assert p.slots.tolist() == [(2 ** 31 - 2) * 256 + j for j in range(3)]
    top = 2 ** 31 - 1
    p = bs.paged_slots(torch.tensor([top - 1, 0], **i32), torch.tensor([5, 1], **i32), torch.full((2, 1), -1, **i32),
                       torch.tensor([3], **i32), 16, 4)
    assert p.lengths.tolist() == [top, 1] and p.positions.tolist() == [top - 1, 0, 0, 0]
    p = bs.paged_slots(torch.tensor([0, 0], **i32), torch.tensor([5, 5], **i32), torch.full((2, 1), -1, **i32),
                       torch.tensor([3, 4], **i32), 16, 7)
    assert p.slots.tolist() == [48, 49, 50, 51, 52, 64, 65] and p.offsets.tolist() == [0, 5, 10]


# ---- the cache ----------------------------------------------------------------------

def filled_cache(bs, g, pages, page, heads, dim, std=1.0):
    cache = bs.new_kv_cache(pages, page, heads, dim)
    k, v = normal(g, pages * page, heads, dim) * std, normal(g, pages * page, heads, dim) * std
    bs.cache_append(cache, k, v, torch.arange(pages * page, device="cuda"))
    return cache


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 64, 16), (17, 3, 128, 16), (300, 8, 128, 64), (129, 2, 64, 256), (50, 5, 128, 32)])
def test_cache_holds_what_quantize_makes(bs, dtype, tokens, heads, dim, page):
    """Bit for bit quantize's elements and scales, at slots in any order; other slots stay as they were."""
    g = gen(tokens)
    pages = tokens // page + 3
    cache = bs.KvCache(*(torch.randint(0, 120, t.shape, device="cuda", generator=g, dtype=torch.uint8) for t in bs.new_kv_cache(pages, page, heads, dim)))
    every = torch.arange(pages * page, device="cuda")
    before = bs.cache_read(cache, every)
    k = (normal(g, tokens, heads, dim) * torch.exp2(torch.randint(-20, 20, (tokens, heads, 1), device="cuda", generator=g).float())).to(dtype)
    v = normal(g, tokens, heads, dim).to(dtype)
    k[0, 0, :32] = 0
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens]
    given = slots.clone()
    if tokens > 4:
        given[1], given[2] = -1, pages * page
    bs.cache_append(cache, k, v, given)
    kept = (given >= 0) & (given < pages * page)
    for got, x, old in zip(bs.cache_read(cache, every), (k, v), before):
        want = old.clone()
        q, sf = bs.quantize(x.reshape(tokens, heads * dim), "mxfp4", scale_format="rowmajor")
        want[slots[kept]] = bs.dequantize(q, sf, "mxfp4", scale_format="rowmajor").view(tokens, heads, dim)[kept]
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    absent = bs.cache_read(cache, torch.tensor([-1, pages * page, 1 << 40], device="cuda"))
    assert not absent[0].any() and not absent[1].any()


def test_cache_layout(bs):
    """The bytes lie as the header says."""
    g = gen(2)
    for dim in (64, 128):
        cache = bs.new_kv_cache(2, 16, 3, dim)
        k, v = normal(g, 5, 3, dim), normal(g, 5, 3, dim)
        slots = torch.tensor([0, 17, 30, 31, 6], device="cuda")
        bs.cache_append(cache, k, v, slots)
        rk, rv = bs.cache_read(cache, slots)
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
        for i, s in enumerate(slots.tolist()):
            p, r = divmod(s, 16)
            for e in range(dim):
                byte = e % 32 // 8 * (dim // 8) + e // 32 * 4 + e % 8 // 2
                code = (cache.k[p, :, r, byte] >> (e % 2 * 4)) & 15
                scale = torch.exp2(cache.k_scale[p, :, r, e // 32].float() - 127)
                assert torch.equal(table[code.long()] * scale, rk[i, :, e].float())
                code = (cache.v[p, :, r // 4, e // 2, r % 4] >> (e % 2 * 4)) & 15
                scale = torch.exp2(cache.v_scale[p, :, r // 4, e // 32, r % 4].float() - 127)
                assert torch.equal(table[code.long()] * scale, rv[i, :, e].float())


def test_cache_append_strides(bs):
    g = gen(6)
    x = normal(g, 20, 6 * 64).to(BF16)
    k, v = x[:, :128].unflatten(1, (2, 64)), x[:, 128:256].unflatten(1, (2, 64))
    slots = torch.arange(40, device="cuda")[::2]
    want = bs.new_kv_cache(3, 16, 2, 64)
    bs.cache_append(want, k.contiguous(), v.contiguous(), slots.contiguous())
    odd = torch.zeros(20 * 128 + 1, device="cuda", dtype=BF16)[1:].view(20, 2, 64)
    odd.copy_(k)
    for kk, vv in ((k, v), (odd, v.transpose(0, 1).contiguous().transpose(0, 1)),
                   (k.transpose(1, 2).contiguous().transpose(1, 2), v)):
        got = bs.new_kv_cache(3, 16, 2, 64)
        bs.cache_append(got, kk, vv, slots)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- attention ----------------------------------------------------------------------

def attention_formula(q, k, v, scale, hidden=None, half=2.0 ** -8, lost=2.0 ** -126):
    """fp64 softmax(scale q k^T) v of [rows, d], [keys, d]: out, lse, and the tolerance of out and of lse.
    Weights are rounded by `half` of theirs and by `lost` of the largest: bf16's 2^-8, and what fp32 cannot hold."""
    q, k, v = q.double(), k.double(), v.double()
    s = scale * q @ k.T
    if hidden is not None:
        s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(torch.isinf(lse)[:, None], torch.zeros_like(s), torch.exp(s - lse[:, None]))
    out, mag = p @ v, p @ v.abs()
    # a score: fp32 sums of dim products (2^-23 each, a truncating adder among what is allowed), its product with the
    # scale, the exponential of a difference (a step of the larger of the two) and its own two steps
    seen = torch.where(torch.isinf(s), torch.zeros_like(s), s).abs()
    e = ((q.shape[1] + 4) * 2.0 ** -23 * scale * (q.abs() @ k.abs().T).amax(-1) + 2 * 2.0 ** -22 * seen.amax(-1) + 2.0 ** -21)[:, None] \
        if k.shape[0] else torch.zeros(q.shape[0], 1, dtype=torch.float64, device=q.device)
    # weights rounded, their error above and below the line: |o' - o| <= d, d = mag (h + 4 e); then o' (not o) to bf16,
    # off by up to h |o'| <= h (|o| + d): with one weight near 1 all three meet, and h d is 2^-16 of the value
    d = mag * (half + 4 * e) + lost * v.abs().sum(0)
    return out, lse, d + HALF[BF16] * (out.abs() + d) + 2.0 ** -126, 2 * e[:, 0] + 2.0 ** -22 * lse.abs()


def cached_rows(bs, cache, table, r, length):
    page = cache.k.shape[2]
    at = table[r, torch.arange(length, device="cuda") // page].long() * page + torch.arange(length, device="cuda") % page
    return bs.cache_read(cache, at)


# Weights are fp16: half a step is 2^-11 of one, or 2^-25 (subnormals); the largest is 2^7 to 2^15.  Beside
# scales that fp16 does not hold they are bf16, half a step 2^-8.
def check_cache_attention(bs, q, cache, table, lengths, out=None, scale=None, half=2.0 ** -11, **kw):
    got = bs.cache_attention(q, cache, table, lengths, scale=scale, **kw) if out is None else out
    heads = cache.k.shape[1]
    group = q.shape[1] // heads
    for r, n in enumerate(lengths.tolist()):
        k, v = cached_rows(bs, cache, table, r, n)
        for h in range(heads):
            rows = slice(h * group, (h + 1) * group)
            want, _, tol, _ = attention_formula(q[r, rows], k[:, h], v[:, h], q.shape[2] ** -0.5 if scale is None else scale,
                                                half=half, lost=2.0 ** -32)
            bad = (got[r, rows].double() - want).abs() > tol
            assert not bad.any(), (r, h, n, int(bad.sum()))
    return got


def paged(bs, g, lengths, page, heads, dim, std=1.0):
    owned = [-(-n // page) for n in lengths]
    pages = sum(owned) + 2
    cache = filled_cache(bs, g, pages, page, heads, dim, std)
    table = torch.full((len(lengths), max(owned) + 1), -1, dtype=torch.int32, device="cuda")
    ids = torch.randperm(pages, device="cuda", generator=g).int()
    for r, n in enumerate(owned):
        table[r, :n], ids = ids[:n], ids[n:]
    return cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (8, 4), (2, 7), (3, 8), (1, 9), (2, 16), (1, 17), (1, 40)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_cache_attention(bs, dim, heads, group, page):
    g = gen(dim + heads + group + page)
    cache, table, lengths = paged(bs, g, [1, 15, 16, 17, 64, 65, 0, 333, 128], page, heads, dim)
    check_cache_attention(bs, normal(g, 9, heads * group, dim).to(BF16) * 2, cache, table, lengths)


@pytest.mark.parametrize("lengths", [[20000], [1, 9000, 64], [2500] * 30, [0, 0], [3] * 400])
def test_cache_attention_split(bs, lengths):
    """One request over all CTAs, requests cut by them, none, many short ones."""
    g = gen(len(lengths))
    cache, table, n = paged(bs, g, lengths, 32, 2, 128)
    q = normal(g, len(lengths), 8, 128).to(BF16)
    got = check_cache_attention(bs, q, cache, table, n)
    assert torch.equal(got, bs.cache_attention(q, cache, table, n))     # the same bits again


def test_cache_attention_scores_of_all_sizes(bs):
    """Scores that grow along the axis (the running maximum moves), sharp ones, a scale of the caller's."""
    g = gen(11)
    n = 700
    cache = bs.new_kv_cache(n // 16 + 1, 16, 1, 128)
    k = normal(g, n, 1, 128) * (torch.arange(n, device="cuda") / 40 + 0.01)[:, None, None]
    bs.cache_append(cache, k, normal(g, n, 1, 128), torch.arange(n, device="cuda"))
    table = torch.arange(n // 16 + 1, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = normal(g, 1, 8, 128).to(BF16)
    for scale in (None, 1.0, 1e-4, 5.0):
        check_cache_attention(bs, q, cache, table, lengths, scale=scale)


@pytest.mark.parametrize("exponent", [-60, -20, 30, 62, 70, 100])
def test_cache_attention_scales_far_from_one(bs, exponent):
    """Values (and keys) of any size, those whose scales pass 2^65 among ordinary ones."""
    g = gen(12)
    cache = bs.new_kv_cache(8, 16, 2, 64)
    k, v = normal(g, 128, 2, 64), normal(g, 128, 2, 64)
    v[::3] *= 2.0 ** exponent
    k[5] *= 2.0 ** min(exponent, 60)
    bs.cache_append(cache, k, v, torch.arange(128, device="cuda"))
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    q = normal(g, 1, 8, 64).to(BF16) * 2.0 ** -abs(min(exponent, 60))
    check_cache_attention(bs, q, cache, table, torch.tensor([128], dtype=torch.int32, device="cuda"), half=2.0 ** -8)


def test_cache_attention_what_lies_behind_a_length(bs):
    """Rows and pages past a request's length do not reach it, NaN scales and bad pages among them."""
    g = gen(13)
    cache, table, lengths = paged(bs, g, [37, 5, 90], 16, 2, 128)
    q = normal(g, 3, 8, 128).to(BF16)
    want = check_cache_attention(bs, q, cache, table, lengths)
    for r, n in enumerate([37, 5, 90]):
        row = n % 16
        page = int(table[r, n // 16])
        if row:
            cache.k_scale[page, :, row:], cache.k[page, :, row:] = 255, 0x77
            for t in range(row, 16):
                cache.v_scale[page, :, t // 4, :, t % 4], cache.v[page, :, t // 4, :, t % 4] = 255, 0xFF
        table[r, -(-n // 16):] = 1 << 30
    assert torch.equal(bs.cache_attention(q, cache, table, lengths), want)
    # a NaN scale inside the length is the request's own
    cache.v_scale[int(table[1, 0]), 0, 0, 0, 2] = 255
    got = bs.cache_attention(q, cache, table, lengths)
    assert got[1, :4, :32].isnan().all() and torch.equal(got[1, 4:], want[1, 4:]) and torch.equal(got[0], want[0])
    # pages that are none: their tokens are absent; a length past the table ends there
    table[2, 1], table[0, 0] = -1, 1 << 20
    got = bs.cache_attention(q, cache, table, torch.tensor([37, 0, 90], dtype=torch.int32, device="cuda"))
    k, v = (torch.cat((x[:16], x[32:])) for x in cached_rows(bs, cache, table.clamp(0, 11), 2, 90))
    out, _, tol, _ = attention_formula(q[2, :4], k[:, 0], v[:, 0], 128 ** -0.5)
    assert ((got[2, :4].double() - out).abs() <= tol).all() and not got[1].any()
    full = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    a = bs.cache_attention(q[:1], cache, full, torch.tensor([48], dtype=torch.int32, device="cuda"))
    b = bs.cache_attention(q[:1], cache, full, torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_cache_attention_strides_and_out(bs):
    g = gen(14)
    cache, table, lengths = paged(bs, g, [40, 77], 16, 2, 64)
    q = normal(g, 2, 8, 64).to(BF16)
    want = bs.cache_attention(q, cache, table, lengths)
    joint = torch.cat((normal(g, 2, 3, 64).to(BF16), q), 1)[:, 3:]
    odd = torch.zeros(2 * 512 + 1, device="cuda", dtype=BF16)[1:].view(2, 8, 64)
    odd.copy_(q)
    wide = torch.stack((table, table), 2).flatten(1)[:, :2 * table.shape[1]].contiguous()
    wide[:, :table.shape[1]] = table
    for x in (joint, odd, q.transpose(1, 2).contiguous().transpose(1, 2), q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(bs.cache_attention(x, cache, wide[:, :table.shape[1]], lengths), want)
    out = torch.full((2, 8, 72), 3.0, device="cuda", dtype=BF16)
    ws = torch.empty(1 << 26, device="cuda", dtype=torch.uint8)
    assert torch.equal(bs.cache_attention(q, cache, table, lengths, out=out[..., 1:65], workspace=ws), want)
    assert (out[..., 0] == 3).all() and (out[..., 65:] == 3).all()
    with pytest.raises(ValueError):
        bs.cache_attention(q, cache, table, lengths, workspace=ws[:100])
    with pytest.raises(bs.BsgemmError):
        bs.cache_attention(q, cache, table, lengths, out=q)
    for call in (lambda: bs.cache_attention(q[:, :7], cache, table, lengths), lambda: bs.cache_attention(q.float(), cache, table, lengths),
                 lambda: bs.cache_attention(q, cache, table.long(), lengths), lambda: bs.cache_attention(q, cache, table, lengths[:1]),
                 lambda: bs.cache_attention(q, cache, table[:1], lengths), lambda: bs.cache_attention(q[..., :32], cache, table, lengths)):
        with pytest.raises(ValueError):
            call()


def test_cache_attention_offsets_past_2_31(bs):
    """A cache whose parts pass 2^31 bytes, with the request's pages at its end."""
    g = gen(15)
    pages = (1 << 31) // (8 * 64 * 64) + 40
    cache = bs.new_kv_cache(pages, 64, 8, 128)
    assert cache.k.numel() > 1 << 31
    slots = torch.arange(200, device="cuda") + (pages - 4) * 64
    bs.cache_append(cache, normal(g, 200, 8, 128), normal(g, 200, 8, 128), slots)
    table = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")[None]
    check_cache_attention(bs, normal(g, 1, 8, 128).to(BF16), cache, table, torch.tensor([200], dtype=torch.int32, device="cuda"))


def packed(g, lengths, hq, h, dim, lengths_k=None):
    lengths_k = lengths if lengths_k is None else lengths_k
    q = normal(g, sum(lengths), hq, dim).to(BF16) * 1.5
    k, v = normal(g, sum(lengths_k), h, dim).to(BF16), normal(g, sum(lengths_k), h, dim).to(BF16)
    offsets = [torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32, device="cuda") for x in (lengths, lengths_k)]
    return q, k, v, *offsets


def check_prompt(q, k, v, offsets, offsets_k, out, lse, causal=True, scale=None):
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5 if scale is None else scale
    a, b = offsets.tolist(), offsets_k.tolist()
    for i in range(len(a) - 1):
        nq, nk = a[i + 1] - a[i], b[i + 1] - b[i]
        hidden = None
        if causal:
            hidden = torch.arange(nk, device="cuda")[None] > torch.arange(nq, device="cuda")[:, None] + nk - nq
        for h in range(q.shape[1]):
            want, wl, tol, ltol = attention_formula(q[a[i]:a[i + 1], h], k[b[i]:b[i + 1], h // group], v[b[i]:b[i + 1], h // group],
                                                    scale, hidden)
            bad = ~((out[a[i]:a[i + 1], h].double() - want).abs() <= tol)
            assert not bad.any(), (i, nq, nk, h, int(bad.sum()), bad.nonzero()[:3].tolist())
            if lse is not None:
                got = lse[a[i]:a[i + 1], h].double()
                assert (torch.isinf(wl) == (got == -math.inf)).all()
                assert ((got - wl).abs() <= ltol)[~torch.isinf(wl)].all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 4), (1, 7), (2, 8), (1, 128), (1, 100), (3, 2)])
def test_prompt_attention(bs, dim, heads, group):
    g = gen(dim + heads + group)
    lengths = [1, 0, 17, 128, 129, 300] if group < 50 else [1, 0, 5, 130]
    q, k, v, o, _ = packed(g, lengths, heads * group, heads, dim)
    out, lse = bs.prompt_attention(q, k, v, o, return_lse=True)
    check_prompt(q, k, v, o, o, out, lse)
    assert torch.equal(out, bs.prompt_attention(q, k, v, o))
    out = bs.prompt_attention(q, k, v, o, causal=False, scale=0.3)
    check_prompt(q, k, v, o, o, out, None, causal=False, scale=0.3)


@pytest.mark.parametrize("dim", [8, 16, 40, 72, 80, 96, 120])
def test_prompt_attention_head_sizes(bs, dim):
    q, k, v, o, _ = packed(gen(dim), [200, 77], 6, 2, dim)
    out, lse = bs.prompt_attention(q, k, v, o, return_lse=True)
    check_prompt(q, k, v, o, o, out, lse)


@pytest.mark.parametrize("heads,group,lengths", [(1, 1, [1500]), (2, 3, [700, 900]), (1, 8, [2100]), (4, 1, [33] * 60), (1, 2, list(range(0, 90, 3))),
                                                 (2, 1, [256, 255, 257, 512])])
def test_prompt_attention_longer(bs, heads, group, lengths):
    """Many key blocks, many items a CTA, sequence ends at and around block borders."""
    q, k, v, o, _ = packed(gen(sum(lengths)), lengths, heads * group, heads, 128)
    out, lse = bs.prompt_attention(q, k, v, o, return_lse=True)
    check_prompt(q, k, v, o, o, out, lse)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attention_other_key_lengths(bs, causal):
    """More keys than queries (a prompt goes on from a cached beginning), fewer (rows that see none), no keys at all."""
    nq, nk = [40, 300, 5, 200, 7, 130, 0, 1], [340, 100, 0, 200, 1, 129, 9, 1000]
    q, k, v, oq, ok = packed(gen(21), nq, 8, 2, 64, nk)
    out, lse = bs.prompt_attention(q, k, v, oq, offsets_k=ok, causal=causal, return_lse=True)
    check_prompt(q, k, v, oq, ok, out, lse, causal=causal)
    none = torch.zeros_like(oq)
    out, lse = bs.prompt_attention(q, k[:0], v[:0], oq, offsets_k=none, causal=causal, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


def test_prompt_attention_scores_of_all_sizes(bs):
    """The running maximum moves often, and by much."""
    g = gen(22)
    q, k, v, o, _ = packed(g, [900], 4, 1, 128)
    k = (k.float() * (torch.arange(900, device="cuda") / 60 + 0.01)[:, None, None]).to(BF16)
    for scale in (None, 1.0, 1e-5):
        out, lse = bs.prompt_attention(q, k, v, o, scale=scale, return_lse=True)
        check_prompt(q, k, v, o, o, out, lse, scale=scale)


def test_prompt_attention_what_lies_outside(bs):
    """Rows of other sequences and rows of none do not reach a sequence, infinities and NaN among them; output rows of none stay."""
    g = gen(23)
    for dim in (64, 128):
        q, k, v, o, _ = packed(g, [50, 131, 20], 4, 2, dim)
        want = bs.prompt_attention(q, k, v, o)
        for bad in (math.nan, math.inf):
            pad = lambda x: torch.cat((torch.full_like(x[:9], bad), x, torch.full_like(x[:140], bad)))
            out = torch.full((q.shape[0] + 149, 4, dim), 5.0, device="cuda", dtype=BF16)
            bs.prompt_attention(pad(q), pad(k), pad(v), o + 9, out=out)
            assert torch.equal(out[9:-140], want) and (out[:9] == 5).all() and (out[-140:] == 5).all()
            # the sequences apart from each other: the middle one is spoilt
            k2, v2 = k.clone(), v.clone()
            k2[50:181], v2[50:181] = bad, bad
            got = bs.prompt_attention(q, k2, v2, o)
            assert torch.equal(got[:50], want[:50]) and torch.equal(got[181:], want[181:]) and got[50:181].isnan().all()
            # a key that is not finite does not reach the rows before it
            k2 = k.clone()
            k2[100] = bad
            got = bs.prompt_attention(q, k2, v, o)
            assert torch.equal(got[:100], want[:100]) and torch.equal(got[181:], want[181:])


def test_prompt_attention_strides_and_out(bs):
    g = gen(24)
    x = normal(g, 150, 12 * 64).to(BF16)
    q, k, v = (x[:, a * 64:b * 64].unflatten(1, (-1, 64)) for a, b in ((0, 8), (8, 10), (10, 12)))
    o = torch.tensor([0, 100, 150], dtype=torch.int32, device="cuda")
    want = bs.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), o)
    odd = torch.zeros(150 * 512 + 1, device="cuda", dtype=BF16)[1:].view(150, 8, 64)
    odd.copy_(q)
    swap = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    for a in ((q, k, v), (odd, k, v), (swap(q), swap(k), swap(v)), (q, k.transpose(1, 2).contiguous().transpose(1, 2), v)):
        assert torch.equal(bs.prompt_attention(*a, o), want)
    one = bs.prompt_attention(q, k[:, :1].expand(150, 2, 64), v[:, :1].expand(150, 2, 64), o)
    assert torch.equal(one, bs.prompt_attention(q, k[:, :1], v[:, :1], o))
    out = torch.full((150, 8, 80), 3.0, device="cuda", dtype=BF16)
    assert torch.equal(bs.prompt_attention(q, k, v, o, out=out[..., 8:72]), want) and (out[..., :8] == 3).all() and (out[..., 72:] == 3).all()
    wide = torch.stack((o, o), 1)[:, 0]
    assert torch.equal(bs.prompt_attention(q, k, v, wide), want)
    for call in (lambda: bs.prompt_attention(q.float(), k, v, o), lambda: bs.prompt_attention(q, k[:149], v[:149], o),
                 lambda: bs.prompt_attention(q, k, v[:, :1], o), lambda: bs.prompt_attention(q[:, :7], k, v, o),
                 lambda: bs.prompt_attention(q, k, v, o.long()), lambda: bs.prompt_attention(q, k, v, o[:0]),
                 lambda: bs.prompt_attention(q, k, v, o, offsets_k=o[:2])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: bs.prompt_attention(q, k, v, o, out=q), lambda: bs.prompt_attention(q, k, v, o, scale=-1.0),
                 lambda: bs.prompt_attention(q, k, v, o, out=out[:, :, 4:68])):
        with pytest.raises(bs.BsgemmError):
            call()


def test_prompt_attention_offsets_that_are_wrong(bs):
    """Past the rows, falling: clamped, never out of bounds; the sound sequences are right."""
    g = gen(25)
    q, k, v, o, _ = packed(g, [60, 70], 4, 1, 64)
    want = bs.prompt_attention(q, k, v, o)
    bad = torch.tensor([0, 60, 1 << 30, -5, 7], dtype=torch.int32, device="cuda")
    got = bs.prompt_attention(q, k, v, bad[:3])
    assert torch.equal(got, want)
    bs.prompt_attention(q, k, v, bad)
    torch.cuda.synchronize()
    assert bs.check_device_error() == 0
