"""The attention operators at the ends of what they accept: padded batches, rows
that see no key at any scale, scores, queries and keys of every size that the
types hold, positions beyond 32 bits, many sequences of unlike lengths, inputs
that are dropped while their call waits."""
import math
from fractions import Fraction

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from test_attention_gpu import BF16, HALF, cached_rows, check_cache_attention, check_prompt, filled_cache, gen, normal, packed, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(cuda):
    yield
    torch.cuda.synchronize()


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- rows of no sequence --------------------------------------------------------------

@pytest.mark.parametrize("rows,heads,group,dim,ends", [
    (400, 2, 4, 64, [0, 40, 75]), (400, 2, 4, 128, [9, 40, 75, 75]), (5, 1, 1, 64, [0, 4]), (3000, 1, 7, 80, [1200, 1201]),
    (257, 3, 2, 40, [0, 0, 0]), (129, 1, 100, 128, [0, 129]), (64, 2, 2, 64, [17]), (20000, 2, 8, 128, [3, 500, 700])])
def test_prompt_attention_rows_of_no_sequence(bs, rows, heads, group, dim, ends):
    """Where the call makes the results, such rows are zeros and -inf; a caller's keep what they hold, lse never."""
    g = gen(rows + dim)
    q = normal(g, rows, heads * group, dim).to(BF16)
    k, v = normal(g, rows, heads, dim).to(BF16), normal(g, rows, heads, dim).to(BF16)
    o = i32(*ends)
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    inside[ends[0]:ends[-1]] = True
    given = torch.full_like(q, 3.0)
    for lse_too in (False, True):
        # what the allocator hands out next holds sevens
        old = [torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")]
        del old
        got = bs.prompt_attention(q, k, v, o, return_lse=lse_too)
        out, lse = got if lse_too else (got, None)
        assert not out[~inside].any()
        check_prompt(q, k, v, o, o, out, lse)
        if lse_too:
            assert (lse[~inside] == -math.inf).all()
        del got, lse
        old = [torch.full(q.shape[:2], 7.0, device="cuda"), torch.full(q.shape[:2], 7.0, device="cuda")]
        del old
        same = bs.prompt_attention(q, k, v, o, out=given, return_lse=lse_too)
        if lse_too:
            assert (same[1][~inside] == -math.inf).all()
        assert torch.equal(given[inside], out[inside]) and (given[~inside] == 3).all()


# ---- scores of every size -------------------------------------------------------------

def whole(g, *shape):
    """Whole numbers from -3 to 3, their products' sums exact in fp32."""
    return torch.randint(-3, 4, shape, device="cuda", generator=g).float()


def check_sharp_prompt(q, k, v, offsets, offsets_k, scale, out, lse):
    """Scores so far apart that only the largest count, several that are equal among them: exact in the kernel's sums.  Their
    weight is 1 from scores (in powers of two) of 2^29 on; below it is 2^d, d what fp32 rounds off c times the largest (up to
    2^4), so the weights are off by their rounding to bf16, up to 2^-8 of the values' sum, while their own sum
    is not.  The rest is the division (2^-22) and the output's rounding."""
    group = q.shape[1] // k.shape[1]
    a, b = offsets.tolist(), offsets_k.tolist()
    for i in range(len(a) - 1):
        nq, nk = a[i + 1] - a[i], b[i + 1] - b[i]
        hidden = torch.arange(nk, device="cuda")[None] > torch.arange(nq, device="cuda")[:, None] + nk - nq
        for h in range(q.shape[1]):
            s = (q[a[i]:a[i + 1], h].double() @ k[b[i]:b[i + 1], h // group].double().T).masked_fill(hidden, -math.inf)
            blind = hidden.all(1)
            top = s.amax(1, keepdim=True) if nk else s.new_zeros(nq, 1)
            w = ((s == top) & ~hidden).double()
            n = w.sum(1).clamp(min=1)
            values = v[b[i]:b[i + 1], h // group].double()
            want, mag = w @ values / n[:, None], w @ values.abs() / n[:, None]
            got = out[a[i]:a[i + 1], h].double()
            assert not got[blind].any()
            d = mag * (2.0 ** -20 + HALF[BF16] * (top.abs() * scale * math.log2(math.e) < 2.0 ** 29))
            assert ((got - want).abs() <= d + HALF[BF16] * (want.abs() + d)).all(), (i, h)
            level = lse[a[i]:a[i + 1], h].double()
            assert (level[blind] == -math.inf).all()
            line = scale * top[:, 0] + n.log()
            assert ((level - line).abs() <= 2.0 ** -21 * line.abs())[~blind].all(), (i, h)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("up,scale", [(0, 2.0 ** 28), (0, 1e9), (0, 1e18), (9, None), (14, None), (14, 1.0), (40, None), (55, None)])
def test_prompt_attention_large_scores(bs, dim, up, scale):
    """Scores of up to 2^117, scales of up to the largest that is accepted, and rows that see no key."""
    g = gen(dim + up)
    nq, nk = [5, 200, 150, 40], [2, 100, 300, 40]
    q, k, v, oq, ok = packed(g, nq, 4, 2, dim, nk)
    q, k = (whole(g, *q.shape) * 2.0 ** up).to(BF16), (whole(g, *k.shape) * 2.0 ** up).to(BF16)
    out, lse = bs.prompt_attention(q, k, v, oq, offsets_k=ok, scale=scale, return_lse=True)
    if up == 9:     # neighbouring scores lie 2^18 scale apart
        assert dim ** -0.5 * 2.0 ** 18 > 1000
    check_sharp_prompt(q, k, v, oq, ok, dim ** -0.5 if scale is None else scale, out, lse)


@pytest.mark.parametrize("offset", [1 << 12, 1 << 18, 1 << 21, -(1 << 21)])
def test_prompt_attention_scores_beside_a_large_offset(bs, offset):
    """Scores that lie close together far from zero, a few dozen higher every hundred keys: whole numbers, exact in fp32, so
    the weights are off by their rounding to bf16 and the exponential's 2^-21 alone."""
    g = gen(5)
    q, k, v, o, _ = packed(g, [700], 2, 1, 64)
    q, k = whole(g, *q.shape), whole(g, *k.shape)
    q[..., 0], q[..., 1] = 1024.0, 8.0
    k[..., 0], k[..., 1] = offset / 1024, (torch.arange(700, device="cuda") // 100 * 20).float()[:, None]
    q, k = q.to(BF16), k.to(BF16)
    out, lse = bs.prompt_attention(q, k, v, o, return_lse=True)
    hidden = torch.ones(700, 700, dtype=torch.bool, device="cuda").triu(1)
    for h in range(2):
        s = (q[:, h].double() @ k[:, 0].double().T / 8).masked_fill(hidden, -math.inf)
        assert (s[~hidden] - offset / 8).abs().max() < 2000
        p, level = torch.softmax(s, -1), torch.logsumexp(s, -1)
        want, mag = p @ v[:, 0].double(), p @ v[:, 0].double().abs()
        d = mag * (2.0 ** -8 + 2.0 ** -16)
        assert ((out[:, h].double() - want).abs() <= d + HALF[BF16] * (want.abs() + d)).all()
        assert ((lse[:, h].double() - level).abs() <= 2.0 ** -22 * level.abs()).all()


def test_prompt_attention_scores_far_below_zero(bs):
    """All of a row's scores below -10^30."""
    g = gen(4)
    q, k, v, o, _ = packed(g, [3, 300], 4, 2, 128)
    q, k = (whole(g, *q.shape).abs() + 1) * 2.0 ** 55, -(whole(g, *k.shape).abs() + 1) * 2.0 ** 50
    q, k = q.to(BF16), k.to(BF16)
    out, lse = bs.prompt_attention(q, k, v, o, return_lse=True)
    check_sharp_prompt(q, k, v, o, o, 128 ** -0.5, out, lse)


@pytest.mark.parametrize("scale", [30.0, 200.0, 1e4])
def test_prompt_attention_bits_do_not_depend_on_neighbours(bs, scale):
    """Rows with large scores among rows with small ones: each has the bits that it has with other neighbours."""
    g = gen(6)
    q, k, v, o, _ = packed(g, [260], 4, 1, 64)
    small, large = (q * 2.0 ** -6), q
    a, b = small.clone(), small.clone()
    a[::2], b[::3] = large[::2], large[::3]
    x, y = bs.prompt_attention(a, k, v, o, scale=scale), bs.prompt_attention(b, k, v, o, scale=scale)
    same = (a == b).flatten(1).all(1)
    assert same.sum() > 80 and torch.equal(x[same], y[same])


def whole_cache(bs, g, tokens, heads, dim, k_up, sign=None):
    """A cache whose keys are whole numbers times 2^k_up; each group of 32 has a 6, so that the format holds them."""
    k = whole(g, tokens, heads, dim)
    if sign:
        k = sign * (k.abs() + 1)
    k[..., ::32] = 6.0 * (sign or 1)
    cache = bs.new_kv_cache(-(-tokens // 16), 16, heads, dim)
    bs.cache_append(cache, k * 2.0 ** k_up, normal(g, tokens, heads, dim), torch.arange(tokens, device="cuda"))
    table = torch.arange(cache.k.shape[0], dtype=torch.int32, device="cuda")[None]
    return cache, table, i32(tokens)


def check_sharp_cache(bs, q, cache, table, lengths, scale=None):
    """As check_sharp_prompt, of one request."""
    got = bs.cache_attention(q, cache, table, lengths, scale=scale)[0].double()
    k, v = cached_rows(bs, cache, table, 0, int(lengths[0]))
    heads = k.shape[1]
    for h in range(q.shape[1]):
        s = k[:, h * heads // q.shape[1]].double() @ q[0, h].double()
        w = (s == s.amax()).double()
        values = v[:, h * heads // q.shape[1]].double()
        want, mag = w @ values / w.sum(), w @ values.abs() / w.sum()
        assert ((got[h] - want).abs() <= HALF[BF16] * want.abs() + 2.0 ** -20 * mag).all(), h


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [40, 3000])
@pytest.mark.parametrize("q_up,k_up,scale", [(15, 15, None), (30, 0, 1.0), (60, 40, None), (110, 0, None), (120, -100, None), (0, 90, None), (0, 112, None),
                                             (-100, 119, 1.0), (-60, 119, None), (119, -110, 2.0 ** 55), (0, 20, 1e18)])
def test_cache_attention_large_scores(bs, dim, tokens, q_up, k_up, scale):
    g = gen(dim + tokens)
    cache, table, n = whole_cache(bs, g, tokens, 2, dim, k_up)
    q = (whole(g, 1, 8, dim) * 2.0 ** q_up).to(BF16)
    check_sharp_cache(bs, q, cache, table, n, scale)


def test_cache_attention_scores_far_below_zero(bs):
    for tokens in (40, 3000):
        cache, table, n = whole_cache(bs, gen(tokens), tokens, 2, 128, 50, sign=-1)
        q = ((whole(gen(1), 1, 8, 128).abs() + 1) * 2.0 ** 55).to(BF16)
        check_sharp_cache(bs, q, cache, table, n)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_up,k_up,scale", [(120, -118, None), (125, -119, None), (113, -113, None), (120, 0, 2.0 ** -121), (126, 0, 2.0 ** -127), (-110, 90, 2.0 ** 20),
                                             (-125, 90, 2.0 ** 35), (-131, 96, 2.0 ** 35), (-112, 112, None),
                                             (-120, 119, None), (-128, 121, 8.0), (0, 110, 2.0 ** -112), (-4, 122, 2.0 ** -119)])
def test_cache_attention_queries_and_keys_of_every_size(bs, dim, q_up, k_up, scale):
    """Sizes that cancel in the scores: every finite query that bf16 holds, keys to the format's ends."""
    g = gen(dim + q_up + 200)
    tokens = 200
    cache = bs.new_kv_cache(13, 16, 2, dim)
    bs.cache_append(cache, normal(g, tokens, 2, dim) * 2.0 ** k_up, normal(g, tokens, 2, dim), torch.arange(tokens, device="cuda"))
    table = torch.arange(13, dtype=torch.int32, device="cuda")[None]
    q = (normal(g, 1, 8, dim).double().clamp(-3, 3) * 2.0 ** q_up).to(BF16)
    assert q.isfinite().all()
    got = check_cache_attention(bs, q, cache, table, i32(tokens), scale=scale, half=2.0 ** -8 if k_up > 90 else 2.0 ** -11)
    assert got.isfinite().all()     # (what is compared above does not tell NaN)


def test_cache_attention_weights_of_whole_steps_apart(bs):
    """Scaled scores beyond 2^27, where fp32 holds multiples of 16: a warp's later tokens are 16 above its earlier ones."""
    n = 80000       # several steps for each warp
    cache = bs.new_kv_cache(313, 256, 1, 64)
    k = torch.zeros(n, 1, 64, device="cuda")
    k[:, 0, 0], k[:, 0, 32] = 6.0, 6.0
    k[torch.arange(n, device="cuda") // 128 % 2 == 1, 0, 1] = 1.0
    bs.cache_append(cache, k, normal(gen(3), n, 1, 64), torch.arange(n, device="cuda"))
    q = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    q[0, 0, 0], q[0, 0, 1] = 2.0 ** 25, 16.0
    check_sharp_cache(bs, q, cache, torch.arange(313, dtype=torch.int32, device="cuda")[None], i32(n), scale=1 / math.log2(math.e))


# ---- lengths at the end of 32 bits ----------------------------------------------------

def test_cache_attention_lengths_at_the_end_of_32_bits(bs):
    """A table of 2^31 tokens: the longest length that there is, beside ordinary requests, has its split and theirs right."""
    g = gen(7)
    cache = filled_cache(bs, g, 5, 256, 1, 64)
    columns = 1 << 23
    table = torch.full((3, columns), -1, dtype=torch.int32, device="cuda")
    table[0, :2], table[2, :1] = i32(0, 1), 2
    table[1, 3], table[1, columns - 1] = 3, 4
    q = normal(g, 3, 2, 64).to(BF16)
    top = 2 ** 31 - 1
    # request 1 sees a whole page and, at the end of the table, all but the last token of another
    near = torch.tensor([[3, 4]], dtype=torch.int32, device="cuda")
    for length, left in ((top, 255), (top - 62, 193), (top - 63, 192), (top - 255, 0)):
        lengths = i32(300, length, 77)
        got = bs.cache_attention(q, cache, table, lengths)
        for r, n in ((0, 300), (2, 77)):
            check_cache_attention(bs, q[r:r + 1], cache, table[r:r + 1, :4].contiguous(), i32(n), out=got[r:r + 1])
        check_cache_attention(bs, q[1:2], cache, near, i32(256 + left), out=got[1:2])
        assert got.isfinite().all()
    assert bs.check_device_error() == 0


# ---- positions ------------------------------------------------------------------------

def turn_of_pi(bits):
    """1 / (2 pi) as a fraction, to 2^-bits: Machin's pi = 16 atan(1/5) - 4 atan(1/239)."""
    one = 1 << (bits + 32)

    def atan(x):
        total, term, n = 0, one // x, 1
        while term:
            total += term // n if n % 4 == 1 else -(term // n)
            term //= x * x
            n += 2
        return total
    return Fraction(one, 2 * (16 * atan(5) - 4 * atan(239)))


@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_at_any_position(bs, inverse):
    """Angles of positions to both ends of int64, against exact arithmetic."""
    g = gen(8)
    plan = bs.rotary_plan(64, scaling="yarn", factor=8.0)
    pos = [0, 1, -1, 1 << 20, (1 << 28) + 3, (1 << 31) - 1, (1 << 33) + 5, -(1 << 40) - 7, (1 << 53) + 1, (1 << 58) + 12345, -(1 << 62) + 3,
           (1 << 63) - 1, -(1 << 63)]
    at = torch.tensor(pos, device="cuda")
    q = normal(g, len(pos), 2, 64)
    got = bs.rotary(q, None, at, plan, inverse=inverse)[0].double()
    inv, sign = turn_of_pi(256), -1 if inverse else 1
    turns = [[float((sign * p * Fraction(f) * inv) % 1) for f in plan.frequencies.tolist()] for p in pos]
    t = torch.tensor(turns, dtype=torch.float64, device="cuda")[:, None] * (2 * math.pi)
    c, s = t.cos() * plan.factor, t.sin() * plan.factor
    a, b = q.double().split(32, -1)
    want = torch.cat((a * c - b * s, b * c + a * s), -1)
    mag = torch.cat((a.abs() + b.abs(),) * 2, -1) * plan.factor
    # as at small positions: the fraction of a turn, cosine and sine, factor, products and sum in fp32
    assert ((got - want).abs() <= 8 * 2.0 ** -24 * mag + 2.0 ** -24 * want.abs()).all()


# ---- many sequences -------------------------------------------------------------------

@pytest.mark.parametrize("heads,group,lengths", [
    (2, 8, [1500] + [1 + i % 5 for i in range(40)]),
    (1, 16, [(37 * i) % 211 for i in range(64)]),
    (1, 4, [(131 * i) % 97 * (i % 7 == 0) for i in range(300)] + [2100]),
    (1, 1, [900 if i in (3, 31, 32, 70, 99) else i % 3 for i in range(100)]),
    (1, 128, [(i * 13) % 40 for i in range(33)]),
    (3, 2, [0] * 50 + [700] + [0] * 50 + [65] * 30)])
def test_prompt_attention_many_sequences_of_several_levels(bs, heads, group, lengths):
    """More than 32 sequences, some of many items and most of few or none, in any order."""
    for order in (lengths, lengths[::-1]):
        q, k, v, o, _ = packed(gen(sum(lengths)), order, heads * group, heads, 64)
        out, lse = bs.prompt_attention(q, k, v, o, return_lse=True)
        check_prompt(q, k, v, o, o, out, lse)
    assert bs.check_device_error() == 0


def test_prompt_attention_one_long_among_many_short(bs):
    """1023 sequences of a token beside one of 24576 cost what they take, not a look at each for every block of the long one."""
    g = gen(9)
    n = 24576
    q, k, v = (normal(g, n + 1023, h, 64).to(BF16) for h in (8, 1, 1))
    alone = i32(0, n)
    among = torch.cat((i32(0), torch.arange(n, n + 1024, dtype=torch.int32, device="cuda")))
    out = torch.zeros_like(q)

    def time(offsets):
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            bs.prompt_attention(q, k, v, offsets, out=out)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    lone = time(alone)
    want = out[:n].clone()
    assert time(among) < 1.5 * lone
    assert torch.equal(out[:n], want) and torch.equal(out[n:], v[n:].expand(1023, 8, 64))


# ---- results and inputs ---------------------------------------------------------------

def test_results_are_made_through_the_dispatcher(bs):
    """A dispatch mode sees the allocations of every operator."""
    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    g = gen(10)
    x = normal(g, 8, 256).to(BF16)
    q, k = normal(g, 8, 4, 64).to(BF16), normal(g, 8, 2, 64).to(BF16)
    cache, table, n = paged(bs, g, [20] * 8, 16, 2, 64)
    plan = bs.rotary_plan(64)
    e, sf = bs.quantize(x, "mxfp8")
    w, wsf = bs.quantize(normal(g, 128, 256).to(BF16), "mxfp8")
    for call in (lambda: bs.layer_norm(x), lambda: bs.layer_norm(x, out_format="mxfp8"), lambda: bs.linear_a8w8_mxfp8(e, w, sf, wsf),
                 lambda: bs.rotary(q, k, i32(*range(8)), plan), lambda: bs.paged_slots(n, n, table, i32(1, 2, 3), 16, 200),
                 lambda: bs.cache_read(cache, torch.arange(8, device="cuda")), lambda: bs.cache_attention(q, cache, table, n),
                 lambda: bs.prompt_attention(q, k, k, i32(0, 8), return_lse=True)):
        Seen.names.clear()
        with Seen():
            call()
        assert any("aten.empty" in name for name in Seen.names), Seen.names


CALLS = ["rotary strided", "rotary positions", "rotary", "slots", "append offset", "append slots", "append", "read slots", "cache offset", "cache lengths",
         "cache", "prompt offset", "prompt offsets", "prompt keys", "prompt"]


@pytest.mark.parametrize("what", CALLS)
def test_inputs_dropped_while_their_call_waits(bs, what):
    """A tensor of one stream, used on another that is busy and dropped at once: its memory is not handed on before the call
    (or the copy that it makes first) has run."""
    g = gen(11)
    q, k, v, o, _ = packed(g, [700, 300], 8, 2, 64)
    cache, table, n = paged(bs, g, [90, 40, 7], 16, 2, 64)
    plan, pos = bs.rotary_plan(64), torch.arange(1000, device="cuda") * 3
    slots = torch.randperm(cache.k.shape[0] * 16, device="cuda", generator=g)[:80]
    q3 = normal(g, 3, 8, 64).to(BF16)
    rows = normal(g, 80, 2, 64).to(BF16)
    three, free = i32(3, 3, 3), i32(7, 8)

    def off(t):     # one element behind an aligned address
        return torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)

    def apart(t):   # every second of a buffer
        return torch.stack((t, t), -1)[..., 0]

    def append(kk, ss):
        fresh = bs.KvCache(*(torch.zeros_like(t) for t in cache))
        bs.cache_append(fresh, kk, rows, ss)
        return tuple(fresh)

    make, use = {
        "rotary strided": (lambda: apart(q), lambda t: bs.rotary(t, None, pos, plan)),
        "rotary positions": (lambda: apart(pos), lambda t: bs.rotary(q, None, t, plan)),
        "rotary": (lambda: q.clone(), lambda t: bs.rotary(t, None, pos, plan)),
        "slots": (lambda: apart(n), lambda t: bs.paged_slots(t, three, table.clone(), free, 16, 12)),
        "append offset": (lambda: off(rows), lambda t: append(t, slots)),
        "append slots": (lambda: apart(slots), lambda t: append(rows, t)),
        "append": (lambda: rows.clone(), lambda t: append(t, slots)),
        "read slots": (lambda: apart(slots), lambda t: bs.cache_read(cache, t)),
        "cache offset": (lambda: off(q3), lambda t: bs.cache_attention(t, cache, table, n)),
        "cache lengths": (lambda: apart(n), lambda t: bs.cache_attention(q3, cache, table, t)),
        "cache": (lambda: q3.clone(), lambda t: bs.cache_attention(t, cache, table, n)),
        "prompt offset": (lambda: off(q), lambda t: bs.prompt_attention(t, k, v, o)),
        "prompt offsets": (lambda: apart(o), lambda t: bs.prompt_attention(q, k, v, t)),
        "prompt keys": (lambda: off(k), lambda t: bs.prompt_attention(q, t, v, o)),
        "prompt": (lambda: q.clone(), lambda t: bs.prompt_attention(t, k, v, o)),
    }[what]
    list_of = lambda r: [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None]
    want = [t.clone() for t in list_of(use(make()))]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        use(make())     # loads its kernels and its stream's memory, which would outlast the wait below
    for _ in range(3):
        t = make()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)   # about 10 ms
            got = list_of(use(t))
        size, at = t.untyped_storage().nbytes(), t.untyped_storage().data_ptr()
        del t
        over = torch.full((size,), 1, dtype=torch.uint8, device="cuda")     # the first stream goes on at once
        if not side.query():    # the call has not run yet
            assert over.untyped_storage().data_ptr() != at
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
