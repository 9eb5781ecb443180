"""Workloads of the attention half of a block as it is served: rotary positions,
block tables and slot maps from request lengths, a cache of keys and values in 4
bits (written, and attended to by single tokens) and causal attention over
packed prompts with grouped heads.

A pass of each is run either in its plain form (elementary torch operations in
fp32, positions' angles in fp64, rounded once at the end) or, with ``own`` set,
by this library's kernels.  Both take the same tensors, the cache in the
library's layout among them: E2M1 elements with one E8M0 scale per 32.
"""
import importlib
import math
import random

import torch

own = False

GROUP = 32            # elements per E8M0 scale
MOST_FLOPS = 1.11e12  # of one pass; the largest listed case has 1.10e12
MOST_BYTES = 1.0e9    # what a drawn case reads and writes at most
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}


def listed():
    return [
        # queries and keys of one decoded token: 32 query heads on 8 key heads
        {"name": "rotary one token", "op": "rotary", "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "inverse": False, "far": 4096, "scaling": "none"},
        # a prompt batch at positions far behind the trained length, frequencies stretched for it
        {"name": "rotary prompt", "op": "rotary", "tokens": 16384, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "inverse": False, "far": 131072, "scaling": "yarn"},
        # the gradient's rotation in a small fp32 model that turns neighbouring pairs in a third of each head
        {"name": "rotary part", "op": "rotary", "tokens": 1023, "q_heads": 9, "kv_heads": 3, "dim": 96, "rot": 32,
         "dtype": "fp32", "interleaved": True, "inverse": True, "far": 8192, "scaling": "linear"},
        # a decode step: each of 64 requests adds one token
        {"name": "slots decode", "op": "slots", "requests": 64, "page": 64, "most_cached": 8192, "most_new": 1, "pattern": 1},
        # prompts and decoded tokens mixed, small pages
        {"name": "slots mixed", "op": "slots", "requests": 1000, "page": 16, "most_cached": 4096, "most_new": 256, "pattern": 2},
        # a decode step's keys and values go to the cache
        {"name": "append decode", "op": "append", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # those of a prompt batch
        {"name": "append prompt", "op": "append", "tokens": 16384, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one request with a long context behind it: the axis has to be split
        {"name": "cache one request", "op": "cache", "requests": 1, "most": 32768, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "pattern": 3},
        # a decode batch of unequal requests
        {"name": "cache batch", "op": "cache", "requests": 128, "most": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "pattern": 4},
        # a handful of short prompts, one of them empty and one a single token
        {"name": "prompt short", "op": "prompt", "lengths": "17,0,1,40,70", "q_heads": 32, "kv_heads": 8, "dim": 128,
         "lse": False},
        # unequal prompts, heads of 64 in groups of seven
        {"name": "prompt packed", "op": "prompt", "lengths": "1999,5,300,1,777,128,2500,64,1023,33,511,1200", "q_heads": 14,
         "kv_heads": 2, "dim": 64, "lse": True},
        # two long prompts
        {"name": "prompt long", "op": "prompt", "lengths": "8192,8192", "q_heads": 32, "kv_heads": 8, "dim": 128,
         "lse": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("rotary", "slots", "append", "cache", "cache", "prompt", "prompt", "prompt"))
    kv = rng.choice((1, 2, 3, 4, 8))
    q = kv * rng.choice((1, 2, 3, 4, 5, 7, 8, 16) if kv < 4 else (1, 2, 4, 6, 8))
    if op == "rotary":
        dim = rng.choice((64, 80, 96, 128, 256))
        c = {"op": op, "tokens": _log_int(rng, 1, 16384), "q_heads": q, "kv_heads": kv, "dim": dim,
             "rot": rng.choice((dim, dim, dim // 2, 32)), "dtype": rng.choice(("bf16", "bf16", "fp32")),
             "interleaved": rng.random() < 0.4, "inverse": rng.random() < 0.3, "far": _log_int(rng, 1024, 1 << 20),
             "scaling": rng.choice(("none", "linear", "yarn"))}
        while work(c)["bytes"] > MOST_BYTES:
            c["tokens"] //= 2
        return c
    if op == "slots":
        return {"op": op, "requests": _log_int(rng, 1, 2000), "page": rng.choice((16, 32, 64, 128)),
                "most_cached": _log_int(rng, 1, 16384), "most_new": rng.choice((1, 1, _log_int(rng, 1, 256))),
                "pattern": rng.randrange(1 << 30)}
    if op == "append":
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "kv_heads": kv, "dim": rng.choice((64, 128)),
                "page": rng.choice((16, 32, 64, 128)), "dtype": rng.choice(("bf16", "bf16", "fp32"))}
    if op == "cache":
        c = {"op": op, "requests": _log_int(rng, 1, 256), "most": _log_int(rng, 1, 65536), "q_heads": q, "kv_heads": kv,
             "dim": rng.choice((64, 128)), "page": rng.choice((16, 32, 64, 128)), "pattern": rng.randrange(1 << 30)}
        while work(c)["bytes"] > 0.5 * MOST_BYTES:
            c["requests"] = max(1, c["requests"] // 2)
            c["most"] = max(1, c["most"] * 3 // 4)
        return c
    c = {"op": op, "q_heads": q, "kv_heads": kv, "dim": rng.choice((64, 64, 80, 128, 128, 128)),
         "lse": rng.random() < 0.5}
    most = _log_int(rng, 1, 8192)
    lengths = [rng.choice((most, rng.randint(0, most), _log_int(rng, 1, most))) for _ in range(_log_int(rng, 1, 24))]
    c["lengths"] = ",".join(map(str, lengths))
    while work(c)["flops"] > MOST_FLOPS or work(c)["bytes"] > MOST_BYTES:
        lengths = [n * 3 // 4 for n in lengths]
        c["lengths"] = ",".join(map(str, lengths))
    return c


def _prompt_lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _cache_lengths(case):
    """Lengths of the requests of a decode batch: the longest, then anything up to it."""
    rng = random.Random(case["pattern"])
    return [case["most"]] + [rng.randint(max(1, case["most"] // 16), case["most"]) for _ in range(case["requests"] - 1)]


def _slot_lengths(case):
    """(tokens in the cache, tokens to come) of each request; some have none of either."""
    rng = random.Random(case["pattern"])
    cached = [rng.randint(0, case["most_cached"]) for _ in range(case["requests"])]
    new = [rng.choice((1, rng.randint(0, case["most_new"]))) for _ in range(case["requests"])]
    return cached, new


def work(case):
    """Bytes and operations that a pass cannot do without: each input read once,
    each output written once; causal attention computes its lower triangle."""
    op = case["op"]
    if op == "rotary":
        heads, n = case["q_heads"] + case["kv_heads"], case["tokens"]
        return {"bytes": 2 * n * heads * case["dim"] * SIZE[case["dtype"]] + 4 * n + 4 * case["rot"],
                "flops": 3 * n * heads * case["rot"]}
    if op == "slots":
        cached, new = _slot_lengths(case)
        pages = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(cached, new))
        return {"bytes": 20 * len(new) + 12 * sum(new) + 8 * pages, "flops": 4 * sum(new)}
    if op == "append":   # elements read; 4 bits and scales written, read back and their values written
        n = case["tokens"] * case["kv_heads"] * case["dim"] * 2
        return {"bytes": n * (SIZE[case["dtype"]] + 2 * (0.5 + 1 / GROUP) + 2) + 8 * case["tokens"], "flops": 4 * n}
    if op == "cache":
        keys, hq, d = sum(_cache_lengths(case)), case["q_heads"], case["dim"]
        return {"bytes": keys * case["kv_heads"] * d * 2 * (0.5 + 1 / GROUP)
                + 4 * case["requests"] * hq * d, "flops": 4.0 * keys * hq * d}
    lengths, hq, d = _prompt_lengths(case), case["q_heads"], case["dim"]
    return {"bytes": 4 * sum(lengths) * d * (hq + case["kv_heads"]),
            "flops": 4.0 * d * hq * sum(n * (n + 1) // 2 for n in lengths)}


# ---- stored formats -----------------------------------------------------------

def _quantise(x):
    """fp32 [..., dim] -> (E2M1 codes [..., dim], E8M0 bytes [..., dim / 32]): scale
    2^ceil(log2(amax / 6)), elements rounded to nearest even."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    mant, e = torch.frexp(g.abs().amax(-1).double() / 6)
    e = torch.where(mant == 0.5, e - 1, e)
    e = torch.where(mant == 0, torch.zeros_like(e), e).clamp(-127, 127)
    v = torch.ldexp(g, -e.unsqueeze(-1)).reshape(x.shape)
    a = v.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i in range(7):     # a tie goes to the even code
        mid = (E2M1[i] + E2M1[i + 1]) / 2
        code += (a >= mid) if i % 2 else (a > mid)
    return code | torch.signbit(v).to(torch.uint8) << 3, (e + 127).to(torch.uint8)


def _values(code, scale):
    """The fp32 values of E2M1 codes [..., dim] with E8M0 bytes [..., dim / 32]."""
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=code.device)
    s = torch.ldexp(torch.ones_like(scale, dtype=torch.float32), scale.int() - 127)
    return (table[code.int()].reshape(*scale.shape, GROUP) * s.unsqueeze(-1)).reshape(code.shape)


def _pack_keys(code):
    """Codes [pages, heads, page, dim] -> bytes [pages, heads, page, dim / 2]: element
    32 g + 8 c + 2 i + h of a row lies in byte c (dim / 8) + 4 g + i, in its low (h = 0) or high half."""
    b = code[..., 0::2] | code[..., 1::2] << 4
    return b.reshape(*b.shape[:-1], -1, 4, 4).transpose(-3, -2).reshape(b.shape).contiguous()


def _unpack_keys(b):
    n = b.reshape(*b.shape[:-1], 4, -1, 4).transpose(-3, -2).reshape(b.shape)
    return torch.stack((n & 15, n >> 4), dim=-1).flatten(-2)


def _pack_values(code):
    """Codes [pages, heads, page, dim] -> bytes [pages, heads, page / 4, dim / 2, 4]: the
    pairs of elements of four tokens side by side."""
    b = code[..., 0::2] | code[..., 1::2] << 4
    return b.unflatten(2, (-1, 4)).transpose(-2, -1).contiguous()


def _unpack_values(b):
    n = b.transpose(-2, -1).flatten(2, 3)
    return torch.stack((n & 15, n >> 4), dim=-1).flatten(-2)


def _pack_value_scales(s):
    return s.unflatten(2, (-1, 4)).transpose(-2, -1).contiguous()


def _unpack_value_scales(s):
    return s.transpose(-2, -1).flatten(2, 3)


def _empty_cache(pages, page, heads, dim):
    kw = {"dtype": torch.uint8, "device": "cuda"}
    return (torch.zeros((pages, heads, page, dim // 2), **kw), torch.zeros((pages, heads, page, dim // GROUP), **kw),
            torch.zeros((pages, heads, page // 4, dim // 2, 4), **kw), torch.zeros((pages, heads, page // 4, dim // GROUP, 4), **kw))


# ---- inputs -------------------------------------------------------------------

def _frequencies(case):
    """Radians a position of each pair, fp64, and the factor on cosine and sine."""
    rot, base = case["rot"], 10000.0
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "none":
        return f, 1.0
    factor = 8.0
    if case["scaling"] == "linear":
        return f / factor, 1.0
    # by parts: pairs that turn often within the trained length keep their frequency, slow ones are stretched
    trained = 4096

    def pair(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    def channels(heads, dim):   # keys have a few channels that are far larger than the others
        return torch.where(torch.rand((heads, dim), device="cuda", generator=g) < 0.03, 6.0, 1.0)

    s, op = dict(case), case["op"]
    if op == "rotary":
        t, n = DTYPES[case["dtype"]], case["tokens"]
        s["q"] = normal(n, case["q_heads"], case["dim"]).to(t)
        s["k"] = normal(n, case["kv_heads"], case["dim"]).to(t)
        s["positions"] = torch.randint(0, case["far"], (n,), device="cuda", generator=g, dtype=torch.int32)
        f, s["factor"] = _frequencies(case)
        s["frequencies"] = f.cuda()
        return s
    if op == "slots":
        cached, new = _slot_lengths(case)
        page = case["page"]
        owned = [-(-c // page) for c in cached]
        most = max(-(-(c + n) // page) for c, n in zip(cached, new))
        fresh = sum(-(-(c + n) // page) - o for c, n, o in zip(cached, new, owned))
        ids = torch.randperm(sum(owned) + fresh + 8, device="cuda", generator=g).int()
        have = torch.arange(max(most, 1), device="cuda") < torch.tensor(owned, device="cuda")[:, None]
        s["table"] = torch.full(have.shape, -1, dtype=torch.int32, device="cuda")
        s["table"][have] = ids[:sum(owned)]
        s["free"] = ids[sum(owned):].contiguous()
        s["cached"] = torch.tensor(cached, dtype=torch.int32, device="cuda")
        s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        s["tokens"] = sum(new) + 5     # a batch padded by five
        return s
    if op == "append":
        n, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        t = DTYPES[case["dtype"]]
        pages = -(-n // page) + 4
        s["k"], s["v"] = (normal(n, h, d) * channels(h, d)).to(t), normal(n, h, d).to(t)
        at = torch.randperm(pages, device="cuda", generator=g)
        i = torch.arange(n, device="cuda")
        s["slots"] = at[i // page] * page + i % page
        s["cache"] = _empty_cache(pages, page, h, d)
        return s
    if op == "cache":
        lengths = _cache_lengths(case)
        h, d, page = case["kv_heads"], case["dim"], case["page"]
        owned = [-(-n // page) for n in lengths]
        pages = sum(owned) + 3
        s["cache"] = _empty_cache(pages, page, h, d)
        amp = channels(h, d)[:, None]
        step = max(1, (1 << 24) // (h * page * d))
        for p in range(0, pages, step):
            m = min(step, pages - p)
            code, scale = _quantise(normal(m, h, page, d) * amp)
            s["cache"][0][p:p + m], s["cache"][1][p:p + m] = _pack_keys(code), scale
            code, scale = _quantise(normal(m, h, page, d))
            s["cache"][2][p:p + m], s["cache"][3][p:p + m] = _pack_values(code), _pack_value_scales(scale)
        have = torch.arange(max(owned), device="cuda") < torch.tensor(owned, device="cuda")[:, None]
        s["table"] = torch.full(have.shape, -1, dtype=torch.int32, device="cuda")
        s["table"][have] = torch.randperm(pages, device="cuda", generator=g)[:sum(owned)].int()
        s["lengths_host"] = lengths
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = (normal(case["requests"], case["q_heads"], d) * 1.5).bfloat16()
        return s
    lengths, hq, h, d = _prompt_lengths(case), case["q_heads"], case["kv_heads"], case["dim"]
    n = sum(lengths)
    s["q"], s["v"] = (normal(n, hq, d) * 1.5).bfloat16(), normal(n, h, d).bfloat16()
    s["k"] = (normal(n, h, d) * channels(h, d)).bfloat16()
    s["lengths_host"] = lengths
    s["offsets"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")
    return s


# ---- the operators --------------------------------------------------------------

def _turn(x, cos, sin, rot, interleaved):
    y = x.float()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, y[..., rot:]), dim=-1).to(x.dtype)


def _plain(s):
    op = s["op"]
    if op == "rotary":
        angle = s["positions"].double()[:, None, None] * s["frequencies"]
        cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
        if s["inverse"]:
            sin = -sin
        return tuple(_turn(s[x], cos, sin, s["rot"], s["interleaved"]) for x in ("q", "k"))
    if op == "slots":
        page, n, cached, new, table = s["page"], s["tokens"], s["cached"], s["new"], s["table"]
        lengths = cached + new
        offsets = torch.cat((new.new_zeros(1), new.cumsum(0).int()))
        had, has = (cached + page - 1) // page, (lengths + page - 1) // page
        first = (has - had).cumsum(0) - (has - had)
        column = torch.arange(table.shape[1], device="cuda")
        fresh = (column >= had[:, None]) & (column < has[:, None])
        which = (first[:, None] + column - had[:, None]).clamp(0, len(s["free"]) - 1)
        table.copy_(torch.where(fresh, s["free"][which], table))
        token = torch.arange(n, device="cuda", dtype=torch.int32)
        r = (token[:, None] >= offsets[None, 1:]).sum(1).clamp_max(len(new) - 1)
        inside = token < offsets[-1]
        position = torch.where(inside, cached[r] + token - offsets[r], 0)
        slot = table[r, position // page].long() * page + position % page
        return torch.where(inside, slot, -1), position.int(), offsets, lengths, (has - had).sum().int().reshape(1), table
    if op == "append":
        cache, page = s["cache"], s["page"]
        at, row = s["slots"] // page, s["slots"] % page
        (kc, ks), (vc, vs) = _quantise(s["k"].float()), _quantise(s["v"].float())
        kb, vb = _pack_keys(kc[:, :, None])[:, :, 0], vc[..., 0::2] | vc[..., 1::2] << 4
        cache[0][at, :, row], cache[1][at, :, row] = kb, ks
        cache[2][at, :, row // 4, :, row % 4], cache[3][at, :, row // 4, :, row % 4] = vb, vs
        k = _values(_unpack_keys(cache[0][at, :, row]), cache[1][at, :, row])
        b = cache[2][at, :, row // 4, :, row % 4]
        v = _values(torch.stack((b & 15, b >> 4), dim=-1).flatten(-2), cache[3][at, :, row // 4, :, row % 4])
        return k.bfloat16(), v.bfloat16()
    if op == "cache":
        k4, ks, v4, vs = s["cache"]
        out = []
        h, group = s["kv_heads"], s["q_heads"] // s["kv_heads"]
        for i, n in enumerate(s["lengths_host"]):
            at = s["table"][i, :-(-n // s["page"])].long()
            k = _values(_unpack_keys(k4[at]), ks[at]).transpose(0, 1).flatten(1, 2)[:, :n]
            v = _values(_unpack_values(v4[at]), _unpack_value_scales(vs[at])).transpose(0, 1).flatten(1, 2)[:, :n]
            q = s["q"][i].float().unflatten(0, (h, group))
            p = q @ k.transpose(1, 2) * s["dim"] ** -0.5
            p = torch.exp(p - p.amax(-1, keepdim=True))
            out.append((p @ v / p.sum(-1, keepdim=True)).flatten(0, 1))
        return torch.stack(out).bfloat16()
    h, group = s["kv_heads"], s["q_heads"] // s["kv_heads"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], device="cuda")
    first = 0
    for n in s["lengths_host"]:
        if n == 0:
            continue
        rows = slice(first, first + n)
        hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n, device="cuda")[:, None]
        for j in range(h):
            heads = slice(j * group, (j + 1) * group)
            q, k, v = s["q"][rows, heads].float().transpose(0, 1), s["k"][rows, j].float(), s["v"][rows, j].float()
            p = (q @ k.t() * s["dim"] ** -0.5).masked_fill_(hidden, -math.inf)
            top = p.amax(-1, keepdim=True)
            p = p.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            out[rows, heads] = (p @ v / total).transpose(0, 1).bfloat16()
            lse[rows, heads] = (top + torch.log(total)).squeeze(-1).t()
        first += n
    return (out, lse) if s["lse"] else out


def _own(s):
    bs = importlib.import_module("355_1_trans_b200")
    op = s["op"]
    if op == "rotary":
        return bs.rotary(s["q"], s["k"], s["positions"], bs.RotaryPlan(s["frequencies"], s["factor"]),
                         interleaved=s["interleaved"], inverse=s["inverse"])
    if op == "slots":
        p = bs.paged_slots(s["cached"], s["new"], s["table"], s["free"], s["page"], s["tokens"])
        return p.slots, p.positions, p.offsets, p.lengths, p.pages_taken, s["table"]
    if op == "append":
        cache = bs.KvCache(*s["cache"])
        bs.cache_append(cache, s["k"], s["v"], s["slots"])
        return bs.cache_read(cache, s["slots"])
    if op == "cache":
        return bs.cache_attention(s["q"], bs.KvCache(*s["cache"]), s["table"], s["lengths"])
    return bs.prompt_attention(s["q"], s["k"], s["v"], s["offsets"], return_lse=s["lse"])


def run(s):
    """One pass through the case's operator."""
    return _own(s) if own else _plain(s)


# ---- the definition in 64 bits ----------------------------------------------------

def _f64(code, scale):
    """E2M1 codes [..., dim] and E8M0 bytes [..., dim / 32] -> fp64 values, from the bit fields."""
    sign, e, f = (code >> 3).double(), (code >> 1 & 3).double(), (code & 1).double()
    v = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2(e - 1)) * (1 - 2 * sign)
    return v * torch.exp2(scale.double() - 127).repeat_interleave(GROUP, -1)


def _cached_f64(s, request, length):
    """Keys and values [heads, length, dim] of a request, byte by byte from the layout."""
    d, page = s["dim"], s["page"]
    token = torch.arange(length, device="cuda")
    at, row = s["table"][request][token // page].long(), token % page
    e = torch.arange(d, device="cuda")
    half = e % 2 * 4
    byte = e % 32 // 8 * (d // 8) + e // 32 * 4 + e % 8 // 2
    k = s["cache"][0][at, :, row][:, :, byte] >> half & 15
    v = s["cache"][2][at, :, row // 4, :, row % 4][:, :, e // 2] >> half & 15
    k = _f64(k, s["cache"][1][at, :, row])
    return k.transpose(0, 1), _f64(v, s["cache"][3][at, :, row // 4, :, row % 4]).transpose(0, 1)


def exact(case, seed):
    """What run returns, from the definition in fp64.  What the cache holds are
    not computed numbers but the nearest of 16, so there the values before that say nothing."""
    op = case["op"]
    if op == "append":
        return None
    s = prepare(case, seed)
    if op == "rotary":
        rot = case["rot"]
        i = torch.arange(rot // 2, device="cuda")
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
        z = torch.polar(torch.full_like(s["frequencies"], s["factor"]).expand(case["tokens"], -1).contiguous(),
                        s["positions"].double()[:, None] * s["frequencies"] * (-1 if case["inverse"] else 1))[:, None]
        out = []
        for x in (s["q"].double(), s["k"].double()):
            w = torch.complex(x[..., first], x[..., second]) * z
            x[..., first], x[..., second] = w.real, w.imag
            out.append(x)
        return tuple(out)
    if op == "slots":
        cached, new = _slot_lengths(case)
        page, table, free = case["page"], s["table"].tolist(), s["free"].tolist()
        slots, positions, offsets, taken = [], [], [0], 0
        for r, (c, n) in enumerate(zip(cached, new)):
            for t in range(c, c + n):
                if t % page == 0:
                    table[r][t // page] = free[taken]
                    taken += 1
                slots.append(table[r][t // page] * page + t % page)
                positions.append(t)
            offsets.append(offsets[-1] + n)
        spare = s["tokens"] - len(slots)
        lengths = [c + n for c, n in zip(cached, new)]
        return tuple(torch.tensor(x, dtype=t, device="cuda") for x, t in (
            (slots + [-1] * spare, torch.int64), (positions + [0] * spare, torch.int32), (offsets, torch.int32),
            (lengths, torch.int32), ([taken], torch.int32), (table, torch.int32)))
    group, d = case["q_heads"] // case["kv_heads"], case["dim"]
    if op == "cache":
        out = torch.empty((case["requests"], case["q_heads"], d), dtype=torch.float64, device="cuda")
        for r, n in enumerate(s["lengths_host"]):
            k, v = _cached_f64(s, r, n)
            for j in range(case["kv_heads"]):
                q = s["q"][r, j * group:(j + 1) * group].double()
                out[r, j * group:(j + 1) * group] = torch.softmax(q @ k[j].T / math.sqrt(d), dim=-1) @ v[j]
        return out
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    offsets = s["offsets"].tolist()
    for a, b in zip(offsets, offsets[1:]):
        for head in range(case["q_heads"]):
            k, v = s["k"][a:b, head // group].double(), s["v"][a:b, head // group].double()
            for r0 in range(a, b, 2048):     # the keys that a block of rows sees
                r1 = min(b, r0 + 2048)
                score = s["q"][r0:r1, head].double() @ k[:r1 - a].T / math.sqrt(d)
                beyond = torch.ones_like(score, dtype=torch.bool).triu(r0 - a + 1)
                score = score.masked_fill(beyond, -math.inf)
                lse[r0:r1, head] = torch.logsumexp(score, dim=-1)
                out[r0:r1, head] = torch.softmax(score, dim=-1) @ v[:r1 - a]
    return (out, lse) if case["lse"] else out
