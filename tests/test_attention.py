"""The attention operators without a GPU: what their entry points refuse before
any CUDA call, the argument structs, the frequencies of rotary plans."""
import ctypes
import importlib
import math
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
G = 1 << 30


@pytest.fixture(scope="module")
def att(bs):
    return importlib.import_module("355_1_trans_b200.attention")


@pytest.mark.parametrize("struct", ["RotaryArgs", "PagedSlotsArgs", "KvCacheArgs", "CacheRows", "CacheAttentionArgs",
                                    "PromptAttentionArgs"])
def test_structs_match_the_header(att, struct):
    """Field names and order as in include/bsgemm_b200.h."""
    cls = getattr(att, struct)
    name = cls.__doc__.strip()
    text = (ROOT / "include" / "bsgemm_b200.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    assert re.findall(r"(\w+)\s*;", body) == [f for f, _ in cls._fields_]


def filled(cls, base, changes):
    a = cls(**base)
    for key, value in changes.items():
        setattr(a, key, value)
    return ctypes.byref(a)


def test_rotary_refusals(bs, att):
    base = dict(q=G, k=2 * G, q_out=3 * G, k_out=4 * G, positions=5 * G, frequencies=6 * G, q_stride=4096, q_head_stride=128,
                k_stride=1024, k_head_stride=128, q_out_stride=4096, q_out_head_stride=128, k_out_stride=1024,
                k_out_head_stride=128, tokens=10, q_heads=32, k_heads=8, dim=128, rot=128, factor=1.0)

    def status(**kw):
        return bs.lib().bsgemm_rotary(filled(att.RotaryArgs, base, kw), None)

    assert bs.lib().bsgemm_rotary(None, None) == bs.ERR_INVALID_VALUE
    for kw in ({"tokens": -1}, {"q_heads": -1}, {"dim": 0}, {"rot": 0}, {"rot": 3}, {"rot": 130}, {"dtype": 2}, {"positions_64": 2},
               {"interleaved": -1}, {"inverse": 2}, {"factor": math.inf}, {"factor": math.nan}, {"q": None}, {"k_out": None},
               {"positions": None}, {"frequencies": None}, {"q_stride": -4096}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    assert status(dim=1024, rot=1024) == bs.ERR_UNSUPPORTED
    for kw in ({"q": G + 1}, {"positions": 5 * G + 2}, {"positions_64": 1, "positions": 5 * G + 4}, {"frequencies": 6 * G + 4}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw
    # outputs over inputs, each other or themselves
    for kw in ({"q_out": G + 256}, {"q_out": 2 * G}, {"k_out": 3 * G + 128}, {"q_out_stride": 128}, {"q_out_head_stride": 64},
               {"q_out": 5 * G}, {"q_out": G, "q_out_stride": 8192}, {"k_out": 6 * G}, {"k": G, "k_out": G}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    assert status(tokens=0) == bs.OK and status(q_heads=0, k_heads=0) == bs.OK


def test_rotary_takes_parts_of_one_buffer(bs, att):
    """Queries and keys of a joint projection, in place: as far as the device check, and not refused for overlap."""
    base = dict(positions=5 * G, frequencies=6 * G, tokens=10, q_heads=32, k_heads=8, dim=128, rot=128, factor=1.0)
    joint = dict(base, q=G, q_out=G, k=G + 4096 * 2, k_out=G + 4096 * 2, q_stride=6144, k_stride=6144, q_out_stride=6144,
                 k_out_stride=6144, q_head_stride=128, k_head_stride=128, q_out_head_stride=128, k_out_head_stride=128)
    by_head = dict(base, q_heads=8, q=G, q_out=G, k=G + 256, k_out=G + 256, q_stride=8 * 384, k_stride=8 * 384, q_out_stride=8 * 384,
                   k_out_stride=8 * 384, q_head_stride=384, k_head_stride=384, q_out_head_stride=384, k_out_head_stride=384)
    for args in (joint, by_head):
        assert bs.lib().bsgemm_rotary(filled(att.RotaryArgs, args, {}), None) in (bs.ERR_CUDA, bs.ERR_ARCH) \
            if not torch.cuda.is_available() else True
    wide = dict(joint, k=G + 4000 * 2, k_out=G + 4000 * 2)
    assert bs.lib().bsgemm_rotary(filled(att.RotaryArgs, wide, {}), None) == bs.ERR_INVALID_VALUE


def test_paged_slots_refusals(bs, att):
    base = dict(cached=G, fresh=2 * G, block_table=3 * G, free_pages=4 * G, first_free=5 * G, slots=6 * G, positions=7 * G,
                offsets=8 * G, lengths=9 * G, pages_taken=10 * G, table_stride=64, requests=16, columns=64, free_count=100,
                page=64, tokens=500)

    def status(**kw):
        return bs.lib().bsgemm_paged_slots(filled(att.PagedSlotsArgs, base, kw), None)

    assert bs.lib().bsgemm_paged_slots(None, None) == bs.ERR_INVALID_VALUE
    for kw in ({"requests": -1}, {"columns": -1}, {"free_count": -1}, {"page": 0}, {"tokens": -1}, {"table_stride": 63},
               {"offsets": None}, {"pages_taken": None}, {"cached": None}, {"fresh": None}, {"slots": None}, {"positions": None},
               {"block_table": None}, {"free_pages": None}, {"lengths": None}, {"slots": 3 * G + 8}, {"lengths": G},
               {"block_table": 4 * G}, {"positions": 6 * G + 64}, {"pages_taken": 5 * G}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    for kw in ({"cached": G + 2}, {"slots": 6 * G + 4}, {"pages_taken": 10 * G + 1}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw
    assert status(requests=1 << 25, columns=1, table_stride=1) == bs.ERR_UNSUPPORTED


CACHE = dict(k=G, k_scale=2 * G, v=3 * G, v_scale=4 * G, pages=100, page=64, heads=8, dim=128)


@pytest.mark.parametrize("entry", ["bsgemm_cache_append", "bsgemm_cache_read", "bsgemm_cache_attention"])
def test_cache_refusals(bs, att, entry):
    """The cache's own description, the same in all three."""
    args = {"bsgemm_cache_attention": att.CacheAttentionArgs}.get(entry, att.CacheRows)()

    def status(**kw):
        return getattr(bs.lib(), entry)(filled(att.KvCacheArgs, CACHE, kw), ctypes.byref(args), None)

    assert getattr(bs.lib(), entry)(None, ctypes.byref(args), None) == bs.ERR_INVALID_VALUE
    assert getattr(bs.lib(), entry)(filled(att.KvCacheArgs, CACHE, {}), None, None) == bs.ERR_INVALID_VALUE
    for kw in ({"pages": -1}, {"page": 0}, {"heads": 0}, {"dim": 0}, {"k": None}, {"v_scale": None}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    for kw in ({"dim": 96}, {"dim": 256}, {"page": 8}, {"page": 48}, {"page": 512}):
        assert status(**kw) == bs.ERR_UNSUPPORTED, kw
    for kw in ({"k": G + 8}, {"k_scale": 2 * G + 4}, {"v": 3 * G + 1}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw


@pytest.mark.parametrize("append", [True, False])
def test_cache_rows_refusals(bs, att, append):
    base = dict(k=6 * G, v=7 * G, slots=8 * G, k_stride=1024, k_head_stride=128, v_stride=1024, v_head_stride=128, tokens=10)
    fn = bs.lib().bsgemm_cache_append if append else bs.lib().bsgemm_cache_read

    def status(**kw):
        return fn(filled(att.KvCacheArgs, CACHE, {}), filled(att.CacheRows, base, kw), None)

    for kw in ({"tokens": -1}, {"dtype": 2}, {"k": None}, {"v": None}, {"slots": None}, {"k_stride": -8}, {"k": G + 1024},
               {"v": 3 * G}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    for kw in ({"k": 6 * G + 8}, {"k_stride": 1028}, {"v_head_stride": 132}, {"slots": 8 * G + 4}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw
    assert status(tokens=0) == bs.OK
    if not append:
        assert status(dtype=1) == bs.ERR_UNSUPPORTED
        assert status(v=6 * G + 64) == bs.ERR_INVALID_VALUE
        assert status(k_head_stride=64) == bs.ERR_INVALID_VALUE


def test_cache_attention_refusals(bs, att):
    base = dict(q=6 * G, out=7 * G, block_table=8 * G, lengths=9 * G, workspace=10 * G, workspace_bytes=1 << 29, q_stride=4096,
                q_head_stride=128, out_stride=4096, out_head_stride=128, table_stride=32, requests=4, q_heads=32, columns=32,
                scale=0.1)

    def status(**kw):
        return bs.lib().bsgemm_cache_attention(filled(att.KvCacheArgs, CACHE, {}), filled(att.CacheAttentionArgs, base, kw), None)

    for kw in ({"requests": -1}, {"columns": -1}, {"q_heads": 0}, {"q_heads": 30}, {"scale": 0.0}, {"scale": -1.0},
               {"scale": math.nan}, {"scale": math.inf}, {"q": None}, {"out": None}, {"lengths": None}, {"block_table": None},
               {"table_stride": 31}, {"out_head_stride": 64}, {"out_stride": 128}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    for kw in ({"q": 6 * G + 8}, {"q_stride": 4100}, {"q_head_stride": 132}, {"out": 7 * G + 1}, {"lengths": 9 * G + 1}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw
    assert status(requests=0) == bs.OK


def test_prompt_attention_refusals(bs, att):
    base = dict(q=G, k=2 * G, v=3 * G, out=4 * G, lse=5 * G, offsets=6 * G, q_stride=4096, q_head_stride=128, k_stride=1024,
                k_head_stride=128, v_stride=1024, v_head_stride=128, out_stride=4096, out_head_stride=128, tokens=100,
                tokens_k=100, sequences=3, q_heads=32, heads=8, dim=128, causal=1, scale=0.1)

    def status(**kw):
        return bs.lib().bsgemm_prompt_attention(filled(att.PromptAttentionArgs, base, kw), None)

    assert bs.lib().bsgemm_prompt_attention(None, None) == bs.ERR_INVALID_VALUE
    for kw in ({"tokens": -1}, {"tokens_k": 99}, {"sequences": -1}, {"q_heads": 30}, {"heads": 0}, {"dim": 0}, {"causal": 2},
               {"scale": 0.0}, {"scale": math.nan}, {"q": None}, {"k": None}, {"v": None}, {"out": None}, {"offsets": None},
               {"q_stride": -8}, {"out": G}, {"out": 2 * G + 1024}, {"out": 3 * G}, {"out": 6 * G}, {"lse": G}, {"lse": 4 * G},
               {"out_stride": 2048}, {"out_head_stride": 120}):
        assert status(**kw) == bs.ERR_INVALID_VALUE, kw
    for kw in ({"dim": 132, "q_head_stride": 136}, {"dim": 256}, {"dim": 100}, {"q_heads": 8 * 136}):
        assert status(**kw) == bs.ERR_UNSUPPORTED, kw
    for kw in ({"q": G + 8}, {"k": 2 * G + 2}, {"q_stride": 4100}, {"v_head_stride": 132}, {"k_stride": 0}, {"k_head_stride": 0},
               {"offsets": 6 * G + 2}, {"lse": 5 * G + 2}, {"out_stride": 4100}):
        assert status(**kw) == bs.ERR_ALIGNMENT, kw
    assert status(tokens=0, tokens_k=0) == bs.OK and status(sequences=0) == bs.OK


def test_python_refuses_tensors_off_the_gpu(bs):
    x = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    cache = bs.new_kv_cache(2, 16, 8, 64, device="cpu")
    plan = bs.rotary_plan(64, device="cpu")
    for call in (lambda: bs.rotary(x, x, i, plan), lambda: bs.paged_slots(i, i, i[None], i, 16, 4),
                 lambda: bs.cache_append(cache, x, x, i.long()), lambda: bs.cache_read(cache, i.long()),
                 lambda: bs.cache_attention(x, cache, i[:, None], i), lambda: bs.prompt_attention(x, x, x, i)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        bs.prompt_attention(1, x, x, i)
    for kw in (dict(dim=96), dict(page_size=8), dict(page_size=24)):
        with pytest.raises(ValueError):
            bs.new_kv_cache(**{**dict(pages=2, page_size=16, heads=1, dim=64, device="cpu"), **kw})


# ---- rotary plans -------------------------------------------------------------------

def test_rotary_plan_frequencies(bs):
    f, by = bs.rotary_plan(8, 10000.0, device="cpu")
    assert by == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(bs.rotary_plan(8, scaling="linear", factor=4.0, device="cpu").frequencies, f / 4)
    ntk = bs.rotary_plan(8, scaling="ntk", factor=4.0, device="cpu").frequencies
    assert ntk[0] == 1.0 and abs(ntk[3] / (f[3] / 4) - 1) < 1e-13      # the slowest pair is divided by the factor


@pytest.mark.parametrize("scaling", ["yarn", "wavelength"])
def test_rotary_plan_by_parts(bs, scaling):
    """Fast pairs keep their frequency, slow ones are divided, those between lie between and in order."""
    rot, factor, trained = 128, 16.0, 4096
    plain = bs.rotary_plan(rot, 500000.0, device="cpu").frequencies
    f, by = bs.rotary_plan(rot, 500000.0, scaling=scaling, factor=factor, trained_length=trained, device="cpu")
    turns = trained * plain / (2 * math.pi)
    fast, slow = (32, 1) if scaling == "yarn" else (4, 1)
    ratio = plain / f
    assert (ratio[turns > 1.3 * fast] == 1).all()
    assert torch.allclose(ratio[turns < slow / 1.3], torch.tensor(factor, dtype=torch.float64), rtol=1e-12)
    assert (ratio.diff() >= -1e-12).all() and ((ratio > 1.01) & (ratio < factor * 0.99)).sum() > 2
    assert by == (pytest.approx(0.1 * math.log(factor) + 1) if scaling == "yarn" else 1.0)


def test_rotary_plan_refusals(bs):
    for args, kw in (((7,), {}), ((0,), {}), ((8, -1.0), {}), ((8,), {"scaling": "other"}), ((8,), {"scaling": "linear", "factor": 0.5}),
                     ((2,), {"scaling": "ntk", "factor": 2.0}), ((8,), {"trained_length": 0, "scaling": "yarn"})):
        with pytest.raises(ValueError):
            bs.rotary_plan(*args, device="cpu", **kw)


def test_rotary_refuses_tokens_past_32_bits(bs, att):
    """Elements of one token's heads are counted in 32 bits."""
    base = dict(q=G, q_out=1 << 50, positions=1 << 49, frequencies=1 << 48, q_stride=1 << 33, q_head_stride=1 << 12,
                q_out_stride=1 << 33, q_out_head_stride=1 << 12, tokens=1, q_heads=1 << 20, dim=1 << 12, rot=64, factor=1.0)
    assert bs.lib().bsgemm_rotary(filled(att.RotaryArgs, base, {}), None) == bs.ERR_UNSUPPORTED
    if not torch.cuda.is_available():
        assert bs.lib().bsgemm_rotary(filled(att.RotaryArgs, base, {"q_heads": 1 << 17}), None) in (bs.ERR_CUDA, bs.ERR_ARCH)
