"""The attention operators without a GPU: refusals at the ends of what they accept."""
import ctypes
import importlib
import math

import pytest
import torch

G = 1 << 30


def test_prompt_attention_fill_refusals(bs):
    """Its flags, and what the form without them refuses; no rows are nothing to fill."""
    att = importlib.import_module("355_1_trans_b200.attention")
    base = dict(q=G, k=2 * G, v=3 * G, out=4 * G, lse=5 * G, offsets=6 * G, q_stride=4096, q_head_stride=128, k_stride=1024,
                k_head_stride=128, v_stride=1024, v_head_stride=128, out_stride=4096, out_head_stride=128, tokens=100,
                tokens_k=100, sequences=3, q_heads=32, heads=8, dim=128, causal=1, scale=0.1)

    def status(fill_out=1, fill_lse=1, **kw):
        return bs.lib().bsgemm_prompt_attention_fill(ctypes.byref(att.PromptAttentionArgs(**{**base, **kw})), fill_out, fill_lse, None)

    assert bs.lib().bsgemm_prompt_attention_fill(None, 1, 1, None) == bs.ERR_INVALID_VALUE
    assert status(fill_out=2) == status(fill_lse=-1) == bs.ERR_INVALID_VALUE
    assert status(sequences=0, out=None) == status(sequences=0, offsets=None) == status(out=G) == bs.ERR_INVALID_VALUE
    assert status(tokens=0, tokens_k=0) == status(0, 0, sequences=0) == status(0, 1, sequences=0, lse=None) == bs.OK


def test_prompt_attention_refuses_sequences_past_its_walk(bs):
    """Each CTA looks at every sequence: more than 2^24 would take longer than its waits."""
    att = importlib.import_module("355_1_trans_b200.attention")
    args = att.PromptAttentionArgs(q=G, k=2 * G, v=3 * G, out=4 * G, offsets=6 * G, q_stride=64, q_head_stride=64, k_stride=64, k_head_stride=64,
                                   v_stride=64, v_head_stride=64, out_stride=64, out_head_stride=64, tokens=100, tokens_k=100,
                                   sequences=(1 << 24) + 1, q_heads=1, heads=1, dim=64, causal=1, scale=0.1)
    assert bs.lib().bsgemm_prompt_attention(ctypes.byref(args), None) == bs.ERR_UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(scaling="yarn", base=1.0), dict(scaling="yarn", base=0.5), dict(scaling="yarn", slow=0.0), dict(scaling="yarn", fast=1.0, slow=1.0), dict(scaling="yarn", fast=1.0, slow=2.0),
    dict(scaling="wavelength", fast=1.0, slow=1.0), dict(scaling="wavelength", fast=2.0, slow=3.0), dict(scaling="wavelength", slow=-1.0),
    dict(scaling="yarn", fast=math.nan), dict(scaling="wavelength", slow=math.nan), dict(scaling="wavelength", fast=math.inf),
    dict(base=math.inf), dict(base=math.nan), dict(scaling="linear", factor=math.inf), dict(scaling="yarn", factor=math.nan),
    dict(scaling="yarn", trained_length=math.inf)])
def test_rotary_plan_refuses_what_has_no_frequencies(bs, kw):
    with pytest.raises(ValueError):
        bs.rotary_plan(64, device="cpu", **kw)


def test_rotary_plan_ends_of_its_ranges(bs):
    """A base of 1 without parts, no slow end of the wavelengths: finite frequencies."""
    assert torch.equal(bs.rotary_plan(8, 1.0, device="cpu").frequencies, torch.ones(4, dtype=torch.float64))
    f = bs.rotary_plan(64, scaling="wavelength", factor=8.0, slow=0.0, device="cpu").frequencies
    plain = bs.rotary_plan(64, device="cpu").frequencies
    assert f.isfinite().all() and (f <= plain).all() and (f >= plain / 8).all()
