"""The attention half of a block as it is served: rotary positions, block tables
and slots from request lengths, a paged cache of keys and values in 4 bits,
attention of single tokens over it, and attention over packed prompts.

A step of a serving loop, prompts and decoded tokens of any requests mixed in
the cache::

    p = paged_slots(cached, new, block_table, free_pages, page_size, tokens)
    q, k = rotary(q, k, p.positions, plan)
    cache_append(cache, k, v, p.slots)
    o = prompt_attention(q, k, v, p.offsets)                       # prompts from their beginning
    o = cache_attention(q, cache, block_table, p.lengths)          # one new token a request

As the operators in ``ops.py``, the functions launch on the current stream,
raise ValueError for a wrong tensor and BsgemmError for a status of the library,
and are no autograd functions; there is no fallback.  Their checks are in
``csrc/binding.cpp``.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from .ops import native

_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong


class RotaryArgs(ctypes.Structure):
    """bsgemm_rotary_args"""
    _fields_ = [(n, _P) for n in ("q", "k", "q_out", "k_out", "positions", "frequencies")] + \
               [(n, _L) for n in ("q_stride", "q_head_stride", "k_stride", "k_head_stride", "q_out_stride",
                                  "q_out_head_stride", "k_out_stride", "k_out_head_stride")] + \
               [(n, _I) for n in ("tokens", "q_heads", "k_heads", "dim", "rot", "dtype", "positions_64", "interleaved",
                                  "inverse")] + [("factor", ctypes.c_float)]


class PagedSlotsArgs(ctypes.Structure):
    """bsgemm_paged_slots_args"""
    _fields_ = [(n, _P) for n in ("cached", "fresh", "block_table", "free_pages", "first_free", "slots", "positions",
                                  "offsets", "lengths", "pages_taken")] + [("table_stride", _L)] + \
               [(n, _I) for n in ("requests", "columns", "free_count", "page", "tokens", "reserved")]


class KvCacheArgs(ctypes.Structure):
    """bsgemm_kv_cache"""
    _fields_ = [(n, _P) for n in ("k", "k_scale", "v", "v_scale")] + [("pages", _L)] + \
               [(n, _I) for n in ("page", "heads", "dim", "reserved")]


class CacheRows(ctypes.Structure):
    """bsgemm_cache_rows"""
    _fields_ = [(n, _P) for n in ("k", "v", "slots")] + \
               [(n, _L) for n in ("k_stride", "k_head_stride", "v_stride", "v_head_stride")] + \
               [("tokens", _I), ("dtype", _I)]


class CacheAttentionArgs(ctypes.Structure):
    """bsgemm_cache_attention_args"""
    _fields_ = [(n, _P) for n in ("q", "out", "block_table", "lengths", "workspace")] + \
               [("workspace_bytes", ctypes.c_size_t)] + \
               [(n, _L) for n in ("q_stride", "q_head_stride", "out_stride", "out_head_stride", "table_stride")] + \
               [("requests", _I), ("q_heads", _I), ("columns", _I), ("scale", ctypes.c_float)]


class PromptAttentionArgs(ctypes.Structure):
    """bsgemm_prompt_attention_args"""
    _fields_ = [(n, _P) for n in ("q", "k", "v", "out", "lse", "offsets", "offsets_k")] + \
               [(n, _L) for n in ("q_stride", "q_head_stride", "k_stride", "k_head_stride", "v_stride", "v_head_stride",
                                  "out_stride", "out_head_stride")] + \
               [(n, _I) for n in ("tokens", "tokens_k", "sequences", "q_heads", "heads", "dim", "causal")] + \
               [("scale", ctypes.c_float)]


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

class RotaryPlan(NamedTuple):
    """frequencies: radians a position of each pair, float64 [rot / 2] on the GPU;
    factor: what cosine and sine are multiplied by."""
    frequencies: torch.Tensor
    factor: float = 1.0


SCALINGS = (None, "linear", "ntk", "yarn", "wavelength")


def rotary_plan(rot: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                trained_length: int = 4096, fast: float | None = None, slow: float | None = None, device="cuda") -> RotaryPlan:
    """The plan of heads whose first `rot` elements turn: base^(-2 i / rot) radians a position.

    scaling stretches it by `factor` for contexts beyond the trained length:
    "linear" divides every frequency; "ntk" raises the base to base *
    factor^(rot / (rot - 2)); "yarn" keeps pairs that turn more than `fast`
    times (32) within trained_length, divides those that turn less than `slow`
    times (1), goes linearly in the pair's index between (NTK by parts), and multiplies cosine
    and sine by 0.1 ln factor + 1; "wavelength" goes linearly in the number of
    turns between `slow` (1) and `fast` (4) instead, without that factor.  fast is above slow."""
    if rot < 2 or rot % 2:
        raise ValueError("rot must be even and at least 2")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if not (0 < base < math.inf and 1 <= factor < math.inf and 0 < trained_length < math.inf):
        raise ValueError("base and trained_length must be positive and finite, factor at least 1")
    if scaling in ("yarn", "wavelength"):
        fast = (32.0 if scaling == "yarn" else 4.0) if fast is None else fast
        slow = 1.0 if slow is None else slow
        if not 0 <= slow < fast < math.inf:
            raise ValueError("fast must be above slow, slow at least 0, both finite")
        if scaling == "yarn" and not (base > 1 and slow > 0):
            raise ValueError("scaling 'yarn' needs a base above 1 and slow above 0")
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk":
        if rot == 2:
            raise ValueError("scaling 'ntk' needs more than one pair")
        base = base * factor ** (rot / (rot - 2))
    f = torch.tensor(float(base), dtype=torch.float64) ** (-2 * i / rot)
    by = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair(turns):
            return rot * math.log(trained_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
        stretch = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - stretch) + f / factor * stretch
        by = 0.1 * math.log(factor) + 1
    elif scaling == "wavelength":
        keep = ((trained_length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return RotaryPlan(f.to(device), by)


def rotary(q, k, positions, plan: RotaryPlan, *, interleaved: bool = False, inverse: bool = False, out=None):
    """(q, k) with the first rot elements of each head turned by position * frequency.

    q [tokens, heads, dim] and k (its own heads, or None) bf16 or fp32, any
    strides with a unit inner one; positions [tokens] int32 or int64.  Pairs are
    (i, i + rot / 2), or (2 i, 2 i + 1) where interleaved; elements behind rot pass
    through.  inverse turns back: applied to the gradients of the results it gives
    those of q and k.  Angles are exact to 2^-24 of a turn at any position, to
    the ends of int64 (frequencies up to 64).  out: (q, k)
    to write, which may be the inputs themselves; q and k may be parts of one buffer."""
    oq, ok = (None, None) if out is None else out
    return native().rotary(q, k, positions, plan.frequencies, plan.factor, bool(interleaved), bool(inverse), oq, ok)


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------

class PagedSlots(NamedTuple):
    slots: torch.Tensor          # int64 [tokens]: page * page_size + row, -1 without one
    positions: torch.Tensor      # int32 [tokens]
    offsets: torch.Tensor        # int32 [requests + 1]: first token of each request
    lengths: torch.Tensor        # int32 [requests]: cached + new
    pages_taken: torch.Tensor    # int32 [1]


def paged_slots(cached, new, block_table, free_pages, page_size: int, tokens: int, *, first_free=None) -> PagedSlots:
    """Block tables and slots of a step's tokens from the requests' lengths, in one launch without the host.

    cached and new [requests] int32: tokens in the cache and to come.  A request's
    first ceil(cached / page_size) entries of block_table [requests, columns]
    int32 are its pages so far; the pages that its new tokens begin are taken from
    free_pages int32, from first_free (int32 [1] on the GPU, default 0) on, in the
    order of the requests, and written to the table.  tokens is the size of the
    results: the sum of new or more; tokens behind the last request's have
    slot -1 and position 0.  Where free_pages or the table's row do not reach, the
    entry and the slots are -1, and pages_taken says what the step asked for."""
    return PagedSlots(*native().paged_slots(cached, new, block_table, free_pages, page_size, tokens, first_free))


class KvCache(NamedTuple):
    """Keys and values of `pages` pages in MXFP4 (include/bsgemm_b200.h says how they lie); uint8, contiguous."""
    k: torch.Tensor          # [pages, heads, page_size, dim / 2]
    k_scale: torch.Tensor    # [pages, heads, page_size, dim / 32]
    v: torch.Tensor          # [pages, heads, page_size / 4, dim / 2, 4]
    v_scale: torch.Tensor    # [pages, heads, page_size / 4, dim / 32, 4]


def new_kv_cache(pages: int, page_size: int, heads: int, dim: int, *, device="cuda") -> KvCache:
    """A cache of zeros: heads of 64 or 128 elements, pages of 16, 32, 64, 128 or 256 tokens."""
    if dim not in (64, 128) or page_size not in (16, 32, 64, 128, 256):
        raise ValueError("dim must be 64 or 128, page_size 16, 32, 64, 128 or 256")
    shapes = ((page_size, dim // 2), (page_size, dim // 32), (page_size // 4, dim // 2, 4), (page_size // 4, dim // 32, 4))
    return KvCache(*(torch.zeros((pages, heads, *s), dtype=torch.uint8, device=device) for s in shapes))


def cache_append(cache: KvCache, k, v, slots) -> None:
    """Quantises k and v [tokens, heads, dim] (bf16 or fp32, copied first where they
    lie off 16 bytes) into the cache at slots (int64, distinct), as quantize does for
    "mxfp4"; tokens whose slot is -1 or past the cache are left out."""
    native().cache_append(*cache, k, v, slots)


def cache_read(cache: KvCache, slots):
    """(k, v) [tokens, heads, dim] bf16: the values that the cache holds at slots, zeros where a slot is -1 or past it."""
    return native().cache_read(*cache, slots)


def cache_attention(q, cache: KvCache, block_table, lengths, *, scale: float | None = None, out=None, workspace=None):
    """softmax(scale q K^T) V of one query token a request over its cached tokens.

    q [requests, q_heads, dim] bf16 (copied first where it lies off 16 bytes), q_heads a
    multiple of the cache's heads: head h reads the cache's head h / (q_heads / heads).  Request r
    has lengths[r] tokens (int32) on the pages block_table[r, 0 ..]; one of length 0 gets zeros.
    scale: dim^-1/2, or a positive number.  Sums are fp32; the weights are rounded
    to fp16 before they meet the values (bf16 beside values whose scales are outside 2^-14 .. 2^13 and keys
    whose scales are 2^97 or more; a scale byte of 0 counts as 0).
    Tokens on pages outside the cache do not count.  The same inputs give the same bits.  workspace:
    bsgemm_cache_attention_workspace_size bytes, allocated when omitted; calls that
    may run at the same time must not share one."""
    return native().cache_attention(q, *cache, block_table, lengths, scale, out, workspace)


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------

def prompt_attention(q, k, v, offsets, *, offsets_k=None, causal: bool = True, scale: float | None = None, out=None,
                     return_lse: bool = False):
    """softmax(scale q K^T) V over packed sequences of any lengths.

    q [tokens, q_heads, dim], k and v [tokens_k, heads, dim] bf16 (copied first
    where they lie off 16 bytes), dim a multiple of 8 up to 128, q_heads a multiple of heads.
    Sequence i has the rows offsets[i] .. offsets[i + 1] (int32 [sequences + 1] on the GPU) of q,
    and those of offsets_k (default: the same) of k and v.  causal: its last query row
    sees all its keys, each row before it one fewer.  A row that sees none gets zeros.
    Rows outside every sequence are zeros (lse: -inf), but a caller's out is left as it is there.  Sums are fp32;
    the weights are rounded to bf16 before they meet the values, which must be finite (keys need not be where
    no row sees them).  return_lse: (out, lse), lse fp32 [tokens, q_heads] the
    logarithm of the sum of exp(scale q k), -inf for a row without keys.  No
    gradients: this is the attention of serving."""
    return native().prompt_attention(q, k, v, offsets, offsets_k, bool(causal), scale, out, bool(return_lse))
