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
