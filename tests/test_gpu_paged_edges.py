"""The paged serving kernels where their numbers leave the ordinary: single keys of NaN and infinity, scores beyond what fp32 resolves."""

import math

import pytest
import torch

from tests.paged_cases import attention_oracle, cache_case, check_attention, fill
from tests.test_gpu_paged import _clean_status, prefix_room, run_attention  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


# 4, 30 and 90 sequences of 3 query heads a kv head, prefixes of 300 tokens: 16 rows at a time, the keys in two halves, 256 rows
@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B,H,Hkv,hd", [(4, 6, 2, 64), (30, 6, 2, 64), (90, 6, 2, 64), (30, 8, 2, 128)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_one_key_that_is_no_number(B, H, Hkv, hd, value):
    """A key with a NaN makes every row of its kv head NaN, wherever in a tile it lies (the first keys, a later full tile, the last,
    partial one); one with an infinity makes those NaN whose query has the component's sign, and is passed over by the others."""
    c = cache_case([5] * B, H, Hkv, hd, 16, prefix_lens=[300], seed=B)
    gqa, keys = H // Hkv, c["ks"][B].clone()
    c["q"][:, :, 3] += torch.where(c["q"][:, :, 3] < 0, -0.1, 0.1).bfloat16()  # no zeros
    up = c["q"][:, :gqa, 3] > 0
    for at in [*range(8), *range(136, 144), 255, 256, 298, 299]:
        k = keys.clone()
        k[at, 0, 3] = value
        fill(c["k_pages"], c["prefix_table"], [300], [k])
        o, lse = (t.cpu() for t in run_attention(c))
        bad = torch.ones_like(up) if math.isnan(value) else up
        assert torch.equal(torch.isnan(o[:, :gqa]).all(-1), bad) and torch.equal(torch.isnan(lse[:, :gqa]), bad), at
        assert torch.isfinite(o[:, gqa:]).all() and torch.isfinite(o[:, :gqa][~bad]).all()
    if math.isinf(value):  # at the last position above: rows that pass the key over see the other 299
        want = attention_oracle(c["q"], c["ks"][:B] + [keys[:299]], c["vs"][:B] + [c["vs"][B][:299]], [0] * B)
        rows = torch.zeros(B, H, dtype=torch.bool)
        rows[:, :gqa] = ~up
        check_attention(o[rows], lse[rows], tuple(t[rows] for t in want), hd)
