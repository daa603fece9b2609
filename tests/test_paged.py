"""CPU statements of the paged serving operators (ops/reference.py) against 64-bit oracles, and their refusals."""

import pytest
import torch

from sample_efficient_gpt_b200 import ops
from sample_efficient_gpt_b200.models.rope import rope_tables

from tests.paged_cases import append_oracle, attention_oracle, cache_case, check_attention, logits_oracle, make_pool, make_tables


@pytest.mark.parametrize("P", [1, 5, 16])
def test_append_cpu(P):
    torch.manual_seed(P)
    H, Hkv, hd, new, past = 4, 2, 32, [3, 0, 7, 1], [0, 4, 9, 2]
    cos, sin = rope_tables(64, 10000, hd)
    total = [a + b for a, b in zip(new, past)]
    table, used = make_tables(total, P, torch.randperm(60).tolist())
    kp, vp = make_pool(60, P, Hkv, hd, dtype=torch.float32), make_pool(60, P, Hkv, hd, "head", dtype=torch.float32)
    T = sum(new) + 2  # two rows behind the last sequence
    qkv, v1 = torch.randn(T, (H + 2 * Hkv) * hd), torch.randn(T, Hkv, hd)
    one = lambda v: torch.tensor([v])  # noqa: E731
    cu = torch.tensor([0, 3, 3, 10, 11], dtype=torch.int32)
    base = torch.tensor([5, 0, 1, 7], dtype=torch.int32)
    q, k, v = ops.qkv_post_paged(qkv, v1, cos, sin, one(1.2), one(0.8), one(0.3), one(1.1), H, Hkv, hd, True, kp, vp, table,
                                 torch.tensor(past, dtype=torch.int32), cu, base, want_k=True, want_v=True)
    seq = [b for b in range(4) for _ in range(new[b])]
    own = torch.tensor([past[b] + i for b in range(4) for i in range(new[b])])
    qo, ko, vo = append_oracle(qkv[:11], v1[:11], cos, sin, 1.2, 0.8, 0.3, 1.1, H, Hkv, hd, True, own + base.long()[seq])
    for got, want in ((q, qo), (k, ko), (v, vo)):
        assert torch.allclose(got[:11].double(), want, atol=2e-6, rtol=2e-6) and (got[11:] == 0).all()
    at = (table.long()[seq, own // P], own % P)
    assert torch.equal(kp[at], k[:11]) and torch.equal(vp[at], v[:11])
    assert int(torch.isfinite(kp).all(-1).all(-1).sum()) == 11  # nothing else was written
    with pytest.raises(ValueError, match="page table"):
        ops.qkv_post_paged(qkv, v1, cos, sin, one(1.2), one(0.8), one(0.3), one(1.1), H, Hkv, hd, True, kp, vp, table, torch.tensor([0, 4, 60, 2]), cu)
    with pytest.raises(ValueError, match="page numbers"):
        ops.qkv_post_paged(qkv, v1, cos, sin, one(1.2), one(0.8), one(0.3), one(1.1), H, Hkv, hd, True, kp, vp, table.clone().fill_(60),
                           torch.tensor(past), cu)
    with pytest.raises(ValueError, match="one token"):
        ops.qkv_post_paged(qkv, v1, cos, sin, one(1.2), one(0.8), one(0.3), one(1.1), H, Hkv, hd, True, kp, vp, table, torch.tensor(past))


@pytest.mark.parametrize("P,layout", [(1, "token"), (7, "head"), (16, "token")])
def test_attention_cpu(P, layout):
    lens, plens, rows = [1, 0, 33, 16, 0, 5], [20, 0, 9], torch.tensor([0, 3, 4, 6], dtype=torch.int32)
    c = cache_case(lens, 6, 2, 32, P, layout, plens, seed=P)
    args = (c["q"], c["k_pages"], c["v_pages"], c["page_table"], c["seq_lens"])
    o, lse = ops.paged_attention(*args, c["prefix_table"], c["prefix_lens"], rows)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [0, 0, 0, 1, 2, 2]), 32)
    o, lse = ops.paged_attention(*args)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"]), 32)
    assert (o[1] == 0).all() and torch.isinf(lse[1]).all()  # a row that sees nothing
    with pytest.raises(ValueError, match="does not fit"):
        ops.paged_attention(*args[:4], c["seq_lens"] + 1000)
    with pytest.raises(ValueError, match="ascend"):
        ops.paged_attention(*args, c["prefix_table"], c["prefix_lens"], torch.tensor([0, 4, 3, 6]))
    with pytest.raises(ValueError, match="page numbers"):
        ops.paged_attention(*args[:3], torch.full_like(c["page_table"], -1), c["seq_lens"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_cpu(dtype):
    torch.manual_seed(2)
    B, V, L = 4, 77, 12
    x = (torch.randn(B, V) * 3).to(dtype)
    tokens = torch.randint(-1, V + 1, (B, L))
    lens, prompts = torch.tensor([12, 0, 1, 9], dtype=torch.int32), torch.tensor([5, 3, 0, 20], dtype=torch.int32)
    rep, pres, freq = torch.tensor([1.3, 0.8, 1.0, 2.0]), torch.tensor([0.4, 0.1, -0.2, 0.3]), torch.tensor([0.2, 0.0, 0.1, -0.1])
    ids = torch.tensor([[3, 3, -1], [V, 0, 1], [5, 6, 5], [-7, -1, -1]], dtype=torch.int32)
    bias = torch.randn(B, 3)
    mask = torch.randint(-2**31, 2**31, (2, 3), dtype=torch.int64).int()
    mask[1] = 0
    rows = torch.tensor([0, 1, -1, 0], dtype=torch.int32)
    y = ops.process_logits(x, tokens, prompts, lens, rep, pres, freq, ids, bias, mask, rows)
    want, mag = logits_oracle(x, tokens, prompts, lens, rep, pres, freq, ids, bias, mask, rows)
    assert torch.equal(torch.isfinite(y), torch.isfinite(want)) and (y[1] == -float("inf")).all()
    fine = torch.isfinite(want)
    assert ((y.double() - want).abs()[fine] <= (2.0**-22 * mag + (2.0**-8 * want.abs() if dtype == torch.bfloat16 else 0))[fine]).all()
    z = x.clone()
    assert ops.process_logits(z, tokens, prompts, lens, rep, pres, freq, ids, bias, mask, rows, out=z) is z and torch.equal(z, y)
    with pytest.raises(ValueError, match="history length"):
        ops.process_logits(x, tokens, prompts, lens + 1)
    with pytest.raises(ValueError, match="mask rows"):
        ops.process_logits(x, mask=mask, mask_rows=rows + 1)
