"""The append kernel that brings groups of tokens through shared memory, with every option that a prefill uses, and borders that fit nothing."""

import pytest
import torch

from sample_efficient_gpt_b200 import ops

from tests.paged_cases import append_oracle
from tests.test_gpu_paged import _clean_status, append_case, check_append, i32, one, run_append, take_status  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu

# query heads, kv heads, dims, tokens: beyond four CTAs' items an SM (148 * 4 * 256 pieces of 16 elements); 8, 16, 2 and 1 tokens a stage
MANY = [(18, 6, 64, 1400), (8, 8, 32, 3300), (32, 8, 128, 450), (96, 16, 128, 160)]


def ragged(tokens):
    new = [tokens // 2, 1, 0, tokens // 3, 5, 0]
    return new + [tokens - sum(new)], [0, 5, 100, 2, 31, 0, 63], [0, 7, 0, 300, 1, 2, 1000]


@pytest.mark.parametrize("H,Hkv,hd,tokens", MANY)
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("qknorm", [True, False])
@pytest.mark.parametrize("P,layout,base", [(64, "head", False), (24, "token", True)])
def test_many_tokens(H, Hkv, hd, tokens, first, qknorm, P, layout, base):
    assert tokens * (H + 2 * Hkv) * (hd // 16) > 148 * 4 * 256
    new, past, bases = ragged(tokens)
    bases = bases if base else None
    c = append_case(new, past, H, Hkv, hd, P, layout, first=first, pad=24, base=bases, behind=3, seed=tokens)
    out = run_append(c, H, Hkv, hd, qknorm, want_k=True, want_v=True)
    check_append(c, out, new, past, H, Hkv, hd, P, qknorm, bases)


@pytest.mark.parametrize("want_k,want_v", [(True, False), (False, True), (False, False)])
def test_many_tokens_with_fewer_results(want_k, want_v):
    H, Hkv, hd, tokens = MANY[0]
    new, past, _ = ragged(tokens)
    c = append_case(new, past, H, Hkv, hd, 16, "head", first=want_v)
    out = run_append(c, H, Hkv, hd, want_k=want_k, want_v=want_v)
    assert (out[1] is not None) == want_k and (out[2] is not None) == want_v
    check_append(c, out, new, past, H, Hkv, hd, 16, True)


@pytest.mark.parametrize("H,Hkv,hd,tokens", MANY)
def test_many_sequences_of_one_token(H, Hkv, hd, tokens):
    past = [(7 * b) % 50 for b in range(tokens)]
    c = append_case([1] * tokens, past, H, Hkv, hd, 16, "token", pad=24)
    check_append(c, run_append(c, H, Hkv, hd, cu=False), [1] * tokens, past, H, Hkv, hd, 16, True)


@pytest.mark.parametrize("H,Hkv,hd,tokens", [(4, 2, 64, 7), *MANY])
def test_borders_that_reach_outside(H, Hkv, hd, tokens):
    """Cumulative rows from before the first to far behind the last row: rows that exist go to the place that the borders give them, or
    nowhere where the page table has none for it; nothing else is touched."""
    c = append_case([tokens, 0, 30], [0, 0, 10], H, Hkv, hd, 16, "token", first=True)
    T, P, width = tokens + 30, 16, c["page_table"].size(1)
    pages = c["k_pages"].size(0)
    c["page_table"][:] = -1
    need = [2, 1, 3]  # pages that each sequence has
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    at = 0
    for b, n in enumerate(need):
        c["page_table"][b, :n] = i32(order[at : at + n])
        at += n
    c["seq_lens"][:] = i32([3, 0, 10])
    cu = [-5, 1, 2, 10**9]
    c["cu"][:] = i32(cu)
    q, k, v = run_append(c, H, Hkv, hd, want_k=True, want_v=True)
    code = take_status()
    place = {}  # row -> (sequence, position)
    for t in range(T):
        b = max(i for i in range(3) if cu[i] <= t)
        pos = [3, 0, 10][b] + t - cu[b]
        if pos < need[b] * P and pos < c["cos"].size(0):
            place[t] = (b, pos)
    assert 0 < len(place) < T and code in ((51, 52) if T > len(place) else (0,)) and width >= 3
    rows = sorted(place)
    pos = torch.tensor([place[t][1] for t in rows])
    seq = torch.tensor([place[t][0] for t in rows])
    want = append_oracle(c["qkv"][rows], None, c["cos"], c["sin"], one(1.3), one(0.8), one(0.35), one(1.1), H, Hkv, hd, True, pos)
    slot = (c["page_table"].cpu().long()[seq, pos // P], pos % P)
    kp, vp = c["k_pages"].cpu(), c["v_pages"].cpu()
    for got, w in ((q.cpu()[rows], want[0]), (k.cpu()[rows], want[1]), (v.cpu()[rows], want[2]), (kp[slot], want[1]), (vp[slot], want[2])):
        # one rounding to bf16 and fp32 arithmetic before it, as for all of this kernel's results
        assert ((got.double() - w).abs() <= 2.0**-8 * w.abs() + 2.0**-20 * w.abs().amax(-1, keepdim=True)).all()
    gone = torch.ones(T, dtype=torch.bool)
    gone[rows] = False
    assert (q.cpu()[gone] == 0).all() and (k.cpu()[gone] == 0).all() and (v.cpu()[gone] == 0).all()
    written = torch.zeros(kp.shape[:2], dtype=torch.bool)
    written[slot] = True
    for pool in (kp, vp):
        assert torch.equal(torch.isfinite(pool).all(-1).all(-1), written)


def test_a_long_prefill_leaves_out_what_does_not_fit():
    """The ring goes on over tokens without a place: a page outside the pool, lengths beyond the table, and none of a group's tokens."""
    H, Hkv, hd, tokens = MANY[0]
    new, past = [tokens, 64, 64], [0, 5, 3]
    c = append_case(new, past, H, Hkv, hd, 16, "head", first=False)
    good = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    want = run_append(good, H, Hkv, hd, want_k=True, want_v=True)
    c["page_table"][0, 2:40] = c["k_pages"].size(0) + 7
    c["seq_lens"][1] = -1
    got = run_append(c, H, Hkv, hd, want_k=True, want_v=True)
    assert take_status() in (51, 52)
    out = torch.zeros(sum(new), dtype=torch.bool, device=c["qkv"].device)
    out[32:640], out[tokens : tokens + 64] = True, True
    for a, b in zip(got, want):
        assert torch.equal(a[~out], b[~out]) and (a[out] == 0).all()
    assert ops.has_kernel("paged_append")
