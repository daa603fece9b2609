"""The paged serving kernels where their numbers leave the ordinary: single keys of NaN and infinity, scores beyond what fp32 resolves."""

import math

import pytest
import torch

from sample_efficient_gpt_b200 import ops

from tests.paged_cases import attention_oracle, cache_case, check_attention, fill, make_pool, make_tables
from tests.test_gpu_paged import DEV, _clean_status, i32, prefix_room, run_attention, to_dev  # noqa: F401  (fixtures)

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


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B,H,Hkv,hd", [(4, 6, 2, 64), (30, 6, 2, 64), (90, 6, 2, 64), (30, 8, 2, 128), (4, 4, 2, 32)])
@pytest.mark.parametrize("scale", [1e7, 1e8, 1e10, 1e13])
def test_scores_beyond_their_own_rounding(B, H, Hkv, hd, scale):
    """Finite scores of 1e8 to 1e15 differ by more than the rounding of any of them, so each row is its best key's value - which
    lies in several places, so that several tiles hold it."""
    c = cache_case([40] * B, H, Hkv, hd, 16, prefix_lens=[700], seed=B)
    for b in range(B):  # own keys that are the prefix's: the maximum again, in another part and another tile
        c["ks"][b], c["vs"][b] = c["ks"][B][300:340], c["vs"][B][300:340]
    c["ks"][B][600:640], c["vs"][B][600:640] = c["ks"][B][300:340], c["vs"][B][300:340]
    for pool, lists in ((c["k_pages"], c["ks"]), (c["v_pages"], c["vs"])):
        fill(pool, c["page_table"], [40] * B, lists[:B])
        fill(pool, c["prefix_table"], [700], lists[B:])
    o, lse = (t.double().cpu() for t in run_attention(c, scale=scale))
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    gqa, sure = H // Hkv, 0
    for b in range(B):
        for h in range(H):
            k, q = c["ks"][B][:, h // gqa].double(), c["q"][b, h].double()
            s, v = k @ q * scale, c["vs"][B][:, h // gqa].double()
            off = (hd + 8) * 2.0**-24 * float((k.abs() @ q.abs()).max()) * scale  # of a score, natural units
            best = int(s.argmax())
            top, second = float(s[best]), float(s[(k != k[best]).any(-1)].max())
            # the score's error, two roundings of the result (2^-23 in all, half a step each), log(740) for keys alike, a cut at 8 log(2)
            assert abs(float(lse[b, h]) - top) <= off + 2.0**-23 * abs(top) + 13
            if top - second > 2 * off + 100:
                # one rounding of the weight to bf16 next to its fp32 sum, one of the result: 2^-8 each
                sure += 1
                assert ((o[b, h] - v[best]).abs() <= 2.0**-7 * v[best].abs() + 2.0**-40).all()
    assert sure > B * H // 2


@pytest.mark.parametrize("H,Hkv,hd,groups", [(32, 32, 128, 3000), (64, 16, 64, 4000), (34, 2, 64, 700)])
def test_scratch_of_many_small_groups(H, Hkv, hd, groups):
    """Parts take the rows that there are, however the groups divide them: 17 query heads a kv head, one, or four."""
    sizes = [1] * groups
    sizes[groups // 2], sizes[groups // 3] = 0, 5
    rows = [0]
    for n in sizes:
        rows.append(rows[-1] + n)
    B = rows[-1]
    plens = [(7 * g) % 40 for g in range(groups)]
    c = cache_case([b % 3 for b in range(B)], H, Hkv, hd, 16, "token", plens, seed=groups)
    d = to_dev(c)
    args = d["q"], d["k_pages"], d["v_pages"], d["page_table"], d["seq_lens"], d["prefix_table"], d["prefix_lens"], i32(rows)
    o, lse = ops.paged_attention(*args)
    torch.cuda.synchronize()
    del o, lse
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    o, lse = ops.paged_attention(*args)
    used = torch.cuda.max_memory_allocated() - before
    # (m, l, fp32 row) of every row for its prefix and for its own tokens (16 rows for every 17), and of 16 rows a warp for each; results
    room = 2.0 * (B * H * (32 / 17 if H == 34 else 1) + 148 * 16 * 16) * (hd * 4 + 8) + B * H * (hd * 2 + 4) + 64 * Hkv * B + (4 << 20)
    assert used <= room, (used, room)
    group = [g for g, n in enumerate(sizes) for _ in range(n)]
    some = torch.tensor(sorted({0, 1, B // 3 - 2, B // 3, groups // 3, groups // 3 + 3, B // 2, B - 1}))
    picked = [int(b) for b in some]
    lists = [c["ks"][b] for b in picked] + c["ks"][B:], [c["vs"][b] for b in picked] + c["vs"][B:]
    want = attention_oracle(c["q"][some], *lists, [group[b] for b in picked], len(picked))
    check_attention(o[some.to(DEV)], lse[some.to(DEV)], want, hd)


@pytest.mark.parametrize("H,Hkv,hd", [(8, 8, 32), (40, 2, 32), (18, 6, 64), (32, 8, 128)])
def test_pages_read_with_and_without_boxes_give_the_same_bits(H, Hkv, hd):
    """Pages of 8 are read as boxes, pages of 4 and 6 with a copy a lane, four stages deep at 32 dims: the same steps over the same keys,
    in items of one step, of many, and cut between warps, with a prefix and without."""
    lens = [0, 1, 33, 700, 31, 64, 2, 0, 260, 5] * 12
    c = cache_case(lens, H, Hkv, hd, 8, prefix_lens=[70, 0, 500], seed=hd)
    rows, B = [0, 50, 60, 110], len(lens)
    want = {pre: None for pre in (False, True)}
    for P in (8, 4, 6):
        a = {**cache_case([0] * B, H, Hkv, hd, P, prefix_lens=[0, 0, 0]), "q": c["q"], "seq_lens": c["seq_lens"], "prefix_lens": c["prefix_lens"]}
        total = sum(-(-n // P) for n in lens + [70, 0, 500])
        order = torch.randperm(total, generator=torch.Generator().manual_seed(P)).tolist()
        # tables for as many tokens in every case: the plan goes by them
        a["page_table"], used = make_tables(lens, P, order, 744 // P)
        a["prefix_table"], _ = make_tables([70, 0, 500], P, order[used:], 504 // P)
        a["k_pages"], a["v_pages"] = make_pool(total, P, Hkv, hd), make_pool(total, P, Hkv, hd)
        for pool, lists in ((a["k_pages"], c["ks"]), (a["v_pages"], c["vs"])):
            fill(pool, a["page_table"], lens, lists[:B])
            fill(pool, a["prefix_table"], [70, 0, 500], lists[B:])
        for pre in want:
            got = run_attention(a, rows) if pre else run_attention({**a, "prefix_table": None, "prefix_lens": None})
            if want[pre] is None:
                want[pre] = got
                group = [0] * 50 + [1] * 10 + [2] * 50 + [-1] * 10 if pre else None
                check_attention(*got, attention_oracle(c["q"], c["ks"], c["vs"], group, B), hd)
            assert torch.equal(got[0], want[pre][0]) and torch.equal(got[1], want[pre][1]), (P, pre)


def test_a_scale_that_32_bits_cannot_hold_is_refused():
    d = to_dev(cache_case([4, 7], 4, 2, 64, 16, seed=1))
    for scale in (1e39, -3e38, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="finite"):
            ops.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"], d["seq_lens"], scale=scale)
    o, _ = ops.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"], d["seq_lens"], scale=1e30)
    assert torch.isfinite(o).all()


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B,H,Hkv,hd", [(4, 6, 2, 64), (30, 6, 2, 64), (90, 6, 2, 64), (30, 8, 2, 128)])
@pytest.mark.parametrize("scale", [None, 200.0])
def test_one_value_that_is_no_number(B, H, Hkv, hd, scale):
    """A NaN among the values makes its component NaN in all rows of its kv head, also where the key's weight has underflowed beside
    another part's (scores of thousands), and leaves the others as they are."""
    c = cache_case([5] * B, H, Hkv, hd, 16, prefix_lens=[300], seed=B)
    gqa = H // Hkv
    clean, lse0 = (t.cpu() for t in run_attention(c, scale=scale))
    for at in (0, 6, 7, 100, 255, 299):
        v = c["vs"][B].clone()
        v[at, 0, 3] = math.nan
        fill(c["v_pages"], c["prefix_table"], [300], [v])
        o, lse = (t.cpu() for t in run_attention(c, scale=scale))
        bad = torch.zeros(B, H, hd, dtype=torch.bool)
        bad[:, :gqa, 3] = True
        assert torch.equal(torch.isnan(o), bad), at
        assert torch.equal(o[~bad], clean[~bad]) and torch.equal(lse, lse0)


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B,H,Hkv,hd", [(4, 6, 2, 64), (30, 6, 2, 64), (90, 6, 2, 64), (30, 8, 2, 128)])
@pytest.mark.parametrize("low", [0.0, 1e-8, -math.inf])
@pytest.mark.parametrize("scale", [1.0, 1e7, 1e10, -1e10])
def test_scores_that_become_large_on_the_way(B, H, Hkv, hd, low, scale):
    """Tiles of small scores (or of none: keys that no query can prefer), then tiles whose maximum climbs over every border, then small
    ones again: each row is its best key's value, or, with a scale of one, what the formula says."""
    n = 900
    c = cache_case([3] * B, H, Hkv, hd, 16, prefix_lens=[n], seed=B)
    c["q"][:, :, 0] = c["q"][:, :, 0].abs() + 0.1
    keys = c["ks"][B].float()
    size = torch.ones(n)
    size[:300], size[300:600], size[700:] = 1e-8, torch.logspace(-8, 0, 300), 1e-3
    keys = keys * size[:, None, None]
    if low == 0.0:
        keys[:300] = 0.0
    elif low == -math.inf:
        keys[:300, :, 0] = low if scale > 0 else math.inf
    c["ks"][B] = keys.bfloat16()
    for b in range(B):
        c["ks"][b] = (c["ks"][b].float() * 1e-6).bfloat16()
    fill(c["k_pages"], c["page_table"], [3] * B, c["ks"][:B])
    fill(c["k_pages"], c["prefix_table"], [n], [c["ks"][B]])
    o, lse = run_attention(c, scale=scale)
    live = c["ks"][B][300:], c["vs"][B][300:]
    if scale == 1.0:
        lists = (c["ks"][:B] + [live[0]], c["vs"][:B] + [live[1]]) if low == -math.inf else (c["ks"], c["vs"])
        check_attention(o, lse, attention_oracle(c["q"], *lists, [0] * B, B, scale=scale), hd)
        return
    o, lse = o.double().cpu(), lse.double().cpu()
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    gqa, sure = H // Hkv, 0
    for b in range(B):
        for h in range(H):
            k = torch.cat((live[0], c["ks"][b]))[:, h // gqa].double()
            v = torch.cat((live[1], c["vs"][b]))[:, h // gqa].double()
            q = c["q"][b, h].double()
            s = k @ q * scale
            off = (hd + 8) * 2.0**-24 * float((k.abs() @ q.abs()).max()) * abs(scale)
            best = int(s.argmax())
            top, second = float(s[best]), float(s.topk(2).values[1])
            if top - second > 2 * off + 100 and top > 2 * off + 100:  # above the keys of zero as well
                sure += 1
                assert abs(float(lse[b, h]) - top) <= off + 2.0**-23 * abs(top) + 13
                assert ((o[b, h] - v[best]).abs() <= 2.0**-7 * v[best].abs() + 2.0**-40).all()
    assert sure > B * H // 2
