"""The paged serving kernels (csrc/paged_append.cu, paged_attn.cu, logits.cu) against 64-bit oracles, and their refusals."""

import functools
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from sample_efficient_gpt_b200 import ops
from sample_efficient_gpt_b200.models.rope import rope_tables

from tests.paged_cases import append_oracle, attention_oracle, cache_case, check_attention, logits_oracle, make_pool, make_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean_status():
    assert ops.ext() is not None, f"extension not built: {ops.ext_error()!r}"
    from sample_efficient_gpt_b200.ops import gemm

    assert gemm.status() == 0
    yield
    code = gemm.status()
    ops.ext().gemm_reset_status(torch.cuda.current_device())
    assert code == 0, f"status word {code}"


def take_status():
    from sample_efficient_gpt_b200.ops import gemm

    code = gemm.status()
    ops.ext().gemm_reset_status(torch.cuda.current_device())
    return code


@functools.lru_cache(None)  # made once: a captured step may not copy from the host
def one(v):
    return torch.tensor([v], device=DEV)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------------------------ append
def append_case(new, past, H, Hkv, hd, P, layout, first=False, pad=0, base=None, behind=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in zip(new, past)]
    n_pages = sum(-(-n // P) for n in total) + 2
    table, _ = make_tables(total, P, torch.randperm(n_pages, generator=g).tolist())
    T, width = sum(new) + behind, (H + 2 * Hkv) * hd
    wide = torch.randn(T, width + pad, generator=g).to(BF16).to(DEV)
    cos, sin = rope_tables(max(total) + max(base or [0]) + 1, 10000, hd)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return dict(qkv=wide[:, :width], v1=None if first else torch.randn(T, Hkv, hd, generator=g).to(BF16).to(DEV), cos=cos.to(DEV), sin=sin.to(DEV),
                k_pages=make_pool(n_pages, P, Hkv, hd, layout, device=DEV), v_pages=make_pool(n_pages, P, Hkv, hd, layout, device=DEV),
                page_table=table.to(DEV), seq_lens=i32(past), cu=i32(cu), pos_base=None if base is None else i32(base))


def run_append(c, H, Hkv, hd, qknorm=True, cu=True, **kw):
    return ops.qkv_post_paged(c["qkv"], c["v1"], c["cos"], c["sin"], one(1.3), one(0.8), one(0.35), one(1.1), H, Hkv, hd, qknorm, c["k_pages"], c["v_pages"],
                              c["page_table"], c["seq_lens"], c["cu"] if cu else None, c["pos_base"], **kw)


def check_append(c, out, new, past, H, Hkv, hd, P, qknorm, base=None):
    n = sum(new)
    seq = torch.tensor([b for b in range(len(new)) for _ in range(new[b])], dtype=torch.long)
    own = torch.tensor([past[b] + i for b in range(len(new)) for i in range(new[b])], dtype=torch.long)
    rot = own + (torch.tensor(base)[seq] if base is not None else 0)
    v1 = c["v1"][:n] if c["v1"] is not None else None
    oracle = append_oracle(c["qkv"][:n], v1, c["cos"], c["sin"], one(1.3), one(0.8), one(0.35), one(1.1), H, Hkv, hd, qknorm, rot)
    at = (c["page_table"].cpu().long()[seq, own // P], own % P)
    kp, vp = c["k_pages"].cpu(), c["v_pages"].cpu()
    for got, want in ((out[0][:n], oracle[0]), (kp[at], oracle[1]), (vp[at], oracle[2])):
        # one rounding to bf16 (half a step, 2^-8), fp32 arithmetic before it (a few 2^-24 of the row's largest value)
        tol = 2.0**-8 * want.abs() + 2.0**-20 * want.abs().amax(-1, keepdim=True)
        assert ((got.double().cpu() - want).abs() <= tol).all()
    written = torch.zeros(kp.shape[:2], dtype=torch.bool)
    written[at] = True
    for pool in (kp, vp):
        assert torch.equal(torch.isfinite(pool).all(-1).all(-1), written), "other slots were touched"
    assert (out[0][n:] == 0).all()
    if out[1] is not None:
        assert torch.equal(out[1][:n].cpu(), kp[at]) and (out[1][n:] == 0).all()
    if out[2] is not None:
        assert torch.equal(out[2][:n].cpu(), vp[at]) and (out[2][n:] == 0).all()


@pytest.mark.parametrize("H,Hkv,hd", [(18, 6, 64), (4, 4, 32), (32, 8, 128), (130, 10, 128), (1, 1, 64)])
@pytest.mark.parametrize("P,layout", [(16, "token"), (24, "head"), (1, "token")])
def test_append_ragged(H, Hkv, hd, P, layout):
    new, past, base = [0, 1, 37, 0, 130, 5, 0], [3, 0, 15, 0, 64, 23, 1], [0, 9, 0, 4, 2, 100, 0]
    c = append_case(new, past, H, Hkv, hd, P, layout, pad=24, base=base, behind=3)
    out = run_append(c, H, Hkv, hd, want_k=True, want_v=True)
    check_append(c, out, new, past, H, Hkv, hd, P, True, base)


@pytest.mark.parametrize("qknorm", [True, False])
@pytest.mark.parametrize("B", [1, 3, 700])
def test_append_decode(B, qknorm):
    past = [(7 * b) % 50 for b in range(B)]
    c = append_case([1] * B, past, 18, 6, 64, 16, "token", first=True, pad=24)
    out = run_append(c, 18, 6, 64, qknorm, cu=False, want_v=True)
    assert out[1] is None
    check_append(c, out, [1] * B, past, 18, 6, 64, 16, qknorm)


def test_append_many_tokens():
    new, past = [4096, 1, 2049, 0, 1777], [0, 5, 100, 2, 31]
    c = append_case(new, past, 18, 6, 64, 64, "head", pad=24)
    check_append(c, run_append(c, 18, 6, 64), new, past, 18, 6, 64, 64, True)


def test_append_leaves_out_what_does_not_fit():
    c = append_case([2, 2, 2], [0, 14, 5], 4, 2, 64, 16, "token", behind=1)
    before = c["k_pages"].clone()
    c["page_table"][0, 0] = c["k_pages"].size(0)  # beyond the pool
    c["seq_lens"][2] = 40  # beyond the page table
    q, k, v = run_append(c, 4, 2, 64, want_k=True, want_v=True)
    assert take_status() in (51, 52)
    assert (q[:2] == 0).all() and (q[4:] == 0).all() and (q[2:4] != 0).any() and (k[:2] == 0).all() and (v[4:] == 0).all()
    own = c["page_table"][1, 0].long()
    rest = torch.arange(before.size(0), device=DEV) != own
    assert torch.isnan(c["k_pages"][rest]).all() and torch.isfinite(c["k_pages"][own, 14:]).all()
    c["seq_lens"][:] = i32([-1, -5, -(2**31)])
    q, _, _ = run_append(c, 4, 2, 64)
    assert take_status() == 51 and (q == 0).all()
    # cumulative rows that reach outside the projection: only rows that exist are touched
    c["seq_lens"][:] = 0
    c["page_table"][0, 0] = own
    c["cu"][:] = i32([-5, 1, 2, 10**9])
    run_append(c, 4, 2, 64)
    assert take_status() in (0, 51, 52)


# --------------------------------------------------------------------------------------------------------------- attention
def to_dev(c):
    return {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}


def dev_pool(t):
    """A pool on the GPU with the strides that it has on the CPU (``.to`` keeps them only for dense layouts)."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
    return out.copy_(t)


ROOM = [1]


@pytest.fixture(params=[1, 2**19])
def prefix_room(request):
    """Tokens that the prefix tables have room for at least: the kernel that walks over a prefix is chosen by it."""
    ROOM[0] = request.param
    yield
    ROOM[0] = 1


def run_attention(c, rows=None, **kw):
    kp, vp = dev_pool(c["k_pages"]), dev_pool(c["v_pages"])
    d = to_dev(c)
    if d["prefix_table"] is not None:
        more = ROOM[0] // kp.size(1) - d["prefix_table"].size(1)
        d["prefix_table"] = torch.nn.functional.pad(d["prefix_table"], (0, max(0, more)), value=-1)
    pre = (d["prefix_table"], d["prefix_lens"], None if rows is None else i32(rows)) if rows is not None or d["prefix_table"] is not None else (None,) * 3
    return ops.paged_attention(d["q"], kp, vp, d["page_table"], d["seq_lens"], *pre, **kw)


@pytest.mark.parametrize("H,Hkv,hd", [(18, 6, 64), (4, 4, 32), (32, 8, 128), (40, 2, 64), (9, 1, 128), (16, 1, 32)])
@pytest.mark.parametrize("P,layout", [(16, "token"), (24, "head"), (1, "head"), (128, "token")])
def test_attention_lengths(H, Hkv, hd, P, layout):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 130, 257, 0, 1000]
    c = cache_case(lens, H, Hkv, hd, P, layout, seed=hd + P)
    o, lse = run_attention(c)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"]), hd)


@pytest.mark.parametrize("B,H,Hkv,hd,P,most", [(200, 18, 6, 64, 16, 90), (1500, 4, 4, 32, 8, 9), (120, 32, 8, 128, 24, 300), (30, 40, 1, 64, 12, 2000), (70, 17, 1, 64, 16, 700),
                                               (1300, 1, 1, 64, 16, 40), (1200, 1, 1, 128, 1, 2)])
def test_attention_many_rows_without_prefix(B, H, Hkv, hd, P, most):
    """Rows whose sequences are empty, whole in a worker's range, or cut between two or many."""
    lens = [(37 * b * b) % most if b % 7 else 0 for b in range(B)]
    lens[B // 2] = 5 * most
    c = cache_case(lens, H, Hkv, hd, P, "head", seed=B)
    want = attention_oracle(c["q"], c["ks"], c["vs"])
    torch.full((B * H * hd * 4,), float("nan"), device=DEV)  # what the allocator hands out next is not zero
    o, lse = run_attention(c)
    check_attention(o, lse, want, hd)
    again = run_attention(c)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("H,Hkv,hd", [(18, 6, 64), (4, 4, 32), (32, 8, 128), (40, 2, 64)])
@pytest.mark.parametrize("P,layout", [(16, "head"), (24, "token"), (64, "token"), (256, "head")])
def test_attention_shared_prefix(H, Hkv, hd, P, layout):
    lens = [0, 3, 100, 1, 0, 0, 17, 64, 5, 9, 2, 33, 0]
    plens, rows = [300, 0, 77, 64], [0, 5, 5, 8, 12]  # the last row is in no group, the second group has no rows
    c = cache_case(lens, H, Hkv, hd, P, layout, plens, seed=hd + P)
    o, lse = run_attention(c, rows)
    group = [0] * 5 + [2] * 3 + [3] * 4 + [-1]
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], group), hd)


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B,plen,H,Hkv,hd,P", [(1, 5000, 18, 6, 64, 16), (7, 129, 12, 12, 64, 16), (64, 1000, 18, 6, 64, 64), (100, 2100, 24, 2, 64, 32), (70, 513, 32, 8, 128, 128),
                                               (33, 700, 16, 4, 64, 40), (20, 900, 18, 6, 64, 16), (11, 127, 18, 6, 64, 8), (45, 128, 18, 6, 64, 128),
                                               (40, 300, 18, 6, 64, 12)])
def test_attention_one_prefix_for_all(B, plen, H, Hkv, hd, P):
    lens = [(13 * b) % 70 for b in range(B)]
    c = cache_case(lens, H, Hkv, hd, P, "token", [plen], seed=B)
    o, lse = run_attention(c)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [0] * B), hd)


# rows of a kv head per group: few (16 at a time), tens (128, the keys in two halves), hundreds (256)
@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("H,Hkv,hd,P,layout", [(18, 6, 64, 16, "token"), (24, 2, 64, 24, "head"), (32, 8, 128, 32, "head"), (64, 2, 128, 8, "token"), (40, 1, 64, 256, "token")])
def test_attention_large_groups(H, Hkv, hd, P, layout):
    sizes, plens = [40, 0, 1, 44], [1500, 64, 129, 700]
    rows = [0, 40, 40, 41, 85]
    lens = [(17 * b) % 90 for b in range(88)]  # three rows without a prefix, some rows without tokens of their own
    c = cache_case(lens, H, Hkv, hd, P, layout, plens, seed=hd + P)
    o, lse = run_attention(c, rows)
    group = [g for g, n in enumerate(sizes) for _ in range(n)] + [-1] * 3
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], group), hd)


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("H,Hkv,hd", [(16, 1, 64), (20, 1, 128)])
def test_attention_many_groups(H, Hkv, hd):
    sizes = [(5 * g) % 4 for g in range(900)]
    rows = [0]
    for n in sizes:
        rows.append(rows[-1] + n)
    plens = [(11 * g) % 40 for g in range(900)]
    c = cache_case([b % 3 for b in range(rows[-1])], H, Hkv, hd, 16, "token", plens, seed=hd)
    o, lse = run_attention(c, rows)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [g for g, n in enumerate(sizes) for _ in range(n)]), hd)


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B,H,Hkv,hd", [(4, 6, 2, 64), (30, 6, 2, 64), (90, 6, 2, 64), (30, 8, 2, 128)])
@pytest.mark.parametrize("scale", [0.125, -0.4, 0.0])
def test_attention_maximum_that_grows(B, H, Hkv, hd, scale):
    """Scores whose maximum climbs from tile to tile, by little and by a lot, and falls again."""
    n = 1000
    c = cache_case([3] * B, H, Hkv, hd, 16, prefix_lens=[n], seed=B)
    climb = torch.cat((torch.linspace(0.1, 2, 400), torch.linspace(2, 40, 300), torch.full((299,), 0.5), torch.tensor([100.0])))
    c["ks"][B] = (c["ks"][B].float() * climb[:, None, None]).bfloat16()
    from tests.paged_cases import fill

    fill(c["k_pages"], c["prefix_table"], [n], [c["ks"][B]])
    o, lse = run_attention(c, scale=scale)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [0] * B, scale=scale), hd)


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("B", [4, 30, 90])
def test_attention_prefix_special_values(B):
    """A key that no query can prefer (-inf scores), a query of NaN, a page that does not exist - in every form."""
    c = cache_case([0] * B, 6, 2, 64, 16, prefix_lens=[300], seed=B)
    c["q"][:, :, 0] = c["q"][:, :, 0].abs() + 0.1
    from tests.paged_cases import fill

    c["ks"][B][5:200, :, 0] = float("-inf")
    fill(c["k_pages"], c["prefix_table"], [300], [c["ks"][B]])
    want = attention_oracle(c["q"], [k[:0] for k in c["ks"][:B]] + [torch.cat((c["ks"][B][:5], c["ks"][B][200:]))],
                            [v[:0] for v in c["vs"][:B]] + [torch.cat((c["vs"][B][:5], c["vs"][B][200:]))], [0] * B)
    o, lse = run_attention(c)
    check_attention(o, lse, want, 64)
    c["q"][B - 1, 3] = float("nan")
    bad = torch.isnan(run_attention(c)[0]).any(-1).cpu()
    assert int(bad.sum()) == 1 and bool(bad[B - 1, 3])
    c["ks"][B][:, :, 0] = float("-inf")  # nothing can be preferred at all
    fill(c["k_pages"], c["prefix_table"], [300], [c["ks"][B]])
    o, lse = run_attention(c)
    assert (o[: B - 1] == 0).all() and (lse[: B - 1] == -math.inf).all()
    c["prefix_table"][0, 3] = 10**7
    run_attention(c)
    assert take_status() == 54


@pytest.mark.usefixtures("prefix_room")
def test_attention_is_the_same_every_time():
    for lens in ([5, 900, 0, 2000, 1], list(range(40)), list(range(120))):
        c = cache_case(lens, 18, 6, 64, 16, "token", [2900], seed=3)
        first = run_attention(c)
        for _ in range(3):
            again = run_attention(c)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_attention_scale_and_large_scores(scale):
    c = cache_case([200, 3], 4, 2, 64, 16, seed=5, scale=6.0)
    o, lse = run_attention(c, scale=scale)
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], scale=scale), 64)


def test_attention_strided_queries_and_wide_tables():
    c = cache_case([40, 7, 100], 6, 2, 64, 16, seed=6, width=300)
    want = attention_oracle(c["q"], c["ks"], c["vs"])
    wide = torch.zeros(3, 9, 128, dtype=BF16)
    wide[:, 1:7, 64:] = c["q"]
    d = to_dev(c)
    q = wide.to(DEV)[:, 1:7, 64:]
    table = torch.full((3, 400), -1, dtype=torch.int32, device=DEV)[:, :300]
    table.copy_(d["page_table"])
    both = torch.stack((c["k_pages"], c["v_pages"]), dim=1).to(DEV)  # keys and values of a page side by side
    o, lse = ops.paged_attention(q, both[:, 0], both[:, 1], table, d["seq_lens"])
    check_attention(o, lse, want, 64)


def test_attention_not_a_number_only_where_it_is_seen():
    c = cache_case([40, 40, 40], 4, 2, 64, 16, seed=7)
    c["q"][1, 2] = float("nan")
    o, _ = run_attention(c)
    bad = torch.isnan(o).any(-1).cpu()
    assert bad.tolist() == [[False] * 4, [False, False, True, False], [False] * 4]


def test_attention_reports_what_does_not_fit():
    c = cache_case([40, 40, 40], 4, 2, 64, 16, seed=8)
    c["seq_lens"][0] = 1000
    o, lse = run_attention(c)
    assert take_status() in (53, 54)  # cut to the table's 48 slots
    c["seq_lens"][:] = torch.tensor([-3, 40, 40])
    o, lse = run_attention(c)
    assert take_status() == 53 and (o[0] == 0).all() and torch.isinf(lse[0]).all()
    c["seq_lens"][0] = 40
    c["page_table"][2, 1] = 10**6
    o, lse = run_attention(c)
    assert take_status() == 54
    want = attention_oracle(c["q"], c["ks"], c["vs"])
    check_attention(o[:2], lse[:2], tuple(t[:2] for t in want), 64)
    c = cache_case([40, 40, 40], 4, 2, 64, 16, prefix_lens=[20, 30], seed=8)
    run_attention(c, [0, 4, 3])
    assert take_status() == 55
    run_attention(c, [2, 1, 3])
    assert take_status() == 55


@pytest.mark.usefixtures("prefix_room")
@pytest.mark.parametrize("H,rows", [(4, [0, 40, 0, 40, 40]), (4, [0, 40, 40, 40, 30]), (32, [0, 40, 0, 40]), (128, [3, 40, 0, 40])])
def test_groups_out_of_order_leave_no_prefix(H, rows):
    """Overlapping groups would hold more rows than the call has; with them no row has a prefix."""
    lens = [(7 * i) % 50 for i in range(40)]
    c = cache_case(lens, H, 2, 64, 16, prefix_lens=[200] * (len(rows) - 1), seed=14)
    o, lse = run_attention(c, rows)
    assert take_status() == 55
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [-1] * 40), 64)


def test_overlapping_groups_of_a_long_prefix():
    """Their tiles together would pass 32 bits: nothing of them is walked over."""
    c = cache_case([5] * 2048, 1, 1, 64, 16, prefix_lens=[16], seed=15)
    d = to_dev(c)
    wide = d["prefix_table"][:, :1].expand(2048, 2**14).contiguous()
    rows = i32([0, 2048] * 1024 + [0])
    o, lse = ops.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"], d["seq_lens"], wide, i32([2**18] * 2048), rows)
    assert take_status() == 55
    check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [-1] * 2048), 64)


# ------------------------------------------------------------------------------------------------------------------ logits
def logits_case(B, V, L, K, M, dtype, seed=0, tok=torch.int32):
    g = torch.Generator().manual_seed(seed)
    tokens = ((V + 1.0) ** torch.rand(B, L, generator=g) - 2).to(tok)  # from -1 (padding) on; small ids often
    lens = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
    u = lambda a, b: a + (b - a) * torch.rand(B, generator=g)  # noqa: E731
    return dict(logits=(torch.randn(B, V, generator=g) * 3).to(dtype), tokens=tokens, prompt_lens=(lens * torch.rand(B, generator=g)).int(), token_lens=lens,
                repetition=u(0.7, 1.5), presence=u(-0.5, 1), frequency=u(-0.1, 0.5), bias_ids=torch.randint(-2, V + 2, (B, K), generator=g, dtype=torch.int32),
                bias_values=torch.randn(B, K, generator=g) * 4, mask=torch.randint(-2**31, 2**31, (M, -(-V // 32)), generator=g, dtype=torch.int64).int(),
                mask_rows=torch.randint(-1, M, (B,), generator=g, dtype=torch.int32))


def oracle_of(c):
    return logits_oracle(*(c.get(k) for k in ("logits", "tokens", "prompt_lens", "token_lens", "repetition", "presence", "frequency", "bias_ids", "bias_values",
                                              "mask", "mask_rows")))


def check_logits(y, c):
    want, mag = oracle_of(c)
    y = y.cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(y), fine) and (y[~fine] == -math.inf).all()
    # at most four fp32 operations, each half a step (2^-24) of a partial sum below mag; bf16 rounds once more
    tol = 2.0**-22 * mag + (2.0**-8 * want.abs() if y.dtype == BF16 else 0)
    assert ((y.double() - want).abs()[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("B,V,L,K,M", [(1, 1, 1, 1, 1), (3, 33, 40, 5, 2), (2, 8192, 300, 64, 1), (5, 8193, 1, 7, 3), (2, 20011, 2048, 300, 4),
                                        (500, 33, 40, 5, 2), (150, 17003, 100, 12, 3)])
def test_logits(B, V, L, K, M, dtype):
    c = logits_case(B, V, L, K, M, dtype, seed=V)
    if K > 4:
        c["bias_ids"][:, 3] = c["bias_ids"][:, 1]  # an id twice
        c["bias_ids"][:, K - 1] = c["bias_ids"][:, 1]
    c["mask"][0] = 0  # a mask that leaves nothing
    d = to_dev(c)
    y = ops.process_logits(**d)
    check_logits(y, c)
    z = d["logits"].clone()
    assert ops.process_logits(**{**d, "logits": z}, out=z) is not None and torch.equal(z, y)  # in place


@pytest.mark.parametrize("keep", [(), ("bias_ids", "bias_values"), ("mask", "mask_rows"), ("tokens", "token_lens", "presence"), ("tokens", "token_lens", "repetition"),
                                  ("tokens", "token_lens", "prompt_lens", "frequency"), ("tokens", "token_lens")])
def test_logits_each_step_alone(keep):
    c = logits_case(4, 9001, 500, 20, 3, torch.float32, seed=1, tok=torch.int64)
    c = {k: v for k, v in c.items() if k == "logits" or k in keep}
    check_logits(ops.process_logits(**to_dev(c)), c)


def test_logits_rows_of_wider_buffers_and_special_values():
    c = logits_case(3, 1000, 64, 8, 2, torch.float32, seed=9)
    c["logits"][0, :4] = torch.tensor([float("-inf"), 0.0, -0.0, 3e38])
    c["bias_ids"][c["bias_ids"] < 4] = 5
    c["tokens"][c["tokens"] < 4] = 6
    buf = torch.zeros(3, 1003, device=DEV)
    buf[:, 2:1002] = c["logits"].to(DEV)
    d = to_dev(c)
    out = torch.full((3, 1500), 7.0, device=DEV)
    tokens = torch.zeros(3, 100, dtype=torch.int32, device=DEV)
    tokens[:, 20:84] = d["tokens"]
    y = ops.process_logits(**{**d, "logits": buf[:, 2:1002], "tokens": tokens[:, 20:84]}, out=out[:, 3:1003])
    check_logits(y, c)
    assert (out[:, :3] == 7).all() and (out[:, 1003:] == 7).all()
    # what the mask hides does not matter, and what it shows stays as it is
    x = torch.full((1, 64), float("nan"), device=DEV)
    x[0, 5] = 2.0
    m = torch.tensor([[32, 0]], dtype=torch.int32, device=DEV)
    y = ops.process_logits(x, mask=m, mask_rows=i32([0]))
    assert float(y[0, 5]) == 2.0 and int(torch.isinf(y).sum()) == 63


def test_logits_reports_what_does_not_fit():
    c = to_dev(logits_case(2, 500, 10, 3, 2, torch.float32, seed=4))
    full = ops.process_logits(**{**c, "token_lens": i32([10, 0])})
    y = ops.process_logits(**{**c, "token_lens": i32([11, -1])})
    assert take_status() == 56 and torch.equal(y, full)
    y = ops.process_logits(**{**c, "mask_rows": i32([2, 10**9])})
    assert take_status() == 57 and torch.isfinite(y).all()


# ------------------------------------------------------------------------------------------- refusals, streams, graphs
def test_refusals():
    c = append_case([1, 1], [0, 3], 4, 2, 64, 16, "token")
    good = lambda **kw: run_append({**c, **kw}, 4, 2, 64, cu=False)  # noqa: E731
    good()
    for kw, text in [(dict(qkv=c["qkv"].float()), "bfloat16"), (dict(qkv=c["qkv"][:, :-8]), "qkv must be"), (dict(k_pages=c["k_pages"].expand(2, *c["k_pages"].shape)[0].float()), "bfloat16"),
                     (dict(v_pages=c["v_pages"][:1]), "shape"), (dict(page_table=c["page_table"].long()), "int32"), (dict(page_table=c["page_table"][:1]), "page_table"),
                     (dict(seq_lens=c["seq_lens"].long()), "seq_lens"), (dict(seq_lens=c["seq_lens"].cpu()), "seq_lens must be on"), (dict(cos=c["cos"][:, :16].contiguous()), "cos"),
                     (dict(v1=c["v1"][:1]), "v1"), (dict(pos_base=i32([1])), "pos_base"), (dict(k_pages=c["k_pages"][:, :, :, 1:]), "k_pages")]:
        with pytest.raises(RuntimeError, match=text):
            good(**kw)
    with pytest.raises(RuntimeError, match="one token"):
        run_append(append_case([2, 1], [0, 3], 4, 2, 64, 16, "token"), 4, 2, 64, cu=False)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.qkv_post_paged(torch.zeros(1, 8 * 48, device=DEV, dtype=BF16), None, c["cos"], c["sin"], one(1.0), one(1.0), one(0.0), one(1.0), 4, 2, 48, True,
                           c["k_pages"], c["v_pages"], c["page_table"][:1], c["seq_lens"][:1])
    a = to_dev(cache_case([40, 7], 4, 2, 64, 16, prefix_lens=[9], seed=1))
    call = lambda *pre, **kw: ops.paged_attention(*({**a, **kw}[k] for k in ("q", "k_pages", "v_pages", "page_table", "seq_lens")), *pre)  # noqa: E731
    call(a["prefix_table"], a["prefix_lens"])
    for kw, text in [(dict(q=a["q"].float()), "bfloat16"), (dict(q=a["q"][:, :3]), "multiple"), (dict(q=a["q"][..., :32].contiguous()), "k_pages"), (dict(k_pages=a["k_pages"].cpu()), "on"),
                     (dict(seq_lens=a["seq_lens"][:1]), "seq_lens"), (dict(page_table=a["page_table"].t()), "page_table")]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    for pre, text in [((a["prefix_table"],), "together"), ((a["prefix_table"].repeat(2, 1), i32([9, 9])), "group_rows"), ((None, None, i32([0, 2])), "prefix_table"),
                      ((a["prefix_table"], a["prefix_lens"], i32([0, 1, 2])), "group_rows")]:
        with pytest.raises(RuntimeError, match=text):
            call(*pre)
    with pytest.raises(RuntimeError, match="2\\^30"):
        call(page_table=torch.zeros(2, 2**26, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="2\\^30"):
        good(page_table=torch.zeros(2, 2**26, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="too large"):  # 128 heads x 2^29 tokens in steps of 32
        ops.paged_attention(torch.zeros(1, 128, 64, device=DEV, dtype=BF16), a["k_pages"], a["v_pages"], torch.zeros(1, 2**25, dtype=torch.int32, device=DEV), i32([0]))
    with pytest.raises(RuntimeError, match="finite"):
        ops.paged_attention(a["q"], a["k_pages"], a["v_pages"], a["page_table"], a["seq_lens"], scale=float("nan"))
    x = torch.zeros(2, 64, device=DEV)
    tok, n = torch.zeros(2, 4, dtype=torch.int32, device=DEV), i32([1, 1])
    for args, text in [(dict(logits=x.half()), "float32 or bfloat16"), (dict(tokens=tok), "together"), (dict(repetition=x[:, 0].contiguous()), "penalties need"),
                       (dict(tokens=tok, token_lens=n, presence=one(1.0)), "presence"), (dict(bias_ids=tok), "together"), (dict(mask=tok, mask_rows=n), "mask must be"),
                       (dict(tokens=tok.float(), token_lens=n), "tokens must be"), (dict(out=x[:, :32]), "out must"), (dict(logits=x[:, :32], out=x.view(-1)[8:72].view(2, 32)), "memory of its own"),
                       (dict(out=x[:1].expand(2, 64)), "overlap")]:
        with pytest.raises(RuntimeError, match=text):
            ops.process_logits(**{"logits": x, **args})


def test_first_call_of_a_process_is_not_captured():
    """It would put the status word into the graph's memory."""
    code = """if True:
        import torch
        from sample_efficient_gpt_b200 import ops
        x = torch.zeros(2, 64, device="cuda")
        g = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(g):
                ops.process_logits(x)
        except RuntimeError as e:
            assert "cannot be captured" in str(e), e
        else:
            raise SystemExit("captured")
        ops.process_logits(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.process_logits(x)
        x.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert (y == 3).all()
    """
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0, r.stdout + r.stderr


def test_empty_batches():
    kp = torch.zeros(2, 16, 2, 64, device=DEV, dtype=BF16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    o, lse = ops.paged_attention(torch.zeros(0, 4, 64, device=DEV, dtype=BF16), kp, kp, torch.zeros(0, 3, dtype=torch.int32, device=DEV), none)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    cos, sin = (t.to(DEV) for t in rope_tables(8, 10000, 64))
    for rows, cu in ((0, None), (0, i32([0])), (3, i32([0]))):
        q, _, _ = ops.qkv_post_paged(torch.ones(rows, 8 * 64, device=DEV, dtype=BF16), None, cos, sin, one(1.0), one(1.0), one(0.0), one(1.0), 4, 2, 64, True, kp, kp.clone(),
                                     torch.zeros(0, 3, dtype=torch.int32, device=DEV), none, cu)
        assert q.shape == (rows, 4, 64) and (q == 0).all()
    assert ops.process_logits(torch.zeros(0, 10, device=DEV)).shape == (0, 10)


def _decode(c, H, Hkv, hd, rows):
    """One step as the decoder runs it: append, attention over own pages and prefix."""
    q, _, _ = run_append(c, H, Hkv, hd, cu=False)
    return ops.paged_attention(q, c["k_pages"], c["v_pages"], c["page_table"], c["seq_lens"] + 1, c["prefix_table"], c["prefix_lens"], rows)


def _decode_case(seed):
    H, Hkv, hd, P, B = 18, 6, 64, 16, 5
    a = cache_case([3, 0, 15, 16, 40], H, Hkv, hd, P, "token", [50, 20], seed=seed, width=4)
    c = append_case([1] * B, [3, 0, 15, 16, 40], H, Hkv, hd, P, "token", pad=24, base=[50, 50, 20, 20, 20], seed=seed)
    spare = list(set(range(a["k_pages"].size(0) + 5)) - set(a["page_table"].flatten().tolist()) - set(a["prefix_table"].flatten().tolist()))
    k, v = (torch.cat((t, make_pool(5, P, Hkv, hd))) for t in (a["k_pages"], a["v_pages"]))
    table = a["page_table"].clone()
    table[1, 0], table[3, 1] = spare[0], spare[1]  # the new token opens a page
    d = to_dev(a)
    c.update(k_pages=k.to(DEV), v_pages=v.to(DEV), page_table=table.to(DEV), prefix_table=d["prefix_table"], prefix_lens=d["prefix_lens"], seq_lens=d["seq_lens"])
    return c, a


def test_decode_step_as_it_is_used():
    """The operators one after the other: appended keys and values are the ones that the attention then reads."""
    c, a = _decode_case(1)
    rows = i32([0, 2, 5])
    o, lse = _decode(c, 18, 6, 64, rows)
    own, group = c["seq_lens"].cpu().long(), [0, 0, 1, 1, 1]
    q, k, v = append_oracle(c["qkv"], c["v1"], c["cos"], c["sin"], one(1.3), one(0.8), one(0.35), one(1.1), 18, 6, 64, True, own + c["pos_base"].cpu())
    ks = [torch.cat((a["ks"][b], k[b : b + 1].bfloat16())) for b in range(5)] + a["ks"][5:]
    vs = [torch.cat((a["vs"][b], v[b : b + 1].bfloat16())) for b in range(5)] + a["vs"][5:]
    want = attention_oracle(q, ks, vs, group, 5)
    # the operands q, k and v were rounded to bf16 once each (2^-8): scores move by at most 2 * 2^-8 of their absolute sums
    assert ((o.double().cpu() - want[0]).abs() <= (2.0**-6 * want[3][..., None] + 2.0**-6) * want[2] + 2.0**-8 * want[0].abs()).all()
    assert torch.isfinite(lse).all()


def test_side_stream_and_graphs():
    """The step on a side stream, and captured: two graphs that replay in turn on new lengths and on new inputs."""
    rows = i32([0, 2, 5])
    cases = [_decode_case(s)[0] for s in (1, 2)]
    want = []
    for c in cases:
        keep = (c["k_pages"].clone(), c["v_pages"].clone())
        want.append([t.clone() for t in _decode(c, 18, 6, 64, rows)])
        c["k_pages"].copy_(keep[0])
        c["v_pages"].copy_(keep[1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _decode(cases[0], 18, 6, 64, rows)
    side.synchronize()
    assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, lse = _decode(c, 18, 6, 64, rows)
            y = ops.process_logits(o.view(5, -1).float(), out=None)
        graphs.append(g)
        outs.append((o, lse, y))
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (o, lse, y), w in zip(outs, want):
        assert torch.equal(o, w[0]) and torch.equal(lse, w[1]) and torch.equal(y, w[0].view(5, -1).float())
    c = cases[0]
    c["seq_lens"].copy_(i32([0, 0, 1, 2, 3]))  # shorter sequences through the same graph
    graphs[0].replay()
    now = _decode(c, 18, 6, 64, rows)
    assert torch.equal(outs[0][0], now[0])


def test_two_streams_at_once():
    """Calls that overlap on the GPU: each has its own workspace, and neither waits for the other."""
    cases = [cache_case([(13 * b) % 70 for b in range(n)], 18, 6, 64, 16, prefix_lens=[p], seed=n) for n, p in ((60, 3000), (90, 2000))]
    dev = [to_dev(c) for c in cases]
    room = [torch.nn.functional.pad(d["prefix_table"], (0, 2**15 - d["prefix_table"].size(1)), value=-1) for d in dev]
    x = torch.randn(64, 5000, device=DEV)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for d, table, stream in zip(dev, room, streams):
            with torch.cuda.stream(stream):
                got.append(ops.paged_attention(d["q"], d["k_pages"], d["v_pages"], d["page_table"], d["seq_lens"], table, d["prefix_lens"]))
                ops.process_logits(x)
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        check_attention(o, lse, attention_oracle(cases[i % 2]["q"], cases[i % 2]["ks"], cases[i % 2]["vs"], [0] * len(cases[i % 2]["q"])), 64)
        assert torch.equal(o, got[i % 2][0]) and torch.equal(lse, got[i % 2][1])


def test_logits_empty_lists():
    x = torch.randn(3, 70, device=DEV)
    empty = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    y = ops.process_logits(x, tokens=empty, token_lens=i32([0, 0, 0]), repetition=torch.full((3,), 2.0, device=DEV), bias_ids=empty, bias_values=empty.float(),
                           mask=torch.zeros(0, 3, dtype=torch.int32, device=DEV), mask_rows=i32([-1, -1, -1]))
    assert torch.equal(x, y)
