"""The paged serving kernels at the ends of what their documentation allows: caches beyond 2^31 elements, the most sequences and groups of a
call, large pages, pools of two layouts, long histories and many biases."""

import math

import pytest
import torch

from sample_efficient_gpt_b200 import ops
from sample_efficient_gpt_b200.models.rope import rope_tables

from tests.paged_cases import append_oracle, attention_oracle, cache_case, check_attention, fill, make_pool, make_tables
from tests.test_gpu_paged import BF16, DEV, _clean_status, check_logits, i32, logits_case, one, oracle_of, run_attention, to_dev  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P,layout", [(64, "token"), (64, "head"), (60, "head")])
def test_a_cache_beyond_32_bit_offsets(P, layout):
    """Pages of the last 2 % of pools of 2.3e9 elements: appended to, then read by themselves and as a prefix, in both walks over prefixes."""
    H, Hkv, hd, n_pages = 16, 8, 64, 72000 * 64 // P
    shape = (n_pages, P, Hkv, hd) if layout == "token" else (n_pages, Hkv, P, hd)
    kp, vp = (torch.empty(shape, dtype=BF16, device=DEV) for _ in range(2))
    if layout == "head":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    assert kp.numel() > 2**31
    g = torch.Generator().manual_seed(P)
    new = [300, 1, 70] + [2] * 40
    order = (n_pages - 1 - torch.randperm(n_pages // 50, generator=g)).tolist()
    table, _ = make_tables(new, P, order)
    T = sum(new)
    qkv = torch.randn(T, (H + 2 * Hkv) * hd, generator=g).to(BF16).to(DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(512, 10000, hd))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    table_d, none = table.to(DEV), torch.zeros(len(new), dtype=torch.int32, device=DEV)
    q, k, v = ops.qkv_post_paged(qkv, None, cos, sin, one(1.0), one(1.0), one(0.0), one(1.0), H, Hkv, hd, True, kp, vp, table_d, none, i32(cu), want_k=True, want_v=True)
    pos = torch.cat([torch.arange(n) for n in new])
    want = append_oracle(qkv, None, cos, sin, one(1.0), one(1.0), one(0.0), one(1.0), H, Hkv, hd, True, pos)
    for got, w in ((q, want[0]), (k, want[1]), (v, want[2])):
        assert ((got.double().cpu() - w).abs() <= 2.0**-8 * w.abs() + 2.0**-20 * w.abs().amax(-1, keepdim=True)).all()
    last = torch.tensor([n - 1 for n in cu[1:]])
    ks, vs = ([t[a:b].cpu() for a, b in zip(cu, cu[1:])] for t in (k, v))
    queries = q[last.to(DEV)]
    o, lse = ops.paged_attention(queries, kp, vp, table_d, i32(new))
    check_attention(o, lse, attention_oracle(queries.cpu(), ks, vs), hd)
    for room in (table.size(1), 2**20 // P):  # the first sequence's pages as all rows' prefix
        prefix = torch.full((1, room), -1, dtype=torch.int32, device=DEV)
        prefix[0, : table.size(1)] = table_d[0]
        o, lse = ops.paged_attention(queries, kp, vp, table_d, i32(new), prefix, i32([new[0]]))
        check_attention(o, lse, attention_oracle(queries.cpu(), ks + [ks[0]], vs + [vs[0]], [0] * len(new), len(new)), hd)


@pytest.mark.parametrize("B,G,H,Hkv,hd", [(8191, 1, 2, 1, 64), (4096, 4096, 4, 2, 32), (1, 8191, 4, 2, 64), (8192, 0, 1, 1, 128)])
def test_the_most_sequences_and_groups(B, G, H, Hkv, hd):
    lens, plens = [(b * 5) % 7 for b in range(B)], [(g * 3) % 9 for g in range(G)]
    rows = [g * B // G for g in range(G + 1)] if G else None
    c = cache_case(lens, H, Hkv, hd, 8, prefix_lens=plens, seed=B)
    o, lse = run_attention(c, rows) if G else run_attention(c)
    group = [g for g in range(G) for _ in range(rows[g + 1] - rows[g])] if G else None
    some = sorted({0, 1 % B, B // 3, B // 2, B - 1, *range(0, B, max(1, B // 97))})
    pick = torch.tensor(some)
    want = attention_oracle(c["q"][pick], [c["ks"][b] for b in some] + c["ks"][B:], [c["vs"][b] for b in some] + c["vs"][B:],
                            [group[b] for b in some] if G else None, len(some))
    check_attention(o[pick.to(DEV)], lse[pick.to(DEV)], want, hd)
    assert torch.isfinite(o).all()
    with pytest.raises(RuntimeError, match="8192"):
        ops.paged_attention(*(to_dev(cache_case([0] * 8193, 1, 1, 64, 8))[k] for k in ("q", "k_pages", "v_pages", "page_table", "seq_lens")))


@pytest.mark.parametrize("P", [4096, 65536, 1000])
def test_large_pages(P):
    c = cache_case([900, 0, 1, 300], 6, 2, 64, P, prefix_lens=[1100], seed=P)
    want = attention_oracle(c["q"], c["ks"], c["vs"], [0] * 4)
    check_attention(*run_attention(c), want, 64)


@pytest.mark.parametrize("P", [16, 12])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pools_of_two_layouts_and_of_some_heads(P, hd):
    """Keys by token, values by head, both some heads of wider pools; many rows on a prefix too, for the walk that wants boxes."""
    for room in (1, 2**18):
        c = cache_case([(9 * b) % 50 for b in range(30)], 8, 2, hd, P, prefix_lens=[400], seed=hd)
        d = to_dev(c)
        n = c["k_pages"].size(0)
        kp = torch.full((n, P, 5, hd), math.nan, dtype=BF16, device=DEV)[:, :, 2:4]
        vp = torch.full((n, 7, P, 2 * hd), math.nan, dtype=BF16, device=DEV)[:, 3:5, :, hd:].transpose(1, 2)
        kp.copy_(d["k_pages"])
        vp.copy_(d["v_pages"])
        prefix = torch.nn.functional.pad(d["prefix_table"], (0, max(0, room // P - d["prefix_table"].size(1))), value=-1)
        o, lse = ops.paged_attention(d["q"], kp, vp, d["page_table"], d["seq_lens"], prefix, d["prefix_lens"])
        check_attention(o, lse, attention_oracle(c["q"], c["ks"], c["vs"], [0] * 30), hd)


def test_one_page_for_everyone():
    """The same page in every table, twice in some: it is read as often as it is listed."""
    k = torch.randn(16, 2, 64).bfloat16()
    v = torch.randn(16, 2, 64).bfloat16()
    q = torch.randn(5, 4, 64).bfloat16()
    kp, vp = make_pool(1, 16, 2, 64), make_pool(1, 16, 2, 64)
    fill(kp, torch.zeros(1, 1, dtype=torch.int32), [16], [k])
    fill(vp, torch.zeros(1, 1, dtype=torch.int32), [16], [v])
    lens = [16, 3, 32, 0, 20]
    o, lse = ops.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), torch.zeros(5, 2, dtype=torch.int32, device=DEV), i32(lens),
                                 torch.zeros(1, 3, dtype=torch.int32, device=DEV), i32([40]))
    twice = lambda t, n: torch.cat((t, t, t))[:n]  # noqa: E731
    check_attention(o, lse, attention_oracle(q, [twice(k, n) for n in [*lens, 40]], [twice(v, n) for n in [*lens, 40]], [0] * 5, 5), 64)


@pytest.mark.parametrize("B,V,L,K,M,dtype,tok", [(65535, 9, 3, 1, 2, torch.float32, torch.int32), (2, 262147, 50000, 40, 2, BF16, torch.int64),
                                                 (1, 5000, 10, 6000, 1, torch.float32, torch.int32), (3, 70001, 17, 513, 1, BF16, torch.int32)])
def test_logits_at_their_ends(B, V, L, K, M, dtype, tok):
    c = logits_case(B, V, L, K, M, dtype, seed=V, tok=tok)
    if K >= 513:
        c["bias_ids"][:, 512:] = torch.randint(0, 40, (B, K - 512), dtype=torch.int32)  # thousands of values on few ids
        c["bias_values"] /= 8
    if B * V > 2**19 or B > 1000:  # the oracle goes entry by entry: of many rows some, and no masks where they are wide
        del c["mask"], c["mask_rows"]
    y = ops.process_logits(**to_dev(c))
    some = torch.tensor(sorted({0, B // 2, B - 1}))
    part = {k: (v[some] if k != "mask" else v) for k, v in c.items()}
    if K >= 513:
        want, mag = oracle_of(part)
        got = y.cpu().double()[some.tolist()]
        fine = torch.isfinite(want)
        # as many additions as an id has values, each half a step (2^-24) of a partial sum below mag
        tol = (K + 4) * 2.0**-24 * mag + (2.0**-8 * want.abs() if dtype == BF16 else 0)
        assert torch.equal(torch.isfinite(got), fine) and ((got - want).abs()[fine] <= tol[fine]).all()
    else:
        check_logits(y[some.to(DEV)], part)
