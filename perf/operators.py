"""Cases of the serving operators: the paged key/value cache with its one-token attention, and the logits on their way to
the sampler.

* ``append``    - ``ops.qkv_post_paged``: the packed qkv projection of new tokens becomes rotated, normalised queries, and
  finished keys and values in the pages of a cache (rotary embedding, QK-norm, value residual).
* ``attention`` - ``ops.paged_attention``: one query token per sequence against its pages and against the pages of a prefix
  that the sequences of a group share.
* ``logits``    - ``ops.process_logits``: penalties for repeated tokens, sparse biases and a bit mask of allowed tokens.

``own`` false: elementary torch operations in 32 bits, rounded once at the end; true: this package's calls.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
QK_EPS = 1e-6
MIX_EPS = 1e-8
BF16 = torch.bfloat16


# ----------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one conversation in a chat: a decode step of the flagship's first block (18 query and 6 key/value heads of 64; the
        # projection's row also holds the gate logits); launch latency is all there is
        dict(name="append_chat_1", op="append", decode=True, seqs=1, tokens=1, past=700, H=18, Hkv=6, hd=64, page=16, layout="token", first=True, pad=24),
        # a decode step of a busy server, a later block (value residual from the first block's values)
        dict(name="append_decode_256", op="append", decode=True, seqs=256, tokens=256, past=2047, H=18, Hkv=6, hd=64, page=16, layout="head", first=False, pad=24),
        # prompts of odd lengths prefilled together behind what their sequences hold already; heads of 128
        dict(name="append_ragged_128", op="append", decode=False, seqs=37, tokens=8191, past=1500, H=32, Hkv=8, hd=128, page=24, layout="head", first=False, pad=0),
        # the training batch's size as a prefill: 16 sequences, 32768 tokens
        dict(name="append_prefill_32k", op="append", decode=False, seqs=16, tokens=32768, past=0, H=18, Hkv=6, hd=64, page=64, layout="token", first=False, pad=24),
        # one conversation of a few hundred tokens: latency
        dict(name="attn_chat_1", op="attention", seqs=1, least=700, most=700, groups=0, prefix=0, H=18, Hkv=6, hd=64, page=16, layout="token"),
        # eight continuations of one chat prompt at the evaluations' context limit; a key/value head for every query head
        dict(name="attn_samples_8", op="attention", seqs=8, least=1, most=257, groups=1, prefix=1791, H=12, Hkv=12, hd=64, page=16, layout="token"),
        # a server's batch of unequal sequences without a common prefix: bound by the cache's bytes
        dict(name="attn_ragged_64", op="attention", seqs=64, least=1, most=8192, groups=0, prefix=0, H=18, Hkv=6, hd=64, page=16, layout="head"),
        # several prompts with several continuations each, heads of 128, an odd page size
        dict(name="attn_groups_128", op="attention", seqs=96, least=0, most=600, groups=7, prefix=4001, H=32, Hkv=8, hd=128, page=24, layout="head"),
        # a long document that 256 requests ask about: the prefix's products outweigh the bytes
        dict(name="attn_document_256", op="attention", seqs=256, least=1, most=1024, groups=1, prefix=32768, H=18, Hkv=6, hd=64, page=64, layout="head"),
        # one conversation's logits: latency
        dict(name="logits_chat_1", op="logits", rows=1, vocab=49152, history=700, dtype="float32", penalties=True, bias=8, masks=1),
        # a batch with all of it, in the compute dtype
        dict(name="logits_batch_64", op="logits", rows=64, vocab=49152, history=2048, dtype="bfloat16", penalties=True, bias=300, masks=16),
        # many long sequences over an odd, large vocabulary
        dict(name="logits_long_512", op="logits", rows=512, vocab=100003, history=8192, dtype="float32", penalties=True, bias=32, masks=40),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "logits"])
    if op == "logits":
        vocab = rng.choice([10000, 32000, 49152, _log(rng, 1000, 100003)])
        rows = _log(rng, 1, max(1, min(512, 512 * 100003 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, history=_log(rng, 1, 8192), dtype=rng.choice(["float32", "bfloat16"]), penalties=rng.random() < 0.8,
                    bias=rng.choice([0, 1, 8, 32, 300]), masks=rng.choice([0, 1, 5, 40]))
    H, Hkv, hd = rng.choice([(18, 6, 64), (16, 8, 64), (12, 12, 64), (32, 8, 128), (24, 2, 64), (8, 8, 32)])
    page, layout = rng.choice([8, 16, 24, 32, 64, 100, 128]), rng.choice(["token", "head"])
    if op == "append":
        decode = rng.random() < 0.4
        width = (H + 2 * Hkv) * hd
        tokens = _log(rng, 1, 512) if decode else _log(rng, 1, 32768 * 1920 // max(width, 1920))
        seqs = tokens if decode else _log(rng, 1, 64)
        return dict(op=op, decode=decode, seqs=seqs, tokens=tokens, past=rng.choice([0, _log(rng, 1, 4000)]), H=H, Hkv=Hkv, hd=hd, page=page, layout=layout,
                    first=rng.random() < 0.3, pad=rng.choice([0, 24, 64]))
    seqs = _log(rng, 1, 256)
    groups = rng.choice([0, 1, min(seqs, _log(rng, 1, 16))])
    heads = Hkv * hd / 384
    most = _log(rng, 1, max(1, min(8192, int(262144 / seqs / max(1.0, heads)))))
    prefix = 0
    if groups:
        prefix = _log(rng, 1, max(1, min(32768, int(32768 * 256 * 18 * 64 / (seqs * H * hd) / 2), int(262144 / groups / max(1.0, heads)))))
    return dict(op=op, seqs=seqs, least=rng.choice([0, 1, most]), most=most, groups=groups, prefix=prefix, H=H, Hkv=Hkv, hd=hd, page=page, layout=layout)


# ------------------------------------------------------------------------------------------------------------- the inputs
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread: their sum does not depend on the seed, only their order."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _group_sizes(seqs, groups):
    """Uneven shares of the sequences, each at least one where there are enough of them."""
    if not groups:
        return []
    cut = [seqs * i * (i + groups) // (2 * groups * groups) for i in range(groups + 1)]
    return [b - a for a, b in zip(cut, cut[1:])]


def _prefix_lens(case):
    return _spread(case["prefix"] - case["prefix"] // 4, case["prefix"], case["groups"]) if case["groups"] else []


def _new_tokens(case, rng):
    """Tokens that each sequence brings: uneven, some none."""
    B, T = case["seqs"], case["tokens"]
    cuts = sorted(rng.randint(0, T) for _ in range(B - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [T])]


def _pool(pages, case, gen):
    """[pages, page, Hkv, hd] of random values, its memory ordered by token or by head."""
    P, Hkv, hd = case["page"], case["Hkv"], case["hd"]
    if case["layout"] == "token":
        return torch.randn(pages, P, Hkv, hd, device=DEV, dtype=BF16, generator=gen)
    return torch.randn(pages, Hkv, P, hd, device=DEV, dtype=BF16, generator=gen).transpose(1, 2)


def _tables(lens, page, first_page, order):
    """Page table [len(lens), widest] over pages order[first_page:]; -1 where a sequence has no page."""
    need = [-(-n // page) for n in lens]
    width = max(1, max(need, default=1))
    flat, rows = first_page, []
    for n in need:
        rows.append(order[flat:flat + n] + [-1] * (width - n))
        flat += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), flat


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "logits": _prepare_logits}[case["op"]](case, rng, gen)


def _prepare_append(case, rng, gen):
    H, Hkv, hd, B, T, page = (case[k] for k in ("H", "Hkv", "hd", "seqs", "tokens", "page"))
    new = [1] * B if case["decode"] else _new_tokens(case, rng)
    past = _spread(0, case["past"], B)
    rng.shuffle(past)
    total = [a + b for a, b in zip(past, new)]
    n_pages = (T + sum(past)) // page + B + 3  # enough however the tokens fall to the sequences
    order = list(range(n_pages))
    rng.shuffle(order)
    table, _ = _tables(total, page, 0, order)
    width = (H + 2 * Hkv) * hd
    qkv = torch.randn(T, width + case["pad"], device=DEV, dtype=BF16, generator=gen)[:, :width]
    v1 = None if case["first"] else torch.randn(T, Hkv, hd, device=DEV, dtype=BF16, generator=gen)
    i = torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    ang = torch.arange(max(8192, max(total)), device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / hd)
    scalar = lambda v: torch.tensor([v], device=DEV)  # noqa: E731
    cu = None
    if not case["decode"]:
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
    return dict(case=case, qkv=qkv, v1=v1, cos=ang.cos().float(), sin=ang.sin().float(), qgain=scalar(1.3), a1=scalar(0.8), a2=scalar(0.35), vscale=scalar(1.1),
                k_pages=_pool(n_pages, case, gen), v_pages=_pool(n_pages, case, gen), table=table, lens=_i32(past), cu=None if cu is None else _i32(cu))


def _prepare_attention(case, rng, gen):
    H, hd, B, page = (case[k] for k in ("H", "hd", "seqs", "page"))
    lens = _spread(case["least"], case["most"], B)
    rng.shuffle(lens)
    plens, sizes = _prefix_lens(case), _group_sizes(B, case["groups"])
    n_pages = sum(-(-n // page) for n in lens + plens) + 3
    order = list(range(n_pages))
    rng.shuffle(order)
    table, used = _tables(lens, page, 0, order)
    s = dict(case=case, q=torch.randn(B, H, hd, device=DEV, dtype=BF16, generator=gen), k_pages=_pool(n_pages, case, gen), v_pages=_pool(n_pages, case, gen),
             table=table, lens=_i32(lens), prefix_table=None, prefix_lens=None, group_rows=None, most=max(lens), prefix_most=0, group_most=0)
    if case["groups"]:
        rows = [0]
        for n in sizes:
            rows.append(rows[-1] + n)
        s.update(prefix_table=_tables(plens, page, used, order)[0], prefix_lens=_i32(plens), group_rows=_i32(rows), prefix_most=max(plens), group_most=max(sizes))
    return s


def _prepare_logits(case, rng, gen):
    B, V, L = case["rows"], case["vocab"], case["history"]
    dtype = getattr(torch, case["dtype"])
    logits = (torch.randn(B, V, device=DEV, generator=gen) * 3).to(dtype)
    s = dict(case=case, logits=logits, tokens=None, prompt_lens=None, token_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None,
             bias_values=None, mask=None, mask_rows=None)
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(B, device=DEV, generator=gen)  # noqa: E731
    if case["penalties"]:
        # a text's tokens: few of them make up most of it
        u = torch.rand(B, L, device=DEV, generator=gen)
        tokens = ((V + 1.0) ** u - 1).long().clamp_(0, V - 1)
        lens = _spread(1, L, B)
        rng.shuffle(lens)
        s.update(tokens=tokens.int(), token_lens=_i32(lens), prompt_lens=_i32([n * rng.randint(0, 4) // 4 for n in lens]), repetition=uniform(0.9, 1.4),
                 presence=uniform(-0.5, 0.8), frequency=uniform(0.0, 0.3))
    if case["bias"]:
        K = case["bias"]
        ids = torch.randint(0, V, (B, K), device=DEV, generator=gen, dtype=torch.int32)
        ids[:, K // 2 + 1:][torch.rand(B, K - K // 2 - 1, device=DEV, generator=gen) < 0.3] = -1  # requests with fewer entries
        s.update(bias_ids=ids, bias_values=torch.randn(B, K, device=DEV, generator=gen) * 4)
    if case["masks"]:
        words = torch.randint(-2**31, 2**31, (case["masks"], -(-V // 32)), device=DEV, generator=gen, dtype=torch.int64).to(torch.int32)
        s.update(mask=words, mask_rows=torch.randint(0 if B == 1 else -1, case["masks"], (B,), device=DEV, generator=gen, dtype=torch.int32))
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    return {"append": _run_append, "attention": _run_attention, "logits": _run_logits}[s["case"]["op"]](s)


def _run_append(s):
    c = s["case"]
    if own:
        from sample_efficient_gpt_b200 import ops

        q, _, v = ops.qkv_post_paged(s["qkv"], s["v1"], s["cos"], s["sin"], s["qgain"], s["a1"], s["a2"], s["vscale"], c["H"], c["Hkv"], c["hd"], True,
                                     s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], want_v=c["first"])
        return [q, v, s["k_pages"], s["v_pages"]]
    H, Hkv, hd, page = c["H"], c["Hkv"], c["hd"], c["page"]
    T = s["qkv"].size(0)
    t = torch.arange(T, device=DEV)
    if s["cu"] is None:
        seq, pos = t, s["lens"].long()
    else:
        seq = torch.searchsorted(s["cu"][1:].contiguous(), t.int(), right=True)
        pos = s["lens"].long()[seq] + t - s["cu"].long()[seq]
    x = s["qkv"].float().view(T, H + 2 * Hkv, hd) if s["qkv"].is_contiguous() else s["qkv"].float().reshape(T, H + 2 * Hkv, hd)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    x1, x2 = x[:, :H + Hkv, :hd // 2], x[:, :H + Hkv, hd // 2:]
    r = torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos), -1)
    r = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + QK_EPS)
    q, k, v = r[:, :H] * s["qgain"], r[:, H:], x[:, H + Hkv:]
    v = s["vscale"] * torch.rsqrt(s["a1"] ** 2 + s["a2"] ** 2 + MIX_EPS) * (s["a1"] * v + s["a2"] * (v if s["v1"] is None else s["v1"].float()))
    where = (s["table"].long()[seq, pos // page], pos % page)
    s["k_pages"][where] = k.to(BF16)
    s["v_pages"][where] = v.to(BF16)
    return [q.to(BF16), v.to(BF16) if c["first"] else None, s["k_pages"], s["v_pages"]]


def _rows(pages, table, n, page):
    """The first n tokens of every row of a page table, [rows, n, Hkv, hd] in 32 bits."""
    i = torch.arange(n, device=DEV)
    return pages[table.long()[:, i // page].clamp_min(0), i % page].float()


def _run_attention(s):
    c = s["case"]
    if own:
        from sample_efficient_gpt_b200 import ops

        return list(ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["prefix_table"], s["prefix_lens"], s["group_rows"]))
    B, H, Hkv, hd, page, n = c["seqs"], c["H"], c["Hkv"], c["hd"], c["page"], s["most"]
    q = s["q"].float().view(B, Hkv, H // Hkv, hd) / math.sqrt(hd)
    score = torch.einsum("bkgd,bnkd->bkgn", q, _rows(s["k_pages"], s["table"], n, page))
    score = score.masked_fill((torch.arange(n, device=DEV) >= s["lens"][:, None])[:, None, None], -math.inf)
    m = score.amax(-1) if n else torch.full((B, Hkv, H // Hkv), -math.inf, device=DEV)
    if s["prefix_table"] is not None:  # the groups' rows side by side, so that each prefix is read once
        b = torch.arange(B, device=DEV)
        group = torch.searchsorted(s["group_rows"][1:].contiguous(), b.int(), right=True)
        member = b - s["group_rows"].long()[group]
        np_ = s["prefix_most"]
        side = q.new_zeros(c["groups"], s["group_most"], Hkv, H // Hkv, hd)
        side[group, member] = q
        shared = torch.einsum("amkgd,ankd->amkgn", side, _rows(s["k_pages"], s["prefix_table"], np_, page))
        shared = shared.masked_fill((torch.arange(np_, device=DEV) >= s["prefix_lens"][:, None])[:, None, None, None], -math.inf)
        m = torch.maximum(m, shared.amax(-1)[group, member])
        top = torch.where(m == -math.inf, 0.0, m)
        tops = side.new_zeros(side.shape[:-1])
        tops[group, member] = top
        shared = (shared - tops[..., None]).exp()
        total = shared.sum(-1)[group, member]
        out = torch.einsum("amkgn,ankd->amkgd", shared, _rows(s["v_pages"], s["prefix_table"], np_, page))[group, member]
    else:
        top = torch.where(m == -math.inf, 0.0, m)
        total, out = 0.0, 0.0
    score = (score - top[..., None]).exp()
    total = total + score.sum(-1)
    out = out + torch.einsum("bkgn,bnkd->bkgd", score, _rows(s["v_pages"], s["table"], n, page))
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    return [out.reshape(B, H, hd).to(BF16), (top + total.log()).reshape(B, H)]


def _run_logits(s):
    if own:
        from sample_efficient_gpt_b200 import ops

        return ops.process_logits(s["logits"], s["tokens"], s["prompt_lens"], s["token_lens"], s["repetition"], s["presence"], s["frequency"], s["bias_ids"],
                                  s["bias_values"], s["mask"], s["mask_rows"])
    x = s["logits"].float()
    B, V = x.shape
    if s["tokens"] is not None:
        i = torch.arange(s["tokens"].size(1), device=DEV)
        there, prompt = i < s["token_lens"][:, None], i < s["prompt_lens"][:, None]
        tokens = s["tokens"].long()
        said = x.new_zeros(B, V).scatter_add_(1, tokens, (there & ~prompt).float())
        seen = x.new_zeros(B, V).scatter_add_(1, tokens, there.float()) > 0
        rep = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["frequency"][:, None] * said - s["presence"][:, None] * (said > 0)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long()
        x = x.scatter_add(1, ids.clamp_min(0), torch.where(ids >= 0, s["bias_values"], 0.0))
    if s["mask"] is not None:
        v = torch.arange(V, device=DEV)
        allowed = (s["mask"][s["mask_rows"].long().clamp_min(0)][:, v // 32] >> (v % 32)) & 1
        x = x.masked_fill((allowed == 0) & (s["mask_rows"] >= 0)[:, None], -math.inf)
    return x.to(s["logits"].dtype)


# -------------------------------------------------------------------------------------------------- what a pass cannot avoid
def work(case):
    if case["op"] == "append":
        T, H, Hkv, hd = (case[k] for k in ("tokens", "H", "Hkv", "hd"))
        row, kv = (H + 2 * Hkv) * hd, Hkv * hd
        # the projection in, queries and cache rows out; the first block also stores its values, the others read them
        return {"bytes": 2 * T * (2 * row + kv) + min(T, 8192) * hd * 4, "flops": T * ((H + Hkv) * hd * 6 + kv * 4)}
    if case["op"] == "attention":
        B, H, Hkv, hd = (case[k] for k in ("seqs", "H", "Hkv", "hd"))
        lens, plens, sizes = _spread(case["least"], case["most"], B), _prefix_lens(case), _group_sizes(B, case["groups"])
        seen = sum(lens) + sum(n * p for n, p in zip(sizes, plens))
        held = sum(lens) + sum(p for n, p in zip(sizes, plens) if n)
        return {"bytes": 4 * Hkv * hd * held + 4 * B * H * hd + 4 * B * H, "flops": 4 * H * hd * seen}
    B, V = case["rows"], case["vocab"]
    n = 2 if case["dtype"] == "bfloat16" else 4
    history = sum(_spread(1, case["history"], B)) if case["penalties"] else 0
    return {"bytes": 2 * n * B * V + 4 * history + 8 * B * case["bias"] + min(B, case["masks"]) * V // 8, "flops": 4 * B * V}


# --------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](case, s)


def _exact_append(case, s):
    H, Hkv, hd, page = (case[k] for k in ("H", "Hkv", "hd", "page"))
    half = hd // 2
    x = s["qkv"].double().reshape(-1, H + 2 * Hkv, hd)
    T = x.size(0)
    starts = list(range(T + 1)) if s["cu"] is None else s["cu"].tolist()
    past = s["lens"].tolist()
    pos = torch.tensor([past[b] + i for b in range(len(past)) for i in range(starts[b + 1] - starts[b])], dtype=torch.long, device=DEV)
    seq = torch.tensor([b for b in range(len(past)) for _ in range(starts[b + 1] - starts[b])], dtype=torch.long, device=DEV)
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
    z = torch.complex(x[:, :H + Hkv, :half].contiguous(), x[:, :H + Hkv, half:].contiguous()) * turn
    rms = ((z.abs() ** 2).sum(-1, keepdim=True) / hd + QK_EPS).sqrt()
    z = z / rms
    qk = torch.cat((z.real, z.imag), -1)
    a1, a2, vs = (float(s[k].double()) for k in ("a1", "a2", "vscale"))
    v = x[:, H + Hkv:]
    v = vs / math.sqrt(a1 * a1 + a2 * a2 + MIX_EPS) * (a1 * v + a2 * (v if s["v1"] is None else s["v1"].double()))
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    page_of = s["table"].long()[seq, torch.div(pos, page, rounding_mode="floor")]
    kp[page_of, pos % page] = qk[:, H:]
    vp[page_of, pos % page] = v
    return [qk[:, :H] * float(s["qgain"].double()), v if case["first"] else None, kp, vp]


def _exact_attention(case, s):
    H, Hkv, hd, page, B = (case[k] for k in ("H", "Hkv", "hd", "page", "seqs"))
    out = torch.zeros(B, H, hd, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=DEV)
    lens, rows = s["lens"].tolist(), s["group_rows"].tolist() if case["groups"] else [0]

    def tokens(table, n):
        i = torch.arange(n, device=DEV)
        at = (table.long()[torch.div(i, page, rounding_mode="floor")], i % page)
        return s["k_pages"][at].double(), s["v_pages"][at].double()

    shared = (None, None)
    for b in range(B):
        if case["groups"]:
            for g in range(case["groups"]):
                if rows[g] <= b < rows[g + 1] and (b == rows[g]):
                    shared = tokens(s["prefix_table"][g], int(s["prefix_lens"][g]))
        k, v = tokens(s["table"][b], lens[b])
        if shared[0] is not None:
            k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
        if not k.size(0):
            continue
        q = s["q"][b].double().view(Hkv, H // Hkv, hd)
        score = torch.bmm(q, k.permute(1, 2, 0)) / math.sqrt(hd)
        lse[b] = torch.logsumexp(score, -1).reshape(H)
        out[b] = torch.bmm(score.softmax(-1), v.transpose(0, 1)).reshape(H, hd)
    return [out, lse]


def _exact_logits(case, s):
    x = s["logits"].double()
    B, V = x.shape
    if s["tokens"] is not None:
        tokens, lens, prompts = s["tokens"].long(), s["token_lens"].tolist(), s["prompt_lens"].tolist()
        for b in range(B):
            row = x[b]
            rep, pres, freq = (float(s[k][b].double()) for k in ("repetition", "presence", "frequency"))
            all_ = torch.bincount(tokens[b, :lens[b]], minlength=V)
            said = torch.bincount(tokens[b, prompts[b]:max(lens[b], prompts[b])], minlength=V)
            row = torch.where(all_ > 0, row * torch.where(row > 0, 1.0 / rep, rep), row)
            x[b] = row - (freq * said + pres * said.clamp_max(1))
    if s["bias_ids"] is not None:
        for j in range(case["bias"]):
            ids = s["bias_ids"][:, j].long()
            has = torch.nonzero(ids >= 0).flatten()
            x[has, ids[has]] += s["bias_values"][has, j].double()
    if s["mask"] is not None:
        bits = (s["mask"].long()[:, :, None] >> torch.arange(32, device=DEV)) & 1
        bits = bits.flatten(1)[:, :V] > 0
        for b, m in enumerate(s["mask_rows"].tolist()):
            if m >= 0:
                x[b][~bits[m]] = -math.inf
    return x
