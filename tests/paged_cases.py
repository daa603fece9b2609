"""Inputs and 64-bit oracles shared by the CPU and GPU tests of the paged serving operators."""

import math

import torch


def make_pool(n_pages, P, Hkv, hd, layout="token", dtype=torch.bfloat16, device="cpu", seed=0):
    """[n_pages, P, Hkv, hd] of NaN: a slot that nobody has written must never count."""
    shape = (n_pages, P, Hkv, hd) if layout == "token" else (n_pages, Hkv, P, hd)
    t = torch.full(shape, float("nan"), dtype=dtype, device=device)
    return t if layout == "token" else t.transpose(1, 2)


def make_tables(lens, P, order, width=None):
    """(table [B, W] int32, -1 behind the last page; pages used) handing out the pages of ``order`` one after the other."""
    need = [-(-n // P) for n in lens]
    width = width or max(1, max(need, default=1))
    out, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        out[b, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    return out, at


def fill(pool, table, lens, values):
    """Writes values[b] ([len, Hkv, hd]) into the sequences' pages."""
    P = pool.size(1)
    for b, n in enumerate(lens):
        if n:
            i = torch.arange(n, device=pool.device)
            pool[table[b].to(pool.device).long()[i // P], i % P] = values[b].to(pool)


def cache_case(lens, H, Hkv, hd, P, layout="token", prefix_lens=(), seed=0, scale=1.0, width=None):
    """A filled cache on the CPU: dict with q, pools, tables and the plain keys / values of every list."""
    g = torch.Generator().manual_seed(seed)
    lists = list(lens) + list(prefix_lens)
    n_pages = sum(-(-n // P) for n in lists) + 2
    order = torch.randperm(n_pages, generator=g).tolist()
    table, used = make_tables(lens, P, order, width)
    ptable, _ = make_tables(prefix_lens, P, order[used:]) if len(prefix_lens) else (None, 0)
    kp, vp = make_pool(n_pages, P, Hkv, hd, layout), make_pool(n_pages, P, Hkv, hd, layout)
    ks = [torch.randn(n, Hkv, hd, generator=g).mul(scale).bfloat16() for n in lists]
    vs = [torch.randn(n, Hkv, hd, generator=g).bfloat16() for n in lists]
    B = len(lens)
    fill(kp, table, lens, ks[:B])
    fill(vp, table, lens, vs[:B])
    if ptable is not None:
        fill(kp, ptable, prefix_lens, ks[B:])
        fill(vp, ptable, prefix_lens, vs[B:])
    return dict(q=torch.randn(B, H, hd, generator=g).bfloat16(), k_pages=kp, v_pages=vp, page_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32),
                prefix_table=ptable, prefix_lens=torch.tensor(prefix_lens, dtype=torch.int32) if ptable is not None else None, ks=ks, vs=vs)


def attention_oracle(q, ks, vs, group=None, n_seqs=None, scale=None):
    """64 bits: (o, lse, a = sum p |v|, s = largest sum |q k| scale of a row) with the rows' keys in ks[b], and the prefix of row b in
    ks[n_seqs + group[b]]."""
    B, H, hd = q.shape
    n_seqs = B if n_seqs is None else n_seqs
    scale = 1 / math.sqrt(hd) if scale is None else scale
    o = torch.zeros(B, H, hd, dtype=torch.float64)
    a, lse, s = torch.zeros_like(o), torch.full((B, H), -math.inf, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        k, v = ks[b], vs[b]
        if group is not None and group[b] >= 0:
            k, v = torch.cat((ks[n_seqs + group[b]], k)), torch.cat((vs[n_seqs + group[b]], v))
        if not len(k):
            continue
        k, v = k.double().cpu(), v.double().cpu()
        rep = H // k.size(1)
        for h in range(H):
            x = q[b, h].double().cpu()
            z = k[:, h // rep] @ x * scale
            p = torch.softmax(z, 0)
            lse[b, h] = torch.logsumexp(z, 0)
            o[b, h] = p @ v[:, h // rep]
            a[b, h] = p @ v[:, h // rep].abs()
            s[b, h] = (k[:, h // rep].abs() @ x.abs() * abs(scale)).max()
    return o, lse, a, s


def check_attention(o, lse, oracle, hd):
    """Weights are rounded to bf16 before the second product (half a step, 2^-8, of each), the result once more (2^-8); scores
    and sums are fp32: a score is off by at most (hd + 8) 2^-24 of its absolute sum, which shifts the weights by as much."""
    oo, ll, a, s = oracle
    o, lse = o.double().cpu(), lse.double().cpu()
    off = (hd + 8) * 2.0**-24 * s + 2.0**-20
    assert torch.equal(torch.isfinite(lse), torch.isfinite(ll)) and not torch.isnan(o).any()
    tol = 2.0**-8 * (a + oo.abs()) + 2.1 * off[..., None] * a + 2.0**-40
    assert ((o - oo).abs() <= tol).all(), float(((o - oo).abs() / tol).max())
    fine = torch.isfinite(ll)
    assert (lse[~fine] == -math.inf).all()
    tol = (off + 2.0**-23 * ll.abs())[fine]
    assert ((lse[fine] - ll[fine]).abs() <= tol).all(), float(((lse[fine] - ll[fine]).abs() / tol).max())


def append_oracle(qkv, v1, cos, sin, qgain, a1, a2, vs, H, Hkv, hd, qknorm, pos):
    """64 bits: (q, k, v) of rows at rotation positions ``pos``."""
    x = qkv.double().cpu().reshape(-1, H + 2 * Hkv, hd)
    half = hd // 2
    c, s = cos.double().cpu()[pos][:, None], sin.double().cpu()[pos][:, None]
    x1, x2 = x[:, : H + Hkv, :half], x[:, : H + Hkv, half:]
    r = torch.cat((x1 * c - x2 * s, x1 * s + x2 * c), -1)
    q, k = r[:, :H], r[:, H:]
    if qknorm:
        q = q / (q.square().mean(-1, keepdim=True) + 1e-6).sqrt() * float(qgain)
        k = k / (k.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    v = x[:, H + Hkv :]
    a1, a2, vs = float(a1), float(a2), float(vs)
    v = vs / math.sqrt(a1 * a1 + a2 * a2 + 1e-8) * (a1 * v + a2 * (v if v1 is None else v1.double().cpu().reshape(v.shape)))
    return q, k, v


def logits_oracle(x, tokens, prompts, lens, rep, pres, freq, ids, bias, mask, rows):
    """64 bits, entry by entry: (y, bound on the rounding of fp32 arithmetic)."""
    B, V = x.shape
    y = x.double().cpu().clone()
    mag = y.abs()
    for b in range(B):
        if tokens is not None:
            n = int(lens[b])
            hist = tokens[b, :n].tolist()
            p0 = min(n, int(prompts[b])) if prompts is not None else 0
            for v in set(t for t in hist if 0 <= t < V):
                if rep is not None:
                    r = float(rep[b])
                    y[b, v] = y[b, v] / r if y[b, v] > 0 else y[b, v] * r
                    mag[b, v] = torch.maximum(mag[b, v], y[b, v].abs())
                c = hist[p0:].count(v)
                f = float(freq[b]) * c if freq is not None else 0.0
                q = float(pres[b]) if pres is not None and c else 0.0
                y[b, v] -= f + q
                mag[b, v] += abs(f) + abs(q)
        if ids is not None:
            for i, w in zip(ids[b].tolist(), bias[b].tolist()):
                if 0 <= i < V:
                    y[b, i] += w
                    mag[b, i] += abs(w)
        if mask is not None and int(rows[b]) >= 0:
            m = mask[int(rows[b])].tolist()
            for v in range(V):
                if not (m[v // 32] >> (v % 32)) & 1:
                    y[b, v] = -math.inf
    return y, mag
