"""Batched KV-cache text generation on this package's own model - the serving path behind the chat evaluation and the
web chat server (the reference delegates this to vLLM in evals/chat_eval.py:289-310 and to ``transformers.generate`` in
evals/chat_web.py:89-110).

* ``StaticKVCache``: keys/values in buffers allocated once for ``max_len`` positions and written in place - a decode
  step appends one column instead of re-concatenating the whole cache.
* ``SamplingParams``: n, max_tokens, temperature, top_k, top_p, stop_token_ids (the subset of vLLM's the evaluations use), and
  penalties, biases and constraints on the tokens.
* ``GraphDecoder``: the one-token decode step of a dense model as a CUDA graph over static buffers (token, position,
  per-layer K/V caches of ``max_len`` positions, a position mask): the ~12 small kernels per layer of a decode step are
  launch-bound, a graph replay issues them in one call.  The prompt is prefilled eagerly into the same buffers.
* ``EngineDecoder``: the same step on the training engine's fused kernels and bf16 weight shadows (default on a GPU).
* ``PagedDecoder`` (``ChatEngine(paged=True)``): prompts of any lengths in one batch over a paged cache; the ``n`` continuations
  of a prompt share its pages, so a prompt is prefilled, stored and read once.  Keys and values are appended by
  ``ops.qkv_post_paged`` and read by ``ops.paged_attention``; the one-token step is a CUDA graph.
* ``LogitsProcessor``: the repetition / presence / frequency penalties, ``logit_bias``, ``allowed_token_ids`` and ``choices`` of
  ``SamplingParams`` through ``ops.process_logits``.
* ``ChatEngine``: renders conversations (tokenizer chat template, else the ``<|user_start|>...`` special-token format,
  else a plain-text fallback), runs prompts of equal length as one batch (the model has no padding mask), samples on the
  device, and checks for "all rows finished" every few steps so the decode loop does not synchronise per token.
  ``stream`` yields tokens one by one for a single conversation.
"""

from __future__ import annotations

import threading
import warnings
from contextlib import nullcontext
from dataclasses import dataclass, field, replace
from pathlib import Path

import torch
from torch import Tensor

from sample_efficient_gpt_b200.models.attention import KVCache


class StaticKVCache(KVCache):
    def __init__(self, max_len: int):
        super().__init__()
        self.max_len = max_len
        self._k: Tensor | None = None
        self._v: Tensor | None = None
        self._n = 0

    @property
    def length(self) -> int:
        return self._n

    def append(self, k: Tensor, v: Tensor):
        if self._k is None:
            b, h, _, d = k.shape
            # zero-filled: positions beyond the current length are masked in attention, but 0 x NaN would still poison it
            self._k = k.new_zeros(b, h, self.max_len, d)
            self._v = v.new_zeros(b, h, self.max_len, d)
        s = k.size(2)
        if self._n + s > self.max_len:
            raise ValueError(f"KV cache overflow: {self._n}+{s} > {self.max_len}")
        self._k[:, :, self._n : self._n + s] = k
        self._v[:, :, self._n : self._n + s] = v
        self._n += s
        self.keys, self.values = self._k[:, :, : self._n], self._v[:, :, : self._n]
        return self.keys, self.values


class GraphDecoder:
    """Static-shape decode step ``(token [B,1], position) -> logits [B,V]`` captured in a CUDA graph.

    Same math as models/attention.py with every shape fixed: the new key/value are written at ``pos`` with ``index_copy_``,
    attention runs over all ``max_len`` cached positions under the mask ``arange(max_len) <= pos``.  Dense blocks only.
    """

    def __init__(self, model, batch: int, max_len: int, device, autocast):
        import torch.nn.functional as F

        self.model, self.B, self.max_len, self.device, self.autocast, self.F = model, batch, max_len, torch.device(device), autocast, F
        at = model.blocks[0].attn
        if any(b.is_moe for b in model.blocks) or at.gating not in (False, "per-head"):
            raise ValueError("graph decode supports dense blocks with per-head (or no) gating")
        self.caches = [StaticKVCache(max_len) for _ in range(model.n_layers)]
        self.token = torch.zeros(batch, 1, dtype=torch.long, device=self.device)
        self.pos = torch.zeros(1, dtype=torch.long, device=self.device)
        self.arange = torch.arange(max_len, device=self.device)
        self.logits: Tensor | None = None
        self.graph: torch.cuda.CUDAGraph | None = None

    def reset(self):
        for c in self.caches:
            c._n = 0
            c.keys = c.values = None

    def _step(self) -> Tensor:
        """The caches hold *finished* keys and values (rotated + QK-normalised keys, mixed values): per position these
        transformations do not depend on later tokens, so they are applied once, when a position is written."""
        from sample_efficient_gpt_b200.models.rope import apply_rope

        F, model, pos = self.F, self.model, self.pos
        mask = (self.arange <= pos).view(1, 1, 1, self.max_len)
        x = model.embedding(self.token)
        v1 = None
        for blk, cache in zip(model.blocks, self.caches):
            at = blk.attn
            b, h, hkv, hd = self.B, at.n_heads, at.n_kv_heads, at.head_dim
            n1 = blk.ln1(x)
            q, k, v = at.qkv(n1).split((h * hd, hkv * hd, hkv * hd), dim=-1)
            q = q.view(b, 1, h, hd).transpose(1, 2)
            k = k.view(b, 1, hkv, hd).transpose(1, 2)
            v = v.view(b, 1, hkv, hd).transpose(1, 2)
            cos, sin = at.rope.cos.index_select(0, pos), at.rope.sin.index_select(0, pos)
            q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
            vm = at.mix_values(v, v if v1 is None else v1)
            if v1 is None:
                v1 = vm
            if at.qknorm:
                q, k = at.sdpa_qknorm.normalize(q, k)
            cache._k.index_copy_(2, pos, k.to(cache._k.dtype))
            cache._v.index_copy_(2, pos, vm.to(cache._v.dtype))
            o = F.scaled_dot_product_attention(q, cache._k.to(q.dtype), cache._v.to(q.dtype), attn_mask=mask, enable_gqa=True).transpose(1, 2)
            if at.gating:
                o = (2.0 * at.attn_gate(n1).sigmoid()).unsqueeze(-1) * o
            y = x + at.out(o.reshape(b, 1, h * hd))
            x = y + blk.ffn(blk.ln2(y))
        logits = model.lm_head(model.final_norm(x))[:, -1, :]
        return logits * model.output_mult if model.output_mult != 1.0 else logits

    @torch.inference_mode()
    def prefill(self, prompt: Tensor) -> Tensor:
        """Eager forward of the prompt [B,S] into the static caches (raw: rotated keys, un-mixed values, as the model's own
        KV cache keeps them), then one pass that finishes them in place; returns the last position's logits."""
        self.reset()
        with self.autocast:
            logits, _ = self.model(prompt, kv_cache=self.caches)
            S = prompt.size(1)
            v1 = None
            for blk, cache in zip(self.model.blocks, self.caches):
                at = blk.attn
                raw_v = cache._v[:, :, :S]
                vm = at.mix_values(raw_v, raw_v if v1 is None else v1)
                if v1 is None:
                    v1 = vm.clone()
                cache._v[:, :, :S] = vm.to(cache._v.dtype)
                if at.qknorm:
                    kk = cache._k[:, :, :S]
                    cache._k[:, :, :S] = at.sdpa_qknorm.normalize(kk, kk)[1].to(cache._k.dtype)
        self.pos.fill_(prompt.size(1))
        return logits[:, -1, :]

    @torch.inference_mode()
    def step(self, tokens: Tensor) -> Tensor:
        """Feed one token per row at the current position; returns logits [B,V] (a static buffer) and advances."""
        self.token.copy_(tokens.view(self.B, 1))
        if self.device.type != "cuda":  # no graphs on the CPU: the same static-shape step, eagerly
            with self.autocast:
                self.logits = self._step()
            self.pos.add_(1)
            return self.logits
        if self.graph is None:
            side = torch.cuda.Stream(device=self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side), self.autocast:  # warm-up outside the capture (lazy initialisations, autotuning)
                for _ in range(2):
                    self._step()
            torch.cuda.current_stream(self.device).wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph), self.autocast:
                self.logits = self._step()
        self.graph.replay()
        self.pos.add_(1)
        return self.logits


class EngineDecoder:
    """Decode step on the fused kernels of the training engine (bf16 weight shadows, fused qkv+gate projection, one
    kernel each for add+RMSNorm, RoPE/QK-norm/value-mix at the cache position, gate, SwiGLU) captured in a CUDA graph:
    about a dozen launches per block instead of the several dozen of the module path.  Caches hold finished keys and values
    token-major, ``[B, max_len, Hkv, hd]``; the prompt is prefilled with the engine's forward."""

    def __init__(self, model, batch: int, max_len: int, device, engine=None):
        import torch.nn.functional as F

        from sample_efficient_gpt_b200.training.engine import FusedEngine

        self.F, self.model, self.B, self.max_len, self.device = F, model, batch, max_len, torch.device(device)
        self.eng = engine if engine is not None else FusedEngine(model, torch.bfloat16)  # bf16 copies of the weights
        at = model.blocks[0].attn
        self.H, self.Hkv, self.hd = at.n_heads, at.n_kv_heads, at.head_dim
        mk = lambda: torch.zeros(batch, max_len, self.Hkv, self.hd, dtype=torch.bfloat16, device=self.device)  # noqa: E731
        self.kc, self.vc = [mk() for _ in model.blocks], [mk() for _ in model.blocks]
        self.token = torch.zeros(batch, dtype=torch.long, device=self.device)
        self.pos = torch.zeros(1, dtype=torch.long, device=self.device)
        self.pos32 = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.arange = torch.arange(max_len, device=self.device)
        # host copies of the per-block norm scales: reading a device scalar is not allowed while a graph is captured
        self.scales = [float(b.ln1.position_scale) for b in model.blocks]
        self.final_scale = float(model.final_norm.position_scale)
        self.logits: Tensor | None = None
        self.graph: torch.cuda.CUDAGraph | None = None

    def _final(self, res, delta):
        from sample_efficient_gpt_b200 import ops

        fn = self.model.final_norm
        _, hf, _, _ = ops.add_rmsnorm_fwd(res, delta, fn.gain, self.final_scale, fn.eps, torch.bfloat16, False)
        logits = ops.matmul_nt(hf, self.eng._w(self.model.lm_head.linear.weight)).float()
        return logits * self.model.output_mult if self.model.output_mult != 1.0 else logits

    @torch.inference_mode()
    def prefill(self, prompt: Tensor) -> Tensor:
        eng, model = self.eng, self.model
        B, S = prompt.shape
        res = model.embedding.weight.detach()[prompt.reshape(-1)].float()
        delta, v1 = None, None
        for i in range(model.n_layers):
            res, delta, v, _, saved = eng._layer_fwd(i, res, delta, v1, B, S, want_kurt=False, train=False)
            if v1 is None:
                v1 = v
            self.kc[i][:, :S].copy_(saved[6].view(B, S, self.Hkv, self.hd))  # finished keys / values of the prompt
            self.vc[i][:, :S].copy_(saved[7].view(B, S, self.Hkv, self.hd))
        last = torch.arange(B, device=self.device) * S + (S - 1)
        self.pos.fill_(S)
        self.pos32.fill_(S)
        return self._final(res[last], delta[last])

    def _step(self) -> Tensor:
        from sample_efficient_gpt_b200 import ops

        eng, model, F = self.eng, self.model, self.F
        B, H, Hkv, hd, lp = self.B, self.H, self.Hkv, self.hd, torch.bfloat16
        mask = (self.arange <= self.pos).view(1, 1, 1, self.max_len)
        res = model.embedding.weight.detach()[self.token].float()
        delta, v1 = None, None
        for i, blk in enumerate(model.blocks):
            at = blk.attn
            scale = self.scales[i]
            x, n1, _, _ = ops.add_rmsnorm_fwd(res, delta, blk.ln1.gain, scale, blk.ln1.eps, lp, False)
            if i in eng.qkvz_w:
                n_qkv = at.qkv.linear.weight.size(0)
                qkvz = ops.matmul_nt(n1, eng.qkvz_w[i])
                qkv, z = qkvz[:, :n_qkv], qkvz[:, n_qkv : n_qkv + H].contiguous()
            else:
                qkv = ops.matmul_nt(n1, eng._w(at.qkv.linear.weight))
                z = ops.matmul_nt(n1, eng._w(at.attn_gate.linear.weight)) if at.gating else None
            qgain = at.sdpa_qknorm.gain if at.qknorm else eng._ones
            q, k, v = ops.qkv_post_fwd(qkv, v1, at.rope.cos, at.rope.sin, qgain, at.alpha1, at.alpha2, at.scale, B, 1, H, Hkv, hd, at.qknorm,
                                       pos=self.pos32)
            if v1 is None:
                v1 = v
            self.kc[i].index_copy_(1, self.pos, k)
            self.vc[i].index_copy_(1, self.pos, v)
            o = F.scaled_dot_product_attention(q.transpose(1, 2), self.kc[i].transpose(1, 2), self.vc[i].transpose(1, 2), attn_mask=mask,
                                               enable_gqa=True)
            o = o.transpose(1, 2).reshape(B, H, hd)
            g = ops.gate_fwd(o, z) if at.gating else o.reshape(B, H * hd)
            a = ops.matmul_nt(g, eng._w(at.out.linear.weight))
            y, n2, _, _ = ops.add_rmsnorm_fwd(x, a, blk.ln2.gain, scale, blk.ln2.eps, lp, False)
            _, f = ops.up_swiglu(n2, eng._w(blk.ffn.up.linear.weight))
            m = ops.matmul_nt(f, eng._w(blk.ffn.down.linear.weight))
            res, delta = y, m
        return self._final(res, delta)

    @torch.inference_mode()
    def step(self, tokens: Tensor) -> Tensor:
        self.token.copy_(tokens.view(self.B))
        if self.graph is None:
            side = torch.cuda.Stream(device=self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side):
                for _ in range(2):
                    self._step()
            torch.cuda.current_stream(self.device).wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.logits = self._step()
        self.graph.replay()
        self.pos.add_(1)
        self.pos32.add_(1)
        return self.logits


class PagedDecoder:
    """Prefill and one-token steps over a paged cache, dense blocks with per-head (or no) gating.

    ``start(prompts, n, budget)`` prefills the prompts (any lengths, each once) and gives the first logits of ``len(prompts) * n``
    rows; ``step(tokens)`` feeds one token per row.  With ``n`` > 1 a prompt's pages are a prefix that its rows share, and each row has
    pages of its own for ``budget`` tokens; with one row per prompt both lie in the row's pages.  The pools are kept between calls
    and replaced when a call needs more pages; tables and graph are kept for the last few shapes of a call (rows, prompts and the
    tables' widths), so that a call's kernels, and with them its results, do not depend on what was asked for before.  On a GPU bf16; on
    the CPU the statements of each op, fp32."""

    PREFILL_TOKENS = 32768  # tokens that one prefill pass takes at most (a longer prompt goes by itself)
    KEPT_SHAPES = 4  # each with a graph, whose activations and logits take up to about 0.2 GB at 256 rows

    def __init__(self, model, device, engine=None, page_size: int = 64):
        from sample_efficient_gpt_b200.training.engine import FusedEngine

        at = model.blocks[0].attn
        if any(b.is_moe for b in model.blocks) or at.gating not in (False, "per-head"):
            raise ValueError("paged decode supports dense blocks with per-head (or no) gating")
        self.model, self.device, self.P = model, torch.device(device), page_size
        self.lp = torch.bfloat16 if self.device.type == "cuda" else torch.float32
        self.eng = engine if engine is not None else FusedEngine(model, self.lp)
        self.H, self.Hkv, self.hd = at.n_heads, at.n_kv_heads, at.head_dim
        self.scales = [float(b.ln1.position_scale) for b in model.blocks]
        self.final_scale = float(model.final_norm.position_scale)
        self.pages, self.shape = 0, None
        self.graph: torch.cuda.CUDAGraph | None = None
        self.logits: Tensor | None = None
        self._kept: dict[tuple, dict] = {}  # buffers of the shapes before the present one, the latest last

    # ---- buffers
    _BUFFERS = ("token", "lens", "place", "last", "pos_base", "table", "prefix_table", "prefix_lens", "group_rows", "graph", "logits")

    @staticmethod
    def _width(pages: int) -> int:
        """A table's width for so many pages: the next 2^k or 3 * 2^k, so that neighbouring lengths share a graph."""
        power = 1 << max(0, pages - 1).bit_length()
        return 3 * power // 4 if power >= 4 and pages <= 3 * power // 4 else power

    def _reserve(self, pages: int, rows: int, width: int, groups: int, prefix_width: int):
        i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device=self.device)  # noqa: E731
        if pages > self.pages:
            # by head, so that a page's tokens of one head lie next to each other
            mk = lambda n: [torch.zeros(n, self.Hkv, self.P, self.hd, dtype=self.lp, device=self.device).transpose(1, 2) for _ in self.model.blocks]  # noqa: E731
            self.graph = None
            self._kept.clear()  # their graphs read the old pools
            ample = max(pages, self.pages * 3 // 2)
            self.pages = 0  # should they not fit
            for n in (ample, pages):  # room for larger calls to come, where there is any
                self.kp = self.vp = None  # before the new pools take their place
                try:
                    self.kp, self.vp = mk(n), mk(n)
                except torch.OutOfMemoryError:
                    if n == pages:
                        raise
                    continue
                self.pages = n
                break
        shape = (rows, self._width(width), groups, self._width(prefix_width))
        if shape == self.shape:
            return
        if self.shape is not None:
            self._kept[self.shape] = {name: getattr(self, name) for name in self._BUFFERS}
        buffers = self._kept.pop(shape, None)
        if buffers is None:
            while len(self._kept) >= self.KEPT_SHAPES:
                del self._kept[next(iter(self._kept))]
            buffers = dict(token=torch.zeros(rows, dtype=torch.long, device=self.device), lens=i32(rows), place=i32(rows), last=i32(rows), pos_base=i32(rows),
                           table=i32(rows, shape[1]), prefix_table=i32(groups, shape[3]) if groups else None, prefix_lens=i32(groups) if groups else None,
                           group_rows=i32(groups + 1) if groups else None, graph=None, logits=None)
        for name, value in buffers.items():
            setattr(self, name, value)
        self.shape = shape

    def _tables(self, prompts: list[list[int]], n: int, budget: list[int]):
        """Hands out pages and fills the tables; returns the table that the prompts are written through."""
        P, need = self.P, lambda t: -(-t // self.P)
        rows, groups = len(prompts) * n, len(prompts) if n > 1 else 0
        lens = [len(x) for x in prompts]
        own = [need(b) for b in budget for _ in range(n)] if groups else [need(t + b) for t, b in zip(lens, budget)]
        shared = [need(t) for t in lens] if groups else []
        self._reserve(sum(own) + sum(shared), rows, max(own), groups, max(shared, default=0))
        at = 0

        def fill(table: Tensor, counts: list[int]):
            nonlocal at
            host = torch.full(table.shape, -1, dtype=torch.int32)
            for i, c in enumerate(counts):
                host[i, :c] = torch.arange(at, at + c, dtype=torch.int32)
                at += c
            table.copy_(host)

        fill(self.table, own)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        if groups:
            fill(self.prefix_table, shared)
            self.prefix_lens.copy_(i32(lens))
            self.group_rows.copy_(i32([g * n for g in range(groups + 1)]))
            self.lens.zero_()
            self.pos_base.copy_(i32([t for t in lens for _ in range(n)]))
            self.last.copy_(i32([b - 1 for b in budget for _ in range(n)]))
            return self.prefix_table
        self.lens.copy_(i32(lens))
        self.pos_base.zero_()
        self.last.copy_(i32([t + b - 1 for t, b in zip(lens, budget)]))
        return self.table

    # ---- model
    def _block(self, i: int, res, delta, v1, attend):
        """One block; ``attend(i, qkv, v1, qgain)`` -> (o [T, H, hd], v1)."""
        from sample_efficient_gpt_b200 import ops

        eng, blk = self.eng, self.model.blocks[i]
        at, scale, T = blk.attn, self.scales[i], res.size(0)
        x, n1, _, _ = ops.add_rmsnorm_fwd(res, delta, blk.ln1.gain, scale, blk.ln1.eps, self.lp, False)
        if i in eng.qkvz_w:
            n_qkv = at.qkv.linear.weight.size(0)
            qkvz = ops.matmul_nt(n1, eng.qkvz_w[i])
            qkv, z = qkvz[:, :n_qkv], qkvz[:, n_qkv : n_qkv + self.H].contiguous()
        else:
            qkv = ops.matmul_nt(n1, eng._w(at.qkv.linear.weight))
            z = ops.matmul_nt(n1, eng._w(at.attn_gate.linear.weight)) if at.gating else None
        o, v1 = attend(i, qkv, v1, at.sdpa_qknorm.gain if at.qknorm else eng._ones)
        g = ops.gate_fwd(o, z) if at.gating else o.reshape(T, self.H * self.hd)
        a = ops.matmul_nt(g, eng._w(at.out.linear.weight))
        y, n2, _, _ = ops.add_rmsnorm_fwd(x, a, blk.ln2.gain, scale, blk.ln2.eps, self.lp, False)
        _, f = ops.up_swiglu(n2, eng._w(blk.ffn.up.linear.weight))
        return y, ops.matmul_nt(f, eng._w(blk.ffn.down.linear.weight)), v1

    def _append(self, i: int, qkv, v1, qgain, table, lens, cu, pos_base, want_k: bool, want_v: bool):
        from sample_efficient_gpt_b200 import ops

        at = self.model.blocks[i].attn
        return ops.qkv_post_paged(qkv, v1, at.rope.cos, at.rope.sin, qgain, at.alpha1, at.alpha2, at.scale, self.H, self.Hkv, self.hd, at.qknorm,
                                  self.kp[i], self.vp[i], table, lens, cu, pos_base, want_k=want_k, want_v=want_v)

    def _final(self, res, delta) -> Tensor:
        from sample_efficient_gpt_b200 import ops

        fn = self.model.final_norm
        _, hf, _, _ = ops.add_rmsnorm_fwd(res, delta, fn.gain, self.final_scale, fn.eps, self.lp, False)
        logits = ops.matmul_nt(hf, self.eng._w(self.model.lm_head.linear.weight)).float()
        return logits * self.model.output_mult if self.model.output_mult != 1.0 else logits

    def _prefill(self, prompts: list[list[int]], table: Tensor) -> Tensor:
        from sample_efficient_gpt_b200 import ops

        starts = [0]
        for x in prompts:
            starts.append(starts[-1] + len(x))
        ids = torch.tensor([t for x in prompts for t in x], dtype=torch.long, device=self.device)
        cu = torch.tensor(starts, dtype=torch.int32, device=self.device)
        none = torch.zeros(len(prompts), dtype=torch.int32, device=self.device)

        def attend(i, qkv, v1, qgain):
            q, k, v = self._append(i, qkv, v1, qgain, table, none, cu, None, True, True)
            o = torch.empty_like(q)
            for a, b in zip(starts, starts[1:]):  # causal over each prompt's own tokens, from the finished keys and values
                o[a:b] = ops.attention_fwd(q[None, a:b], k[None, a:b], v[None, a:b], True, 0, for_backward=False)[0][0]
            return o, v if v1 is None else v1

        res, delta, v1 = self.model.embedding.weight.detach()[ids].float(), None, None
        for i in range(self.model.n_layers):
            res, delta, v1 = self._block(i, res, delta, v1, attend)
        last = cu[1:].long() - 1
        return self._final(res[last], delta[last])

    def _step(self) -> Tensor:
        from sample_efficient_gpt_b200 import ops

        lens = self.place + 1  # with the token of this step

        def attend(i, qkv, v1, qgain):
            q, _, v = self._append(i, qkv, v1, qgain, self.table, self.place, None, self.pos_base, False, v1 is None)
            o, _ = ops.paged_attention(q, self.kp[i], self.vp[i], self.table, lens, self.prefix_table, self.prefix_lens, self.group_rows)
            return o, v if v1 is None else v1

        res, delta, v1 = self.model.embedding.weight.detach()[self.token].float(), None, None
        for i in range(self.model.n_layers):
            res, delta, v1 = self._block(i, res, delta, v1, attend)
        return self._final(res, delta)

    @torch.inference_mode()
    def start(self, prompts: list[list[int]], n: int, budget: int | list[int]) -> Tensor:
        """Logits [len(prompts) * n, V] after the prompts, with the model's weights as they are now; the rows of a prompt lie next to each
        other.  ``budget``: tokens that rows may take, one number or one for each prompt; a row that has taken them must not be active
        any more."""
        budget = [budget] * len(prompts) if isinstance(budget, int) else list(budget)
        if not prompts or not all(prompts) or n < 1 or len(budget) != len(prompts) or min(budget) < 1:
            raise ValueError("start() needs prompts of at least one token, n >= 1 and budget >= 1")
        vocab = self.model.embedding.weight.size(0)
        if any(min(x) < 0 or max(x) >= vocab for x in prompts):  # on the device a failing index would end the process
            raise ValueError(f"a prompt's tokens lie in [0, {vocab})")
        longest = max(len(x) + b for x, b in zip(prompts, budget))
        if longest > self.model.blocks[0].attn.rope.cos.size(0):
            raise ValueError(f"{longest} positions do not fit the model's rotation table")
        self.eng.refresh_shadows()  # gains and embeddings are read where they are, the matrices through copies
        table, out, a = self._tables(prompts, n, budget), [], 0
        while a < len(prompts):
            b, tokens = a + 1, len(prompts[a])
            while b < len(prompts) and tokens + len(prompts[b]) <= self.PREFILL_TOKENS:
                tokens += len(prompts[b])
                b += 1
            out.append(self._prefill(prompts[a:b], table[a:b]))
            a = b
        return torch.cat(out).repeat_interleave(n, dim=0)

    @torch.inference_mode()
    def step(self, tokens: Tensor, active: Tensor | None = None) -> Tensor:
        """Feed one token per row; logits [R, V] (a static buffer).  Rows that are not ``active`` stay where they are: their tokens go to
        the place behind their last one, or, where they have taken their whole budget, to the last."""
        if self.shape is None:
            raise ValueError("start() comes before step()")
        if tokens.numel() != self.token.numel() or (active is not None and active.shape != self.token.shape):
            raise ValueError(f"step() takes one token for each of {self.token.numel()} rows, and as many flags")
        self.token.copy_(tokens.view(-1))
        if active is None:
            self.place.copy_(self.lens)
        else:
            torch.minimum(self.lens, self.last, out=self.place)
            torch.where(active.to(torch.bool), self.lens, self.place, out=self.place)
        if self.device.type != "cuda":
            self.logits = self._step()
        else:
            with torch.cuda.device(self.device):  # a capture records the current device's streams
                if self.graph is None:
                    side = torch.cuda.Stream()
                    side.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.stream(side):
                        for _ in range(2):
                            self._step()
                    torch.cuda.current_stream().wait_stream(side)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        self.logits = self._step()
                    self.graph = graph  # only a capture that came to its end is replayed
                self.graph.replay()
        self.lens.add_(1 if active is None else active.to(torch.bool))
        return self.logits


@dataclass
class SamplingParams:
    n: int = 1
    max_tokens: int = 512
    temperature: float = 0.0
    top_k: int | None = 50
    top_p: float = 1.0
    stop_token_ids: list[int] = field(default_factory=list)
    seed: int | None = None
    repetition_penalty: float = 1.0  # on tokens of the prompt and the answer: > 1 makes them less likely
    presence_penalty: float = 0.0  # on tokens of the answer, once
    frequency_penalty: float = 0.0  # on tokens of the answer, per occurrence
    logit_bias: dict[int, float] | None = None
    allowed_token_ids: list[int] | None = None  # no other token is sampled (stop tokens neither, unless they are listed)
    choices: list[list[int]] | None = None  # the answer is one of these token sequences, none of which begins another

    @property
    def penalised(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0


class LogitsProcessor:
    """What ``SamplingParams`` asks to be done to a batch's logits before sampling, and the state that it needs."""

    def __init__(self, p: SamplingParams, rows: list[list[int]], budget: int, vocab: int, device):
        self.p, self.device = p, device
        R, i32 = len(rows), lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        full = lambda v: torch.full((R,), float(v), device=device)  # noqa: E731
        self.args: dict = {}
        if p.penalised:
            # 1e30 times a count of 2^29 and a logit of 1e8 stay finite in fp32.  A row whose allowed tokens all overflow to -inf could not be
            # sampled: on the device that is a failing assertion.
            if not 1e-30 <= p.repetition_penalty <= 1e30:
                raise ValueError("repetition_penalty must be positive, finite and within 1e-30 .. 1e30")
            if not all(abs(v) <= 1e29 for v in (p.presence_penalty, p.frequency_penalty)):
                raise ValueError("presence and frequency penalties must be finite, 1e29 at most")
            lens = [len(x) for x in rows]
            history = torch.full((R, max(lens) + budget), -1, dtype=torch.int32)
            for r, x in enumerate(rows):
                history[r, : len(x)] = torch.tensor(x, dtype=torch.int32)
            self.args.update(tokens=history.to(device), prompt_lens=i32(lens), token_lens=i32(lens), repetition=full(p.repetition_penalty),
                             presence=full(p.presence_penalty), frequency=full(p.frequency_penalty))
        if p.logit_bias:
            if any(not 0 <= t < vocab or not abs(v) <= 1e38 for t, v in p.logit_bias.items()):
                raise ValueError(f"logit_bias takes finite values, 1e38 at most, for tokens in [0, {vocab})")
            self.args.update(bias_ids=i32(list(p.logit_bias)).expand(R, -1).contiguous(),
                             bias_values=torch.tensor(list(p.logit_bias.values()), dtype=torch.float32, device=device).expand(R, -1).contiguous())
        self.state: Tensor | None = None
        if p.allowed_token_ids is not None or p.choices is not None:
            if p.allowed_token_ids is not None and p.choices is not None:
                raise ValueError("allowed_token_ids and choices exclude each other")
            nodes = [dict.fromkeys(p.allowed_token_ids)] if p.allowed_token_ids is not None else self._trie(p.choices)
            if not nodes[0] or any(not 0 <= t < vocab for node in nodes for t in node):
                raise ValueError(f"the answer must be allowed at least one token, all in [0, {vocab})")
            bits = torch.zeros(len(nodes), (vocab + 31) // 32 * 32, dtype=torch.bool)
            for i, node in enumerate(nodes):
                bits[i, list(node)] = True
            words = (bits.view(len(nodes), -1, 32).long() << torch.arange(32)).sum(-1)
            self.args.update(mask=torch.where(words >= 2**31, words - 2**32, words).to(torch.int32).to(device), mask_rows=i32([0] * R))
            if p.choices is not None:
                # the next node of every node and child token; node len(nodes): the answer is complete (all tokens allowed, none used)
                wide = max(len(node) for node in nodes)
                self.children = torch.tensor([list(node) + [-1] * (wide - len(node)) for node in nodes] + [[-1] * wide], device=device)
                self.next = torch.tensor([list(node.values()) + [0] * (wide - len(node)) for node in nodes] + [[len(nodes)] * wide], device=device)
                self.end, self.state = len(nodes), torch.zeros(R, dtype=torch.long, device=device)

    @staticmethod
    def _trie(choices: list[list[int]]) -> list[dict[int, int]]:
        """Nodes as {token: next node}; the node behind a choice's last token is len(nodes)."""
        nodes: list[dict[int, int | None]] = [{}]
        for choice in choices:
            at = 0
            for k, t in enumerate(choice):
                last = k == len(choice) - 1
                if t in nodes[at] and (last or nodes[at][t] is None):
                    if last and nodes[at][t] is None:
                        break  # the same choice again
                    raise ValueError("no choice may begin another one")
                if t not in nodes[at]:
                    nodes[at][t] = None if last else len(nodes)
                    if not last:
                        nodes.append({})
                if not last:
                    at = nodes[at][t]
        if not all(choices):
            raise ValueError("a choice has at least one token")
        return [{t: len(nodes) if nxt is None else nxt for t, nxt in node.items()} for node in nodes]

    def __call__(self, logits: Tensor) -> Tensor:
        from sample_efficient_gpt_b200 import ops

        if not self.args:
            return logits
        return ops.process_logits(logits.float() if logits.dtype == torch.float16 else logits, **self.args)

    def push(self, tokens: Tensor) -> Tensor | None:
        """Take the sampled tokens [R] into account; rows whose choice is complete (or None)."""
        if self.p.penalised:
            self.args["tokens"].scatter_(1, self.args["token_lens"].long()[:, None].clamp(max=self.args["tokens"].size(1) - 1), tokens[:, None].to(torch.int32))
            self.args["token_lens"] = (self.args["token_lens"] + 1).clamp(max=self.args["tokens"].size(1))
        if self.state is None:
            return None
        hit = self.children[self.state] == tokens[:, None]
        self.state = torch.where(hit, self.next[self.state], 0).sum(-1).where(self.state != self.end, self.state)
        self.args["mask_rows"] = torch.where(self.state == self.end, -1, self.state).to(torch.int32)
        return self.state == self.end


def sample_next(logits: Tensor, p: SamplingParams, gen: torch.Generator | None = None) -> Tensor:
    """logits [B,V] -> token ids [B]."""
    if p.temperature <= 0:
        return logits.argmax(-1)
    logits = logits.float() / p.temperature
    if p.top_k and p.top_k < logits.size(-1):
        kth = logits.topk(p.top_k, dim=-1).values[:, -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    probs = logits.softmax(-1)
    if p.top_p < 1.0:
        sp, si = probs.sort(-1, descending=True)
        keep = sp.cumsum(-1) - sp < p.top_p  # always keeps the most likely token
        probs = torch.zeros_like(probs).scatter_(-1, si, sp * keep)
        probs = probs / probs.sum(-1, keepdim=True)
    return torch.multinomial(probs, 1, generator=gen).squeeze(-1)


SPECIAL_FORMAT = ("<|bos|>", "<|user_start|>", "<|user_end|>", "<|assistant_start|>", "<|assistant_end|>")


def _message_text(content) -> str:
    if isinstance(content, str):
        return content
    return "".join(part.get("text", "") for part in content)


class ChatEngine:
    def __init__(self, model, tokenizer, device="cpu", max_model_len: int = 2048, chat_template: str | None = None,
                 dtype: torch.dtype | None = None, sync_every: int = 16, cuda_graphs: bool | None = None, cast_weights: bool = False,
                 fused_decode: bool | None = None, paged: bool = False):
        """``paged``: decode over a paged cache (``PagedDecoder``), prompts of any lengths in one batch."""
        self.model, self.tokenizer, self.device = model.to(device).eval(), tokenizer, torch.device(device)
        self.max_model_len, self.chat_template, self.sync_every = max_model_len, chat_template, sync_every
        self.autocast = (torch.autocast("cuda", dtype=dtype or torch.bfloat16) if self.device.type == "cuda" else nullcontext())
        if cast_weights and self.device.type == "cuda" and (dtype or torch.bfloat16) != torch.float32:
            # serving: keep the weights in the compute dtype instead of re-casting fp32 masters on every decode step
            for prm in self.model.parameters():  # matrices only: gains, scalars, rotary tables and norm scales stay fp32
                if prm.ndim >= 2:
                    prm.data = prm.data.to(dtype or torch.bfloat16)
        vocab = tokenizer.get_vocab() if hasattr(tokenizer, "get_vocab") else {}
        self._special = {t: vocab[t] for t in SPECIAL_FORMAT if t in vocab}
        dense = not any(b.is_moe for b in self.model.blocks) and self.model.blocks[0].attn.gating in (False, "per-head")
        self.cuda_graphs = (self.device.type == "cuda" and dense) if cuda_graphs is None else (cuda_graphs and self.device.type == "cuda")
        self._decoders: dict = {}  # batch size -> decoder (caches for max_model_len positions)
        # decode on the engine's fused kernels when they are built and apply (bf16, dense, per-head or no gate)
        from sample_efficient_gpt_b200 import ops as _ops

        can_fuse = (self.cuda_graphs and (dtype or torch.bfloat16) == torch.bfloat16 and _ops.ext() is not None
                    and self.model.blocks[0].attn.head_dim % 16 == 0)
        self.fused_decode = can_fuse if fused_decode is None else (fused_decode and can_fuse)
        if paged and not dense:
            raise ValueError("paged decode supports dense blocks with per-head (or no) gating")
        if paged and self.device.type == "cuda" and (dtype or torch.bfloat16) != torch.bfloat16:
            raise ValueError("paged decode runs in bfloat16 on a GPU")
        self.paged = PagedDecoder(self.model, self.device) if paged else None
        self._paged_turn = threading.Lock()

    # ---- prompt rendering -------------------------------------------------------------------------------------------
    def render(self, messages: list[dict]) -> list[int]:
        tok = self.tokenizer
        template = self.chat_template or getattr(tok, "chat_template", None)
        if template:
            out = tok.apply_chat_template(messages, chat_template=template, add_generation_prompt=True, tokenize=True)
            return list(out["input_ids"] if hasattr(out, "keys") else out)
        enc = lambda s: list(tok.encode(s, add_special_tokens=False))
        if len(self._special) == len(SPECIAL_FORMAT):
            sp = self._special
            ids = [sp["<|bos|>"]]
            for m in messages:
                role = "user" if m["role"] in ("user", "system") else "assistant"
                ids += [sp[f"<|{role}_start|>"]] + enc(_message_text(m["content"])) + [sp[f"<|{role}_end|>"]]
            return ids + [sp["<|assistant_start|>"]]
        text = "".join(f"{m['role'].capitalize()}: {_message_text(m['content'])}\n" for m in messages) + "Assistant:"
        return enc(text)

    def default_stop_ids(self) -> list[int]:
        vocab = self.tokenizer.get_vocab() if hasattr(self.tokenizer, "get_vocab") else {}
        ids = [vocab[t] for t in ("<|endoftext|>", "<|assistant_end|>") if t in vocab]
        eos = getattr(self.tokenizer, "eos_token_id", None)
        return ids + ([eos] if eos is not None and eos not in ids else [])

    # ---- decoding ---------------------------------------------------------------------------------------------------
    @torch.inference_mode()
    def _decode_batch(self, prompt: Tensor, p: SamplingParams, gen=None, on_token=None) -> list[list[int]]:
        """prompt [B,S] (same length for every row) -> new token ids per row (stop token excluded)."""
        B, S = prompt.shape
        budget = min(p.max_tokens, self.max_model_len - S)
        if budget <= 0:
            return [[] for _ in range(B)]
        stop = torch.tensor(sorted(set(p.stop_token_ids)), device=self.device, dtype=torch.long)
        out = torch.zeros(B, budget, dtype=torch.long, device=self.device)
        done = torch.zeros(B, dtype=torch.bool, device=self.device)
        rows = prompt.tolist() if p.penalised else [[]] * B  # a copy from the device only where it is needed
        process = LogitsProcessor(p, rows, budget, self.model.vocab_size, self.device)
        step_in, steps = prompt, 0
        decoder = None
        if self.cuda_graphs:
            decoder = self._decoders.get(B)
            if decoder is None:
                if self.fused_decode:
                    shared = next((d.eng for d in self._decoders.values() if isinstance(d, EngineDecoder)), None)
                    decoder = self._decoders[B] = EngineDecoder(self.model, B, self.max_model_len, self.device, shared)
                else:
                    decoder = self._decoders[B] = GraphDecoder(self.model, B, self.max_model_len, self.device, self.autocast)
        else:
            caches = [StaticKVCache(S + budget) for _ in range(self.model.n_layers)]
        with self.autocast:
            for t in range(budget):
                if decoder is not None:
                    last = decoder.prefill(prompt) if t == 0 else decoder.step(step_in)
                else:
                    last = self.model(step_in, kv_cache=caches)[0][:, -1, :]
                nxt = sample_next(process(last), p, gen)
                if stop.numel():
                    done = done | torch.isin(nxt, stop)
                out[:, t] = torch.where(done, torch.full_like(nxt, -1), nxt)
                complete = process.push(nxt)
                if complete is not None:
                    done = done | complete
                step_in, steps = nxt[:, None], t + 1
                if on_token is not None:
                    token = int(out[0, t])
                    if token == -1:
                        break
                    if on_token(token) or (complete is not None and bool(complete[0])):
                        break
                elif (t + 1) % self.sync_every == 0 and bool(done.all()):
                    break
        rows = out[:, :steps].cpu().tolist()
        return [row[: row.index(-1)] if -1 in row else row for row in rows]

    MAX_PAGED_ROWS = 256

    def _kernel_status(self) -> int:
        """The package's status word of this engine's device, which is cleared by reading."""
        if self.device.type != "cuda":
            return 0
        from sample_efficient_gpt_b200.ops import gemm

        return gemm.take_status(self.device.index)

    def _decode_paged(self, prompts: list[list[int]], p: SamplingParams, gen=None, on_token=None) -> list[list[list[int]]]:
        """Prompts of any lengths, ``p.n`` rows each -> new token ids per prompt and row (stop token excluded).  Calls from several threads,
        an unfinished stream's among them, take turns: they share the decoder's tables."""
        with self._paged_turn:
            return self._decode_paged_now(prompts, p, gen, on_token)

    @torch.inference_mode()
    def _decode_paged_now(self, prompts: list[list[int]], p: SamplingParams, gen, on_token) -> list[list[list[int]]]:
        room = [min(p.max_tokens, self.max_model_len - len(x)) for x in prompts]
        live = [i for i, r in enumerate(room) if r > 0]
        results: list[list[list[int]]] = [[[] for _ in range(p.n)] for _ in prompts]
        if not live:
            return results
        budget, R = max(room[i] for i in live), len(live) * p.n
        rows = [prompts[i] for i in live for _ in range(p.n)]
        limit = torch.tensor([room[i] for i in live for _ in range(p.n)], device=self.device)
        stop = torch.tensor(sorted(set(p.stop_token_ids)), device=self.device, dtype=torch.long)
        out = torch.full((R, budget), -1, dtype=torch.long, device=self.device)
        done = torch.zeros(R, dtype=torch.bool, device=self.device)
        process = LogitsProcessor(p, rows, budget, self.model.vocab_size, self.device)
        if (code := self._kernel_status()) != 0:  # not this generation's, which is judged by what it does itself
            warnings.warn(f"a kernel had reported status {code} before this generation", RuntimeWarning, stacklevel=2)
        logits, steps = self.paged.start([prompts[i] for i in live], p.n, [room[i] for i in live]), 0
        for t in range(budget):
            if t > 0:
                logits = self.paged.step(nxt, ~done)
            nxt = sample_next(process(logits), p, gen)
            if stop.numel():
                done = done | torch.isin(nxt, stop)
            out[:, t] = torch.where(done, torch.full_like(nxt, -1), nxt)
            complete = process.push(nxt)
            done = done | (limit <= t + 1)
            if complete is not None:
                done = done | complete
            steps = t + 1
            if on_token is not None:  # one row
                token = int(out[0, t])
                if token == -1 or on_token(token) or (complete is not None and bool(complete[0])):
                    break
            elif (t + 1) % self.sync_every == 0 and bool(done.all()):
                break
        tokens = out[:, :steps].cpu().tolist()
        if (code := self._kernel_status()) != 0:
            raise RuntimeError(f"a kernel reported status {code} during generation")
        for j, i in enumerate(live):
            for k in range(p.n):
                row = tokens[j * p.n + k]
                results[i][k] = row[: row.index(-1)] if -1 in row else row
        return results

    def generate_ids(self, prompts: list[list[int]], p: SamplingParams) -> list[list[list[int]]]:
        """For each prompt, ``p.n`` continuations (token ids)."""
        gen = None
        if p.seed is not None:
            gen = torch.Generator(device=self.device).manual_seed(p.seed)
        if self.paged is not None:
            for i, ids in enumerate(prompts):
                prompts[i] = ids[-(self.max_model_len - 1):]
            at_once, rows = max(1, self.MAX_PAGED_ROWS // p.n), []
            for a in range(0, len(prompts), at_once):
                rows += self._decode_paged(prompts[a : a + at_once], p, gen)
            return rows
        results: list[list[list[int]] | None] = [None] * len(prompts)
        by_len: dict[int, list[int]] = {}
        for i, ids in enumerate(prompts):
            ids = ids[-(self.max_model_len - 1):]
            prompts[i] = ids
            by_len.setdefault(len(ids), []).append(i)
        for _, members in sorted(by_len.items()):
            batch = torch.tensor([prompts[i] for i in members for _ in range(p.n)], dtype=torch.long, device=self.device)
            rows = self._decode_batch(batch, p, gen)
            for j, i in enumerate(members):
                results[i] = rows[j * p.n : (j + 1) * p.n]
        return results  # type: ignore[return-value]

    def chat(self, conversations: list[list[dict]], p: SamplingParams) -> list[list[str]]:
        ids = self.generate_ids([self.render(c) for c in conversations], p)
        return [[self.tokenizer.decode(r, skip_special_tokens=True) for r in rows] for rows in ids]

    def stream(self, messages: list[dict], p: SamplingParams):
        """Generator of text pieces for one conversation (decodes the growing id list so multi-byte characters that span
        tokens come out whole).  Decoding ends with the answer or when the generator is closed."""
        import queue

        q: queue.Queue = queue.Queue()
        prompt = self.render(messages)[-(self.max_model_len - 1):]
        closed = threading.Event()

        def on_token(token: int) -> bool:
            q.put(token)
            return closed.is_set()

        def run():
            try:
                if self.paged is not None:
                    self._decode_paged([prompt], replace(p, n=1), None, on_token)
                else:
                    self._decode_batch(torch.tensor([prompt], dtype=torch.long, device=self.device), p, None, on_token)
            except BaseException as e:  # raised where the answer is read
                q.put(e)
            else:
                q.put(None)

        threading.Thread(target=run, daemon=True).start()
        ids: list[int] = []
        shown = ""
        try:
            while (tok := q.get()) is not None:
                if isinstance(tok, BaseException):
                    raise tok
                ids.append(tok)
                text = self.tokenizer.decode(ids, skip_special_tokens=True)
                if text.endswith("�"):
                    continue
                if len(text) > len(shown):
                    yield text[len(shown):]
                    shown = text
        finally:
            closed.set()


def load_chat_template(tokenizer_dir) -> str | None:
    """The tokenizer's own template, else a ``chat_template.jinja`` beside it (evals/chat_eval.py:25-34 of the reference)."""
    from transformers import AutoTokenizer

    tok = AutoTokenizer.from_pretrained(str(tokenizer_dir), local_files_only=True, trust_remote_code=False)
    if getattr(tok, "chat_template", None):
        return tok.chat_template
    f = Path(tokenizer_dir) / "chat_template.jinja"
    return f.read_text() if f.is_file() else None


def load_engine(checkpoint: str, device="cuda", dtype: str = "bfloat16", max_model_len: int = 2048, paged: bool = False) -> ChatEngine:
    """``checkpoint`` is a converted HF directory (config.json + weights + tokenizer) or a native ``.pt`` file.  ``paged``: see
    ``ChatEngine``."""
    path = Path(checkpoint)
    if path.is_dir():
        from transformers import AutoTokenizer

        from sample_efficient_gpt_b200.scripts.hf.run_imu1_hf import load_native_from_hf

        model, _ = load_native_from_hf(path)
        tokenizer = AutoTokenizer.from_pretrained(str(path), local_files_only=True, trust_remote_code=False)
        template = load_chat_template(path)
    else:
        from sample_efficient_gpt_b200.training.trainer import Trainer

        tr = Trainer(load_from=str(path), load_components="infer", **{"trainer.device": str(device)})
        model, tokenizer, template = tr.model, tr.tokenizer, None
    torch_dtype = {"float32": torch.float32, "bfloat16": torch.bfloat16, "auto": None}[dtype]
    return ChatEngine(model, tokenizer, device, max_model_len, template, torch_dtype, cast_weights=True, paged=paged)
