"""The paged decoder and the chat engine on the GPU around failures: status words, captures, what earlier calls leave behind."""

import warnings

import pytest
import torch

from sample_efficient_gpt_b200 import ops
from sample_efficient_gpt_b200.evals.generation import ChatEngine, PagedDecoder, SamplingParams
from sample_efficient_gpt_b200.ops import gemm

from tests.test_gpu_paged_generation import gpu_model
from tests.test_paged_generation import PROMPTS, Tok
from tests.test_streaming import TALK, ChatTok

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status():
    assert ops.ext() is not None and gemm.status() == 0
    yield
    assert gemm.take_status() == 0


def test_a_status_is_reported_once(monkeypatch):
    eng = ChatEngine(gpu_model(), Tok(), "cuda", max_model_len=64, paged=True)
    run = lambda: eng.generate_ids([list(x) for x in PROMPTS], SamplingParams(max_tokens=8, temperature=0.0))  # noqa: E731
    want = run()
    # a report that is not the generation's own
    ops.process_logits(torch.zeros(1, 64, device="cuda"), mask=torch.zeros(1, 2, dtype=torch.int32, device="cuda"),
                       mask_rows=torch.ones(1, dtype=torch.int32, device="cuda"))
    with pytest.warns(RuntimeWarning, match="status 57 before"):
        assert run() == want
    # a generation that fails: page numbers beyond the pool, which the kernels leave out
    tables = PagedDecoder._tables

    def beyond(self, *args):
        table = tables(self, *args)
        table.fill_(10**7)
        return table

    monkeypatch.setattr(PagedDecoder, "_tables", beyond)
    with pytest.raises(RuntimeError, match="status 5[24] during"):
        run()
    monkeypatch.undo()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert run() == want and run() == want


def test_results_do_not_depend_on_what_was_served_before():
    """100 rows on one prompt: behind a prompt of 16000 tokens the same short one keeps its kernels, its graph and its bits."""
    dec = PagedDecoder(gpu_model(max_seq_len=20000), "cuda")
    tokens = torch.arange(100, device="cuda")

    def served(prompt):
        out = [dec.start([prompt], 100, 40).clone()]
        for _ in range(3):
            out.append(dec.step(tokens).clone())
        return out

    short, long = [3, 4, 5, 6, 7] * 20, [i % 500 for i in range(16000)]
    want = served(short)
    graph, width = dec.graph, dec.prefix_table.size(1)
    first = served(long)
    again = served(short)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    assert dec.prefix_table.size(1) == width
    assert all(torch.equal(a, b) for a, b in zip(first, served(long)))  # and the other way round
    served(short)
    kept = dec.graph
    served(long)
    served(short)
    assert graph is not None and dec.graph is kept  # captured once for both shapes in turn


def test_a_capture_that_fails_is_made_again(monkeypatch):
    dec = PagedDecoder(gpu_model(), "cuda", page_size=16)
    tokens = torch.tensor([5, 6], device="cuda")
    dec.start(PROMPTS[:2], 1, 8)
    want = dec.step(tokens).clone()
    dec = PagedDecoder(gpu_model(), "cuda", page_size=16)
    dec.start(PROMPTS[:2], 1, 8)
    block, calls = PagedDecoder._block, []

    def fails(self, i, *args):
        calls.append(i)
        if len(calls) == 2 * self.model.n_layers + 2:  # both warm-up steps pass, the captured one ends in its second block
            raise MemoryError("no room")
        return block(self, i, *args)

    monkeypatch.setattr(PagedDecoder, "_block", fails)
    with pytest.raises(MemoryError):
        dec.step(tokens)
    monkeypatch.undo()
    assert torch.equal(dec.step(tokens), want)
    assert torch.equal(dec.step(tokens), dec.logits) and dec.graph is not None


@pytest.mark.parametrize("n", [1, 2])
def test_a_row_that_has_taken_its_budget_is_left_alone(n):
    """Nothing is reported for it, and the rows beside it get what they get by themselves."""
    m = gpu_model(max_seq_len=48)
    both, alone = PagedDecoder(m, "cuda", page_size=16), PagedDecoder(m, "cuda", page_size=16)
    prompts, budget = [list(range(32)), [7, 8, 9]], [16, 45]  # up to the rotation table's end, one of them in full pages
    both.start(prompts, n, budget)
    alone.start(prompts, n, budget)
    limit = torch.tensor([b for b in budget for _ in range(n)], device="cuda")
    for t in range(45):
        nxt = torch.arange(2 * n, device="cuda") + t
        a = both.step(nxt, limit > t)
        if t < 16:
            alone.step(nxt)
        else:  # the same rows with the first ones put back to where they were
            with torch.inference_mode():
                alone.lens[:n] -= 1
            assert torch.equal(a[n:], alone.step(nxt)[n:])
    assert gemm.status() == 0


def test_streams_of_a_paged_engine():
    """Captured on the stream's own thread; the same tokens as the whole answer, again and beside other calls."""
    eng = ChatEngine(gpu_model(), ChatTok(), "cuda", max_model_len=96, paged=True)
    p = SamplingParams(max_tokens=24, temperature=0.0)
    parts = "".join(eng.stream(TALK, p))
    assert parts == eng.chat([TALK], p)[0][0] == "".join(eng.stream(TALK, p)) and len(parts.split()) == 24
    stream = eng.stream(TALK, p)
    head = next(stream)
    other = eng.generate_ids([list(PROMPTS[2])], SamplingParams(n=3, max_tokens=12, temperature=0.0))  # waits for its turn
    assert head + "".join(stream) == parts and other[0][0] == other[0][2]
    choice = "".join(eng.stream(TALK, SamplingParams(max_tokens=24, temperature=0.0, choices=[[10, 11, 12], [20]])))
    assert choice in ("10 11 12", "20")
    assert not eng._decoders  # no static caches beside the pages


def test_constraints_of_an_engine_in_half_precision():
    """Its logits are fp16, which the kernel does not take."""
    eng = ChatEngine(gpu_model(), Tok(), "cuda", max_model_len=64, dtype=torch.float16)
    run = lambda **kw: eng.generate_ids([[3, 4, 5], [3, 4, 5, 6]], SamplingParams(**{**dict(max_tokens=8, temperature=0.0), **kw}))  # noqa: E731
    assert {t for r in run(allowed_token_ids=[7, 200, 511], temperature=1.0, seed=0) for t in r[0]} <= {7, 200, 511}
    assert all(set(r[0]) == {33} for r in run(logit_bias={33: 1e9}))  # beyond fp16
    assert all(len(set(r[0])) == 8 for r in run(frequency_penalty=1e6))


@pytest.mark.parametrize("kw", [dict(attn_qknorm=False), dict(attn_val_residual=False), dict(attn_qknorm=False, attn_gating=False, attn_val_residual=False),
                                dict(n_heads=8, n_kv_heads=8), dict(n_heads=2, n_kv_heads=1), dict(weight_tying=False)])
@pytest.mark.parametrize("n", [1, 3])
def test_logits_of_other_models_track_the_module_path(kw, n):
    """Without QK-norm, value residual or gate; heads of 32 and of 128: bf16 kernels against the fp32 module path, as the default model is
    held to it."""
    m = gpu_model(**kw)
    dec = PagedDecoder(m, "cuda", page_size=16)
    rows = [list(x) for x in PROMPTS for _ in range(n)]
    logits = dec.start(PROMPTS, n, 24)
    g = torch.Generator().manual_seed(0)
    for _ in range(12):
        with torch.no_grad():
            want = torch.stack([m(torch.tensor([r], device="cuda"))[0][0, -1] for r in rows])
        assert torch.allclose(logits.float(), want, atol=0.15, rtol=0.05), float((logits - want).abs().max())
        nxt = torch.randint(0, 512, (len(rows),), generator=g)
        for r, t in zip(rows, nxt.tolist()):
            r.append(t)
        logits = dec.step(nxt.cuda())


def test_a_prefill_of_many_tokens_is_the_module_paths():
    """Prompts long enough for the append kernel's ring in every layer, over page borders; then a few steps."""
    m = gpu_model(max_seq_len=4096)
    dec = PagedDecoder(m, "cuda", page_size=64)
    prompts = [[(7 * i + b) % 512 for i in range(n)] for b, n in enumerate((3000, 1, 1501, 64))]
    rows = [list(x) for x in prompts]
    logits = dec.start(prompts, 1, 8)
    for t in range(4):
        with torch.no_grad():
            want = torch.stack([m(torch.tensor([r], device="cuda"))[0][0, -1] for r in rows])
        assert torch.allclose(logits.float(), want, atol=0.15, rtol=0.05), float((logits - want).abs().max())
        nxt = torch.arange(4) + t
        for r, x in zip(rows, nxt.tolist()):
            r.append(x)
        logits = dec.step(nxt.cuda())


@pytest.mark.parametrize("cast", [False, True])
def test_weights_that_change_between_calls(cast):
    m = gpu_model()
    eng = ChatEngine(m, Tok(), "cuda", max_model_len=64, paged=True, cast_weights=cast)
    dec = eng.paged
    dec.start(PROMPTS, 2, 5)
    dec.step(torch.arange(8, device="cuda"))
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(0.75)
    fresh = PagedDecoder(m, "cuda")
    assert torch.equal(dec.start(PROMPTS, 2, 5), fresh.start(PROMPTS, 2, 5))
    for _ in range(3):  # the step captured before
        assert torch.equal(dec.step(torch.arange(8, device="cuda")), fresh.step(torch.arange(8, device="cuda")))
