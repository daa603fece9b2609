"""The paged decoder on the CPU (fp32 statements of each op): what earlier calls leave behind, rows at their limits."""

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from sample_efficient_gpt_b200.evals.generation import ChatEngine, LogitsProcessor, PagedDecoder, SamplingParams

from tests.test_paged_generation import PROMPTS, Tok, model


@pytest.mark.parametrize("n", [1, 3])
def test_buffers_do_not_depend_on_earlier_calls(n):
    """The kernels are chosen by the tables' widths: a short batch after a long one is laid out as it would be by itself."""
    m = model()
    dec, fresh = PagedDecoder(m, "cpu", page_size=4), PagedDecoder(m, "cpu", page_size=4)
    short, long = [[3, 4, 5], [6, 7]], [[1 + i % 50 for i in range(300)], [2] * 200]
    want = fresh.start(short, n, 5)
    dec.start(long, n, 9)
    assert torch.equal(dec.start(short, n, 5), want)
    for name in ("table", "prefix_table", "lens", "token"):
        a, b = getattr(dec, name), getattr(fresh, name)
        assert (a is None) == (b is None) and (a is None or (a.shape == b.shape and torch.equal(a, b)))
    # many shapes in turn: only the last few are kept, and each gives its own results again
    firsts = [dec.start([p], n, 4) for p in PROMPTS]
    for b in range(2, 9):
        dec.start([[5] * (7 * b)] * b, n, 4)
    assert len(dec._kept) <= dec.KEPT_SHAPES
    for p, want in zip(PROMPTS, firsts):
        assert torch.equal(dec.start([p], n, 4), want)


def test_width_of_a_table():
    got = [PagedDecoder._width(n) for n in range(1, 34)]
    assert got == [1, 2, 3, 4, 6, 6, 8, 8] + [12] * 4 + [16] * 4 + [24] * 8 + [32] * 8 + [48]


@pytest.mark.parametrize("n", [1, 2])
def test_a_row_that_has_taken_its_budget_beside_others(n):
    """It must not be active any more; the others go on, up to the last position of the rotation table."""
    m = model(max_seq_len=12)
    dec = PagedDecoder(m, "cpu", page_size=4)
    prompts, budget = [[3, 4, 5, 6], [7, 8]], [8, 6]  # 12 and 8 positions; full pages where a prompt has one row
    rows = [list(x) for x in prompts for _ in range(n)]
    limit = torch.tensor([b for b in budget for _ in range(n)])
    dec.start(prompts, n, budget)
    for t in range(10):
        nxt = torch.arange(len(rows)) + t
        active = limit > t
        logits = dec.step(nxt, active)
        for r, ids in enumerate(rows):
            if bool(active[r]):
                ids.append(int(nxt[r]))
                assert torch.allclose(logits[r], m(torch.tensor([ids]))[0][0, -1], atol=2e-4, rtol=1e-4)
    assert [len(x) for x in rows] == [12] * n + [8] * n


def test_two_calls_at_once():
    """Two threads on one engine: each gets what it gets by itself."""
    eng = ChatEngine(model(), Tok(), "cpu", max_model_len=40, paged=True)
    p = SamplingParams(max_tokens=12, temperature=0.0)
    asked = [[list(x)] for x in PROMPTS[:3]] + [[list(x) for x in PROMPTS[1:3]]]
    want = [eng.generate_ids([list(x) for x in a], p) for a in asked]
    with ThreadPoolExecutor(len(asked)) as pool:
        for _ in range(3):
            assert list(pool.map(lambda a: eng.generate_ids([list(x) for x in a], p), asked)) == want


def test_parameters_that_32_bits_cannot_hold_are_refused():
    mk = lambda **kw: LogitsProcessor(SamplingParams(**kw), [[1], [2]], 4, 61, "cpu")  # noqa: E731
    for kw in (dict(repetition_penalty=1e39), dict(presence_penalty=-1e39), dict(frequency_penalty=1e39), dict(logit_bias={1: 1e39}), dict(logit_bias={1: -1e40})):
        with pytest.raises(ValueError, match="finite"):
            mk(**kw)
    with pytest.raises(ValueError, match="positive"):
        mk(repetition_penalty=1e-50)


def test_allowed_tokens_stay_finite():
    """Whatever the parameters, an allowed token can be sampled: 2^29 occurrences is the most that a history counts."""
    for kw in (dict(frequency_penalty=1e38), dict(frequency_penalty=-3e38), dict(presence_penalty=2e38), dict(repetition_penalty=3e38), dict(repetition_penalty=1e-38),
               dict(logit_bias={5: -3e38})):
        with pytest.raises(ValueError):
            LogitsProcessor(SamplingParams(allowed_token_ids=[5], **kw), [[5] * 40], 4, 61, "cpu")
    largest = dict(frequency_penalty=1e29, presence_penalty=1e29, logit_bias={5: -1e38})
    for kw in (dict(repetition_penalty=1e30, **largest), dict(repetition_penalty=1e-30, **largest)):
        proc = LogitsProcessor(SamplingParams(allowed_token_ids=[5], **kw), [[5] * 40], 4, 61, "cpu")
        for x in (torch.full((1, 61), -1e8), torch.full((1, 61), 1e8)):
            for _ in range(4):
                proc.push(torch.tensor([5]))
            y = proc(x)
            assert torch.isfinite(y[0, 5]) and int(torch.isfinite(y).sum()) == 1
    assert 1e29 * 2.0**29 + 1e29 + 1e38 + 1e38 < torch.finfo(torch.float32).max


@pytest.mark.parametrize("token", [-1, 61, 10**9])
def test_prompts_of_tokens_that_do_not_exist_are_refused(token):
    dec = PagedDecoder(model(), "cpu")
    want = dec.start(PROMPTS, 2, 5)
    with pytest.raises(ValueError, match="tokens lie in"):
        dec.start([[3, 4], [5, token, 6]], 2, 5)
    assert torch.equal(dec.start(PROMPTS, 2, 5), want)


def test_steps_that_do_not_fit_the_rows_are_refused():
    """One token for several rows would have been taken by all of them."""
    dec = PagedDecoder(model(), "cpu")
    with pytest.raises(ValueError, match="start"):
        dec.step(torch.tensor([1]))
    dec.start(PROMPTS, 1, 5)
    for tokens, active in ((torch.tensor([1]), None), (torch.arange(5), None), (torch.arange(4), torch.tensor([True])), (torch.arange(4), torch.ones(4, 1, dtype=torch.bool))):
        with pytest.raises(ValueError, match="4 rows"):
            dec.step(tokens, active)
    assert dec.step(torch.arange(4)[:, None], torch.ones(4, dtype=torch.bool)).shape == (4, 61)


def test_pools_that_grow_take_what_there_is(monkeypatch):
    """Half as much again is room for later calls, not a need: a call that fits without it is served."""
    dec = PagedDecoder(model(), "cpu", page_size=4)
    dec.start([[3] * 40], 1, 40)  # 20 pages
    make, asked = torch.zeros, []

    def limited(*size, **kw):
        if len(size) == 4:
            asked.append(size[0])
            if size[0] > 25:
                raise torch.OutOfMemoryError("no room")
        return make(*size, **kw)

    monkeypatch.setattr(torch, "zeros", limited)
    got = dec.start([[3] * 48], 1, 40)  # 22 pages
    assert dec.pages == 22 and asked[0] == 30 and len(dec.kp) == len(dec.vp) == 3
    with pytest.raises(torch.OutOfMemoryError):
        dec.start([[3] * 80], 1, 40)
    assert dec.pages == 0
    assert torch.equal(dec.start([[3] * 48], 1, 40), got)


def test_weights_that_change_between_calls():
    """Each call runs with all of the model's weights as they are, not with some of an earlier time."""
    m = model()
    dec = PagedDecoder(m, "cpu", page_size=4)
    dec.start(PROMPTS, 2, 5)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(1.25).add_(0.01)
    fresh = PagedDecoder(m, "cpu", page_size=4)
    assert torch.equal(dec.start(PROMPTS, 2, 5), fresh.start(PROMPTS, 2, 5))
    for _ in range(3):
        assert torch.equal(dec.step(torch.arange(8)), fresh.step(torch.arange(8)))
    want = torch.stack([m(torch.tensor([x]))[0][0, -1] for x in PROMPTS]).repeat_interleave(2, 0)
    assert torch.allclose(dec.start(PROMPTS, 2, 5), want, atol=2e-4, rtol=1e-4)


@pytest.mark.parametrize("dtype", [torch.bool, torch.int32, torch.int64, torch.float32])
def test_flags_of_any_type(dtype):
    """Whatever is not zero is active, by one token."""
    dec = PagedDecoder(model(), "cpu", page_size=4)
    dec.start(PROMPTS, 1, 5)
    flags = torch.tensor([1, 0, 3, 0]).to(dtype)
    before = dec.lens.clone()
    dec.step(torch.arange(4), flags)
    assert torch.equal(dec.lens - before, torch.tensor([1, 0, 1, 0], dtype=torch.int32))
