"""Generation over a paged cache and the processing of logits in the chat engine, on the CPU (fp32 statements of each op)."""

import pytest
import torch

from sample_efficient_gpt_b200.config_schema import ModelConfig
from sample_efficient_gpt_b200.evals.generation import ChatEngine, LogitsProcessor, PagedDecoder, SamplingParams
from sample_efficient_gpt_b200.models import build_model


class Tok:
    eos_token_id = None
    chat_template = None

    def get_vocab(self):
        return {}

    def decode(self, ids, skip_special_tokens=True):
        return " ".join(map(str, ids))


def model(**kw):
    torch.manual_seed(0)
    cfg = dict(d_model=64, d_ff=128, n_layers=3, n_heads=4, n_kv_heads=2, vocab_size=61, attn_qknorm=True, attn_val_residual=True, attn_gating="per-head",
               layernorm_scaling=True)
    m = build_model(ModelConfig(**{**cfg, **kw})).eval()
    with torch.no_grad():  # the mix of first and later values, the query gain: not their neutral starting values
        for i, b in enumerate(m.blocks):
            for name, v in (("alpha1", 0.9), ("alpha2", 0.3 + 0.1 * i), ("scale", 1.1)):
                if isinstance(getattr(b.attn, name), torch.nn.Parameter):
                    getattr(b.attn, name).fill_(v)
            if b.attn.qknorm:
                b.attn.sdpa_qknorm.gain.fill_(1.4)
    return m


PROMPTS = [[3, 4, 5, 6, 7], [9, 8], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [9, 8]]


@pytest.mark.parametrize("kw", [dict(), dict(attn_qknorm=False, attn_gating=False), dict(attn_val_residual=False, n_kv_heads=4)])
def test_paged_greedy_is_the_plain_decode(kw):
    m = model(**kw)
    plain, paged = ChatEngine(m, Tok(), "cpu", max_model_len=40), ChatEngine(m, Tok(), "cpu", max_model_len=40, paged=True)
    paged.paged.P = 4  # pages that end inside prompts and answers
    p = SamplingParams(max_tokens=14, temperature=0.0)
    a = plain.generate_ids([list(x) for x in PROMPTS], p)
    assert paged.generate_ids([list(x) for x in PROMPTS], p) == a
    # continuations that share their prompt's pages: greedy, so all alike
    assert paged.generate_ids([list(x) for x in PROMPTS], SamplingParams(n=3, max_tokens=14, temperature=0.0)) == [[r[0]] * 3 for r in a]
    # the same buffers again, for fewer and shorter rows
    assert paged.generate_ids([list(PROMPTS[1])], p) == [a[1]]


def test_a_long_prompt_beside_a_short_one():
    """Each row stops where its own prompt leaves no room, up to the last position of the rotation table."""
    m = model(max_seq_len=40)
    prompts = [[5] * 37, [7, 8, 9]]
    for n in (1, 2):
        p = SamplingParams(n=n, max_tokens=100, temperature=0.0)
        a = ChatEngine(m, Tok(), "cpu", max_model_len=40).generate_ids([list(x) for x in prompts], p)
        engine = ChatEngine(m, Tok(), "cpu", max_model_len=40, paged=True)
        engine.paged.P = 4
        assert engine.generate_ids([list(x) for x in prompts], p) == a and [len(r[0]) for r in a] == [3, 37]


def test_decoder_survives_pools_that_do_not_fit(monkeypatch):
    m = model()
    dec = PagedDecoder(m, "cpu", page_size=4)
    want = dec.start(PROMPTS[:2], 1, 3).clone()
    make = torch.zeros

    def limited(*size, **kw):
        if len(size) == 4:
            raise torch.OutOfMemoryError("no room")
        return make(*size, **kw)

    monkeypatch.setattr(torch, "zeros", limited)
    with pytest.raises(torch.OutOfMemoryError):
        dec.start(PROMPTS, 3, 9)
    monkeypatch.undo()
    assert torch.equal(dec.start(PROMPTS[:2], 1, 3), want)


def test_paged_step_logits_match_the_full_forward():
    m = model()
    dec = PagedDecoder(m, "cpu", page_size=3)
    prompts = [[3, 4, 5, 6], [7, 8], [9]]
    rows = [list(x) for x in prompts for _ in range(2)]
    logits = dec.start(prompts, 2, 6).clone()
    g = torch.Generator().manual_seed(1)
    for t in range(6):
        for r, ids in enumerate(rows):
            want = m(torch.tensor([ids]))[0][0, -1]
            assert torch.allclose(logits[r], want, atol=2e-4, rtol=1e-4)
        nxt = torch.randint(0, 61, (6,), generator=g)
        active = torch.arange(6) != 3 if t >= 2 else None  # a row that stays where it is does not disturb the others
        if t < 5:
            logits = dec.step(nxt, active).clone()
            for r in range(6):
                if active is None or bool(active[r]):
                    rows[r].append(int(nxt[r]))
            if active is not None:
                logits[3] = m(torch.tensor([rows[3]]))[0][0, -1]


def test_paged_limits_stops_and_long_prompts():
    m = model()
    eng = ChatEngine(m, Tok(), "cpu", max_model_len=16, paged=True, sync_every=1)
    out = eng.generate_ids([list(range(1, 31)), [4, 5], list(range(1, 13))], SamplingParams(max_tokens=50, temperature=0.0))
    assert [len(r[0]) for r in out] == [1, 14, 4]  # the room that each prompt leaves
    first = out[1][0]
    cut = eng.generate_ids([[4, 5]], SamplingParams(max_tokens=10, temperature=0.0, stop_token_ids=[first[3]]))[0][0]
    assert cut == first[: first.index(first[3])]
    many = eng.generate_ids([[3, 4, 5], [6, 7]], SamplingParams(n=3, max_tokens=4, temperature=1.0, seed=1))
    assert [len(r) for r in many] == [3, 3] and all(len(x) == 4 for r in many for x in r)
    assert eng.generate_ids([[3]], SamplingParams(n=2, max_tokens=0)) == [[[], []]]
    dec = PagedDecoder(m, "cpu")
    dec.PREFILL_TOKENS = 5  # prompts in several passes
    want = torch.stack([m(torch.tensor([x]))[0][0, -1] for x in PROMPTS])
    assert torch.allclose(dec.start(PROMPTS, 1, 3), want, atol=2e-4, rtol=1e-4)
    with pytest.raises(ValueError, match="rotation table"):
        dec.start([[1] * 8000], 1, 500)
    with pytest.raises(ValueError, match="at least one token"):
        dec.start([[1], []], 1, 5)
    with pytest.raises(ValueError, match="dense blocks"):
        ChatEngine(model(attn_gating="elementwise"), Tok(), "cpu", paged=True)


@pytest.mark.parametrize("paged", [False, True])
def test_constraints_and_penalties(paged):
    m = model()
    eng = ChatEngine(m, Tok(), "cpu", max_model_len=40, paged=paged)
    run = lambda **kw: eng.generate_ids([[3, 4, 5], [3, 4, 5, 6]], SamplingParams(**{**dict(max_tokens=8, temperature=0.0), **kw}))  # noqa: E731
    plain = run()
    assert run(repetition_penalty=1.0, logit_bias={}) == plain
    allowed = run(allowed_token_ids=[7, 20, 60], temperature=1.0, seed=0)
    assert {t for r in allowed for t in r[0]} <= {7, 20, 60}
    banned = plain[0][0][0]
    assert all(banned not in r[0] for r in run(logit_bias={banned: -1e9}))
    assert all(set(r[0]) == {33} for r in run(logit_bias={33: 1e9}))
    # a penalty so large that no token comes twice
    for kw in (dict(frequency_penalty=1e6), dict(presence_penalty=1e6)):
        assert all(len(set(r[0])) == 8 for r in run(**kw))
    choices = [[10, 11, 12], [10, 13], [14]]
    for seed in range(4):
        for r in run(choices=choices, temperature=1.0, seed=seed):
            assert r[0] in choices
    assert run(choices=[[10, 11, 12], [10, 11, 12]])[0][0] == [10, 11, 12]


def test_refused_constraints():
    mk = lambda **kw: LogitsProcessor(SamplingParams(**kw), [[1], [2]], 4, 61, "cpu")  # noqa: E731
    for kw, text in [(dict(repetition_penalty=0.0), "positive"), (dict(presence_penalty=float("nan")), "finite"), (dict(logit_bias={61: 1.0}), "logit_bias"),
                     (dict(logit_bias={1: float("-inf")}), "finite"), (dict(allowed_token_ids=[]), "at least one"), (dict(allowed_token_ids=[-1]), "at least one"),
                     (dict(choices=[]), "at least one"), (dict(choices=[[]]), "at least one"), (dict(choices=[[1, 2], [1]]), "begin"), (dict(choices=[[1], [1, 2]]), "begin"),
                     (dict(choices=[[1]], allowed_token_ids=[1]), "exclude")]:
        with pytest.raises(ValueError, match=text):
            mk(**kw)


def test_processor_history_is_prompt_and_answer():
    p = SamplingParams(repetition_penalty=2.0, frequency_penalty=0.5, presence_penalty=0.25)
    proc = LogitsProcessor(p, [[1, 2], [5]], 3, 8, "cpu")
    x = torch.tensor([[4.0, -4.0, 4.0, 1.0, 1.0, 1.0, 1.0, 1.0]] * 2)
    assert torch.allclose(proc(x)[0], torch.tensor([4.0, -8.0, 2.0, 1, 1, 1, 1, 1])) and torch.allclose(proc(x)[1, 5], torch.tensor(0.5))
    proc.push(torch.tensor([0, 5]))
    proc.push(torch.tensor([0, 2]))
    y = proc(x)
    assert torch.allclose(y[0], torch.tensor([4 / 2 - 2 * 0.5 - 0.25, -8.0, 2.0, 1, 1, 1, 1, 1]))
    assert torch.allclose(y[1], torch.tensor([4, -4, 4 / 2 - 0.75, 1, 1, 0.5 - 0.75, 1, 1.0]))
