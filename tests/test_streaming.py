"""Streaming from the chat engine on the CPU."""

import threading

import pytest
import torch

from sample_efficient_gpt_b200.evals.generation import ChatEngine, SamplingParams

from tests.test_paged_generation import Tok, model


class ChatTok(Tok):
    def encode(self, text, add_special_tokens=False):
        return [ord(c) % 61 for c in text]


TALK = [{"role": "user", "content": "hello"}]


def engine(paged=False, **kw):
    return ChatEngine(model(), ChatTok(), "cpu", max_model_len=64, paged=paged, **kw)


def streamed(eng, **kw):
    return "".join(eng.stream(TALK, SamplingParams(**{**dict(max_tokens=8, temperature=0.0), **kw})))


@pytest.mark.parametrize("kw", [dict(), dict(choices=[[10, 11, 12], [10, 13], [14]]), dict(choices=[[20]]), dict(allowed_token_ids=[7, 20], temperature=1.0),
                                dict(frequency_penalty=1e6), dict(max_tokens=1)])
def test_a_stream_is_the_whole_answer(kw):
    eng = engine()
    torch.manual_seed(3)
    want = eng.chat([TALK], SamplingParams(**{**dict(max_tokens=8, temperature=0.0), **kw}))[0][0]
    torch.manual_seed(3)
    assert streamed(eng, **kw) == want


def test_a_stream_ends_at_a_stop_token():
    eng = engine()
    answer = [int(t) for t in streamed(eng).split()]
    assert [int(t) for t in streamed(eng, stop_token_ids=[answer[3]]).split()] == answer[: answer.index(answer[3])]


def test_a_refusal_reaches_the_reader(monkeypatch):
    eng = engine()
    with pytest.raises(ValueError, match="at least one token"):
        streamed(eng, allowed_token_ids=[])
    with pytest.raises(ValueError, match="finite"):
        streamed(eng, frequency_penalty=float("nan"))
    forward, calls = eng.model.forward, []

    def fails(*args, **kw):
        calls.append(1)
        if len(calls) == 3:
            raise RuntimeError("no more")
        return forward(*args, **kw)

    monkeypatch.setattr(eng.model, "forward", fails)
    pieces = []
    with pytest.raises(RuntimeError, match="no more"):
        for piece in eng.stream(TALK, SamplingParams(max_tokens=8, temperature=0.0)):
            pieces.append(piece)
    monkeypatch.undo()
    assert len(pieces) == 2 and streamed(eng).startswith("".join(pieces))


def test_a_paged_engine_streams_over_its_pages(monkeypatch):
    plain, eng = engine(), engine(paged=True)
    monkeypatch.setattr(eng, "_decode_batch", None)  # the static caches are not used
    for kw in (dict(), dict(n=3), dict(max_tokens=100), dict(choices=[[10, 11, 12], [10, 13], [14]]), dict(max_tokens=0)):
        assert streamed(eng, **kw) == streamed(plain, **kw)
    answer = [int(t) for t in streamed(eng).split()]
    assert [int(t) for t in streamed(eng, stop_token_ids=[answer[3]]).split()] == answer[: answer.index(answer[3])]
    with pytest.raises(ValueError, match="at least one token"):
        streamed(eng, allowed_token_ids=[])


def test_a_stream_that_is_closed_stops_decoding(monkeypatch):
    eng = engine(paged=True)
    seen, taken = eng.paged.step, threading.Event()
    steps = []

    def step(*args):
        taken.wait(10)  # the reader has its first piece and closes before the second step
        steps.append(1)
        return seen(*args)

    monkeypatch.setattr(eng.paged, "step", step)
    stream = eng.stream(TALK, SamplingParams(max_tokens=40, temperature=0.0))
    next(stream)
    stream.close()
    taken.set()
    with eng._paged_turn:  # free again once the thread has stopped
        assert len(steps) <= 1
    monkeypatch.undo()
    assert streamed(eng) == streamed(engine())
