"""Generation over a paged cache on the GPU: the captured step against the module path and against itself."""

import pytest
import torch

from sample_efficient_gpt_b200.evals.generation import ChatEngine, PagedDecoder, SamplingParams

from tests.test_paged_generation import PROMPTS, Tok, model

pytestmark = pytest.mark.gpu


def gpu_model(**kw):
    return model(**{**dict(d_model=256, d_ff=512, n_layers=3, n_heads=4, n_kv_heads=2, vocab_size=512), **kw}).cuda()


@pytest.mark.parametrize("n", [1, 3])
def test_logits_track_the_module_path(n):
    """bf16 kernels against the fp32 module path on the same token stream: as close as the static bf16 decoder is held to be."""
    m = gpu_model()
    dec = PagedDecoder(m, "cuda", page_size=16)
    rows = [list(x) for x in PROMPTS for _ in range(n)]
    logits = dec.start(PROMPTS, n, 40)
    g = torch.Generator().manual_seed(0)
    for _ in range(20):
        with torch.no_grad():
            want = torch.stack([m(torch.tensor([r], device="cuda"))[0][0, -1] for r in rows])
        assert torch.allclose(logits.float(), want, atol=0.15, rtol=0.05), float((logits - want).abs().max())
        nxt = torch.randint(0, 512, (len(rows),), generator=g)
        for r, t in zip(rows, nxt.tolist()):
            r.append(t)
        logits = dec.step(nxt.cuda())
    assert dec.graph is not None


def test_samples_share_a_prompt_and_buffers_are_used_again():
    m = gpu_model()
    eng = ChatEngine(m, Tok(), "cuda", max_model_len=96, paged=True)
    p = SamplingParams(max_tokens=24, temperature=0.0)
    a = eng.generate_ids([list(x) for x in PROMPTS], p)
    graph = eng.paged.graph
    assert eng.generate_ids([list(x) for x in PROMPTS], p) == a and eng.paged.graph is graph  # the captured step again
    assert all(len(r[0]) == 24 for r in a)
    # three samples of one prompt: the same tokens greedily, each step over the shared pages
    b = eng.generate_ids([list(PROMPTS[2])], SamplingParams(n=3, max_tokens=24, temperature=0.0))
    assert b[0][0] == b[0][1] == b[0][2]
    s = eng.generate_ids([list(PROMPTS[0]), list(PROMPTS[2])], SamplingParams(n=20, max_tokens=8, temperature=1.0, top_k=50, seed=3))
    assert [len(x) for x in s] == [20, 20] and all(len(r) == 8 for x in s for r in x)
    many = eng.generate_ids([list(PROMPTS[0])] * 300, SamplingParams(max_tokens=3, temperature=0.0))  # more rows than one batch takes
    assert len(many) == 300 and all(r == many[0] for r in many)


@pytest.mark.parametrize("paged", [False, True])
def test_constraints_on_the_gpu(paged):
    eng = ChatEngine(gpu_model(), Tok(), "cuda", max_model_len=64, paged=paged)
    run = lambda **kw: eng.generate_ids([[3, 4, 5], [3, 4, 5, 6]], SamplingParams(**{**dict(max_tokens=8, temperature=0.0), **kw}))  # noqa: E731
    assert {t for r in run(allowed_token_ids=[7, 200, 511], temperature=1.0, seed=0) for t in r[0]} <= {7, 200, 511}
    assert all(set(r[0]) == {33} for r in run(logit_bias={33: 1e9}))
    assert all(len(set(r[0])) == 8 for r in run(frequency_penalty=1e6))
    choices = [[10, 11, 12], [10, 13], [14]]
    assert all(r[0] in choices for seed in range(3) for r in run(choices=choices, temperature=1.0, seed=seed))


def test_paged_wants_bf16():
    with pytest.raises(ValueError, match="bfloat16"):
        ChatEngine(gpu_model(), Tok(), "cuda", dtype=torch.float32, paged=True)
