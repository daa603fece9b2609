"""The CPU statements of the paged serving operators refuse what the kernels refuse, instead of leaving a part of the call out."""

import pytest
import torch

from sample_efficient_gpt_b200 import ops

from tests.paged_cases import cache_case


def test_logits_refusals():
    x, tok = torch.randn(2, 40), torch.zeros(2, 4, dtype=torch.int32)
    n, one = torch.ones(2, dtype=torch.int32), torch.ones(2)
    for kw, text in [(dict(tokens=tok), "together"), (dict(token_lens=n), "together"), (dict(repetition=one), "penalties need"), (dict(presence=one), "penalties need"),
                     (dict(frequency=one), "penalties need"), (dict(prompt_lens=n), "penalties need"), (dict(bias_ids=tok), "together"),
                     (dict(bias_values=torch.zeros(2, 4)), "together"), (dict(mask=tok), "together"), (dict(mask_rows=n), "together")]:
        with pytest.raises(ValueError, match=text):
            ops.process_logits(x, **kw)
    assert torch.equal(ops.process_logits(x), x)


def test_attention_refusals():
    c = cache_case([4, 7], 4, 2, 32, 16, prefix_lens=[9, 3], seed=1)
    args = [c[k] for k in ("q", "k_pages", "v_pages", "page_table", "seq_lens")]
    rows = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for pre, text in [((c["prefix_table"],), "together"), ((None, c["prefix_lens"]), "together"), ((None, None, rows(0, 2)), "needs"),
                      ((c["prefix_table"], c["prefix_lens"]), "one prefix"), ((c["prefix_table"], c["prefix_lens"], rows(0, 2)), "an entry more")]:
        with pytest.raises(ValueError, match=text):
            ops.paged_attention(*args, *pre)
    ops.paged_attention(*args, c["prefix_table"], c["prefix_lens"], rows(0, 1, 2))
    ops.paged_attention(*args, c["prefix_table"][:1], c["prefix_lens"][:1])
