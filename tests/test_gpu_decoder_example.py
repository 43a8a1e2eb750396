"""The example decoder (examples/hybrid_decoder.py): the operators together. What it computes does not
depend on how a text is cut into steps: the logits after a text decoded and verified in steps are those after the same text
read as one prompt, within what the 8-bit cache's rounding and the bf16 activations leave (a page that
grew in steps has codes rounded twice). Needs an MI355X."""

import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("hybrid_decoder", os.path.join(ROOT, "examples", "hybrid_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_steps_give_what_a_prompt_gives():
    m = _example()
    prompts = (300, 117)
    texts, logprobs, logits = m.generate(prompts=prompts, tokens=6, drafts=3)
    assert [len(t) for t in logprobs] == [6, 6] and all(v <= 0 for t in logprobs for v in t)
    assert torch.isfinite(logits).all()
    # the whole texts, with the token that came last, as prompts of a model of the same weights
    n = len(texts)
    gen = torch.Generator().manual_seed(1)
    for p in prompts:
        torch.randint(m.VOCAB, (p,), generator=gen)
    pages = -(-(max(len(t) for t in texts) + 8) // m.PAGE)
    model = m.Model(4, n * pages, n)
    table = torch.arange(n * pages, dtype=torch.int32).view(n, pages).cuda()
    lens = [len(t) for t in texts]
    x = model(torch.tensor(sum(texts, []), device="cuda"), m.Batch(lens, lens, table, [-1] * n, list(range(n))))
    last = torch.tensor(lens).cumsum(0).cuda() - 1
    nxt = x[last].argmax(-1)
    y = model(nxt, m.Batch([1] * n, [v + 1 for v in lens], table, list(range(n)), list(range(n))))
    cos = torch.nn.functional.cosine_similarity(y.float(), logits.float())
    assert (cos > 0.99).all(), cos


@pytest.mark.parametrize("prompts,tokens,drafts", [((64, 20), 0, 3), ((63, 1), 1, 7), ((100, 30), 2, 0), ((63, 40), 0, 0)])
def test_few_tokens_and_drafts(prompts, tokens, drafts, monkeypatch):
    """No decoded tokens, no drafts, and drafts that start a page: the table has room for every step."""
    m = _example()

    class Batch(m.Batch):
        def __init__(self, *a):
            super().__init__(*a)
            assert self.max_len <= self.table.shape[1] * m.PAGE

    monkeypatch.setattr(m, "Batch", Batch)
    texts, logprobs, logits = m.generate(prompts=prompts, tokens=tokens, drafts=drafts)
    assert [len(t) for t in logprobs] == [tokens] * 2 and torch.isfinite(logits).all()
    assert all(p + tokens < len(t) <= p + tokens + 1 + drafts for p, t in zip(prompts, texts))
