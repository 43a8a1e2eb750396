"""The example decoder over trees of drafts (examples/tree_decoder.py): the operators together. What it computes does not depend on how a
text came to be in the cache: the logits behind kept paths are those of the same text read as one prompt, within what the
8-bit cache's rounding and the bf16 activations leave (a page that grew in steps has codes rounded twice). Needs an MI355X."""

import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("tree_decoder", os.path.join(ROOT, "examples", "tree_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_kept_paths_give_what_a_prompt_gives(example):
    m, prompts = example, (300, 117)
    first, kept, _ = m.generate(prompts=prompts, steps=12, depth=0)
    assert kept == [[1, 1]] * 12 and [len(t) for t in first] == [p + 13 for p in prompts]
    texts, kept, logits = m.generate(prompts=prompts, steps=4, depth=3, known=first)
    assert torch.isfinite(logits).all() and all(1 <= k <= 4 for ks in kept for k in ks)
    assert [len(t) for t in texts] == [p + 1 + sum(k[s] for k in kept) for s, p in enumerate(prompts)]
    assert sum(k > 1 for ks in kept for k in ks) > 0  # some drafts were kept: rows moved, from the second branch
    # the texts, but for the tokens not yet read, as prompts of a model of the same weights
    n, read = len(texts), [t[:-1] for t in texts]
    pages = -(-max(map(len, read)) // m.PAGE)
    model = m.Model(2, n * pages)
    table = torch.arange(n * pages, dtype=torch.int32).view(n, pages).cuda()
    trees = [[i - 1 for i in range(len(t))] for t in read]
    y = model(torch.tensor(sum(read, []), device="cuda"), m.Step(trees, [0] * n, table))
    y = y[torch.tensor([len(t) for t in read]).cumsum(0).cuda() - 1]
    cos = torch.nn.functional.cosine_similarity(y.float(), logits.float())
    assert (cos > 0.99).all(), cos


@pytest.mark.parametrize("prompts,steps,depth", [((1, 1), 2, 1), ((63, 64), 3, 5), ((20, 130), 1, 40), ((5,), 0, 2)])
def test_few_rows_and_deep_trees(example, prompts, steps, depth):
    """Prompts of one token, drafts that start a page, more rows than a word of the mask, no steps."""
    texts, kept, logits = example.generate(layers=1, prompts=prompts, steps=steps, depth=depth)
    assert len(kept) == steps and torch.isfinite(logits).all()
    assert [len(t) for t in texts] == [p + 1 + sum(k[s] for k in kept) for s, p in enumerate(prompts)]
