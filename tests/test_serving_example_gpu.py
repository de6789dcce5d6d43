"""The serving rows together, as examples/verify_drafts.py runs them: the logits
of a drafted token in a tree equal those of its path decoded token by token, and
what follows a kept path does not show how it was drafted."""

import os
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT, TOL, rel_err

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(ROOT, "examples"))


def test_a_tree_equals_its_paths(cuda):
    import verify_drafts as ex

    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (45, 3, 16)]
    trees = [([5, 7, 9, 11, 13], [-1, 0, 0, 1, 2]), ([1], [-1]), ([4, 8, 15, 16, 23, 42], [-1, 0, 1, 2, 1, 4])]
    model = ex.Decoder(len(prompts))
    _, plan = model.forward(prompts)
    model.commit(plan, [list(range(len(p))) for p in prompts])
    logits, plan = model.forward([t for t, _ in trees], [p for _, p in trees])
    got = logits.cpu().numpy()
    kept = [[0, 2, 4], [0], [0, 1, 4, 5]]
    model.commit(plan, kept)
    after, _ = model.forward([[100], [200], [300]])
    after = after.cpu().numpy()

    def path(parents, i):
        return path(parents, parents[i]) + [i] if i >= 0 else []

    row = 0
    for r, (tokens, parents) in enumerate(trees):
        for i in range(len(tokens)):
            text = prompts[r] + [tokens[j] for j in path(parents, i)]
            alone = ex.Decoder(1)
            want = alone.forward([text])[0][-1:].cpu().numpy()
            assert rel_err(got[row:row + 1], want) <= TOL
            row += 1
        text = prompts[r] + [tokens[j] for j in kept[r]] + [100 * (r + 1)]
        alone = ex.Decoder(1)
        for t in text:  # token by token
            want, plan = alone.forward([[t]])
            alone.commit(plan, [[0]])
        assert rel_err(after[r:r + 1], want.cpu().numpy()) <= TOL


def test_example_runs(cuda, capsys, monkeypatch):
    import verify_drafts as ex

    monkeypatch.setattr(sys, "argv", ["verify_drafts.py", "--steps", "3"])
    ex.main()
    assert "request 2" in capsys.readouterr().out
    torch.cuda.synchronize()
