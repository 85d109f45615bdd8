"""The example of several answers to each prompt: it runs, its books come out, and its draws repeat."""
import os
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_many_answers_run():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import many_answers
    prompts, answers, steps, block = (67, 33), 3, 20, 16
    got = many_answers.run(prompts=prompts, answers=answers, steps=steps, vocab=300)
    tokens = got["tokens"]
    assert tokens.shape == (6, steps) and int(tokens.min()) >= 0 and int(tokens.max()) < 300
    # whole pages of a prompt once, what follows them by answer
    want = sum(n // block + answers * (-(-(n + steps) // block) - n // block) for n in prompts)
    assert got["pages"] == want and got["alone"] == sum(answers * -(-(n + steps) // block) for n in prompts)
    assert len({tuple(t) for t in tokens.tolist()}) == 6  # each its own answer
    assert torch.equal(many_answers.run(prompts=prompts, answers=answers, steps=steps, vocab=300)["tokens"], tokens)
