"""Beam search's selection over values where numbers that are equal have more than one form.  Against the definition of test_beam_search_gpu.py, with its bounds."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES
from test_beam_search_gpu import _check, _problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocabulary", [6, 300, 8192, 20000, 600000])
def test_zeros_of_either_sign_are_equal(vocabulary, dtype):
    """As a 0/1 mask leaves them, or small negative values rounded to 16 bits: few, and more than are ordered at once."""
    g = torch.Generator(device="cuda").manual_seed(vocabulary)
    for zeros, keep in ((4, 2), (vocabulary // 2, 3), (vocabulary, 8)):
        p = _problem(3, 2, vocabulary, dtype, seed=zeros, finished=0)
        z = -1 - p["logits"].abs()
        at = torch.arange(vocabulary, device="cuda") * zeros // vocabulary
        place = torch.cat([at.new_zeros(1), (at.diff() > 0).nonzero().flatten() + 1])[:zeros]
        sign = torch.where(torch.rand(3, 2, len(place), device="cuda", generator=g) < 0.5, -0.0, 0.0).to(dtype)
        sign[..., 0], sign[0, 0] = -0.0, torch.where(torch.arange(len(place), device="cuda") < len(place) // 2, -0.0, 0.0).to(dtype)
        z[..., place] = sign
        p["scores"][1] = -0.5                          # (hypotheses of one score)
        _check(p, f"{zeros} of {vocabulary}", logits=z, beams=keep)


def test_scores_of_zero_of_either_sign_are_equal():
    """Finished hypotheses keep their scores, and the lower one comes first."""
    p = _problem(4, 6, 500, seed=3, finished=2)
    p["scores"] = torch.where(torch.arange(24, device="cuda").view(4, 6) % 3 < 2, -0.0, 0.0)
    p["scores"][1, 2:] = -0.0
    p["finished"][2, 4] = False                         # (whose best continuation is worse than a certain one)
    scores, parents, tokens, finished = fl.beam_select(**p)
    want = torch.arange(6, device="cuda").repeat(4, 1)
    want[2] = torch.tensor([0, 1, 2, 3, 5, 4], device="cuda")
    assert torch.equal(parents, want) and bool((scores[want != 4] == 0).all()) and bool((tokens[want != 4] == p["end"]).all())
    # a hypothesis whose only continuation is certain, behind one that is finished and in front of it
    for done in (0, 1):
        flags = torch.arange(2, device="cuda")[None] == done
        scores, parents, tokens, finished = fl.beam_select(torch.zeros(1, 2, 1, device="cuda"), torch.tensor([[-0.0, 0.0]], device="cuda"), end=0, finished=flags)
        assert parents.tolist() == [[0, 1]] and scores.tolist() == [[0, 0]] and tokens.tolist() == [[0, 0]]
        scores, parents, tokens, finished = fl.beam_select(torch.zeros(1, 2, 1, device="cuda"), torch.tensor([[0.0, -0.0]], device="cuda"), end=0, finished=flags)
        assert parents.tolist() == [[0, 1]] and scores.tolist() == [[0, 0]] and tokens.tolist() == [[0, 0]]
