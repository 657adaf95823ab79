"""Beam search's selection over values where numbers that are equal have more than one form, and where sums of exponentials leave the range of 32 bits
on the way.  Against the definition of test_beam_search_gpu.py, with its bounds."""
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [1e7, 1e9, 3e9, 1e10, 3e11, 1e12, 1e15, 3e18, 1e20, 1e25, 1e30, 1e38])
def test_logits_of_any_size(size, dtype):
    """Masks of a large negative value, over some or all of a row or over whole parts of it, and a row whose largest logit is as large."""
    for vocabulary in (40, 9000, 50001):
        p = _problem(5, 3, vocabulary, dtype, seed=17, finished=0)
        z, half = p["logits"], vocabulary // 3
        z[0, :, half:] = -size                          # the first tokens alone
        z[1, :, :-2] = -size                            # the last ones alone
        z[2, 1] = -size                                 # a row of nothing else
        z[3] = -size * (1 + torch.rand(3, vocabulary, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).to(dtype)
        z[4, 1, half] = size
        z[4, 2, ::2] = size
        _check(p, f"{size} of {vocabulary} {dtype}")
        _check(p, f"{size} of {vocabulary} {dtype}, its negative", logits=-z)
