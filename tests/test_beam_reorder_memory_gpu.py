"""Beam search's reordering of states whose rows lie between each other's: taken where they share no memory, whatever their strides, and refused before any of it
moves where they do."""
import random

import pytest
import torch

import flashlstm_poc_amd as fl

pytestmark = pytest.mark.gpu


def _rows(room, begin, stride, width, rows):
    return room.as_strided((rows, width), (stride, 1), begin)


def _reordered(state, parents):
    n, beams = parents.shape
    return state[(parents + beams * torch.arange(n, device="cuda")[:, None]).flatten()]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float32, torch.float64], ids=str)
def test_rows_between_each_other(dtype):
    r = random.Random(5)
    seen = [0, 0]
    parents = torch.tensor([[1, 0, 1], [2, 2, 0]], device="cuda")
    for _ in range(400):
        first, second = sorted(r.sample(range(2, 40), 2)) if r.random() < 0.8 else [r.randrange(2, 40)] * 2
        extents = [(r.randrange(0, 30), stride, r.randint(1, max(1, stride // r.choice([1, 2, 4])))) for stride in (first, second)]
        r.shuffle(extents)
        places = [{b + i * s + j for i in range(6) for j in range(w)} for b, s, w in extents]
        shared = bool(places[0] & places[1])
        room = torch.arange(300, device="cuda").to(dtype)
        states, before = [_rows(room, *e, 6) for e in extents], room.clone()
        if shared:
            with pytest.raises(ValueError, match="share"):
                fl.beam_reorder(parents, *states)
            assert torch.equal(room, before)
        else:
            fl.beam_reorder(parents, *states)
            for e in extents:
                _rows(before, *e, 6).copy_(_reordered(_rows(before, *e, 6), parents))
            assert torch.equal(room, before), extents
        seen[shared] += 1
    assert min(seen) > 40


def test_parents_beside_rows():
    room = torch.zeros(40, device="cuda", dtype=torch.int64)
    parents, state = room[:6].view(2, 3), _rows(room, 6, 5, 2, 6)
    parents.copy_(torch.tensor([[1, 0, 1], [2, 2, 0]], device="cuda"))
    state.copy_(torch.arange(12, device="cuda").view(6, 2))
    want = _reordered(state.clone(), parents)
    fl.beam_reorder(parents, state)
    assert torch.equal(state, want)
    with pytest.raises(ValueError, match="share"):
        fl.beam_reorder(parents, _rows(room, 5, 5, 2, 6))
