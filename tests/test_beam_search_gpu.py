"""Beam search's selection against a sort of all continuations in 64 bits, and the reordering of states against indexing.

Bounds: a score is one rounding to 32 bits of a sum in 64, off by the logarithm of the sum of exponentials alone.  An exponential's argument -d is
rounded (d u of the term, and d exp(-d) < 0.4), the hardware's exponential is off by 2 u, and a thread's chain of sums and the tree behind it are
under 45 additions: 48 u of the logarithm.  Which continuations come, and in which order, is compared whole: the inputs' values leave gaps that
are far wider than that, or none at all."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within, offset_copy

pytestmark = pytest.mark.gpu
INF = float("inf")


def _problem(sequences, beams, vocabulary, dtype=torch.float32, seed=0, finished=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return dict(logits=(2.5 * torch.randn(sequences, beams, vocabulary, device="cuda", generator=g)).to(dtype),
                scores=-20 * torch.rand(sequences, beams, device="cuda", generator=g),
                finished=torch.rand(sequences, beams, device="cuda", generator=g) < finished, end=vocabulary // 3)


def _definition(logits, scores, finished=None, end=None, beams=None):
    n, hypotheses, vocabulary = logits.shape
    keep = hypotheses if beams is None else beams
    z = logits.double()
    z = torch.where(z.isnan(), -INF, z.clamp(max=3.4028234663852886e38))
    most = z.amax(-1, keepdim=True).clamp(min=-3.5e38)
    value = (z - most) - (z - most).exp().sum(-1, keepdim=True).log() + scores.double()[..., None]
    value = torch.where((z > -INF) & (scores > -INF)[..., None], value, -INF)
    if finished is not None:
        value = torch.where(finished[..., None], -INF, value)
        value[..., end] = torch.where(finished, scores.double(), value[..., end])
    value, place = torch.sort(value.flatten(1), dim=1, descending=True, stable=True)
    there = torch.nn.functional.pad(value, (0, keep), value=-INF)[:, :keep]
    place = torch.nn.functional.pad(place, (0, keep))[:, :keep]
    none = there == -INF
    slot = torch.arange(keep, device="cuda").expand(n, keep)
    parents = torch.where(none, torch.where(slot < hypotheses, slot, 0), place // vocabulary)
    tokens = torch.where(none, -1, place % vocabulary)
    return there, parents, tokens, None if end is None else none | (tokens == end)


def _check(p, label, **more):
    p = {**p, **more}
    got, want = fl.beam_select(**p), _definition(**p)
    for a, b, name in zip(got[1:], want[1:], ("parents", "tokens", "finished")):
        assert (a is None and b is None) or torch.equal(a, b), f"{label} {name}: {a.tolist()} instead of {b.tolist()}"
    dead = want[0] == -INF
    assert torch.equal(got[0] == -INF, dead)
    assert_within(torch.where(dead, 0, got[0]), torch.where(dead, 0, want[0]), torch.full_like(want[0], 48 * U32), f"{label} scores")
    return got


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocabulary", [1, 2, 7, 8, 9, 255, 1000, 2049, 8191, 8192, 8193, 16385, 50001])
def test_vocabularies(vocabulary, dtype):
    for sequences, beams in ((1, 1), (1, 4), (5, 3), (3, 8)):
        _check(_problem(sequences, beams, vocabulary, dtype, seed=vocabulary), f"{sequences} x {beams} x {vocabulary} {dtype}")


@pytest.mark.parametrize("hypotheses,keep", [(1, 1), (1, 5), (1, 32), (4, 1), (32, 32), (31, 17), (16, 16), (2, 32)])
def test_beams(hypotheses, keep):
    for vocabulary in (3, 40, 9000):
        _check(_problem(2, hypotheses, vocabulary, seed=keep, finished=0.1), f"{hypotheses} to {keep} of {vocabulary}", beams=keep)


def test_many_sequences_and_large_vocabularies():
    _check(_problem(3000, 4, 300, torch.float16, seed=1), "many")
    for vocabulary in (70000, 600000, 1100001):   # (beyond 524288 a workgroup takes more than one round of logits)
        _check(_problem(2, 3, vocabulary, torch.bfloat16, seed=2), f"of {vocabulary}")


def test_without_an_end():
    p = _problem(4, 5, 600, seed=3)
    for more in (dict(finished=None, end=None), dict(finished=None)):
        _check({**p, **more}, "alive")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_equal_logits_come_lowest_first(dtype):
    for vocabulary in (5, 3000, 20000):
        p = _problem(3, 4, vocabulary, dtype, seed=4, finished=0)
        p["logits"][:] = 0.5
        p["scores"][0], p["scores"][1, 2:] = -1.25, -INF
        _check(p, "equal")
        p["logits"][:, :, ::7] = 1.0
        _check(p, "two values")
        p["logits"][:] = p["logits"][:, :1]     # beams of one score and the same logits
        _check(p, "same beams")
        p["logits"] = torch.randint(0, 4, p["logits"].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(dtype)
        _check(p, "few values")


@pytest.mark.parametrize("rising", [True, False])
def test_sorted_logits(rising):
    for vocabulary in (300, 8192, 30000):
        p = _problem(2, 6, vocabulary, seed=6, finished=0)
        p["logits"] = torch.sort(p["logits"], -1, descending=not rising).values
        _check(p, f"{vocabulary}", beams=32)


def test_best_logits_beside_each_other():
    """All of the best with one thread, one wave, or one part."""
    for begin, step in ((0, 1), (8, 1), (0, 2048), (5, 256), (8190, 1), (0, 8)):
        p = _problem(2, 2, 20000, seed=7, finished=0)
        at = (begin + step * torch.arange(40, device="cuda")) % 20000
        p["logits"][:, :, at] += 30
        _check(p, f"{begin} + {step}", beams=32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masks(dtype):
    lowest = torch.finfo(dtype).min
    for mask in (-INF, lowest, float("nan")):
        p = _problem(6, 4, 9000, dtype, seed=8, finished=0)
        p["logits"][0, :, 100:], p["logits"][1, :2], p["logits"][2] = mask, mask, mask
        p["logits"][3, :, 3:], p["logits"][4, 1, ::2] = mask, mask
        p["scores"][3, 1:] = -INF
        p["scores"][5] = -INF
        _check(p, f"{mask}")
        p["finished"][2, 1] = p["finished"][5, 2] = p["finished"][1, 0] = True
        _check(p, f"{mask}, some finished")
    p = _problem(3, 3, 500, dtype, seed=9, finished=0)
    p["logits"][0, 1, 77] = p["logits"][1, 2, 5] = p["logits"][1, 2, 8] = INF
    _check(p, "infinite")
    p = _problem(2, 3, 500, dtype, seed=10, finished=0)
    p["scores"][0, 1] = float("nan")
    got = fl.beam_select(**p)
    assert not bool((got[1][0] == 1).any()) and bool(got[0].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_few_allowed_among_many_equal(dtype):
    """Masks that leave logits where the threads' groups do not all find one, with everything else at one value."""
    for vocabulary, low in ((8192, torch.finfo(dtype).min), (30000, 0.0), (1100001, -7.0)):
        for allowed in (slice(0, 1), slice(5000, 5003), slice(0, None, 16), slice(8, None, 4096), slice(1, None, 2)):
            p = _problem(2, 2, vocabulary, dtype, seed=15, finished=0)
            masked = torch.full_like(p["logits"], low)
            masked[..., allowed] = p["logits"][..., allowed] + 20
            _check({**p, "logits": masked}, f"{allowed} of {vocabulary}", beams=11)


def test_all_finished():
    p = _problem(3, 4, 800, seed=11, finished=2)
    p["logits"][:] = float("nan")
    scores, parents, tokens, finished = _check(p, "finished")
    assert bool(finished.all()) and bool((tokens == p["end"]).all()) and torch.equal(scores, p["scores"].sort(-1, descending=True).values)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides_and_alignment(dtype):
    p = _problem(4, 3, 2500, dtype, seed=12)
    want = fl.beam_select(**p)
    same = lambda got: [torch.equal(a, b) or pytest.fail("differs") for a, b in zip(got, want)]
    wide = torch.zeros(4, 3, 2511, device="cuda", dtype=dtype)
    wide[..., 3:2503] = p["logits"]
    same(fl.beam_select(**{**p, "logits": wide[..., 3:2503]}))
    same(fl.beam_select(**{**p, "logits": offset_copy(p["logits"])}))
    same(fl.beam_select(**{**p, "logits": p["logits"].transpose(0, 1).contiguous().transpose(0, 1), "scores": p["scores"].t().contiguous().t(),
                           "finished": p["finished"].t().contiguous().t()}))
    same(fl.beam_select(**{**p, "logits": p["logits"].permute(2, 0, 1).contiguous().permute(1, 2, 0)}))
    _check({**p, "logits": p["logits"][:1, :1].expand(4, 3, 2500)}, "shared row")
    one = _problem(1, 1, 2500, dtype, seed=13)
    _check(one, "one")


def test_empty():
    p = _problem(0, 3, 50)
    got = fl.beam_select(**p)
    assert got[0].shape == got[1].shape == got[2].shape == got[3].shape == (0, 3)
    fl.beam_reorder(got[1], torch.zeros(0, 4, device="cuda"))


def test_graphs_and_streams():
    p = _problem(5, 4, 9000, torch.float16, seed=14)
    state = torch.randn(20, 33, device="cuda")
    want = fl.beam_select(**p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fl.beam_select(**p)
    here = fl.beam_select(**p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(got, want, here))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fl.beam_select(**p)
        fl.beam_reorder(got[1], state)
    for seed in range(4):
        fresh = _problem(5, 4, 9000, torch.float16, seed=seed)
        for name in ("logits", "scores", "finished"):
            p[name].copy_(fresh[name])
        state.normal_()
        before = state.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = fl.beam_select(**p)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        fl.beam_reorder(want[1], before)
        assert torch.equal(before, state)


# ---- the states

def _reordered(state, parents):
    n, beams = parents.shape
    slot = torch.arange(beams, device="cuda")
    parents = torch.where((parents >= 0) & (parents < beams), parents, slot)
    rows = (parents + beams * torch.arange(n, device="cuda")[:, None]).flatten()
    flat = state.reshape(n * beams, -1) if state.numel() else state
    return flat[rows].view(state.shape) if state.numel() else state.clone()


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32])
def test_reorder(beams):
    g = torch.Generator(device="cuda").manual_seed(beams)
    for sequences in (1, 3, 40):
        parents = torch.randint(0, beams, (sequences, beams), device="cuda", generator=g)
        parents[0] = torch.arange(beams, device="cuda")
        if sequences > 2:
            parents[1, 0], parents[2, -1] = -1, beams
            parents[2, 0] = 2 ** 40
        rows = sequences * beams
        states = [torch.randn(rows, 1024, device="cuda", generator=g).half(), torch.randn(rows, 3, 7, device="cuda", generator=g),
                  torch.randint(0, 100, (sequences, beams, 5), device="cuda", generator=g), torch.randn(rows, 5000, device="cuda", generator=g).bfloat16(),
                  torch.randint(0, 2, (rows, 1), device="cuda", generator=g).bool(), torch.randn(rows, device="cuda", generator=g, dtype=torch.float64),
                  offset_copy(torch.randn(rows, 19, device="cuda", generator=g).half()), torch.empty(rows, 0, device="cuda")]
        want = [_reordered(s, parents) for s in states]
        versions = [s._version for s in states]
        fl.beam_reorder(parents, *states)
        for i, (a, b) in enumerate(zip(states, want)):
            assert torch.equal(a, b), (beams, sequences, i)
        assert all(s._version > v for s, v in zip(states, versions))


def test_reorder_leaves_the_rest():
    g = torch.Generator(device="cuda").manual_seed(0)
    parents = torch.randint(0, 4, (6, 4), device="cuda", generator=g)
    room = torch.randn(24, 100, device="cuda", generator=g)
    before = room.clone()
    view = room[:, 7:60]
    fl.beam_reorder(parents, view)
    assert torch.equal(view, _reordered(before[:, 7:60], parents))
    assert torch.equal(room[:, :7], before[:, :7]) and torch.equal(room[:, 60:], before[:, 60:])
    many = [torch.randn(24, 3, device="cuda", generator=g) for _ in range(40)]     # more than one launch takes
    want = [_reordered(s, parents) for s in many]
    fl.beam_reorder(parents, *many)
    assert all(torch.equal(a, b) for a, b in zip(many, want))
    fl.beam_reorder(parents)
    lots = torch.randn(24, 3, 400000, device="cuda", generator=g)
    want = _reordered(lots, parents)
    fl.beam_reorder(parents, lots)
    assert torch.equal(lots, want)


def test_reorder_of_shared_memory():
    """What a call would move twice is refused before any of it moves; rows between each other's are each other's neighbours only."""
    g = torch.Generator(device="cuda").manual_seed(1)
    parents = torch.randint(0, 4, (6, 4), device="cuda", generator=g)
    room = torch.randn(24, 100, device="cuda", generator=g)
    before, others = room.clone(), [torch.randn(24, 3, device="cuda", generator=g) for _ in range(20)]
    kept = [t.clone() for t in others]
    for bad in ([room, room], [room[:, :50], room[:, 49:]], [others[0], *others], [room, room.flatten()[300:324]],
                [room.view(48, 50)[:24], room.view(48, 50)[23:47]], [*others, parents]):
        with pytest.raises(ValueError, match="share"):
            fl.beam_reorder(parents, *bad)
    assert torch.equal(room, before) and all(torch.equal(a, b) for a, b in zip(others, kept))
    fl.beam_reorder(parents, room[:, :50], room[:, 50:99])
    assert torch.equal(room[:, :99], _reordered(before, parents)[:, :99]) and torch.equal(room[:, 99], before[:, 99])


def test_refusals():
    p = _problem(2, 3, 50)
    for bad, match in ((dict(logits=p["logits"].cpu()), "CUDA"), (dict(logits=p["logits"].double()), "dtype"), (dict(logits=p["logits"][0]), "logits"),
                       (dict(scores=p["scores"].half()), "scores"), (dict(scores=p["scores"][:1]), "scores"), (dict(end=50), "end"), (dict(end=-1), "end"),
                       (dict(end=None), "end"), (dict(finished=p["finished"].int()), "finished"), (dict(finished=p["finished"][:1]), "finished"),
                       (dict(finished=p["finished"].cpu()), "finished"), (dict(beams=0), "between"), (dict(beams=33), "between"),
                       (dict(logits=torch.zeros(2, 33, 50, device="cuda")), "between"), (dict(logits=torch.zeros(2, 3, 0, device="cuda")), "logits")):
        with pytest.raises(ValueError, match=match):
            fl.beam_select(**{**p, **bad})
    parents, state = torch.zeros(2, 3, device="cuda", dtype=torch.int64), torch.zeros(6, 8, device="cuda")
    for bad, match in (((parents.int(), state), "parents"), ((parents.cpu(), state), "parents"), ((parents[0], state), "parents"),
                       ((torch.zeros(1, 33, device="cuda", dtype=torch.int64), state), "parents"), ((parents, state[:5]), "rows"),
                       ((parents, state.cpu()), "state 0"), ((parents, state, state.t().contiguous().t()), "state 1"),
                       ((parents, state[:1].expand(6, 8)), "state 0"), ((parents, state.clone().requires_grad_()), "gradient")):
        with pytest.raises(ValueError, match=match):
            fl.beam_reorder(*bad)
