"""The results of the embedding, the gated recurrence and beam search are allocated past torch's dispatch only where nothing looks at that: the same results where torch
has no such function or one that takes something else, allocations that a dispatch mode sees, and memory that deterministic algorithms fill."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import flashlstm_poc_amd as fl
from flashlstm_poc_amd import lm_ops

pytestmark = pytest.mark.gpu


def _calls():
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    tokens, table = torch.randint(-1, 50, (9, 7), device="cuda", generator=g), n(50, 24)
    out = [fl.embedding_forward(tokens, table, dtype=torch.float16), fl.embedding_backward(n(9, 7, 24), tokens, 50)]
    x, forget, gate = n(2, 300, 24), n(2, 300, 24), n(2, 300, 24)
    y, state, saved = fl.gated_recurrence_forward(x, forget, gate)
    out += [y, state, saved, *fl.gated_recurrence_backward(n(2, 300, 24), x, forget, gate, saved)]
    out.append(fl.gated_recurrence_step(x[:, 0], forget[:, 0], state.clone(), gate[:, 0]))
    out += fl.beam_select(n(3, 4, 900), -n(3, 4).abs(), end=3)
    return out


def _same(got, want):
    assert len(got) == len(want) and all(torch.equal(a, b) and a.stride() == b.stride() for a, b in zip(got, want))


def test_without_the_function(monkeypatch):
    want = _calls()
    monkeypatch.setattr(lm_ops, "_EMPTY_STRIDED", None)
    _same(_calls(), want)


def test_with_a_function_that_takes_something_else(monkeypatch):
    want = _calls()
    monkeypatch.setattr(lm_ops, "_EMPTY_STRIDED", lambda shape: None)
    _same(_calls(), want)
    assert lm_ops._EMPTY_STRIDED is None


class _Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.empty = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        self.empty += isinstance(out, torch.Tensor) and "empty" in str(func)
        return out


def test_dispatch_modes_see_allocations():
    want = _calls()
    with _Seen() as seen:
        got = _calls()
    _same(got, want)
    assert seen.empty >= len(want)


def test_deterministic_algorithms_fill():
    want = _calls()
    torch.use_deterministic_algorithms(True)
    try:
        got, fresh = _calls(), lm_ops._allocation()((5, 3), torch.float32)
    finally:
        torch.use_deterministic_algorithms(False)
    _same(got, want)
    assert bool(fresh.isnan().all())
