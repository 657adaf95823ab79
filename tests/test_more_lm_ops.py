"""CPU-side checks of the embedding, the gated linear recurrence and beam search: what the C entry points and their Python callers refuse before
any device work."""
import ctypes

import pytest
import torch

import flashlstm_poc_amd as fl
from flashlstm_poc_amd import lm_ops

SOME = ctypes.c_void_p(4096)   # an address that is only compared with null


def test_embedding_refuses_before_device_work():
    lib = lm_ops._bind()

    def problem(**change):
        return lm_ops._EMBEDDING.pack(*{**dict(tokens=4, vocabulary=10, width=8, index=SOME.value, index_64=1, scale=1.0), **change}.values())

    bad = (dict(vocabulary=0), dict(vocabulary=1 << 31), dict(tokens=1 << 31), dict(width=1 << 24), dict(scale=float("nan")), dict(index=0))
    forward = lambda p=problem(), table=SOME, ld=8, kind=0, out=SOME, to=1: lib.flstm_embedding_forward(p, table, ld, kind, out, to, None)
    backward = lambda p=problem(), d=SOME, kind=0, out=SOME, to=1, work=SOME: lib.flstm_embedding_backward(p, d, 8, kind, out, to, work, None)
    for change in bad:
        assert forward(problem(**change)) == 1 and backward(problem(**change)) == 1, change
        assert lib.flstm_embedding_workspace_bytes(problem(**change)) == 0
    assert forward(None) == 1 and forward(table=None) == 1 and forward(out=None) == 1 and forward(ld=7) == 1 and forward(kind=3) == 1 and forward(to=-1) == 1
    assert backward(None) == 1 and backward(d=None) == 1 and backward(out=None) == 1 and backward(kind=3) == 1 and backward(to=9) == 1
    assert backward(work=None) == 1
    assert forward(problem(tokens=0, index=0), None, 8, 0, None) == 0 and forward(problem(width=0), None, 8, 0, None) == 0
    assert backward(problem(width=0), None, 0, None, 0, None) == 0
    assert lib.flstm_embedding_workspace_bytes(problem()) > 0 and lib.flstm_embedding_workspace_bytes(problem(tokens=0, index=0)) == 0


def test_gated_recurrence_refuses_before_device_work():
    lib = lm_ops._bind()
    rows = lambda data=SOME: lm_ops._ROWS.pack(data.value if data else 0, 64, 8, 0)

    def shape(**change):
        return lm_ops._RECURRENCE.pack(*{**dict(sequences=2, tokens=5, cu_seqlens=0, width=8, dtype=1), **change}.values())

    forward = lambda s=shape(), x=rows(), u=rows(), y=rows(): lib.flstm_gated_recurrence_forward(s, x, u, None, None, y, None, None, None, None)
    backward = lambda s=shape(), dy=rows(), x=rows(), g=None, saved=SOME, dg=None: lib.flstm_gated_recurrence_backward(
        s, dy, x, rows(), g, saved, None, rows(), rows(), dg, None, None, None)
    step = lambda s=shape(), x=rows(), y=rows(), state=SOME: lib.flstm_gated_recurrence_step(s, x, rows(), None, y, state, None)
    for change in (dict(dtype=3), dict(dtype=-1), dict(sequences=1 << 31), dict(tokens=1 << 39), dict(width=1 << 28), dict(cu_seqlens=4096, tokens=1 << 31)):
        assert forward(shape(**change)) == 1 and backward(shape(**change)) == 1 and step(shape(**change)) == 1, change
        assert lib.flstm_gated_recurrence_workspace_bytes(shape(**change), 0) == 0 and lib.flstm_gated_recurrence_saved_rows(shape(**change)) == 0
    assert forward(None) == 1 and forward(x=None) == 1 and forward(u=rows(None)) == 1 and forward(y=rows(None)) == 1
    assert forward(shape(sequences=1, tokens=1 << 20)) == 1     # no workspace
    assert backward(None) == 1 and backward(dy=None) == 1 and backward(x=rows(None)) == 1 and backward(saved=None) == 1 and backward(dg=rows()) == 1
    assert step(None) == 1 and step(x=None) == 1 and step(y=rows(None)) == 1 and step(state=None) == 1
    assert forward(shape(sequences=0), None, None, None) == 0 and forward(shape(width=0), None, None, None) == 0
    assert step(shape(sequences=0), None, None, None) == 0
    assert lib.flstm_gated_recurrence_saved_rows(shape()) == 2 and lib.flstm_gated_recurrence_saved_rows(shape(tokens=17)) == 4
    assert lib.flstm_gated_recurrence_saved_rows(shape(tokens=40, cu_seqlens=4096)) == 5
    assert forward(shape(sequences=(1 << 31) - 1, tokens=1, width=1 << 20)) == 2004


def test_beam_search_refuses_before_device_work():
    lib = lm_ops._bind()

    def problem(**change):
        values = dict(sequences=2, beams=3, keep=3, vocabulary=50, logits=SOME.value, ld=50, dtype=0, scores=SOME.value, finished=SOME.value, end=7)
        return lm_ops._BEAMS.pack(*{**values, **change}.values())

    select = lambda p=problem(), scores=SOME, parents=SOME, tokens=SOME, work=SOME: lib.flstm_beam_select(p, scores, parents, tokens, None, work, None)
    for change in (dict(dtype=3), dict(beams=0), dict(beams=33), dict(keep=0), dict(keep=33), dict(vocabulary=0), dict(vocabulary=1 << 31), dict(ld=49),
                   dict(logits=0), dict(scores=0), dict(end=-1), dict(end=50), dict(sequences=1 << 31)):
        assert select(problem(**change)) == 1, change
        assert lib.flstm_beam_select_workspace_bytes(problem(**change)) == 0
    assert select(None) == 1 and select(scores=None) == 1 and select(parents=None) == 1 and select(tokens=None) == 1 and select(work=None) == 1
    assert select(problem(sequences=0, logits=0, scores=0), None, None, None, None) == 0
    state = lambda data=4096, stride=16, size=16: lm_ops._BEAM_STATE.pack(data, stride, size)
    reorder = lambda n=2, beams=3, parents=SOME, states=state(), count=1: lib.flstm_beam_reorder(n, beams, parents, states, count, None)
    assert reorder(beams=0) == 1 and reorder(beams=33) == 1 and reorder(parents=None) == 1 and reorder(states=None) == 1
    assert reorder(count=-1) == 1 and reorder(states=state(0)) == 1 and reorder(states=state(stride=15)) == 1
    assert reorder(n=0, parents=None) == 0 and reorder(count=0, parents=None) == 0 and reorder(beams=1, parents=None) == 0
    assert reorder(states=state(0, 0, 0)) == 0
    assert reorder(n=1 << 20, states=state(stride=1 << 40, size=1 << 40)) == 2004
    # six rows: the same ones twice, begun inside of one, at the last one's last byte, inside unlike strides; parents inside and at the end
    two = lambda a, b, count=2: reorder(parents=1 << 30, states=a + b, count=count)
    assert two(state(), state()) == 1 and two(state(), state(4096 + 33)) == 1 and two(state(), state(4096 - 95)) == 1 and two(state(), state(4096 + 95)) == 1
    assert two(state(stride=32), state(4096 + 16, 48)) == 1 and two(state(stride=32), state(4096 + 15, 32)) == 1 and two(state(stride=32), state(4096 + 17, 32)) == 1
    assert two(b"".join(state(4096 + i * 96) for i in range(20)), state(4096 + 96 + 95), 21) == 1
    assert reorder(parents=4096 + 88) == 1 and reorder(parents=4096 - 40) == 1


def test_host_tensors_are_refused():
    x, tokens = torch.zeros(2, 5, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: fl.embedding_forward(tokens, x[0]), lambda: fl.embedding(tokens, x[0].requires_grad_()), lambda: fl.embedding_backward(x[0], tokens, 5),
                 lambda: fl.gated_recurrence_forward(x, x), lambda: fl.gated_recurrence(x, x), lambda: fl.gated_recurrence_step(x[0], x[0], x[0]),
                 lambda: fl.gated_recurrence_backward(x, x, x, None, x[0]), lambda: fl.beam_select(x, x[..., 0]),
                 lambda: fl.beam_reorder(tokens.view(2, 2), x[0])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
