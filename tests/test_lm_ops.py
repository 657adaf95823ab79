"""CPU-side checks of the language-model operators: the header's functions are exported, and refuse bad arguments before any
device work."""
import ctypes
import os
import re

import pytest
import torch

import flashlstm_poc_amd as fl

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOME = ctypes.c_void_p(4096)   # an address that is only compared with null


def test_header_functions_are_exported():
    text = open(os.path.join(ROOT, "include/flashlstm/lm_ops.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"\b(flstm_\w+)\s*\(", text))
    assert {"flstm_layer_norm_forward", "flstm_layer_norm_backward", "flstm_layer_norm_workspace_bytes",
            "flstm_decay_attention_forward", "flstm_decay_attention_backward", "flstm_decay_attention_step",
            "flstm_distillation_forward", "flstm_distillation_backward", "flstm_distillation_train"} <= names
    for name in sorted(names):
        assert hasattr(fl.load_library(), name), f"{name} declared but not exported"


def test_layer_norm_refuses_before_device_work():
    from flashlstm_poc_amd import lm_ops
    lib = lm_ops._bind()
    forward = lambda rows=4, width=8, x=SOME, residual=None, dtype=0, eps=1e-5, total=None, y=SOME: lib.flstm_layer_norm_forward(
        rows, width, x, width, residual, width, dtype, None, None, eps, total, y, None, None, None)
    assert forward(dtype=3) == 1 and forward(dtype=-1) == 1 and forward(eps=-1.0) == 1 and forward(eps=float("nan")) == 1
    assert forward(x=None) == 1 and forward(y=None) == 1 and forward(residual=SOME) == 1
    assert forward(width=16385) == 2004
    assert forward(rows=0, x=None, y=None) == 0 and forward(width=0, x=None, y=None) == 0
    backward = lambda rows=4, width=8, dtype=0, dy=SOME, dweight=None, workspace=None: lib.flstm_layer_norm_backward(
        rows, width, dy, width, SOME, width, None, 0, dtype, None, SOME, SOME, SOME, dweight, None, workspace, None)
    assert backward(dtype=9) == 1 and backward(dy=None) == 1 and backward(dweight=SOME) == 1 and backward(width=20000) == 2004
    assert lib.flstm_layer_norm_workspace_bytes(0, 8) == 0 and lib.flstm_layer_norm_workspace_bytes(1, 8) == 64


def test_layer_norm_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        fl.layer_norm_forward(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        fl.layer_norm(torch.zeros(2, 8, requires_grad=True))


def test_decay_attention_refuses_before_device_work():
    from flashlstm_poc_amd import lm_ops
    lib = lm_ops._bind()
    rows = lambda data=SOME, token=64: lm_ops._ROWS.pack(data.value if data else 0, 64 * 5, token, 32)

    def shape(**change):
        values = dict(sequences=2, tokens=5, cu_seqlens=0, heads=2, kv_heads=1, dk=32, dv=32, dtype=1, scale=0.5, log_decay=SOME.value)
        return lm_ops._SHAPE.pack(*{**values, **change}.values())

    forward = lambda s=shape(), q=rows(), o=rows(): lib.flstm_decay_attention_forward(s, q, rows(), rows(), None, o, None, None, None)
    for change in (dict(dtype=3), dict(heads=0), dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(dk=7), dict(dk=257), dict(dv=0), dict(dv=300),
                   dict(scale=float("nan")), dict(log_decay=0)):
        assert forward(shape(**change)) == 1, change
    assert forward(q=rows(None)) == 1 and forward(q=None) == 1 and forward(o=rows(None)) == 1 and forward(q=rows(token=1 << 23)) == 2004
    assert lib.flstm_decay_attention_forward(None, rows(), rows(), rows(), None, rows(), None, None, None) == 1
    assert lib.flstm_decay_attention_forward(shape(tokens=1 << 20, heads=1), rows(), rows(), rows(), None, rows(), None, None, None) == 1   # no workspace
    assert lib.flstm_decay_attention_step(shape(), rows(), rows(), rows(), rows(), None, None) == 1
    assert lib.flstm_decay_attention_step(shape(sequences=0), rows(None), rows(None), rows(None), rows(None), None, None) == 0
    assert lib.flstm_decay_attention_workspace_bytes(shape(dk=1), 0) == 0
    assert lib.flstm_decay_attention_workspace_bytes(shape(heads=1), 1) == 0


def test_decay_attention_refuses_host_tensors():
    q = torch.zeros(1, 4, 2, 32)
    with pytest.raises(ValueError, match="CUDA"):
        fl.decay_attention_forward(q, q, q, torch.zeros(2))


def test_distillation_refuses_before_device_work():
    from flashlstm_poc_amd import lm_ops
    lib = lm_ops._bind()

    def problem(**change):
        values = dict(rows=4, vocabulary=100, logits=SOME.value, ld=100, dtype=1, top=5, teacher_logits=SOME.value, teacher_dtype=0,
                      teacher_index=SOME.value, index_64=0, temperature=1.0)
        return lm_ops._PROBLEM.pack(*{**values, **change}.values())

    for change in (dict(dtype=3), dict(teacher_dtype=-1), dict(top=0), dict(top=1025), dict(temperature=0.0), dict(temperature=float("nan")),
                   dict(temperature=float("inf")), dict(temperature=1e-40), dict(vocabulary=0), dict(vocabulary=1 << 31), dict(ld=99),
                   dict(logits=0), dict(teacher_logits=0), dict(teacher_index=0)):
        assert lib.flstm_distillation_forward(problem(**change), SOME, None, None) == 1, change
    assert lib.flstm_distillation_forward(None, SOME, None, None) == 1 and lib.flstm_distillation_forward(problem(), None, None, None) == 1
    assert lib.flstm_distillation_backward(problem(), None, SOME, 1, SOME, 100, None) == 1
    assert lib.flstm_distillation_backward(problem(), SOME, SOME, 1, SOME, 99, None) == 1
    assert lib.flstm_distillation_train(problem(), SOME, 1, SOME, None, 100, None, None) == 1
    assert lib.flstm_distillation_train(problem(vocabulary=200000, ld=200000), SOME, 1, SOME, SOME, 200000, None, None) == 1   # no workspace
    assert lib.flstm_distillation_forward(problem(rows=0, logits=0), None, None, None) == 0
    assert lib.flstm_distillation_workspace_bytes(problem()) == 0
    assert lib.flstm_distillation_workspace_bytes(problem(vocabulary=200000, ld=200000)) == 32


def test_distillation_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        fl.distillation_forward(torch.zeros(2, 8), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int32))


def test_decay_attention_refuses_more_workgroups_than_a_launch_has():
    from flashlstm_poc_amd import lm_ops
    lib = lm_ops._bind()
    rows = lm_ops._ROWS.pack(SOME.value, 64, 64, 32)
    shape = lambda heads: lm_ops._SHAPE.pack(2 ** 24, 1, 0, heads, 1, 32, 32, 1, 0.5, SOME.value)
    assert lib.flstm_decay_attention_step(shape(1), rows, rows, rows, rows, SOME, None) == 2004
    assert lib.flstm_decay_attention_forward(shape(2), rows, rows, rows, None, rows, None, None, None) == 2004
    assert lib.flstm_decay_attention_backward(shape(2), rows, rows, rows, rows, None, None, rows, rows, rows, None, SOME, None) == 2004
