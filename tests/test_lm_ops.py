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
    assert {"flstm_layer_norm_forward", "flstm_layer_norm_backward", "flstm_layer_norm_workspace_bytes"} <= names
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
