"""The gated linear recurrence over tensors beyond what the caches hold, which are written past them, cut into segments and with a gate: every output against
64-bit arithmetic, with the bounds of test_gated_recurrence_gpu.py."""
import pytest
import torch

from test_gated_recurrence_gpu import _check, _problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,sequences,tokens,width", [(torch.float16, 3, 6000, 1024), (torch.float32, 2, 5000, 1000), (torch.bfloat16, 1, 18000, 1026)])
def test_more_than_the_caches_hold_with_a_gate(dtype, sequences, tokens, width):
    assert sequences * tokens * width * torch.empty((), dtype=dtype).element_size() > 32 << 20
    _check(_problem((sequences, tokens, width), dtype, sequences, True, seed=21), f"{sequences} x {tokens} x {width} {dtype}")
