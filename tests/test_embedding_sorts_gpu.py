"""The embedding's gradient by sorts of one to three passes and of all widths, and over tables of more than 32 MiB, whose zeros are written past the caches by all
launches of the sort, against 64-bit arithmetic (bounds as in test_embedding_gpu.py)."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within
from test_embedding_gpu import _check_backward, _generator, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocabulary", [1, 5, 100, 127, 1023, 1024, 4095, 4096, 2 ** 17, 2 ** 18 - 1, 2 ** 20 - 1, 2 ** 20, 1500000])
@pytest.mark.parametrize("count", [8192, 8193, 9000, 20000])
def test_passes_and_bits(vocabulary, count):
    """More than 8192 tokens are sorted in passes: one up to 1023 tokens, two up to 2^20 - 1, then three."""
    for kind in ("text", "rising", "falling"):
        tokens = _tokens(count, vocabulary, vocabulary, kind)
        tokens[count // 2:count // 2 + 5] = vocabulary - 1
        _check_backward(torch.randn(count, 2, device="cuda", generator=_generator(count)), tokens, vocabulary)


@pytest.mark.parametrize("out", DTYPES, ids=str)
@pytest.mark.parametrize("vocabulary,width,count", [(4000, 4200, 9000), (20000, 901, 30001), (1200000, 17, 12345), (50001, 513, 3000)])
def test_tables_of_more_than_32_mib(vocabulary, width, count, out):
    """Every row of a table that held something else, those of tokens and those of none (the last of them sorted in one launch, by ranks)."""
    assert vocabulary * width * torch.empty((), dtype=out).element_size() > 32 << 20
    tokens = _tokens(count, vocabulary, 7)
    tokens[:2], tokens[-1] = vocabulary - 1, 0
    d = torch.randn(count, width, device="cuda", generator=_generator(8)).half()
    room = [torch.full((vocabulary, width), float("nan"), device="cuda", dtype=out) for _ in range(2)]
    del room                                                        # (what the result is likely to lie in)
    got = fl.embedding_backward(d, tokens, vocabulary, scale=0.75, dtype=out)
    held = tokens >= 0
    there = torch.zeros(vocabulary, device="cuda", dtype=torch.bool)
    there[tokens[held]] = True
    assert not bool(got[~there].any())                              # (a NaN is something)
    rows, place = torch.unique(tokens[held], return_inverse=True)
    sums = lambda x: torch.zeros(len(rows), x.shape[1], dtype=torch.float64).index_add_(0, place.cpu(), x.cpu())
    d = d[held].double()
    want, size, many = 0.75 * sums(d), 0.75 * sums(d.abs()), sums(torch.ones_like(d[:, :1]))
    assert_within(got[rows].cpu(), want, U32 * (many + 1) * size, f"{vocabulary} x {width} of {count} to {out}")
