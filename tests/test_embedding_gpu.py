"""The embedding of tokens and its gradient against 64-bit arithmetic.

Bounds: a row times the scale is one rounding in 32 bits and one to the type.  A token's gradient is a sum of k rows, in whatever order, of at
most k additions in a chain, each off by at most an ulp of what is summed (k u times the sum of the magnitudes), then the scale's
rounding and the type's."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within, offset_copy

pytestmark = pytest.mark.gpu


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tokens(count, vocabulary, seed=0, kind="text"):
    g = _generator(seed)
    if kind == "text":   # the n-th most frequent with a share of about 1 / n, some outside
        t = (vocabulary ** torch.rand(count, device="cuda", generator=g, dtype=torch.float64)).long() - 1
        return torch.where(torch.rand(count, device="cuda", generator=g) < 0.05, -1, t.clamp(max=vocabulary - 1))
    if kind == "one":
        return torch.full((count,), vocabulary // 2, device="cuda")
    if kind == "rising":
        return torch.arange(count, device="cuda") % vocabulary
    if kind == "falling":
        return vocabulary - 1 - torch.arange(count, device="cuda") % vocabulary
    if kind == "pairs":
        return torch.arange(count, device="cuda") // 33 % vocabulary
    assert kind == "outside"
    return torch.tensor([-1, vocabulary, 2 ** 31 - 1, -2 ** 31, 2 ** 40, -2 ** 62], device="cuda").repeat(count)[:count]


def _check_forward(tokens, table, scale, dtype):
    got = fl.embedding_forward(tokens, table, scale=scale, dtype=dtype)
    assert got.dtype == (dtype or table.dtype)
    held = (tokens >= 0) & (tokens < len(table))
    scale = float(torch.tensor(scale, dtype=torch.float32))
    want = torch.where(held[..., None], scale * table.double()[torch.where(held, tokens, 0).long()], 0.0)
    assert_within(got, want, U32 * want.abs(), f"{tuple(tokens.shape)} of {tuple(table.shape)} {table.dtype} as {dtype}")


def _check_backward(d_out, tokens, vocabulary, scale=1.0, dtype=torch.float32):
    got = fl.embedding_backward(d_out, tokens, vocabulary, scale=scale, dtype=dtype)
    assert got.dtype == dtype
    flat, d = tokens.reshape(-1), d_out.reshape(-1, d_out.shape[-1]).double()
    held = (flat >= 0) & (flat < vocabulary)
    index = torch.where(held, flat, vocabulary).long()
    scale = float(torch.tensor(scale, dtype=torch.float32))
    index = index.cpu()
    sums = lambda x: torch.zeros(vocabulary + 1, x.shape[1], dtype=torch.float64).index_add_(0, index, x.cpu())[:-1].to(d.device)
    want, size, count = scale * sums(d), abs(scale) * sums(d.abs()), sums(torch.ones_like(d[:, :1]))
    assert_within(got, want, U32 * (count + 1) * size, f"{tuple(tokens.shape)} over {vocabulary} {d_out.dtype} to {dtype}")
    return got


@pytest.mark.parametrize("table", DTYPES, ids=str)
@pytest.mark.parametrize("dtype", [None] + DTYPES, ids=str)
def test_forward_types(table, dtype):
    for width in (1, 3, 8, 33, 64, 257, 1024, 2050):
        rows = torch.randn(50, width, device="cuda", generator=_generator(width)).to(table)
        _check_forward(_tokens(70, 50, width), rows, 1.0 if width % 2 else width ** 0.5, dtype)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_forward_shapes_and_places(index):
    table = torch.randn(300, 130, device="cuda", generator=_generator(0))
    wide = torch.zeros(300, 3, 131, device="cuda")
    view = wide[:, 1, 1:]
    view.copy_(table)
    tokens = _tokens(60, 300).to(index)
    for t in (tokens, tokens.view(4, 15), tokens.view(4, 15).t(), tokens[:1].view(()), offset_copy(tokens)):
        for rows in (table, view, offset_copy(table), table.t().contiguous().t(), table[:1].expand(300, 130)):
            _check_forward(t, rows, 0.37, torch.float16)
    out = fl.embedding_forward(_tokens(7, 300, kind="outside"), table)
    assert not bool(out.any())


@pytest.mark.parametrize("kind", ["text", "one", "rising", "falling", "pairs", "outside"])
@pytest.mark.parametrize("count", [1, 2, 31, 32, 33, 64, 65, 1000, 2048, 2049, 5000, 20000])
def test_backward_orders(kind, count):
    for vocabulary, width in ((1, 9), (70, 40), (1023, 8), (1024, 8), (5000, 17)):
        d = torch.randn(count, width, device="cuda", generator=_generator(count)).half()
        _check_backward(d, _tokens(count, vocabulary, count, kind), vocabulary, 1.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("out", DTYPES, ids=str)
def test_backward_types(dtype, out):
    for width in (1, 3, 8, 33, 64, 257, 1024, 2050):
        d = torch.randn(300, width, device="cuda", generator=_generator(width)).to(dtype)
        _check_backward(d, _tokens(300, 60, width), 60, width ** -0.5, out)


@pytest.mark.parametrize("vocabulary", [2 ** 20 - 1, 2 ** 20, 1500000])
def test_backward_large_vocabularies(vocabulary):
    tokens = _tokens(3000, vocabulary, 1)
    _check_backward(torch.randn(3000, 4, device="cuda", generator=_generator(1)), tokens, vocabulary)
    tokens[:5] = vocabulary - 1
    _check_backward(torch.randn(3000, 4, device="cuda", generator=_generator(2)), tokens, vocabulary)


def test_backward_many_tokens():
    for count, vocabulary, width in ((600000, 3000, 8), (300000, 50001, 33)):
        _check_backward(torch.randn(count, width, device="cuda", generator=_generator(3)).bfloat16(), _tokens(count, vocabulary, 3), vocabulary)


def test_backward_strides():
    tokens = _tokens(600, 50).view(20, 30)
    d = torch.randn(20, 30, 66, device="cuda", generator=_generator(4)).half()
    want = _check_backward(d, tokens, 50)
    wide = torch.zeros(20, 30, 3, 67, device="cuda", dtype=torch.float16)
    view = wide[:, :, 1, 1:]
    view.copy_(d)
    assert torch.equal(fl.embedding_backward(view, tokens.int(), 50), want)
    assert torch.equal(fl.embedding_backward(offset_copy(d), offset_copy(tokens), 50), want)
    assert torch.equal(fl.embedding_backward(d.transpose(0, 1).contiguous().transpose(0, 1), tokens.t().contiguous().t(), 50), want)
    _check_backward(d[:1, :1].expand(20, 30, 66), tokens, 50)


def test_infinities_and_nan_stay_with_their_tokens():
    tokens = _tokens(500, 40)
    d = torch.randn(500, 24, device="cuda", generator=_generator(5))
    d[7, 3], d[100, 5] = float("inf"), float("nan")
    tokens[7], tokens[100], tokens[9] = 3, 4, -1
    d[9] = float("nan")
    got = fl.embedding_backward(d, tokens, 40)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[3, 3] = bad[4, 5] = True
    assert torch.equal(~got.isfinite(), bad)


def test_empty():
    none = torch.empty(0, device="cuda", dtype=torch.int64)
    assert fl.embedding_forward(none, torch.ones(5, 6, device="cuda")).shape == (0, 6)
    got = fl.embedding_backward(torch.empty(0, 6, device="cuda"), none, 5)
    assert got.shape == (5, 6) and not bool(got.any())
    assert fl.embedding_forward(torch.zeros(3, device="cuda", dtype=torch.int64), torch.empty(5, 0, device="cuda")).shape == (3, 0)
    assert fl.embedding_backward(torch.empty(3, 0, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.int64), 5).shape == (5, 0)


def test_same_bits_from_call_to_call_and_on_other_streams():
    tokens, d = _tokens(9000, 700), torch.randn(9000, 65, device="cuda", generator=_generator(6)).half()
    want = fl.embedding_backward(d, tokens, 700)
    for _ in range(3):
        assert torch.equal(fl.embedding_backward(d, tokens, 700), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fl.embedding_backward(d, tokens, 700)
    here = fl.embedding_backward(d, tokens, 700)   # two at a time
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(here, want)


@pytest.mark.parametrize("count", [300, 12000])
def test_captured_in_a_graph(count):
    tokens, table = _tokens(count, 500), torch.randn(500, 64, device="cuda", generator=_generator(7))
    d = torch.randn(count, 64, device="cuda", generator=_generator(8))
    run = lambda: (fl.embedding_forward(tokens, table, dtype=torch.float16), fl.embedding_backward(d, tokens, 500))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(4):
        tokens.copy_(_tokens(count, 500, seed, "text" if seed % 2 else "pairs"))
        d.normal_(generator=_generator(20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run()):
            assert torch.equal(a, b)


def test_autograd():
    tokens = _tokens(40, 30).view(5, 8)
    module = fl.Embedding(30, 20, scale=2.5, dtype=torch.float16)
    out = module(tokens)
    d = torch.randn(5, 8, 20, device="cuda", generator=_generator(9)).half()
    out.backward(d)
    assert out.dtype == torch.float16 and torch.equal(module.weight.grad, fl.embedding_backward(d, tokens, 30, scale=2.5))
    # the result is linear in the table: its gradient against differences, in the direction of a whole table
    table = torch.randn(30, 20, device="cuda", generator=_generator(10), requires_grad=True)
    fl.embedding(tokens, table, scale=0.5).backward(d.float())
    step = torch.randn(30, 20, device="cuda", generator=_generator(11))
    up, down = (fl.embedding(tokens, table.detach() + s * step, scale=0.5).double() for s in (1, -1))
    slope, along = ((up - down) * d.double()).sum() / 2, (table.grad.double() * step.double()).sum()
    # 40 rows of 20 products, each of two values rounded to 2^-24 of some units
    assert abs(float(slope - along)) <= 40 * 20 * 8 * U32 * 4
    half = table.detach().half().requires_grad_()
    fl.embedding(tokens, half).sum().backward()
    assert half.grad.dtype == torch.float16
    with torch.no_grad():
        assert not module(tokens).requires_grad
    torch.manual_seed(3)
    ours = fl.Embedding(9, 4)
    torch.manual_seed(3)
    assert torch.equal(ours.weight, torch.nn.Embedding(9, 4, device="cuda").weight) and list(ours.state_dict()) == ["weight"]


def test_refusals():
    tokens, table = torch.zeros(4, device="cuda", dtype=torch.int64), torch.ones(5, 6, device="cuda")
    for bad, match in ((dict(tokens=tokens.cpu()), "tokens"), (dict(tokens=tokens.float()), "tokens"), (dict(table=table.cpu()), "table"),
                       (dict(table=table.double()), "dtype"), (dict(table=table[0]), "table"), (dict(table=table[:0]), "table"),
                       (dict(dtype=torch.float64), "dtype"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")):
        with pytest.raises(ValueError, match=match):
            fl.embedding_forward(**{**dict(tokens=tokens, table=table), **bad})
    d = torch.ones(4, 6, device="cuda")
    for bad, match in ((dict(d_out=d[:3]), "d_out"), (dict(d_out=d.double()), "dtype"), (dict(vocabulary=0), "vocabulary"),
                       (dict(dtype=torch.int32), "dtype"), (dict(scale=float("nan")), "scale")):
        with pytest.raises(ValueError, match=match):
            fl.embedding_backward(**{**dict(d_out=d, tokens=tokens, vocabulary=5), **bad})
    for bad in ((0, 4), (4, 0)):
        with pytest.raises(ValueError, match=">= 1"):
            fl.Embedding(*bad)
