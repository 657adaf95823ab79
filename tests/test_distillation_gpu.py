"""The distillation loss and its gradient against 64-bit arithmetic.

Bounds: a power of two of an argument a is off by about |a| u (its rounding) and a few ulp, sums by a few ulp of their terms'
magnitudes.  With m the largest |logit| / temperature of a row and its lse: probabilities are off by (32 + 4 m) u relative, the
loss by that times the magnitudes of what it adds up, p (|log p| + |log q|)."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within, offset_copy

pytestmark = pytest.mark.gpu


def _problem(rows, vocabulary, top, dtype, seed=0, temperature=2.0, distinct=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    if distinct and top <= vocabulary:
        index = torch.stack([torch.randperm(vocabulary, device="cuda", generator=g)[:top] for _ in range(rows)]) if rows else torch.zeros(0, top, device="cuda")
    else:
        index = torch.randint(0, vocabulary, (rows, top), device="cuda", generator=g)
    return dict(logits=(2.5 * n(rows, vocabulary)).to(dtype), teacher_logits=2 * n(rows, top) + 3, teacher_index=index.to(torch.int64),
                d_loss=torch.rand(rows, device="cuda", generator=g) + 0.1, temperature=temperature)


def _definition(p):
    tau, index = p["temperature"], p["teacher_index"].long()
    vocabulary = p["logits"].shape[-1]
    z, t = p["logits"].double() / tau, p["teacher_logits"].double() / tau
    held = (index >= 0) & (index < vocabulary) & (t > -float("inf"))
    some = held.any(-1, keepdim=True)
    z = torch.where(some, z, 0.0)
    at = index.clamp(0, vocabulary - 1)
    t = t.masked_fill(~held, -float("inf"))
    log_p = torch.where(some, torch.log_softmax(torch.where(some, t, 0.0), -1), -float("inf"))
    target = log_p.exp() * held
    log_q = torch.log_softmax(z, -1)   # (not z - logsumexp, which loses the sum beside a row of lowest values)
    lse = torch.logsumexp(z, -1, keepdim=True)
    chosen = log_q.gather(1, at)
    parts = torch.where(target > 0, target * (torch.where(target > 0, log_p, 0.0) - chosen), 0.0)
    q = log_q.exp()
    dense = torch.zeros_like(z).scatter_add_(1, at, target)
    factor = p["d_loss"].double().expand(len(z))[:, None] * tau
    grad = torch.where(some, factor * (q - dense), 0.0)
    m = 32 + 4 * (z.abs().where(z.isfinite(), torch.zeros_like(z)).amax(-1, keepdim=True) + lse.abs().nan_to_num(0.0, 0.0, 0.0) +
                  torch.where(held, t.abs(), 0.0).amax(-1, keepdim=True))
    terms = torch.where(target > 0, target * (torch.where(target > 0, log_p, 0.0).abs() + chosen.abs()), 0.0).sum(-1)
    return dict(loss=tau * tau * parts.sum(-1), grad=grad, loss_slack=tau * tau * U32 * m[:, 0] * (terms + 1),
                grad_slack=torch.where(some, factor.abs() * (q + dense) * U32 * m, 0.0))


def _own(p, d_loss=None):
    args = (p["logits"], p["teacher_logits"], p["teacher_index"])
    loss, stats = fl.distillation_forward(*args, temperature=p["temperature"])
    grad = fl.distillation_backward(p["d_loss"], *args, stats, temperature=p["temperature"])
    both = fl.distillation_train(*args, p["d_loss"], temperature=p["temperature"])
    return dict(loss=loss, grad=grad, train_loss=both[0], train_grad=both[1])


def _check(p, got, label=""):
    want = _definition(p)
    for name in ("loss", "train_loss"):
        assert_within(got[name], want["loss"], want["loss_slack"], f"{label} {name}")
    for name in ("grad", "train_grad"):
        assert_within(got[name], want["grad"], want["grad_slack"], f"{label} {name}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocabulary", [1, 2, 7, 8, 9, 100, 2047, 2048, 2055, 5000, 8192, 8193, 16384, 16391, 32000, 50001, 65536, 65543, 131072, 140001])
def test_vocabularies(vocabulary, dtype):
    p = _problem(3, vocabulary, min(vocabulary, 20), dtype, seed=vocabulary)
    _check(p, _own(p), f"{vocabulary}")


@pytest.mark.parametrize("top", [1, 2, 64, 255, 256, 257, 1000, 1024])
@pytest.mark.parametrize("vocabulary", [1024, 20000])
def test_numbers_of_entries(top, vocabulary):
    p = _problem(5, vocabulary, top, torch.bfloat16, seed=top)
    _check(p, _own(p))


@pytest.mark.parametrize("temperature", [0.25, 1.0, 4.0, 50.0])
def test_temperatures(temperature):
    p = _problem(6, 3000, 16, torch.float32, temperature=temperature)
    _check(p, _own(p))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocabulary", [300, 40000, 140000])
def test_entries_that_do_not_count(vocabulary, dtype):
    p = _problem(8, vocabulary, 12, dtype)
    p["teacher_index"][0] = -1                                  # a row without entries
    p["logits"][0] = float("nan")                               # with anything in it
    p["teacher_index"][1, 3:] = -1
    p["teacher_index"][2, 5], p["teacher_index"][2, 6] = vocabulary, 1 << 40
    p["teacher_logits"][3, 2:7] = -float("inf")
    p["teacher_logits"][4] = -float("inf")
    p["teacher_logits"][5, 1] = -2000.0                         # a probability of zero
    p["teacher_index"][7] = -(1 << 40)
    p["d_loss"][7] = float("nan")
    got = _own(p)
    for row in (0, 4, 7):
        assert float(got["loss"][row]) == 0 and not bool(got["grad"][row].any()) and not bool(got["train_grad"][row].any())
    _check(dict(p, d_loss=p["d_loss"].nan_to_num(1.0)), got)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_indices_that_come_twice(dtype):
    p = _problem(4, 50, 40, dtype, distinct=False)
    p["teacher_index"][0] = 7
    p["teacher_index"][1, ::2] = 3
    got = _own(p)
    _check(p, got)
    again = _own(p)
    for name in got:
        assert torch.equal(got[name], again[name]), name
    order = torch.randperm(40, device="cuda")                   # one entry for all, and entries in another order
    p["teacher_index"], p["teacher_logits"] = p["teacher_index"][:, order], p["teacher_logits"][:, order]
    _check(p, _own(p))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masked_vocabularies(dtype):
    p = _problem(5, 9000, 10, dtype)
    low = torch.finfo(dtype).min
    named = torch.zeros(5, 9000, dtype=torch.bool, device="cuda").scatter_(1, p["teacher_index"], True)
    p["logits"][:2] = torch.where(named[:2], p["logits"][:2], -float("inf"))
    p["logits"][2] = torch.where(named[2], p["logits"][2], low)  # the type's lowest value, beside others
    p["logits"][3] = low                                         # and all of a row
    got = _own(p)
    _check(p, got)
    assert bool(torch.isfinite(got["loss"]).all()) and bool(torch.isfinite(got["grad"].float()).all())
    # a row of lowest values alone: the bound above goes by its largest logit, which is that, and allows anything; its tokens are alike
    want = _definition(p)
    for name in ("grad", "train_grad"):
        assert_within(got[name][3], want["grad"][3], 128 * U32 * want["grad"][3].abs(), name)
    assert_within(got["loss"][3], want["loss"][3], 128 * U32 * (want["loss"][3].abs() + 10), "loss")
    # a token that the student rules out and the teacher does not: an infinite loss, a finite gradient
    p["logits"][4, p["teacher_index"][4, 0]] = -float("inf")
    got = _own(p)
    assert float(got["loss"][4]) == float("inf") and float(got["train_loss"][4]) == float("inf")
    assert bool(torch.isfinite(got["grad"][4]).all()) and torch.equal(got["grad"][4], got["train_grad"][4])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides_types_and_shapes(dtype):
    p = _problem(12, 701, 9, dtype)
    want = _own(p)
    room = torch.full((12, 705), float("nan"), device="cuda", dtype=dtype)
    room[:, 2:703].copy_(p["logits"])
    for view in (dict(p, logits=room[:, 2:703]), dict(p, logits=offset_copy(p["logits"]))):   # (where a row begins decides the order of its sums)
        _check(view, _own(view))
    views = [dict(p, logits=p["logits"].t().contiguous().t()), dict(p, teacher_index=p["teacher_index"].to(torch.int32)), dict(p, teacher_logits=p["teacher_logits"].t().contiguous().t()),
             dict(p, teacher_index=p["teacher_index"].t().contiguous().t(), d_loss=torch.stack([p["d_loss"], p["d_loss"]], 1)[:, 0])]
    for view in views:
        got = _own(view)
        for name in want:
            assert torch.equal(want[name], got[name]), name
    half = dict(p, teacher_logits=p["teacher_logits"].to(dtype))
    _check(half, _own(half))
    one = dict(p, d_loss=torch.full((1,), 0.125, device="cuda"))
    all_ = dict(p, d_loss=torch.full((12,), 0.125, device="cuda"))
    assert torch.equal(_own(one)["grad"], _own(all_)["grad"]) and torch.equal(_own(one)["train_grad"], _own(all_)["train_grad"])
    shaped = {name: p[name].view(3, 4, *p[name].shape[1:]) for name in ("logits", "teacher_logits", "teacher_index", "d_loss")}
    got = _own(dict(shaped, temperature=p["temperature"]))
    assert got["loss"].shape == (3, 4) and torch.equal(got["grad"].view(12, 701), want["grad"])
    # one row for all, expanded
    shared = dict(p, logits=p["logits"][:1].expand(12, 701))
    copied = dict(p, logits=p["logits"][:1].expand(12, 701).contiguous())
    assert torch.equal(_own(shared)["grad"], _own(copied)["grad"])


@pytest.mark.parametrize("vocabulary", [500, 33000, 150000])
def test_in_place(vocabulary):
    p = _problem(6, vocabulary, 30, torch.bfloat16, distinct=False)
    want = _own(p)
    room = torch.zeros(6, vocabulary + 3, device="cuda", dtype=torch.bfloat16)
    for logits in (p["logits"].clone(), room[:, 1:-2].copy_(p["logits"])):
        loss, grad = fl.distillation_train(logits, p["teacher_logits"], p["teacher_index"], p["d_loss"], temperature=p["temperature"], in_place=True)
        assert grad is logits
        if logits.is_contiguous():
            assert torch.equal(grad, want["train_grad"]) and torch.equal(loss, want["train_loss"])
        _check(p, dict(want, train_grad=grad, train_loss=loss))
    assert not bool(room[:, 0].any()) and not bool(room[:, -2:].any())
    with pytest.raises(ValueError, match="in place"):
        fl.distillation_train(p["logits"].t().contiguous().t(), p["teacher_logits"], p["teacher_index"], p["d_loss"], in_place=True)


def test_offsets_beyond_32_bits():
    far = (1 << 31) + 40
    room = torch.zeros(far + 3000, device="cuda", dtype=torch.float16)
    p = _problem(2, 3000, 10, torch.float16)
    want = _own(p)
    view = room.as_strided((2, 3000), (far, 1))
    view.copy_(p["logits"])
    got = _own(dict(p, logits=view))
    for name in want:
        assert torch.equal(want[name], got[name]), name


def test_empty():
    p = _problem(0, 30, 4, torch.float16)
    got = _own(p)
    assert got["loss"].shape == (0,) and got["grad"].shape == (0, 30) and got["train_grad"].shape == (0, 30)


def test_gradient_against_differences_and_autograd():
    p = _problem(5, 200, 12, torch.float32, distinct=False)
    logits = p["logits"].clone().requires_grad_()
    loss = fl.distillation_loss(logits, p["teacher_logits"], p["teacher_index"], temperature=2.0)
    loss.backward(p["d_loss"])
    assert torch.equal(logits.grad, _own(p)["grad"])
    for j in range(3):
        direction = torch.randn(5, 200, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(j))
        h = 1e-5
        up, down = (float((_definition(dict(p, logits=p["logits"].double() + s * h * direction))["loss"] * p["d_loss"].double()).sum()) for s in (1, -1))
        products = logits.grad.double() * direction
        # the difference's own error: h^2 times a third derivative of order one, and 64-bit rounding over h
        assert abs(float(products.sum()) - (up - down) / (2 * h)) <= 1e-8 * 200 + 256 * U32 * float(products.abs().sum())
    logits.grad = None
    fl.distillation_loss(logits, p["teacher_logits"], p["teacher_index"]).mean().backward()   # a broadcast gradient
    even = fl.distillation_train(p["logits"], p["teacher_logits"], p["teacher_index"], torch.full((1,), 0.2, device="cuda"))[1]
    assert torch.allclose(logits.grad, even, rtol=1e-5, atol=1e-9)
    with torch.no_grad():
        assert not fl.distillation_loss(logits, p["teacher_logits"], p["teacher_index"]).requires_grad


def test_other_streams_and_graphs():
    p = _problem(20, 40000, 16, torch.float16)
    want = _own(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _own(p)
    torch.cuda.current_stream().wait_stream(side)
    for name in want:
        assert torch.equal(want[name], got[name]), name
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _own(p)
    for seed in range(3):
        fresh = _problem(20, 40000, 16, torch.float16, seed=seed)
        for name in ("logits", "teacher_logits", "teacher_index", "d_loss"):
            p[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        want = _own(p)
        for name in want:
            assert torch.equal(want[name], got[name]), name


def test_refusals():
    p = _problem(4, 100, 5, torch.float16)
    z, t, i, d = p["logits"], p["teacher_logits"], p["teacher_index"], p["d_loss"]
    for args, more, match in (((z.cpu(), t, i), {}, "logits must be a CUDA"), ((z.double(), t, i), {}, "unsupported dtype"), ((z, t, i.short()), {}, "int32 or int64"),
                              ((z, t[:2], i), {}, "shape"), ((z, t[:, :3], i), {}, "shape"), ((z[:2], t, i), {}, "shape"), ((z, t, i.cpu()), {}, "teacher_index"),
                              ((z, t, i), dict(temperature=0.0), "temperature"), ((z, t, i), dict(temperature=float("nan")), "temperature"),
                              ((z, t[:, :0], i[:, :0]), {}, "between 1 and 1024"),
                              ((z, t[:, :1].repeat(1, 1025), i[:, :1].repeat(1, 1025)), {}, "between 1 and 1024")):
        with pytest.raises(ValueError, match=match):
            fl.distillation_forward(*args, **more)
    loss, stats = fl.distillation_forward(z, t, i)
    with pytest.raises(ValueError, match="d_loss"):
        fl.distillation_backward(d[:3], z, t, i, stats)
    with pytest.raises(ValueError, match="d_loss"):
        fl.distillation_train(z, t, i, d.half())
    with pytest.raises(ValueError, match="stats"):
        fl.distillation_backward(d, z, t, i, stats[:2])


def test_more_rows_than_a_launch_has():
    """Rows are launched at most 2^21 at a time."""
    p = _problem(2 ** 21 + 3, 5, 3, torch.bfloat16, distinct=False)
    _check(p, _own(p))


def test_in_place_is_known_to_autograd():
    p = _problem(4, 100, 8, torch.float32)
    logits = p["logits"].requires_grad_()
    kept = logits * 1.0
    square = kept * kept
    fl.distillation_train(kept.detach(), p["teacher_logits"], p["teacher_index"], p["d_loss"], in_place=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.sum().backward()
