"""Layer norm on a residual stream against 64-bit arithmetic.

Bounds: outputs are rounded to their type once.  In front of that, sums of w values in fp32 are off by at most a few ulp of the
sum of their magnitudes (trees over lanes, eight values a lane): 32 u max|x| covers a mean.  The error of y is that of the mean
times rstd times |weight|, plus a few roundings of y itself.  In a gradient the same errors meet factors of rstd, n and h."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within, offset_copy

pytestmark = pytest.mark.gpu
WIDTHS = [1, 3, 8, 63, 64, 65, 128, 200, 257, 512, 650, 1024, 1025, 2048, 2050, 4097, 8192, 8193, 16384]


def _problem(rows, width, dtype, seed=0, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    p = dict(x=(n(rows, width) + 0.5 * n(rows, 1)).to(dtype), residual=n(rows, width).to(dtype) if residual else None,
             weight=1 + 0.2 * n(width), bias=0.3 * n(width), dy=n(rows, width).to(dtype), d_total=n(rows, width).to(dtype))
    return p


def _definition(p, eps=1e-5):
    x = p["x"].double()
    total = x if p["residual"] is None else (x + p["residual"].double()).to(p["x"].dtype).double()
    mean = total.mean(-1, keepdim=True)
    rstd = ((total - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    w = torch.ones_like(total[0]) if p["weight"] is None else p["weight"].double()
    b = torch.zeros_like(w) if p["bias"] is None else p["bias"].double()
    n = (total - mean) * rstd
    dy = p["dy"].double()
    h = dy * w
    dx = rstd * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
    if p["d_total"] is not None:
        dx = dx + p["d_total"].double()
    return dict(total=total, mean=mean, rstd=rstd, n=n, w=w, h=h, y=n * w + b, dx=dx, dweight=(dy * n).sum(0), dbias=dy.sum(0), dy=dy)


def _check(p, got, label):
    r = _definition(p)
    most = r["total"].abs().amax(-1, keepdim=True)
    # (a row without variance: rstd is 1 / sqrt(eps), and so large is the factor on the mean's error)
    shift = 32 * U32 * most * r["rstd"]
    assert_within(got["total"], r["total"], 0 * r["total"], f"{label} total")
    assert_within(got["mean"], r["mean"].flatten(), (32 * U32 * most).flatten(), f"{label} mean")
    assert_within(got["y"], r["y"], shift * r["w"].abs() + 32 * U32 * (r["n"] * r["w"]).abs() + 2 * U32 * r["y"].abs(), f"{label} y")
    if "dx" in got:
        reach = r["h"].abs().amax(-1, keepdim=True) * (1 + r["n"].abs()) * (1 + r["n"].abs().amax(-1, keepdim=True))
        assert_within(got["dx"], r["dx"], r["rstd"] * reach * (64 * U32 + 2 * shift) + 2 * U32 * r["dx"].abs(), f"{label} dx")
        # sums over rows: at most (rows of a lane + partial sums) additions in a chain, each off by an ulp of what is summed
        chain = (64 + len(r["dy"]) / 64) * U32
        assert_within(got["dweight"], r["dweight"], chain * (r["dy"] * r["n"]).abs().sum(0) + (shift * r["dy"].abs()).sum(0) +
                      32 * U32 * (r["dy"] * r["n"]).abs().sum(0), f"{label} dweight")
        assert_within(got["dbias"], r["dbias"], chain * r["dy"].abs().sum(0), f"{label} dbias")


def _own(p, want_d_total=True):
    y, total, mean, rstd = fl.layer_norm_forward(p["x"], p["weight"], p["bias"], residual=p["residual"])
    dx, dw, db = fl.layer_norm_backward(p["dy"], total, p["weight"], mean, rstd, d_total=p["d_total"] if want_d_total else None)
    return dict(y=y, total=total, mean=mean, rstd=rstd, dx=dx, dweight=dw, dbias=db)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width, dtype):
    for rows, residual in ((1, True), (37, False), (260, True)):
        p = _problem(rows, width, dtype, seed=rows, residual=residual)
        _check(p, _own(p), f"{rows} x {width} {dtype}")


@pytest.mark.parametrize("rows,width", [(5000, 64), (14000, 257), (20000, 1000), (9000, 2048), (3000, 5000)])
def test_many_rows(rows, width):
    p = _problem(rows, width, torch.float16, seed=1)
    _check(p, _own(p), f"{rows} x {width}")


def test_without_parameters_and_without_stream_gradient():
    p = _problem(19, 130, torch.bfloat16, residual=False)
    p["weight"] = p["bias"] = p["d_total"] = None
    _check(p, _own(p, False), "bare")
    p = _problem(19, 130, torch.bfloat16)
    y, total, mean, rstd = fl.layer_norm_forward(p["x"], p["weight"], p["bias"], residual=p["residual"])
    dx, dw, db = fl.layer_norm_backward(p["dy"], total, p["weight"], mean, rstd, d_total=p["d_total"], want_parameters=False)
    assert dw is None and db is None and torch.equal(dx, _own(p)["dx"])


def test_rows_without_variance_and_far_from_zero():
    p = _problem(24, 300, torch.float32, residual=False)
    p["x"][:8] = 3.25                      # no variance at all
    p["x"][8:16] = 4096 + p["x"][8:16]     # a mean of thousands of standard deviations
    p["x"][16:] *= 1e-4                    # eps decides
    _check(p, _own(p), "edge rows")
    assert torch.equal(_own(p)["y"][:8], p["bias"].expand(8, -1))


def test_infinities_and_nan_stay_in_their_rows():
    p = _problem(40, 520, torch.float16)
    p["x"][3, 7], p["x"][17, 0], p["residual"][30, 519] = float("inf"), float("nan"), float("-inf")
    got, marked = _own(p), torch.zeros(40, dtype=torch.bool, device="cuda")
    marked[[3, 17, 30]] = True
    assert bool(got["y"][~marked].isfinite().all()) and not bool(got["y"][marked].isfinite().any())
    assert bool(got["dx"][~marked].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides_and_alignment(dtype):
    p = _problem(33, 130, dtype)
    want = _own(p)
    wide = torch.zeros(33, 3, 131, device="cuda", dtype=dtype)
    for name in ("x", "dy"):   # rows of a larger tensor, an odd distance apart
        view = wide.clone()[:, 1, 1:]
        view.copy_(p[name])
        p[name] = view
    p["residual"], p["d_total"] = offset_copy(p["residual"]), p["d_total"].t().contiguous().t()   # columns contiguous, not rows
    got = _own(p)
    for name in want:
        assert torch.equal(want[name], got[name]), name
    # a leading shape, a broadcast residual
    x = p["x"].contiguous().view(11, 3, 130)
    y, total, _, _ = fl.layer_norm_forward(x, p["weight"], p["bias"], residual=p["residual"][:1].expand(33, 130).view(11, 3, 130))
    again = fl.layer_norm_forward(x.view(33, 130), p["weight"], p["bias"], residual=p["residual"][:1].expand(33, 130).contiguous())
    assert y.shape == x.shape and torch.equal(y.view(33, 130), again[0]) and torch.equal(total.view(33, 130), again[1])


def test_empty():
    for shape in ((0, 64), (5, 0)):
        x = torch.empty(shape, device="cuda")
        y, total, mean, rstd = fl.layer_norm_forward(x)
        assert y.shape == shape
    x = torch.empty(0, 64, device="cuda")
    y, total, mean, rstd = fl.layer_norm_forward(x)
    dx, dw, db = fl.layer_norm_backward(x, total, None, mean, rstd)
    assert dx.shape == (0, 64) and not bool(dw.any()) and not bool(db.any()) and dw.shape == (64,)


def test_gradients_against_differences():
    p = _problem(6, 37, torch.float32, seed=5)
    module = fl.LayerNorm(37)
    with torch.no_grad():
        module.weight.copy_(p["weight"])
        module.bias.copy_(p["bias"])
    x, r = p["x"].clone().requires_grad_(), p["residual"].clone().requires_grad_()
    y, total = module(x, r)
    (y * p["dy"] + total * p["d_total"]).sum().backward()

    def loss(x, r, w, b):
        t = (x + r)
        n = torch.nn.functional.layer_norm(t, (37,), w, b, 1e-5)
        return (n * p["dy"].double() + t * p["d_total"].double()).sum()

    at = [t.double() for t in (p["x"], p["residual"], p["weight"], p["bias"])]
    for k, grad in enumerate((x.grad, r.grad, module.weight.grad, module.bias.grad)):
        direction = torch.randn(at[k].shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(k))
        h = 1e-5
        up, down = ([a + s * h * direction if j == k else a for j, a in enumerate(at)] for s in (1, -1))
        slope = float((loss(*up) - loss(*down)) / (2 * h))
        # the difference's own error is h^2 of a third derivative of order 100; total's rounding moves n by an ulp
        assert abs(float((grad.double() * direction).sum()) - slope) <= 1e-4 * max(1.0, float((grad.double() * direction).abs().sum()))


def test_autograd_paths():
    p = _problem(9, 64, torch.float16)
    want = _own(p)
    x = p["x"].clone().requires_grad_()
    y, total = fl.layer_norm(x, p["weight"], p["bias"], residual=p["residual"])
    torch.autograd.backward([y, total], [p["dy"], p["d_total"]])
    assert torch.equal(y, want["y"]) and torch.equal(x.grad, want["dx"])
    x.grad = None
    _, total = fl.layer_norm(x, p["weight"], p["bias"], residual=p["residual"])
    total.backward(p["d_total"])
    assert torch.equal(x.grad, p["d_total"])
    module = fl.LayerNorm(64)
    y = module(p["x"])
    y.backward(p["dy"])
    assert module.weight.grad.shape == (64,) and module.bias.grad.shape == (64,)
    with torch.no_grad():
        assert not module(p["x"]).requires_grad


def test_other_streams_and_repeats():
    p = _problem(700, 513, torch.bfloat16)
    want = _own(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _own(p)
    torch.cuda.current_stream().wait_stream(side)
    for name in want:
        assert torch.equal(want[name], got[name]), name


def test_captured_in_a_graph():
    p = _problem(64, 1024, torch.float16)
    _own(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _own(p)
    for seed in range(3):
        fresh = _problem(64, 1024, torch.float16, seed=seed)
        for name in ("x", "residual", "weight", "bias", "dy", "d_total"):
            p[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        want = _own(p)
        for name in want:
            assert torch.equal(want[name], got[name]), name


def test_in_place_through_the_c_entry_points():
    import ctypes
    lib = fl.load_library()
    p = _problem(50, 96, torch.float16)
    want = _own(p)
    x, r, stats = p["x"].clone(), p["residual"].clone(), torch.empty(2, 50, device="cuda")
    code = lambda t: ctypes.c_void_p(t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    rc = lib.flstm_layer_norm_forward(50, 96, code(x), 96, code(r), 96, 1, code(p["weight"]), code(p["bias"]), 1e-5, code(r), code(x),
                                      code(stats[0]), code(stats[1]), stream)
    assert rc == 0 and torch.equal(x, want["y"]) and torch.equal(r, want["total"])
    dy = p["dy"].clone()
    rc = lib.flstm_layer_norm_backward(50, 96, code(dy), 96, code(r), 96, code(p["d_total"]), 96, 1, code(p["weight"]), code(stats[0]),
                                       code(stats[1]), code(dy), None, None, None, stream)
    assert rc == 0 and torch.equal(dy, want["dx"])


def test_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad, match in ((dict(x=x.cpu()), "CUDA"), (dict(x=x.double()), "dtype"), (dict(x=x, weight=w[:4]), "weight"),
                       (dict(x=x, weight=w.half()), "weight"), (dict(x=x, residual=x.half()), "residual"),
                       (dict(x=x, residual=x[:2]), "residual"), (dict(x=x, eps=-1.0), "eps"), (dict(x=x, eps=float("nan")), "eps")):
        with pytest.raises(ValueError, match=match):
            fl.layer_norm_forward(**bad)
    with pytest.raises(RuntimeError, match="2004"):
        fl.layer_norm_forward(torch.zeros(2, 16385, device="cuda"))
    y, total, mean, rstd = fl.layer_norm_forward(x, w)
    with pytest.raises(ValueError, match="total"):
        fl.layer_norm_backward(x, total[:2], w, mean, rstd)
    with pytest.raises(ValueError, match="mean"):
        fl.layer_norm_backward(x, total, w, mean[:2], rstd)
    with pytest.raises(ValueError, match="width"):
        fl.LayerNorm(0)
