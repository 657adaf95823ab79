"""The gated linear recurrence against 64-bit arithmetic.

Bounds, with u = 2^-24.  A sigmoid's smaller side s of an argument a is off by (|a| + 6) u of itself: the exponential's argument is
rounded (|a| u), the hardware's exponential and reciprocal are off by 2 u each, a sum and a product by u each.  A step of the state therefore
adds (|a| + 8) s M + 2 M times u, where M, the state with all its terms taken as magnitudes, also bounds what a segment adds and what it leaves
of the state in front of it; errors of earlier steps fade as the state does, E_t = f_t E_{t-1} + e_t.  The gradient's recurrence has the same
form.  The factor of two in front of E is for products of errors and the second walk over a segment.
Below 2^-126 fp32 has no more digits but steps of 2^-149, and a rounding there costs up to LEAST = 2^-150 instead of a part of the value (the last one
assert_within counts): a gate's sigmoid (e^-90, say) has two (the exponential brought into that range, and corrected), its slope one more, its product with
dy one, a step of G one (the product with f; sums are exact there), and G's product with c - x one.  What multiplies them afterwards multiplies that."""
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within, offset_copy

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -150


def _problem(shape, dtype, states, gate=True, seed=0, keeps=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    width = shape[-1]
    return dict(x=n(*shape).to(dtype), forget=(n(*shape) + keeps * torch.rand(width, device="cuda", generator=g)).to(dtype),
                gate=n(*shape).to(dtype) if gate else None, state=n(states, width), dy=n(*shape).to(dtype), d_state=n(states, width))


def _one(x, u, g, state, dy, d_state):
    """Sequences of one length (tokens, .., width) token by token: every output with its bound."""
    x, u, dy = x.double(), u.double(), dy.double()
    f, z = torch.sigmoid(u), torch.sigmoid(-u)
    small, rel = torch.minimum(f, z), (u.abs() + 8) * U32
    c, magnitude, error = state.double(), state.double().abs(), torch.zeros_like(state, dtype=torch.float64)
    befores, afters, errors = [], [], [error]
    for t in range(len(x)):
        befores.append(c)
        c = f[t] * c + z[t] * x[t]
        step = rel[t] * small[t] * (magnitude + x[t].abs())
        magnitude = f[t] * magnitude + z[t] * x[t].abs()
        error = f[t] * error + step + 2 * U32 * magnitude
        afters.append(c)
        errors.append(error)
    stack = lambda l: torch.stack(l) if l else torch.zeros_like(x)
    before, after, of_before, of_after = stack(befores), stack(afters), 2 * stack(errors[:-1]), 2 * stack(errors[1:])
    out = dict(state=(c, 2 * error))
    if g is None:
        o, d = torch.ones_like(x), dy
        of_d = torch.zeros_like(x)
        out["y"] = (after, of_after)
    else:
        o = torch.sigmoid(g.double())
        of_o = (g.double().abs() + 8) * U32
        d, of_d = dy * o, (dy * o).abs() * of_o + LEAST * (2 * dy.abs() + 2)
        out["y"] = (o * after, o * of_after + (o * after).abs() * of_o + 2 * LEAST * after.abs())
        slope = o * torch.sigmoid(-g.double())
        out["dgate"] = (dy * after * slope, dy.abs() * slope * of_after + 2 * (dy * after * slope).abs() * of_o + 3 * LEAST * (dy * after).abs())
    carried, size, error = d_state.double(), d_state.double().abs(), torch.zeros_like(c)
    totals, of_totals = [], []
    for t in range(len(x) - 1, -1, -1):
        total, size, error = d[t] + carried, d[t].abs() + size, error + of_d[t] + U32 * (d[t].abs() + size)
        totals.append(total)
        of_totals.append(error)
        carried = f[t] * total
        error = f[t] * error + rel[t] * small[t] * size + 2 * U32 * f[t] * size
        size = f[t] * size
    total, of_total = stack(totals[::-1]), 2 * stack(of_totals[::-1])
    out["dx"] = (z * total, z * of_total + (z * total).abs() * rel)
    way = before - x
    out["dforget"] = (total * way * f * z, f * z * (of_total * way.abs() + total.abs() * (of_before + U32 * (before.abs() + x.abs()))) +
                      2 * (total * way * f * z).abs() * rel + LEAST * f * z)
    out["d_initial"] = (carried, 2 * error)
    return out


def _definition(p, spans):
    names = ("x", "forget", "gate", "dy")
    rows = ("y", "dx", "dforget") + (("dgate",) if p["gate"] is not None else ())
    zeros = torch.zeros(len(spans), p["x"].shape[-1], device="cuda")
    state, d_state = (zeros if p[k] is None else p[k] for k in ("state", "d_state"))
    if p["x"].dim() == 3:   # sequences of one length, all at once
        part = {k: None if p[k] is None else p[k].transpose(0, 1) for k in names}
        one = _one(part["x"], part["forget"], part["gate"], state, part["dy"], d_state)
        return {k: tuple(t.transpose(0, 1) for t in v) if k in rows else v for k, v in one.items()}
    out = {k: (torch.zeros_like(p["x"], dtype=torch.float64), torch.zeros_like(p["x"], dtype=torch.float64)) for k in rows}
    of_states = {"state": ([], []), "d_initial": ([], [])}
    for n, (a, b) in enumerate(spans):
        part = {k: None if p[k] is None else p[k][a:b] for k in names}
        one = _one(part["x"], part["forget"], part["gate"], state[n], part["dy"], d_state[n])
        for k, pair in out.items():
            pair[0][a:b], pair[1][a:b] = one[k]
        for k, pair in of_states.items():
            pair[0].append(one[k][0])
            pair[1].append(one[k][1])
    out.update({k: tuple(torch.stack(l) for l in pair) for k, pair in of_states.items() if pair[0]})
    return out


def _own(p, cu=None):
    y, state, saved = fl.gated_recurrence_forward(p["x"], p["forget"], p["gate"], state=p["state"], cu_seqlens=cu)
    dx, dforget, dgate, d_initial = fl.gated_recurrence_backward(p["dy"], p["x"], p["forget"], p["gate"], saved, d_state=p["d_state"], cu_seqlens=cu)
    out = dict(y=y, state=state, dx=dx, dforget=dforget, d_initial=d_initial)
    if p["gate"] is not None:
        out["dgate"] = dgate
    return out


def _check(p, label, lengths=None, cu=None):
    if lengths is None:
        n, t = p["x"].shape[:2]
        spans = [(i * t, i * t + t) for i in range(n)]
    else:
        ends = torch.tensor([0] + lengths).cumsum(0).tolist()
        spans = list(zip(ends[:-1], ends[1:]))
    got, want = _own(p, cu), _definition(p, spans)
    for name, (value, slack) in want.items():
        assert_within(got[name], value, slack, f"{label} {name}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 128, 129, 200, 333, 1000])
def test_lengths(tokens, dtype):
    for sequences, width, gate in ((1, 64, True), (3, 131, False), (2, 1, True), (5, 2, False), (1, 3, True)):
        _check(_problem((sequences, tokens, width), dtype, sequences, gate, seed=tokens), f"{sequences} x {tokens} x {width} {dtype}")


@pytest.mark.parametrize("sequences,tokens,width", [(200, 40, 1400), (300, 150, 1024), (1, 5000, 257), (1, 20000, 8), (4, 700, 2050), (1, 300, 9000)])
@pytest.mark.parametrize("gate", [True, False])
def test_sizes(sequences, tokens, width, gate):
    for dtype in (torch.float16, torch.float32):
        _check(_problem((sequences, tokens, width), dtype, sequences, gate, seed=1), f"{sequences} x {tokens} x {width} {dtype}")


PACKED = [[5], [0], [1, 0, 0, 7, 16, 0], [64, 1, 300, 0, 17, 2, 129, 63, 65], [900, 3], [0, 0, 250], [16] * 30, [1] * 70]


@pytest.mark.parametrize("lengths", PACKED, ids=str)
@pytest.mark.parametrize("tail", [0, 1, 40])
def test_packed(lengths, tail):
    cu = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
    for dtype, width, gate in ((torch.float32, 33, True), (torch.bfloat16, 130, False), (torch.float16, 1, True)):
        p = _problem((sum(lengths) + tail, width), dtype, len(lengths), gate, seed=len(lengths))
        _check(p, f"{lengths} + {tail}, {width} {dtype}", lengths, cu)   # (the definition has zeros behind the last)


def test_no_sequences():
    cu = torch.zeros(1, device="cuda", dtype=torch.int32)
    p = _problem((9, 20), torch.float16, 0)
    got = _own(p, cu)
    assert got["state"].shape == (0, 20) and not any(bool(got[k].any()) for k in ("y", "dx", "dforget", "dgate"))
    got = _own(_problem((0, 9, 20), torch.float16, 0))
    assert got["y"].shape == (0, 9, 20)
    p = _problem((3, 0, 20), torch.float16, 3)
    got = _own(p)
    assert torch.equal(got["state"], p["state"]) and torch.equal(got["d_initial"], p["d_state"])
    assert fl.gated_recurrence_forward(*[torch.empty(2, 3, 0, device="cuda")] * 2)[0].shape == (2, 3, 0)


def test_without_states():
    for tokens in (20, 400):
        p = _problem((2, tokens, 70), torch.float16, 2)
        p["state"] = p["d_state"] = None
        _check(p, "bare")
        want = _own(p)
        y, state, saved = fl.gated_recurrence_forward(p["x"], p["forget"], p["gate"], want_state=False, want_saved=False)
        assert state is None and saved is None and torch.equal(y, want["y"])
        saved = fl.gated_recurrence_forward(p["x"], p["forget"], p["gate"])[2]
        for i, name in enumerate(("dx", "dforget", "dgate", "d_initial")):
            got = fl.gated_recurrence_backward(p["dy"], p["x"], p["forget"], p["gate"], saved, want=[j == i for j in range(4)])
            assert torch.equal(got[i], want[name]) and all(got[j] is None for j in range(4) if j != i)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens", [50, 300])
def test_strides_and_alignment(tokens, dtype):
    p = _problem((3, tokens, 66), dtype, 3, seed=4)
    want = _own(p)
    same = lambda got: [torch.equal(want[k], got[k]) or pytest.fail(k) for k in want]
    wide = torch.zeros(3, tokens, 3 * 67 + 1, device="cuda", dtype=dtype)     # parts of a projection, at odd places
    views = [wide[..., 1 + 67 * i:67 + 67 * i] for i in range(3)]
    for view, name in zip(views, ("x", "forget", "gate")):
        view.copy_(p[name])
    same(_own(dict(p, x=views[0], forget=views[1], gate=views[2], dy=offset_copy(p["dy"]))))
    across = {k: p[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ("x", "forget", "gate", "dy")}
    got = _own(dict(p, **across))
    same(got)
    assert got["y"].stride() == across["x"].stride()
    channels = {k: p[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("x", "forget", "dy")}
    same(_own(dict(p, **channels)))
    back = {k: p[k].flip(1).contiguous().flip(1) for k in ("x", "gate")}
    same(_own(dict(p, **back)))
    shared = dict(p, forget=p["forget"][:1, :1].expand(3, tokens, 66), dy=p["dy"][:, :1].expand(3, tokens, 66))
    whole = dict(shared, forget=shared["forget"].contiguous(), dy=shared["dy"].contiguous())
    want = _own(whole)
    same(_own(shared))


def test_gates_at_their_ends():
    inf = float("inf")
    p = _problem((2, 300, 64), torch.float32, 2, seed=6)
    p["forget"][0, ::3] = 60.0      # keeps all
    p["forget"][0, 1::3] = -60.0    # keeps nothing
    p["forget"][1, :, ::2] = 12.0   # a memory of 160000 tokens
    p["gate"][0, :, ::4], p["gate"][1, :, 1::4] = -90.0, 90.0
    _check(p, "ends")
    p["forget"][1, 7], p["forget"][1, 9] = inf, -inf
    p["gate"][1, 8], p["gate"][1, 10] = inf, -inf
    got = _own(p)
    assert all(bool(v.isfinite().all()) for v in got.values())
    plain = fl.gated_recurrence_forward(p["x"], p["forget"])[0]
    assert torch.equal(plain[1, 7], plain[1, 6]) and torch.equal(plain[1, 9], p["x"][1, 9])


@pytest.mark.parametrize("tokens", [90, 600])
def test_infinities_and_nan_stay_in_their_channels(tokens):
    p = _problem((2, tokens, 40), torch.bfloat16, 2, seed=7)
    want = _own(p)
    p["x"][0, 50, 3], p["forget"][0, 60, 4], p["state"][1, 5] = float("inf"), float("nan"), float("-inf")
    p["gate"][1, 70, 6], p["dy"][1, 20, 7] = float("nan"), float("inf")
    got = _own(p)
    clean = torch.ones(2, tokens, 40, dtype=torch.bool, device="cuda")
    clean[0, 50:, 3] = clean[0, 60:, 4] = clean[1, :, 5] = clean[1, 70, 6] = False
    assert torch.equal(got["y"][clean], want["y"][clean]) and not bool(got["y"][0, 50, 3].isfinite()) and not bool(got["y"][0, 60:, 4].isfinite().any())
    for name in ("dx", "dforget", "dgate"):   # gradients: nothing but those channels
        assert torch.equal(got[name][..., 8:], want[name][..., 8:]) and torch.equal(got[name][..., :3], want[name][..., :3])
    assert torch.equal(got["dx"][1, 21:, 7], want["dx"][1, 21:, 7]) and not bool(got["dx"][1, :21, 7].isfinite().any())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_single_tokens(dtype):
    for sequences, width, gate in ((1, 64, True), (3, 1, False), (7, 131, True), (300, 1024, False)):
        p = _problem((sequences, 5, width), dtype, sequences, gate, seed=8)
        want = _definition(p, [(i * 5, i * 5 + 5) for i in range(sequences)])
        state = p["state"].clone()
        for t in range(5):
            part = [None if p[k] is None else p[k][:, t] for k in ("x", "forget", "gate")]
            version = state._version
            y = fl.gated_recurrence_step(part[0], part[1], state, part[2])
            assert state._version > version
            assert_within(y, want["y"][0][:, t], want["y"][1][:, t], f"{sequences} x {width} {dtype} token {t}")
        assert_within(state, *want["state"], "state")
    empty = torch.empty(0, 8, device="cuda")
    assert fl.gated_recurrence_step(empty, empty, torch.empty(0, 8, device="cuda")).shape == (0, 8)


def test_a_prompt_in_pieces():
    p = _problem((2, 500, 96), torch.float32, 2, seed=9)
    want, slack = _definition(p, [(0, 500), (500, 1000)])["y"]
    state, parts = p["state"], []
    for a, b in ((0, 1), (1, 130), (130, 131), (131, 499), (499, 500)):
        y, state, _ = fl.gated_recurrence_forward(p["x"][:, a:b], p["forget"][:, a:b], p["gate"][:, a:b], state=state, want_saved=False)
        parts.append(y)
    assert_within(torch.cat(parts, 1), want, slack, "pieces")


def test_gradients_against_differences():
    p = _problem((2, 40, 5), torch.float32, 2, seed=10)
    names = ("x", "forget", "gate", "state")
    leaves = [p[k].clone().requires_grad_() for k in names]
    y, final = fl.gated_recurrence(*leaves[:3], state=leaves[3])
    torch.autograd.backward([y, final], [p["dy"], p["d_state"]])

    def loss(x, u, g, c):
        total = 0
        for t in range(40):
            f = torch.sigmoid(u[:, t])
            c = f * c + (1 - f) * x[:, t]
            total = total + (torch.sigmoid(g[:, t]) * c * p["dy"][:, t].double()).sum()
        return total + (c * p["d_state"].double()).sum()

    at = [p[k].double() for k in names]
    for k, leaf in enumerate(leaves):
        direction = torch.randn(at[k].shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(k))
        h = 1e-5
        up, down = (loss(*[a + s * h * direction if j == k else a for j, a in enumerate(at)]) for s in (1, -1))
        slope, along = float((up - down) / (2 * h)), leaf.grad.double() * direction
        # the difference's own error is h^2 times a third derivative of order 100; the gradient's terms are off by some ulp each
        assert abs(float(along.sum()) - slope) <= 1e-5 * max(1.0, float(along.abs().sum())), names[k]


def test_autograd_paths():
    for tokens in (40, 300):
        p = _problem((2, tokens, 70), torch.float16, 2, seed=11)
        want = _own(p)
        leaves = {k: p[k].clone().requires_grad_() for k in ("x", "forget", "gate", "state")}
        y, final = fl.gated_recurrence(leaves["x"], leaves["forget"], leaves["gate"], state=leaves["state"])
        torch.autograd.backward([y, final], [p["dy"], p["d_state"]])
        for leaf, name in (("x", "dx"), ("forget", "dforget"), ("gate", "dgate"), ("state", "d_initial")):
            assert torch.equal(leaves[leaf].grad, want[name]), name
        x = p["x"].clone().requires_grad_()
        _, final = fl.gated_recurrence(x, p["forget"])
        final.backward(p["d_state"][:1].expand(2, 70))
        assert x.grad.shape == x.shape
        bias = p["forget"][0, 0].clone().requires_grad_()     # one forget gate for all tokens: its gradient is their sum
        y, _ = fl.gated_recurrence(p["x"], bias.expand(2, tokens, 70))
        y.backward(p["dy"])
        assert bias.grad.shape == (70,)
        with torch.no_grad():
            assert not fl.gated_recurrence(x, p["forget"])[0].requires_grad


@pytest.mark.parametrize("tokens", [48, 700])
def test_captured_in_a_graph_and_other_streams(tokens):
    p = _problem((2, tokens, 128), torch.float16, 2, seed=12)
    want = _own(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _own(p)
    here = _own(p)   # two at a time
    torch.cuda.current_stream().wait_stream(side)
    for name in want:
        assert torch.equal(want[name], got[name]) and torch.equal(want[name], here[name]), name
    state = p["state"].clone()
    run = lambda: (_own(p), fl.gated_recurrence_step(p["x"][:, 0], p["forget"][:, 0], state, p["gate"][:, 0]))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, y = run()
    for seed in range(4):
        fresh = _problem((2, tokens, 128), torch.float16, 2, seed=seed)
        for name in ("x", "forget", "gate", "dy", "state", "d_state"):
            p[name].copy_(fresh[name])
        state.copy_(fresh["state"])
        graph.replay()
        torch.cuda.synchronize()
        after = state.clone()
        state.copy_(fresh["state"])
        want, want_y = run()
        assert torch.equal(y, want_y) and torch.equal(after, state)
        for name in want:
            assert torch.equal(want[name], got[name]), name


def test_refusals():
    x, s = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    cu = torch.tensor([0, 2, 5], device="cuda", dtype=torch.int32)
    for bad, match in ((dict(x=x.cpu()), "CUDA"), (dict(x=x.double()), "dtype"), (dict(forget=x[:1]), "forget"), (dict(forget=x.half()), "forget"),
                       (dict(gate=x[..., :4]), "gate"), (dict(gate=x.half()), "gate"), (dict(state=s[:1]), "state"), (dict(state=s.half()), "state"),
                       (dict(x=x[0], forget=x[0]), "axes"), (dict(cu_seqlens=cu), "axes"), (dict(x=x[0], forget=x[0], cu_seqlens=cu.long()), "cu_seqlens"),
                       (dict(x=x[0], forget=x[0], cu_seqlens=cu[:0]), "cu_seqlens"), (dict(x=x[0], forget=x[0], cu_seqlens=cu.cpu()), "cu_seqlens")):
        with pytest.raises(ValueError, match=match):
            fl.gated_recurrence_forward(**{**dict(x=x, forget=x), **bad})
    y, final, saved = fl.gated_recurrence_forward(x, x)
    for bad, match in ((dict(dy=x[:1]), "dy"), (dict(saved=None), "saved"), (dict(saved=saved[:1]), "saved"), (dict(d_state=s[:1]), "state")):
        with pytest.raises(ValueError, match=match):
            fl.gated_recurrence_backward(**{**dict(dy=x, x=x, forget=x, gate=None, saved=saved), **bad})
    for bad, match in ((dict(state=None), "state"), (dict(state=s[:1]), "state"), (dict(x=x), "axes"), (dict(gate=x[0, :1]), "gate")):
        with pytest.raises(ValueError, match=match):
            fl.gated_recurrence_step(**{**dict(x=x[:, 0], forget=x[:, 0], state=s), **bad})
