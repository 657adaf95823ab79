"""Attention with a decaying state against its recurrence in 64 bits, token by token.

Bounds.  The same recurrence over the magnitudes of everything gives, for every output, the sum A of the magnitudes of its terms.
A term is rounded to the tensors' type once on its way (as a score, or as part of the state that the token meets), which costs
unit * A at most, and the result once more; sums in 32 bits and decays as powers of two cost a few ulp of A: 64 u A covers them.
The state is summed in 32 bits from values that are held in parts of 22 bits or more, relative to the largest of a chunk."""
import math

import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, UNIT, assert_within, offset_copy

pytestmark = pytest.mark.gpu


def _recurrence(q, k, v, log_decay, scale, state):
    """(T, H, dk), (T, Hkv, dk), (T, Hkv, dv), state (H, dk, dv), all in 64 bits -> o (T, H, dv), final state."""
    group = q.shape[1] // k.shape[1]
    k, v, g, outs = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1), torch.exp(log_decay)[:, None, None], []
    for t in range(q.shape[0]):
        state = g * state + k[t, :, :, None] * v[t, :, None, :]
        outs.append(scale * (q[t, :, :, None] * state).sum(1))
    return (torch.stack(outs) if outs else q.new_zeros(0, q.shape[1], v.shape[-1])), state


def _definition(p, magnitudes=False):
    """o, final states, and where p has `do` the gradients, of every sequence of a problem; of the magnitudes if asked for."""
    f = (lambda t: t.double().abs()) if magnitudes else (lambda t: t.double())
    out = {name: [] for name in ("o", "state", "dq", "dk", "dv", "d_initial")}
    with torch.enable_grad():
        for n in range(p["sequences"]):
            x = [f(t[p["first"][n]:p["first"][n] + p["lengths"][n]] if p["cu_seqlens"] is not None else t[n]).requires_grad_()
                 for t in (p["q"], p["k"], p["v"])]
            s = f(p["state"][n]).requires_grad_() if p["state"] is not None else \
                torch.zeros(x[0].shape[1], x[0].shape[2], x[2].shape[2], device="cuda", dtype=torch.float64).requires_grad_()
            o, final = _recurrence(*x, p["log_decay"].double(), abs(p["scale"]) if magnitudes else p["scale"], s)
            out["o"].append(o.detach())
            out["state"].append(final.detach())
            if p.get("do") is not None:
                do = f(p["do"][p["first"][n]:p["first"][n] + p["lengths"][n]] if p["cu_seqlens"] is not None else p["do"][n])
                loss = (o * do).sum() + ((final * f(p["d_state"][n])).sum() if p["d_state"] is not None else 0 * final.sum())
                for name, g in zip(("dq", "dk", "dv", "d_initial"), torch.autograd.grad(loss, (*x, s), materialize_grads=True)):
                    out[name].append(g)
    whole = torch.cat if p["cu_seqlens"] is not None else torch.stack
    return {name: (torch.stack(parts) if name in ("state", "d_initial") else whole(parts)) for name, parts in out.items() if parts}


def _problem(sequences, length, heads=2, kv_heads=2, dk=64, dv=64, dtype=torch.bfloat16, lengths=None, seed=0, with_state=True, train=True,
             log_decay=None, scale=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *shape, dtype=dtype: torch.randn(*shape, device="cuda", generator=g).to(dtype)
    p = dict(sequences=sequences, cu_seqlens=None, lengths=lengths, scale=dk ** -0.5 if scale is None else scale)
    lead = (sequences, length)
    if lengths is not None:
        p["first"] = [sum(lengths[:i]) for i in range(sequences)]
        p["cu_seqlens"] = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        lead = (sum(lengths),)
    else:
        p["first"], p["lengths"] = [0] * sequences, [length] * sequences
    p["q"], p["k"], p["v"] = n(*lead, heads, dk), n(*lead, kv_heads, dk), n(*lead, kv_heads, dv)
    p["log_decay"] = -torch.exp(torch.linspace(-0.5, -5.0, heads, device="cuda")) if log_decay is None else torch.tensor(log_decay, device="cuda")
    p["state"] = n(sequences, heads, dk, dv, dtype=torch.float32) if with_state else None
    if train:
        p["do"] = n(*lead, heads, dv)
        p["d_state"] = n(sequences, heads, dk, dv, dtype=torch.float32) if with_state else None
    return p


def _own(p):
    qkv, more = (p["q"], p["k"], p["v"], p["log_decay"]), dict(scale=p["scale"], state=p["state"], cu_seqlens=p["cu_seqlens"])
    out = dict(zip(("o", "state"), fl.decay_attention_forward(*qkv, **more)))
    if p.get("do") is not None:
        out.update(zip(("dq", "dk", "dv", "d_initial"), fl.decay_attention_backward(p["do"], *qkv, d_state=p["d_state"], **more)))
    return out


def _check(p, got, label=""):
    want, most = _definition(p), _definition(p, magnitudes=True)
    unit = UNIT[p["q"].dtype] if p["q"].dtype != torch.float32 else 0.0
    for name, value in want.items():
        if name in ("state", "d_initial"):
            # 2^-21: two parts of 11 bits, the smaller one absolute to the chunk's largest value, taken as four times a column's
            slack = (64 * U32 + (0 if unit == 0 else 2.0 ** -21)) * most[name] + (0 if unit == 0 else 2.0 ** -21) * most[name].amax((-1, -2), keepdim=True)
        else:
            slack = (1.05 * unit + 64 * U32) * most[name]
        assert_within(got[name], value, slack, f"{label} {name}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 100, 128, 200])
def test_lengths(length, dtype):
    p = _problem(2, length, dtype=dtype, seed=length)
    _check(p, _own(p), f"{length}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dk,dv", [(8, 8), (9, 15), (16, 32), (33, 64), (64, 33), (40, 65), (65, 40), (128, 128), (127, 129), (128, 64), (64, 128), (130, 17),
                                   (256, 256), (255, 200), (24, 250), (250, 24)])
def test_head_widths(dk, dv, dtype):
    p = _problem(1, 75, heads=2, kv_heads=1, dk=dk, dv=dv, dtype=dtype, seed=dk + dv)
    _check(p, _own(p), f"{dk} x {dv}")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (4, 1), (6, 2), (8, 4)])
def test_head_groups(heads, kv_heads):
    p = _problem(2, 90, heads=heads, kv_heads=kv_heads, dk=40, dv=48, seed=heads)
    _check(p, _own(p))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lengths", [[70], [1, 64, 0, 129, 3], [0, 0, 5], [200, 0], [0], [65] * 5])
def test_packed(lengths, dtype):
    p = _problem(len(lengths), None, lengths=lengths, dtype=dtype, heads=4, kv_heads=2, dk=32, dv=48, seed=len(lengths))
    got = _own(p)
    _check(p, got)
    for n, length in enumerate(lengths):   # an empty sequence hands its state through
        if length == 0:
            assert torch.equal(got["state"][n], p["state"][n]) and torch.equal(got["d_initial"][n], p["d_state"][n])


@pytest.mark.parametrize("sequences,length,lengths", [(1, 1500, None), (2, 1030, None), (1, 513, None), (4, None, [1300, 1, 0, 700]), (3, None, [512, 1024, 65])])
@pytest.mark.parametrize("kv_heads", [1, 2])
def test_split_along_the_sequence(sequences, length, lengths, kv_heads):
    p = _problem(sequences, length, lengths=lengths, heads=2, kv_heads=kv_heads, dk=40, dv=72, seed=3, dtype=torch.float16)
    got = _own(p)
    _check(p, got)
    again = _own(p)
    for name in got:
        assert torch.equal(got[name], again[name]), name
    p["state"] = p["d_state"] = None
    _check(p, _own(p))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sequences,length,lengths,dk,dv", [(1, 257, None, 64, 64), (2, 300, None, 40, 65), (1, 256, None, 64, 64), (5, None, [64, 128, 0, 63, 65], 65, 40),
                                                            (1, 330, None, 200, 136), (3, None, [257, 1, 190], 16, 256)])
def test_short_segments(sequences, length, lengths, dk, dv, dtype):
    p = _problem(sequences, length, kv_heads=1, dk=dk, dv=dv, dtype=dtype, lengths=lengths, seed=4)
    _check(p, _own(p))


def test_tokens_of_no_sequence():
    p = _problem(2, None, lengths=[40, 70], heads=2, kv_heads=1, dk=32, dv=32)
    want = _own(p)
    fill = lambda t: torch.cat([t, torch.full_like(t, float("nan"))])   # as many tokens again, of no sequence, with anything in them
    p.update(q=fill(p["q"]), k=fill(p["k"]), v=fill(p["v"]), do=fill(p["do"]))
    got = _own(p)
    for name in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[name][:110], want[name]) and not bool(got[name][110:].any()), name
    assert torch.equal(got["state"], want["state"]) and torch.equal(got["d_initial"], want["d_initial"])
    # bounds that make no sense stay inside the tensors
    p["cu_seqlens"] = torch.tensor([-5, 1000, 60], device="cuda", dtype=torch.int32)
    assert _own(p)["o"].shape == (220, 2, 32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("log_decay", [[0.0, -0.001], [-float("inf"), -30.0], [-1e-9, -5.0]])
def test_extreme_decays(log_decay, dtype):
    p = _problem(1, 150, dtype=dtype, log_decay=log_decay, dk=32, dv=32)
    p["log_decay"] = p["log_decay"].clamp(min=-1e4)   # (exp of minus infinity times zero is no derivative; the value is the same, zero)
    want = _definition(p)
    got_p = dict(p, log_decay=torch.tensor(log_decay, device="cuda"))
    got = _own(got_p)
    _check(p, got)
    assert bool(torch.isfinite(want["o"]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("small,large", [(1e-4, 1.0), (1.0, 100.0), (0.01, 300.0)])
def test_magnitudes(small, large, dtype):
    """fp16 operands are brought into that type's range: small gradients keep their bits, large states do not overflow."""
    p = _problem(1, 200, dtype=dtype, dk=64, dv=64, log_decay=[0.0, -0.02], with_state=False, scale=0.01)
    p["do"] = (p["do"] * small).to(dtype)
    p["k"] = (p["k"] * large).to(dtype)
    got = _own(p)
    want = _definition(p)
    fits = {name: bool((want[name].abs() < 60000).all()) for name in want}
    assert bool(torch.isfinite(got["state"]).all()) and bool(torch.isfinite(got["d_initial"]).all())
    if all(fits.values()):
        _check(p, got)


def test_zeros():
    p = _problem(1, 130, dtype=torch.float16, with_state=False)
    p["v"].zero_()
    got = _own(p)
    assert not bool(got["o"].any()) and not bool(got["state"].any())
    _check(p, got)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_nan_and_infinity_reach_later_tokens_alone(dtype):
    p = _problem(1, 150, dtype=dtype, dk=32, dv=48)
    want = _definition(p)
    most = _definition(p, magnitudes=True)
    bad = dict(p, v=p["v"].clone(), do=p["do"].clone())
    bad["v"][0, 80, 0, 5], bad["v"][0, 20, 1, 7] = float("nan"), float("inf")
    bad["do"][0, 100, 0, 3] = float("-inf")
    got = _own(bad)
    unit = UNIT[dtype] if dtype != torch.float32 else 0.0
    clean = torch.ones(want["o"].shape, dtype=torch.bool, device="cuda")
    clean[0, 80:, 0, 5] = clean[0, 20:, 1, 7] = False
    slack = (1.05 * unit + 64 * U32) * most["o"]
    assert_within(torch.where(clean, got["o"], torch.zeros_like(got["o"])), torch.where(clean, want["o"], 0.0), slack, "o")
    assert not bool(torch.isfinite(got["o"][~clean]).any())
    # dv: the bad gradient at token 100 reaches the tokens up to it, in its column
    slack = (1.05 * unit + 64 * U32) * most["dv"]
    clean = torch.ones(want["dv"].shape, dtype=torch.bool, device="cuda")
    clean[0, :101, 0, 3] = False
    assert_within(torch.where(clean, got["dv"], torch.zeros_like(got["dv"])), torch.where(clean, want["dv"], 0.0), slack, "dv")
    # a bad query reaches its own output alone, a bad key no earlier one
    bad = dict(p, q=p["q"].clone(), k=p["k"].clone(), do=None)
    bad["q"][0, 10, 0, 2] = float("nan")
    bad["k"][0, 90, 1, 3] = float("inf")
    o = _own(bad)["o"]
    clean = torch.ones(want["o"].shape, dtype=torch.bool, device="cuda")
    clean[0, 10, 0] = clean[0, 90:, 1] = False
    assert bool(torch.isfinite(o[clean]).all()) and not bool(torch.isfinite(o[0, 10, 0]).any())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_an_infinite_value_leaves_the_others_their_range(dtype):
    p = _problem(1, 150, dtype=dtype, dk=32, dv=48, train=False)
    p["q"][0, 20, 1] *= 1000                                    # (a row whose scores fp16 holds scaled alone)
    want, most = _definition(p), _definition(p, magnitudes=True)
    bad = dict(p, q=p["q"].clone())
    bad["q"][0, 10, 0, 2], bad["q"][0, 70, 1, 3] = float("inf"), float("-inf")
    o = _own(bad)["o"]
    clean = torch.ones(want["o"].shape, dtype=torch.bool, device="cuda")
    clean[0, 10, 0] = clean[0, 70, 1] = False
    unit = UNIT[dtype] if dtype != torch.float32 else 0.0
    # (fp16: the scores of a chunk share a power of two; the smallest that it leaves, 2^-25 of a largest of 2^13, is far below the
    # rounding of the row that decides it)
    slack = (1.05 * unit + 64 * U32) * most["o"] + (2.0 ** -38 * most["o"].amax() if dtype == torch.float16 else 0.0)
    assert_within(torch.where(clean, o, torch.zeros_like(o)), torch.where(clean, want["o"], 0.0), slack, "o")
    assert not bool(torch.isfinite(o[0, 10, 0]).any()) and not bool(torch.isfinite(o[0, 70, 1]).any())


def test_strides_and_alignment():
    for dtype in DTYPES:
        p = _problem(3, 70, heads=4, kv_heads=2, dk=40, dv=24, dtype=dtype)
        want = _own(p)
        # (T, B, H, D) below, one tensor with q, k and v side by side and an odd distance between tokens
        room = torch.zeros(70, 3, 4 * 40 + 2 * 40 + 2 * 24 + 1, device="cuda", dtype=dtype)
        at = 1
        strided = dict(p)
        for name, h, d in (("q", 4, 40), ("k", 2, 40), ("v", 2, 24)):
            view = room[:, :, at:at + h * d].unflatten(2, (h, d)).transpose(0, 1)
            view.copy_(p[name])
            strided[name] = view
            at += h * d
        strided["do"] = offset_copy(p["do"])
        got = _own(strided)
        for name in want:
            assert torch.equal(want[name], got[name]), (dtype, name)
        assert got["o"].stride()[0] < got["o"].stride()[1]     # the memory order of q's rows
        # broadcast keys: one head's, expanded
        wide = dict(p, k=p["k"][:, :, :1].expand(-1, -1, 2, -1), do=None)
        plain = dict(wide, k=wide["k"].contiguous())
        assert torch.equal(_own(wide)["o"], _own(plain)["o"])


def test_offsets_beyond_32_bits():
    far = (1 << 31) + 24
    room = torch.zeros(far + 70 * 2 * 32, device="cuda", dtype=torch.float16)
    p = _problem(2, 70, dk=32, dv=32, dtype=torch.float16)
    want = _own(p)
    for name in ("q", "k", "v", "do"):
        room.zero_()
        view = room.as_strided((2, 70, 2, 32), (far, 64, 32, 1))
        view.copy_(p[name])
        got = _own(dict(p, **{name: view}))
        for key in want:
            assert torch.equal(want[key], got[key]), (name, key)


def test_a_single_token_of_any_stride():
    p = _problem(3, 1, heads=2, kv_heads=1, dk=32, dv=32, train=False)
    wide = {name: p[name].as_strided(p[name].shape, (p[name].stride(0), 1 << 24, *p[name].stride()[2:])) for name in ("q", "k", "v")}
    assert torch.equal(_own(dict(p, **wide))["o"], _own(p)["o"])


def test_a_sequence_in_pieces_and_token_by_token():
    for dtype in DTYPES:
        p = _problem(3, 150, heads=4, kv_heads=2, dk=72, dv=100, dtype=dtype, train=False)
        want, most = _definition(p), _definition(p, magnitudes=True)
        unit = UNIT[dtype] if dtype != torch.float32 else 0.0
        state, outs = p["state"], []
        for a, b in ((0, 1), (1, 70), (70, 70), (70, 150)):
            o, state = fl.decay_attention_forward(p["q"][:, a:b], p["k"][:, a:b], p["v"][:, a:b], p["log_decay"], state=state)
            outs.append(o)
        slack = (1.05 * unit + 64 * U32) * most["o"]
        assert_within(torch.cat(outs, 1), want["o"], slack, "pieces")
        state, outs = p["state"].clone(), []
        for t in range(150):
            outs.append(fl.decay_attention_step(p["q"][:, t], p["k"][:, t], p["v"][:, t], p["log_decay"], state))
        assert_within(torch.stack(outs, 1), want["o"], 64 * U32 * most["o"], "steps")
        assert_within(state, want["state"], 64 * U32 * most["state"], "state after steps")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sequences,heads,kv_heads,dk,dv", [(1, 1, 1, 64, 64), (5, 4, 2, 128, 128), (3, 2, 1, 8, 9), (2, 3, 3, 65, 127), (2, 2, 2, 256, 256), (70, 8, 2, 40, 66)])
def test_step(sequences, heads, kv_heads, dk, dv, dtype):
    p = _problem(sequences, 1, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, dtype=dtype, train=False, seed=dk)
    want, most = _definition(p), _definition(p, magnitudes=True)
    state = p["state"].clone()
    o = fl.decay_attention_step(p["q"][:, 0], p["k"][:, 0], p["v"][:, 0], p["log_decay"], state)
    assert_within(o, want["o"][:, 0], 64 * U32 * most["o"][:, 0], "o")
    assert_within(state, want["state"], 4 * U32 * most["state"], "state")
    again = p["state"].clone()
    assert torch.equal(o, fl.decay_attention_step(offset_copy(p["q"][:, 0]), p["k"].transpose(0, 1)[0], p["v"][:, 0], p["log_decay"], again))
    assert torch.equal(state, again)


def test_nothing_asked_and_nothing_there():
    p = _problem(2, 90)
    want = _own(p)
    o, state = fl.decay_attention_forward(p["q"], p["k"], p["v"], p["log_decay"], state=p["state"], want_state=False)
    assert state is None and torch.equal(o, want["o"])
    names = ("dq", "dk", "dv", "d_initial")
    for wanted in ((True, False, False, False), (False, True, False, False), (False, False, True, True), (False, False, False, True), (False,) * 4):
        got = fl.decay_attention_backward(p["do"], p["q"], p["k"], p["v"], p["log_decay"], state=p["state"], d_state=p["d_state"], want=wanted)
        for name, asked, value in zip(names, wanted, got):
            assert (value is None) if not asked else torch.equal(value, want[name]), name
    for shape in ((0, 5), (3, 0)):
        q = torch.zeros(*shape, 2, 32, device="cuda")
        o, state = fl.decay_attention_forward(q, q, q, p["log_decay"])
        assert o.shape == q.shape and not bool(state.any())
        start = torch.randn(shape[0], 2, 32, 32, device="cuda")
        assert torch.equal(fl.decay_attention_forward(q, q, q, p["log_decay"], state=start)[1], start)
        dq, dk, dv, d0 = fl.decay_attention_backward(q, q, q, q, p["log_decay"], d_state=start)
        assert dq.shape == q.shape and torch.equal(d0, start)
    empty = torch.zeros(0, 2, 32, device="cuda")
    cu = torch.zeros(1, device="cuda", dtype=torch.int32)
    assert fl.decay_attention_forward(empty, empty, empty, p["log_decay"], cu_seqlens=cu)[1].shape == (0, 2, 32, 32)
    assert fl.decay_attention_step(empty, empty, empty, p["log_decay"], torch.zeros(0, 2, 32, 32, device="cuda")).shape == (0, 2, 32)


def test_gradients_against_differences():
    p = _problem(2, 70, heads=2, kv_heads=1, dk=9, dv=11, dtype=torch.float32, seed=2)
    inputs = [p[name].clone().requires_grad_() for name in ("q", "k", "v", "state")]
    o, final = fl.decay_attention(*inputs[:3], p["log_decay"], state=inputs[3])
    ((o * p["do"]).sum() + (final * p["d_state"]).sum()).backward()

    def loss(*x):
        total = 0.0
        for n in range(2):
            o, s = _recurrence(*(t[n] for t in x[:3]), p["log_decay"].double(), 9 ** -0.5, x[3][n])
            total = total + (o * p["do"][n].double()).sum() + (s * p["d_state"][n].double()).sum()
        return float(total)

    at = [p[name].double() for name in ("q", "k", "v", "state")]
    for j, x in enumerate(inputs):
        direction = torch.randn(x.shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(j))
        h = 1e-4   # (the loss is linear in each input by itself: the difference is exact but for 64-bit rounding)
        slope = (loss(*(a + h * direction if i == j else a for i, a in enumerate(at))) - loss(*(a - h * direction if i == j else a for i, a in enumerate(at)))) / (2 * h)
        products = x.grad.double() * direction
        assert abs(float(products.sum()) - slope) <= 64 * U32 * float(products.abs().sum()) * 16 + 1e-6 * abs(slope)


def test_autograd_paths():
    p = _problem(2, 50, heads=4, kv_heads=2, dk=32, dv=40)
    want = _own(p)
    q, k, v = (p[name].clone().requires_grad_() for name in ("q", "k", "v"))
    o, final = fl.decay_attention(q, k, v, p["log_decay"], state=p["state"])
    torch.autograd.backward([o, final], [p["do"], p["d_state"]])
    for x, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        assert torch.equal(x.grad, want[name]), name
    # the output alone; the state alone
    q.grad = None
    o, final = fl.decay_attention(q, k.detach(), v.detach(), p["log_decay"])
    o.backward(p["do"].transpose(0, 1).contiguous().transpose(0, 1))
    alone = fl.decay_attention_backward(p["do"], p["q"], p["k"], p["v"], p["log_decay"], want=(True, False, False, False))[0]
    assert torch.equal(q.grad, alone)
    start = p["state"].clone().requires_grad_()
    _, final = fl.decay_attention(p["q"], p["k"], p["v"], p["log_decay"], state=start)
    final.sum().backward()
    decay = torch.exp(50 * p["log_decay"])[None, :, None, None]
    assert torch.allclose(start.grad, decay.expand_as(start.grad), rtol=1e-5, atol=0)
    with torch.no_grad():
        assert not fl.decay_attention(q, k, v, p["log_decay"])[0].requires_grad


def test_other_streams_and_graphs():
    p = _problem(2, 700, heads=2, kv_heads=1, dk=64, dv=64)
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
    state = p["state"].clone()
    with torch.cuda.graph(graph):
        got = _own(p)
        step = fl.decay_attention_step(p["q"][:, 0], p["k"][:, 0], p["v"][:, 0], p["log_decay"], state)
    for seed in range(3):
        fresh = _problem(2, 700, heads=2, kv_heads=1, dk=64, dv=64, seed=seed)
        for name in ("q", "k", "v", "state", "do", "d_state"):
            p[name].copy_(fresh[name])
        state.copy_(fresh["state"])
        graph.replay()
        torch.cuda.synchronize()
        want = _own(p)
        for name in want:
            assert torch.equal(want[name], got[name]), name
        again = fresh["state"].clone()
        assert torch.equal(step, fl.decay_attention_step(p["q"][:, 0], p["k"][:, 0], p["v"][:, 0], p["log_decay"], again)) and torch.equal(state, again)


def test_more_tokens_than_a_launch_has_rows():
    """The shares of heads are summed for 2^20 tokens at a time.  (Sequences of one token each: their recurrence is a product.)"""
    sequences, heads, width, scale = 2 ** 20 + 5, 2, 8, 0.5
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(sequences, 1, n, width, device="cuda", generator=g).to(torch.bfloat16) for n in (heads, 1, 1, heads))
    decay = torch.tensor([-0.5, -0.25], device="cuda")
    dq, dk, dv, _ = fl.decay_attention_backward(do, q, k, v, decay, scale=scale, want=(True, True, True, False))
    q64, k64, v64, do64 = (t.double() for t in (q, k, v, do))
    slack = lambda most: (1.05 * UNIT[torch.bfloat16] + 64 * U32) * most
    dot = lambda a, b: (a * b).sum(-1, keepdim=True)
    for got, want, most, name in (
            (dq, scale * dot(do64, v64) * k64, scale * dot(do64.abs(), v64.abs()) * k64.abs(), "dq"),
            (dk, (scale * dot(do64, v64) * q64).sum(2, True), (scale * dot(do64.abs(), v64.abs()) * q64.abs()).sum(2, True), "dk"),
            (dv, (scale * dot(q64, k64) * do64).sum(2, True), (scale * dot(q64.abs(), k64.abs()) * do64.abs()).sum(2, True), "dv")):
        assert_within(got, want, slack(most), name)


def test_a_step_is_known_to_autograd():
    p = _problem(2, 1, train=False, dtype=torch.float32)
    state = (p["state"].requires_grad_() * 1.0)
    square = state * state
    fl.decay_attention_step(p["q"][:, 0], p["k"][:, 0], p["v"][:, 0], p["log_decay"], state.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.sum().backward()
    with torch.inference_mode():
        held = torch.zeros_like(p["state"])
    fl.decay_attention_step(p["q"][:, 0], p["k"][:, 0], p["v"][:, 0], p["log_decay"], held)   # (such a tensor has no version)
    assert bool(held.any())


def test_refusals():
    p = _problem(2, 10, heads=4, kv_heads=2, dk=32, dv=32)
    q, k, v, g, s = p["q"], p["k"], p["v"], p["log_decay"], p["state"]
    f = fl.decay_attention_forward
    for args, more, match in (((q.cpu(), k, v, g), {}, "q must be a CUDA"), ((q, k.float(), v, g), {}, "k must be of type"),
                              ((q, k[:, :5], v, g), {}, "leading axes"), ((q, k, v[..., :4], g), {}, "widths"), ((q[..., :16], k, v, g), {}, "q's width"),
                              ((q[:, :, :3], k, v, g), {}, "multiple"), ((q, k, v, g[:2]), {}, "log_decay"), ((q, k, v, g.double()), {}, "log_decay"),
                              ((q, k, v, g), dict(state=s[:1]), "state"), ((q, k, v, g), dict(state=s.half()), "state"),
                              ((q, k, v, g), dict(scale=float("nan")), "scale"), ((q, k, v, g.clone().requires_grad_()), {}, "gradient"),
                              ((q[0], k[0], v[0], g), {}, "4 axes"), ((q, k, v, g), dict(cu_seqlens=torch.zeros(3, device="cuda", dtype=torch.int32)), "3 axes"),
                              ((q[0], k[0], v[0], g), dict(cu_seqlens=torch.zeros(3, device="cuda")), "int32"),
                              ((q.double(), k.double(), v.double(), g), {}, "unsupported dtype")):
        with pytest.raises(ValueError, match=match):
            f(*args, **more)
    with pytest.raises(ValueError, match="do must have shape"):
        fl.decay_attention_backward(p["do"][..., :8], q, k, v, g)
    with pytest.raises(ValueError, match="d_state"):
        fl.decay_attention_backward(p["do"], q, k, v, g, d_state=s[:1])
    with pytest.raises(ValueError, match="state"):
        fl.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, None)
    assert math.isfinite(float(f(q, k, v, g)[0].float().sum()))


def _check_long(p, got, label=""):
    """Like _check, for long walks with tokens of zeros, behind which little but decayed values is left.  A decay by e^-x is exp2 of a
    product that is rounded to 32 bits a few times, 3 u x relative (x up to 104: what is smaller is below 2^-150), and an exp2 and a
    product a chunk cost 4 u; one below 2^-126 is zero, which leaves less than 2^-110 out.  Operands of fp16 are held to 2^-25 at the
    least: as parts of the state (as many as the head is wide) or as scores (64 a chunk), times another operand; in the state's
    update, relative to the largest value of their chunk, 64 a chunk too.  Where no key is zero that value is in the state, whose
    largest is then 1 or more before it decays; beside keys of zero it is not, and the bound is absolute."""
    want, most = _definition(p), _definition(p, magnitudes=True)
    dtype, (dk, dv) = p["q"].dtype, (p["q"].shape[-1], p["v"].shape[-1])
    largest = max(float(p[name].abs().max()) for name in ("q", "k", "v", "do"))
    unit, held = (UNIT[dtype] if dtype != torch.float32 else 0.0), (2.0 ** -25 if dtype == torch.float16 else 0.0)
    decays = U32 * (64 + 312 + max(p["lengths"]) / 8 + 8)
    beside = 64 * held * largest if bool((p["k"] == 0).all(-1).any()) else 0.0
    for name, value in want.items():
        if name in ("state", "d_initial"):
            slack = (decays + (0 if unit == 0 else 2.0 ** -21)) * most[name] + ((0 if unit == 0 else 2.0 ** -21) + 64 * held * largest) * most[name].amax((-1, -2), keepdim=True) + (beside if name == "state" else 0.0)
        else:
            slack = (1.05 * unit + decays) * most[name] + held * largest * max(1.0, abs(p["scale"])) * (64 + max(dk, dv))
        assert_within(got[name], value, slack + 2.0 ** -110, f"{label} {name}")


_DECAYS = [0.2, 0.5, 0.75, 0.9, 0.97, 0.99]


@pytest.mark.parametrize("name", ["v", "do", "k"])
@pytest.mark.parametrize("whole", [False, True], ids=["few heads", "many heads"])
@pytest.mark.parametrize("zeros,dtype", [(64, torch.float16), (130, torch.float16), (320, torch.float16), (1000, torch.float16), (1000, torch.bfloat16), (1000, torch.float32),
                                         (8192, torch.float16)], ids=str)
def test_tokens_of_zeros(zeros, dtype, whole, name):
    """Padding, and tokens without a loss: the state decays beside them, far below anything that is added to it later."""
    heads = 132 if whole else 6          # (more than 128: walked as a whole)
    p = _problem(1, zeros + 140, heads=heads, kv_heads=heads, dk=16, dv=16, dtype=dtype, log_decay=[math.log(g) for g in _DECAYS] * (heads // 6), seed=zeros)
    p[name][:, 70:70 + zeros] = 0        # ordinary tokens on both sides
    _check_long(p, _own(p), f"{zeros} in the middle")
    if zeros <= 1000:
        p[name][:, 70:] = 0
        _check_long(p, _own(p), f"{zeros} at the end")
        p[name][:, :70 + zeros] = 0
        _check_long(p, _own(p), "all")


@pytest.mark.parametrize("dk,dv", [(72, 136), (128, 64), (200, 40)])
def test_tokens_of_zeros_by_width(dk, dv):
    p = _problem(2, 500, heads=6, kv_heads=2, dk=dk, dv=dv, dtype=torch.float16, log_decay=[math.log(g) for g in _DECAYS])
    for name in ("v", "do", "k"):
        bad = dict(p, **{name: p[name].clone()})
        bad[name][0, 30:460] = 0
        bad[name][1, 200:] = 0
        _check_long(bad, _own(bad), name)


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -40, 2.0 ** 20])
def test_tokens_of_zeros_under_other_scales(scale):
    p = _problem(1, 500, heads=6, kv_heads=6, dk=16, dv=16, dtype=torch.float16, log_decay=[math.log(g) for g in _DECAYS], scale=scale)
    if scale > 1:
        p["q"] = (p["q"] * 2.0 ** -14).to(torch.float16)
    for name in ("v", "do", "k"):
        bad = dict(p, **{name: p[name].clone()})
        bad[name][:, 60:440] = 0
        got, want = _own(bad), _definition(bad)
        for key, value in want.items():
            assert not bool(torch.isnan(got[key]).any()), (name, key)
            fits = value.abs() < 60000
            assert bool(torch.isfinite(got[key][fits]).all()), (name, key)
        if scale <= 1:
            _check_long(bad, got, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_a_large_state_that_decays(dtype):
    """An initial state of up to 2^112 and ordinary tokens: outputs are right where they fit their type, states throughout."""
    p = _problem(1, 300, heads=6, kv_heads=6, dk=16, dv=16, dtype=dtype, log_decay=[math.log(g) for g in _DECAYS], train=False)
    p["do"] = torch.zeros_like(p["v"])
    p["d_state"] = None
    p["state"] = p["state"] * 2.0 ** 110
    got, want, most = _own(p), _definition(p), _definition(p, magnitudes=True)
    fits = most["o"] < 60000
    for name in ("o", "dq", "dk", "dv"):
        assert not bool(torch.isnan(got[name]).any()), name
    unit, held = (UNIT[dtype] if dtype != torch.float32 else 0.0), (2.0 ** -25 if dtype == torch.float16 else 0.0)
    slack = (1.05 * unit + U32 * (64 + 312 + 50)) * most["o"] + held * 80 * 5
    assert_within(torch.where(fits, got["o"], torch.zeros_like(got["o"])), torch.where(fits, want["o"], 0.0), torch.where(fits, slack, 0.0), "o")
    slack = (U32 * (64 + 312 + 50) + 2.0 ** -21) * most["state"] + (2.0 ** -21 + 64 * held * 5) * most["state"].amax((-1, -2), keepdim=True)
    assert_within(got["state"], want["state"], slack, "state")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", ["v", "k", "q", "do"])
@pytest.mark.parametrize("length,at", [(150, 80), (150, 149), (1, 0), (65, 64), (600, 301)])
def test_an_infinity_reaches_what_it_should(length, at, name, dtype):
    """What an infinity of an input reaches by the definition is not finite, all else as it was.  (It may be NaN where the definition has
    an infinity: values go into the state in parts, and heads are padded with zeros.)"""
    p = _problem(1, length, dtype=dtype, dk=32, dv=48, seed=at)
    most = _definition(p, magnitudes=True)
    bad = dict(p, **{name: p[name].clone()})
    bad[name][0, at, 0, 5], bad[name][0, at, 1, 7] = float("inf"), float("-inf")
    got, want = _own(bad), _definition(bad)
    unit = UNIT[dtype] if dtype != torch.float32 else 0.0
    for key, value in want.items():
        if key in ("state", "d_initial"):
            slack = (64 * U32 + (0 if unit == 0 else 2.0 ** -21)) * most[key] + (0 if unit == 0 else 2.0 ** -21) * most[key].amax((-1, -2), keepdim=True)
        else:
            slack = (1.05 * unit + 64 * U32) * most[key]
        numbers = torch.isfinite(value)
        assert not bool(torch.isfinite(got[key][~numbers]).any()), (name, key)
        assert_within(torch.where(numbers, got[key], torch.zeros_like(got[key])), torch.where(numbers, value, 0.0), slack, f"{name} {key}")
    if name != "do" and length == 1:   # a single token's form keeps infinities as they are
        state = p["state"].clone()
        o = fl.decay_attention_step(bad["q"][:, 0], bad["k"][:, 0], bad["v"][:, 0], p["log_decay"], state)
        assert torch.equal(torch.isinf(state), torch.isinf(want["state"])) and torch.equal(torch.isfinite(o), torch.isfinite(want["o"][:, 0]))


@pytest.mark.parametrize("packed", [False, True])
def test_tokens_far_apart(packed):
    """Tokens 2^23 elements apart and more, as of a (tokens, sequences, ..) tensor of very many features."""
    p = _problem(2, 5, heads=4, kv_heads=2, dk=32, dv=40, dtype=torch.float16, lengths=[3, 2] if packed else None)
    want = _own(p)
    room = torch.zeros(5 * (1 << 23) + 4096, device="cuda", dtype=torch.float16)
    for name in ("q", "k", "v", "do"):
        t = p[name]
        strides = (1 << 23, *t.stride()[1:]) if packed else (512, 1 << 23, *t.stride()[2:])
        view = room.as_strided(t.shape, strides)
        view.copy_(t)
        got = _own(dict(p, **{name: view}))
        for key in want:
            assert torch.equal(want[key], got[key]), (name, key)
        if not packed and name == "q":   # (outputs keep the memory order of q's rows)
            assert got["o"].stride()[0] < got["o"].stride()[1] and got["dq"].stride()[0] < got["dq"].stride()[1]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("sequences,length,lengths,kv_heads,dk,dv", [(2, 200, None, 2, 64, 64), (1, 130, None, 2, 128, 128), (1, 100, None, 1, 40, 65), (1, 90, None, 2, 256, 200),
                                                                     (1, 70, None, 2, 128, 64), (1, 600, None, 1, 128, 128), (3, None, [300, 1, 64], 2, 72, 136)])
def test_outputs_are_rounded_once(sequences, length, lengths, kv_heads, dk, dv, dtype):
    """The narrower types' outputs are those of 32 bits, rounded: what is an operand on the way is held in two parts, which leaves 2^-18 of a
    term at the most in bf16 (2^-22 in fp16, or 2^-25 times the other operand: a score's, 64 a chunk, or a part of the state's, one
    for each of the head's width), in the state and in the scores."""
    p = _problem(sequences, length, lengths=lengths, heads=2, kv_heads=kv_heads, dk=dk, dv=dv, dtype=dtype, seed=dk)
    got, want, most = _own(p), _definition(p), _definition(p, magnitudes=True)
    largest = max(float(p[name].abs().max()) for name in ("q", "k", "v", "do"))
    for name in ("o", "dq", "dk", "dv"):
        part = 2 * 2.0 ** -18 * most[name] if dtype == torch.bfloat16 else 2 * 2.0 ** -22 * most[name] + 2.0 ** -25 * largest * (64 + max(dk, dv))
        assert_within(got[name], want[name], part + 64 * U32 * most[name], name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("small,large", [(1e-4, 1.0), (1.0, 100.0), (0.01, 300.0), (1.0, 1e4)])
def test_magnitudes_of_what_fits(small, large, dtype):
    """Large keys and small gradients: every output that fits its type is right, whatever the others do.  An operand of fp16 is held to 2^-17
    of the largest beside it (2^-25 where that is 2^-8), and there are two: with terms up to four times a head's mean, less than 2^-13 of
    the largest sum of terms in the head."""
    p = _problem(1, 200, dtype=dtype, dk=64, dv=64, log_decay=[0.0, -0.02], with_state=False, scale=0.01)
    p["do"] = (p["do"] * small).to(dtype)
    p["k"] = (p["k"] * large).to(dtype)
    got, want, most = _own(p), _definition(p), _definition(p, magnitudes=True)
    for name, value in want.items():
        fits = value.abs() < 60000
        if name in ("state", "d_initial"):
            slack = (64 * U32 + 2.0 ** -21) * most[name] + 2.0 ** -21 * most[name].amax((-1, -2), keepdim=True)
        else:
            slack = (1.05 * UNIT[dtype] + 64 * U32) * most[name] + (2.0 ** -13 * most[name].amax((1, 3), keepdim=True) if dtype == torch.float16 else 0.0)
            assert not bool(torch.isnan(got[name]).any()), name
        assert bool(fits.any()), name
        assert_within(torch.where(fits, got[name], torch.zeros_like(got[name])), torch.where(fits, value, 0.0), torch.where(fits, slack, 0.0), name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("length", [256, 257, 449, 512, 513, 577])
def test_around_eight_chunks(length, dtype):
    """Where walks over whole sequences end and segments begin (512 tokens, 256 of fp32)."""
    p = _problem(2, length, heads=2, kv_heads=1, dk=40, dv=72, dtype=dtype, seed=length)
    _check(p, _own(p))
