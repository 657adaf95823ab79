"""The gated linear recurrence with gates that are alike at every token and memories of thousands of them, where a rounding that is the same at every
token adds up.

Bounds, with u = 2^-24 and M the state (the gradient) with all its terms taken as magnitudes.  Cut into segments, a state is put together from what the
16 tokens of a wave, the waves of a segment, 8 segments, 8 groups and all groups of groups in front make of one, and 16 tokens walked.
* Every such step s -> F s + S rounds F, of a state of M at most, and the sum: 2 u M.  The steps inside of a piece do that to the piece's own S, of which
  the pieces have M between them, and a piece keeps of an error no more than F <= 1.  At most 16 + 8 + 8 + 8 + 16 of them and one for each of the
  groups of groups in front, G: 2 (56 + G) u M.
* A token's smaller sigmoid is off by (|a| + 6) u of itself (see test_gated_recurrence_gpu.py), what its step rounds included (|a| + 8) u; and 1 - F by 2 u a
  step more, as its terms have one sign: 2 (16 + 8 + 8 + 8 + G).  A weight of x, s (1 - s)^n, changes by no more than (1 + s n / (1 - s)) of that, and the
  sum over n of s (1 - s)^n s n is below 1, where the values and the state that it starts from are of one size: 2 (|a| + 8) + 4 (40 + G) u M.
Walked whole, one sequence of few channels never is.  Gradients' own products are off as in test_gated_recurrence_gpu.py."""
import numpy as np
import pytest
import torch

import flashlstm_poc_amd as fl
from lm_helpers import DTYPES, U32, assert_within
from test_gated_recurrence_gpu import _check, _problem

pytestmark = pytest.mark.gpu


def _bound(gate, groups):
    return (2 * (56 + groups) + 4 * (40 + groups) + 2 * (gate.abs() + 8)) * U32


def _walked(first, keep, take, x):
    """s_t = keep s_{t-1} + take x_t and the same of magnitudes: what is in front of each token, and behind the last, in 64 bits."""
    s, m = first.copy(), np.abs(first)
    values, sizes = np.empty((len(x) + 1, len(first))), np.empty((len(x) + 1, len(first)))
    for t in range(len(x)):
        values[t], sizes[t] = s, m
        s = keep * s + take * x[t]
        m = keep * m + take * np.abs(x[t])
    values[-1], sizes[-1] = s, m
    return torch.from_numpy(values), torch.from_numpy(sizes)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sign", [1, -1])
def test_gates_that_stay_the_same(dtype, sign):
    tokens, gates = 40000, torch.tensor([-3.0, 0.0, 2.0, 8.0, 9.0, 10.0, 11.0, 12.0], dtype=torch.float64)
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g)
    x, dy = (sign + n(tokens, 8)).to(dtype), (sign + n(tokens, 8)).to(dtype)
    state, d_state = sign + n(8), (sign + n(8)) / torch.sigmoid(-gates).float()    # (of the size that the tokens' sums have)
    f, z = torch.sigmoid(gates).numpy(), torch.sigmoid(-gates).numpy()
    c, of_c = _walked(state.double().numpy(), f, z, x.double().numpy())
    # G_t = dy_t + H_{t+1}, H_t = f G_t: H_t = f H_{t+1} + f dy_t, from the last token on
    h, of_h = (t.flip(0) for t in _walked(d_state.double().numpy(), f, f, dy.double().flip(0).numpy()))
    forget = gates.to("cuda", dtype).expand(1, tokens, 8)                        # (one bias for all tokens)
    y, final, saved = fl.gated_recurrence_forward(x.cuda()[None], forget, state=state.cuda()[None])
    dx, dforget, _, d_initial = fl.gated_recurrence_backward(dy.cuda()[None], x.cuda()[None], forget, None, saved, d_state=d_state.cuda()[None])
    rel = (gates.abs() + 8) * U32
    slack, back = _bound(gates, -(-tokens // 8192)), _bound(gates, -(-tokens // 4096))
    f, z = torch.sigmoid(gates), torch.sigmoid(-gates)
    total, size = dy.double() + h[1:], dy.double().abs() + of_h[1:]
    of_total = (back + U32) * size
    way = c[:-1] - x.double()
    of_way = slack * of_c[:-1] + 2 * U32 * (of_c[:-1] + x.double().abs())
    for name, got, want, bound in (
            ("y", y[0], c[1:], slack * of_c[1:]), ("state", final[0], c[-1], slack * of_c[-1]), ("d_initial", d_initial[0], h[0], back * of_h[0]),
            ("dx", dx[0], z * total, z * (of_total + (rel + 2 * U32) * size)),
            ("dforget", dforget[0], total * way * f * z, f * z * (of_total * way.abs() + size * of_way + (2 * rel + 4 * U32) * size * (of_c[:-1] + x.double().abs())))):
        assert_within(got.cpu(), want, bound, f"{dtype} {name}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gates_of_all_sizes(dtype):
    """Factors of pieces from nothing to one, in every order, over states of all sizes; bounds of test_gated_recurrence_gpu.py."""
    p = _problem((2, 20000, 12), dtype, 2, True, seed=22)
    g = torch.Generator(device="cuda").manual_seed(23)
    sizes = torch.tensor([-60.0, -7.0, -1.0, 0.0, 0.5, 3.0, 9.0, 14.0, 40.0], device="cuda")
    drawn = sizes[torch.randint(0, 9, (2, 20000, 12), device="cuda", generator=g)].to(dtype)
    keeps = torch.rand(2, 20000, 12, device="cuda", generator=g) < torch.tensor([0.0, 0.5, 0.99, 0.999, 0.9999, 1.0], device="cuda").repeat(2)
    p["forget"] = torch.where(keeps, drawn.abs() + 6, drawn)
    p["state"], p["d_state"] = p["state"] * 10.0 ** torch.arange(-6, 6, device="cuda"), p["d_state"] * 10.0 ** torch.arange(5, -7, -1, device="cuda")
    _check(p, f"{dtype}")
