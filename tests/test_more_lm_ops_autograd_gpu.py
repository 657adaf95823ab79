"""What the embedding and the gated linear recurrence say to derivatives that they do not have, and to captured backward passes."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import flashlstm_poc_amd as fl

pytestmark = pytest.mark.gpu


def _calls():
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    tokens = torch.tensor([3, 1, 1, -1], device="cuda")
    return {
        "embedding": (lambda w: fl.embedding(tokens, w, scale=2.0), [n(5, 8)]),
        "gated_recurrence": (lambda x, u, o, s: fl.gated_recurrence(x, u, o, state=s)[0], [n(2, 6, 8), n(2, 6, 8), n(2, 6, 8), n(2, 8)]),
    }


@pytest.mark.parametrize("name", ["embedding", "gated_recurrence"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(name, grad):
    call, inputs = _calls()[name]
    plain = call(*inputs)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        assert torch.equal(call(*inputs), plain)          # none of these carries a derivative
        for i, t in enumerate(inputs):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="jvp"):
                call(*inputs[:i], dual, *inputs[i + 1:])
    assert torch.equal(call(*inputs), plain)


@pytest.mark.parametrize("name", ["embedding", "gated_recurrence"])
def test_second_derivatives_are_refused(name):
    call, inputs = _calls()[name]
    leaves = [t.requires_grad_() for t in inputs]
    grads = torch.autograd.grad(call(*leaves).square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(g.sum() for g in grads).backward()


def test_a_changed_state_is_noticed():
    x, u, s = (torch.randn(2, 8, device="cuda") for _ in range(3))
    w = torch.ones(2, 8, device="cuda", requires_grad=True)
    loss = (w * s).sum()          # its backward pass needs s as it was
    fl.gated_recurrence_step(x, u, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    s = torch.randn(4, 8, device="cuda")
    loss = (torch.ones(4, 8, device="cuda", requires_grad=True) * s).sum()
    fl.beam_reorder(torch.zeros(2, 2, device="cuda", dtype=torch.int64), s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        state = torch.zeros(2, 8, device="cuda")
        fl.gated_recurrence_step(x, u, state)
        fl.beam_reorder(torch.zeros(1, 2, device="cuda", dtype=torch.int64), state)


@pytest.mark.parametrize("tokens", [40, 400])
def test_training_step_captured_in_a_graph(tokens):
    """Forward and backward of embedding and recurrence through autograd in one graph, on leaves of its own."""
    index = torch.randint(0, 30, (2, tokens), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    table = torch.randn(30, 48, device="cuda").requires_grad_()
    dy = torch.randn(2, tokens, 16, device="cuda").half()

    def run():
        x, forget, gate = fl.embedding(index, table, dtype=torch.float16).chunk(3, -1)
        y, state = fl.gated_recurrence(x, forget, gate)
        return y, torch.autograd.grad(y, table, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grad = run()
    for seed in range(4):
        g = torch.Generator(device="cuda").manual_seed(seed + 5)
        index.copy_(torch.randint(-1, 30, index.shape, device="cuda", generator=g))
        dy.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        want, want_grad = run()
        assert torch.equal(y, want) and torch.equal(grad, want_grad)
