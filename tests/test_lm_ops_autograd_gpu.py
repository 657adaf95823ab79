"""What the language-model operators say to derivatives that they do not have."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import flashlstm_poc_amd as fl

pytestmark = pytest.mark.gpu


def _calls():
    g = torch.Generator(device="cuda").manual_seed(0)
    n = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    index = torch.arange(3, device="cuda").expand(4, 3)
    decay = -torch.ones(2, device="cuda")
    return {
        "layer_norm": (lambda x, w, b, r: fl.layer_norm(x, w, b, residual=r), [n(4, 16), n(16), n(16), n(4, 16)]),
        "decay_attention": (lambda q, k, v, s: fl.decay_attention(q, k, v, decay, state=s), [n(1, 5, 2, 8), n(1, 5, 2, 8), n(1, 5, 2, 8), n(1, 2, 8, 8)]),
        "decay_attention's decay": (lambda d: fl.decay_attention(*[torch.ones(1, 5, 2, 8, device="cuda")] * 3, d), [decay]),
        "distillation_loss": (lambda z, t: fl.distillation_loss(z, t, index), [n(4, 20), n(4, 3)]),
    }


@pytest.mark.parametrize("name", ["layer_norm", "decay_attention", "decay_attention's decay", "distillation_loss"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(name, grad):
    call, inputs = _calls()[name]
    first = lambda out: out[0] if isinstance(out, tuple) else out
    plain = first(call(*inputs))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        assert torch.equal(first(call(*inputs)), plain)          # none of these carries a derivative
        for i, t in enumerate(inputs):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="jvp"):
                call(*inputs[:i], dual, *inputs[i + 1:])
    assert torch.equal(first(call(*inputs)), plain)
