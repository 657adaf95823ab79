"""What the tests of the language-model operators share: types, their rounding, and the bound that an output is held to."""
import torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# half a unit in the last place, relative: what one rounding to the type costs at most
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the distance between the smallest numbers of the type
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U32 = UNIT[torch.float32]


def assert_within(got, want, slack, label):
    """|got - want| <= one rounding to got's type + slack, element by element; want and slack in 64 bits."""
    assert tuple(got.shape) == tuple(want.shape), f"{label}: shape {tuple(got.shape)} instead of {tuple(want.shape)}"
    assert want.dtype == torch.float64
    got64 = got.detach().double().to(want.device)
    bound = UNIT[got.dtype] * want.abs() + TINY[got.dtype] + slack
    bad = ~((got64 - want).abs() <= bound)
    if bool(bad.any()):
        over = torch.where(bad, ((got64 - want).abs() / bound).nan_to_num(float("inf")), torch.zeros_like(want))
        at = int(over.argmax())
        raise AssertionError(f"{label}: {int(bad.sum())} of {bad.numel()} outside the bound, the worst at {at}: "
                             f"{float(got64.flatten()[at]):.9g} instead of {float(want.flatten()[at]):.9g}")


def offset_copy(t, by=1):
    """The same values in memory that begins `by` elements behind an allocation's start: no alignment but the type's own."""
    room = torch.empty(t.numel() + by, device=t.device, dtype=t.dtype)
    out = room[by:].view(t.shape)
    out.copy_(t)
    return out
