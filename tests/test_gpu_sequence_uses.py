"""Uses of the event-sequence operators beside the plain call."""
import pytest
import torch
from torch.autograd import forward_ad

import x_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


CALLS = [("embedding", lambda t: x_b200.embedding(t, torch.arange(6, device=DEV))),
         ("dropout", lambda t: x_b200.dropout(t, 0.5, 1)),
         ("dropout, residual", lambda t: x_b200.dropout(randn(6, 4), 0.5, 1, residual=t)),
         ("gate", lambda t: x_b200.linear_recurrence(t, randn(6, 4))),
         ("x", lambda t: x_b200.linear_recurrence(randn(6, 4), t, kind="decay", return_state=True)),
         ("h0", lambda t: x_b200.linear_recurrence(randn(6, 4), randn(6, 4), B=6, h0=t))]


@pytest.mark.parametrize("call", [c for _, c in CALLS], ids=[n for n, _ in CALLS])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_inputs_are_refused(call, grad):
    """A tangent that the operator cannot carry on raises instead of becoming zero, with gradients on or off; plain
    tensors pass at the same level."""
    x, t = randn(6, 4, seed=1), randn(6, 4, seed=2)
    plain = call(x)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
            call(forward_ad.make_dual(x, t))
        again = call(x)
    for a, b in zip((plain, again) if torch.is_tensor(plain) else plain, (again, plain) if torch.is_tensor(again) else again):
        assert torch.equal(a, b)
