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


def test_events_outside_the_sensor_read_zeros_and_train_nothing():
    """Positions with fractions, on the border and outside on every side: the row of the nearest pixel, or zeros."""
    W, H, D = 7, 5, 8
    xy = torch.tensor([[0.0, 0.0], [6.4, 4.4], [2.6, 3.3], [7.0, 1.0], [-1.0, 2.0], [-0.4, 0.4], [3.0, -1.0], [3.0, 5.0],
                       [6.6, 2.0], [2.0, 3.5]], device=DEV)
    want = [0, 34, 24, -1, -1, 0, -1, -1, -1, 4 * W + 2]  # halves to even
    xi, yi = xy.round().long().unbind(1)
    pix = torch.where((xi >= 0) & (xi < W) & (yi >= 0) & (yi < H), yi * W + xi, -1)
    assert pix.tolist() == want
    table = randn(H * W, D, seed=3).requires_grad_()
    out = x_b200.embedding(table, pix)
    (grad,) = torch.autograd.grad(out, [table], torch.ones_like(out))
    count = torch.zeros(H * W, device=DEV)
    for row, n in enumerate(want):
        assert torch.equal(out[row], table[n] if n >= 0 else torch.zeros(D, device=DEV))
        if n >= 0:
            count[n] += 1
    assert torch.equal(grad, count[:, None].expand(H * W, D))
