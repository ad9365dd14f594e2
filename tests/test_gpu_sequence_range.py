"""The recurrence with gates and states far from one: products of gates that leave fp32's range where no state does,
against the float64 statement (tests/sequence_ref.py), whose bounds count the roundings of the row-by-row recurrence."""
import numpy as np
import pytest
import torch

import x_b200
from tests import sequence_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def compare(kind, gate, x, b, B, h0, gh, ghT):
    h, st = x_b200.linear_recurrence(gate, x, b=b, B=B, h0=h0, kind=kind, return_state=True)
    got = (h, st, *torch.autograd.grad([h, st], [gate, x, h0], [gh, ghT]))
    N = x.shape[0]
    bn = b.cpu().numpy() if b is not None else np.repeat(np.arange(B), N // B)
    with np.errstate(all="ignore"):
        r = R.recurrence(kind, R.f64(gate), R.f64(x), bn, B, R.f64(h0), R.f64(gh), R.f64(ghT))
    for name, t in zip(["h", "state", "dgate", "dx", "dh0"], got):
        R.check(t, *r[name], name)
    return got, r


def swings(N, D, up, down, rows, at, seed):
    """Gates of one, but from row `at` on `rows` gates of `up` and as many of `down`; every sign at random."""
    gate = torch.ones(N, D, device=DEV)
    gate[at:at + rows], gate[at + rows:at + 2 * rows] = up, down
    return gate * (torch.randint(0, 2, (N, D), generator=gen(seed), device=DEV) * 2 - 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,at", [(1400, 64, 542), (1400, 40, 542), (4500, 3, 2174), (17000, 4, 8318),
                                    (26000, 2, 16510)])
def test_decay_gates_whose_product_overflows(N, D, at, dtype):
    """A state of 0.01 and 130 doublings: 1e37, and back.  The gates' product over the rows of the swing, 2^130, is not
    an fp32 number, and backward the mirrored swing meets the same product.  Rows are joined in chunks of 512 (the first
    two widths), 2048, 4096 or 8192 rows, groups of 32 inside; the swing lies inside a chunk, its peak at a group's border,
    and states and gradients come from outside the chunk."""
    gate = swings(N, D, 2.0, 0.5, 130, at, 1).to(dtype).requires_grad_()
    x, gh = torch.zeros(N, D, dtype=dtype, device=DEV), torch.zeros(N, D, dtype=dtype, device=DEV)
    x[at - 150] = 0.01
    x[at + 260:] = randn(N - at - 260, D, seed=2, dtype=dtype, scale=1e-3)
    gh[-1], gh[:at] = 0.25, randn(at, D, seed=3, dtype=dtype, scale=1e-3)
    x.requires_grad_()
    h0, ghT = torch.zeros(1, D, device=DEV, requires_grad=True), randn(1, D, seed=4, scale=0.01)
    got, r = compare("decay", gate, x, None, 1, h0, gh, ghT)
    # the bound lets no state behind the swing be lost: about 410 rows of 8 U, 2^-12, of a state that x moves by half
    # of 0.01 at most
    assert (r["h"][1][at + 260] < np.abs(r["h"][0][at + 260]) * 2.0**-8).all()
    assert torch.isfinite(got[0][at + 260:]).all() and torch.isfinite(got[1]).all() and torch.isfinite(got[4]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D,at", [(1500, 3, 300), (1500, 64, 10), (9000, 4, 4000)])
def test_decay_gates_whose_product_vanishes(T, D, at, dtype):
    """A state of 2^100 falls to 2^-100 and comes back: the product over the fall, 2^-200, is no fp32 number, the states
    are; nor is the rise, 2^200, which takes a gradient of 2^-100 to 2^100.  Two windows, so that the swing starts at two
    places of a chunk."""
    gate = torch.cat([swings(T, D, 0.5, 2.0, 200, at, 1), swings(T, D, 0.5, 2.0, 200, at + 37, 2)]).to(dtype)
    gate.requires_grad_()
    x = torch.zeros(2 * T, D, dtype=dtype, device=DEV, requires_grad=True)
    gh = torch.zeros(2 * T, D, dtype=dtype, device=DEV)
    h0 = torch.full((2, D), 2.0**100, device=DEV, requires_grad=True)
    got, _ = compare("decay", gate, x, None, 2, h0, gh, torch.full((2, D), 2.0**-100, device=DEV))
    assert (got[1].abs() == 2.0**100).all() and (got[4].abs() == 2.0**-100).all()


@pytest.mark.parametrize("D", [1, 2, 64])
def test_decay_gates_of_zero_and_at_the_ends_of_fp32(D):
    """Gates of zero, subnormal gates and gates near the largest number, in rows that no group or chunk border marks."""
    N = 2500
    gate = torch.where(torch.rand(N, D, generator=gen(1), device=DEV) < 0.5, -0.75, 0.75)
    for k, at in enumerate(range(40, N - 40, 97)):
        if k % 3 == 0:
            gate[at] = 0.0
        elif k % 3 == 1:  # 2^-130 is subnormal
            gate[at], gate[at + 1] = 2.0**-130, 2.0**126
        else:
            gate[at], gate[at + 1], gate[at + 2] = 2.0**100, 2.0**-120, 2.0**20
    gate.requires_grad_()
    x, h0 = randn(N, D, seed=2).requires_grad_(), randn(1, D, seed=3).requires_grad_()
    gh = torch.zeros(N, D, device=DEV)
    gh[10::400] = randn(len(gh[10::400]), D, seed=4)
    # x is zero where the state stands near the ends
    with torch.no_grad():
        x[(gate.abs() < 0.5) | (gate.abs() > 1)] = 0
    compare("decay", gate, x, None, 1, h0, gh, randn(1, D, seed=5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", [0.0, 2.0**-14, 2.0**-3])
def test_decay_short_memories(low, dtype):
    """Gates that are zero or small in most rows, one among them or all of a group, and rows of ones around them: what
    passes is lost or kept to the bit.  x and gradients are whole numbers; the small gates are powers of two."""
    N, D = 1800, 40
    gate = torch.ones(N, D, device=DEV)
    pick = torch.rand(N, D, generator=gen(1), device=DEV)
    gate[600:1200] = torch.where(pick[600:1200] < 0.3, low, 1.0)
    gate[1300:1340] = low
    gate[::50, ::3] = low
    gate = gate.to(dtype).requires_grad_()
    x = torch.randint(-3, 4, (N, D), generator=gen(2), device=DEV).to(dtype).requires_grad_()
    gh = torch.randint(-3, 4, (N, D), generator=gen(3), device=DEV).to(dtype)
    h0, ghT = randn(1, D, seed=4).requires_grad_(), randn(1, D, seed=5)
    got, r = compare("decay", gate, x, None, 1, h0, gh, ghT)
    if low == 0.0:  # nothing but whole numbers behind a zero
        assert (got[0][1340:1350].float() == got[0][1340:1350].float().round()).all() and torch.equal(got[0][1339], x[1339])


def test_decay_infinite_gate_stays_in_its_column():
    N, D = 900, 4
    gate, x = torch.full((N, D), 0.5, device=DEV), randn(N, D, seed=1)
    clean = x_b200.linear_recurrence(gate, x, kind="decay")
    gate[200, 1], gate[333, 3] = float("inf"), float("nan")
    h = x_b200.linear_recurrence(gate, x, kind="decay")
    assert not torch.isfinite(h[200:, 1]).any() and not torch.isfinite(h[333:, 3]).any()
    assert torch.equal(h[:, [0, 2]], clean[:, [0, 2]]) and torch.equal(h[:200, 1], clean[:200, 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", [-float("inf"), -1000.0, -130.0])
def test_closed_gates_leave_no_trace_of_a_large_state(low, dtype):
    """A gate far below zero takes x and nothing of the state before it, of 2^120 here: exp(-130) 2^120 is below 2^-66."""
    N, D = 700, 40
    gate, x = torch.full((N, D), 20.0, dtype=dtype, device=DEV), randn(N, D, seed=1, dtype=dtype)
    x[100:103] = float(2.0**120) if dtype != torch.float16 else 0.0
    shut = torch.tensor([0, 40, 103, 330, 600], device=DEV)
    gate[shut] = low
    gate[100:103] = -20.0
    gate.requires_grad_(), x.requires_grad_()
    h0 = torch.full((1, D), 2.0**120, device=DEV, requires_grad=True)
    h, st = x_b200.linear_recurrence(gate, x, h0=h0, return_state=True)
    assert torch.equal(h[shut], x[shut])
    assert h.isfinite().all() and (st.abs() < 8).all()
    gg, gx, g0 = torch.autograd.grad(st, [gate, x, h0], torch.ones_like(st))
    assert (gx[:600] == 0).all() and (gg[:600] == 0).all() and (g0 == 0).all() and gg.isfinite().all()
    assert ((gx[600] - 1).abs() < 0.01).all()
