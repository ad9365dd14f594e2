"""The paths that the event-sequence operators take at window sizes: the sort's tiles, passes and scan on both sides of
each border, long runs of one row, rows of several column slabs, and chains of more chunks than threads."""
import numpy as np
import pytest
import torch

import x_b200
from tests import sequence_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ row gradient
def row_gradient_is_exact(N, V, D, dtype, spread):
    """Whole numbers up to 8 and a scale of 1/2: every fp32 sum below 2^24 is exact, so one event lost, doubled or put to
    another row shows.  Some indices lie outside the table."""
    assert N * 8 < 2**24
    idx = (torch.rand(N, generator=gen(N), device=DEV) ** spread * (V + 4)).long() - 2
    g = torch.randint(-8, 9, (N, D), generator=gen(V), device=DEV).to(dtype)
    w = randn(V, D, seed=1, dtype=dtype).requires_grad_()
    out = x_b200.embedding(w, idx, 0.5)
    (gw,) = torch.autograd.grad(out, [w], g)
    ok = (idx >= 0) & (idx < V)
    assert torch.equal(out, torch.where(ok[:, None], w.detach()[idx.clamp(0, V - 1)] * 0.5, 0.0))
    ref = torch.zeros(V + 1, D, dtype=torch.float64, device=DEV)
    ref.index_add_(0, torch.where(ok, idx, V), g.double())
    assert torch.equal(gw, (ref[:V] * 0.5).to(dtype))


@pytest.mark.parametrize("V", [900, 5000, (1 << 20) + 5])  # one, two and three digits
@pytest.mark.parametrize("N", [4096, 4097, 131072, 131073, 200000, 262144, 262145, 700001])
def test_row_gradient_over_the_sorts_borders(N, V):
    """One launch up to 4096 events; up to 131072 each tile's offsets are summed in the placement, above by a scan of their
    own; above 262144 larger tiles; above 524288 more than 128 of them."""
    row_gradient_is_exact(N, V, 2, torch.float32, 1)
    row_gradient_is_exact(N, V, 8, torch.bfloat16, 4)


@pytest.mark.parametrize("N,V,D,dtype", [
    (3000, 700, 264, torch.bfloat16), (3000, 700, 512, torch.float16), (3000, 700, 132, torch.float32),
    (3000, 700, 512, torch.float32), (20000, 2, 264, torch.bfloat16), (20000, 3, 260, torch.float32),
    (20000, 1, 520, torch.float16)])
def test_rows_of_several_aligned_slabs(N, V, D, dtype):
    """16-byte threads and more columns than 32 of them hold; with few rows, runs over many chunks as well."""
    row_gradient_is_exact(N, V, D, dtype, 2)


@pytest.mark.parametrize("N,V,D,dtype", [(300000, 5, 8, torch.float32), (300000, 3, 96, torch.float32),
                                         (1000000, 2, 24, torch.float16), (200000, 40, 256, torch.bfloat16)])
def test_long_runs_keep_the_error_of_their_chunks(N, V, D, dtype):
    """Events are summed in fp32 over chunks of L (a wave of groups on 148 SMs of 3 CTAs), the chunks in 64 bits: an
    event's value takes at most L roundings on its way, then one to fp32 and one for the scale."""
    lanes = max(1, min(32, -(-D // 8)))
    L = max(16, -(-N // (148 * 3 * (256 // lanes))))
    idx = (torch.rand(N, generator=gen(1), device=DEV) ** 4 * V).long()
    g = randn(N, D, seed=2, dtype=dtype, scale=0.1)
    w = randn(V, D, seed=3, dtype=dtype).requires_grad_()
    (gw,) = torch.autograd.grad(x_b200.embedding(w, idx, 0.375), [w], g)
    grad, mag = (torch.zeros(V, D, dtype=torch.float64, device=DEV) for _ in range(2))
    grad.index_add_(0, idx, g.double())
    mag.index_add_(0, idx, g.double().abs())
    ref, bound = R.f64(grad) * 0.375, (L + 2) * R.U * R.f64(mag) * 0.375
    # magnitudes add up to 0.08 an event, sums to 0.1 a root of their number: the bound is far below the values
    assert np.median(bound) < 0.05 * np.median(np.abs(ref))
    R.check(gw, ref, bound)


# ------------------------------------------------------------------------------------------------ recurrence
@pytest.mark.parametrize("N,D,B,kind,dtype,state", [
    (20000, 64, 1, "sigmoid", torch.float32, False), (20000, 64, 4, "decay", torch.bfloat16, True),
    (70001, 33, 1, "sigmoid", torch.float16, True), (70001, 33, 3, "decay", torch.float32, True),
    (140001, 64, 3, "sigmoid", torch.bfloat16, True), (140001, 64, 1, "decay", torch.float32, True),
    (140001, 64, 1, "sigmoid", torch.float32, False), (140001, 64, 2, "decay", torch.bfloat16, False)])
def test_chains_of_many_chunks(N, D, B, kind, dtype, state):
    """40 chunks of 512 rows (more than a warp joins), 274 of 256 or 512 (several to a thread), states and gradients that
    reach over hundreds of rows: past the chunks' borders both ways."""
    rng = np.random.default_rng(N + D)
    cut = np.sort(rng.integers(1, N, B - 1))
    bn = np.searchsorted(cut, np.arange(N), side="right").astype(np.int64)
    if B > 1:
        bn[N - 7:] = -1
    b = torch.from_numpy(bn).to(DEV)
    if kind == "sigmoid":
        gate = (randn(N, D, seed=1) + 6.0).to(dtype)
    else:  # 1 and 1 - 2^-8, which all types hold
        gate = (1.0 - 2.0**-8 * torch.randint(0, 2, (N, D), generator=gen(1), device=DEV)).to(dtype)
    gate.requires_grad_()
    x, gh = randn(N, D, seed=2, dtype=dtype).requires_grad_(), randn(N, D, seed=3, dtype=dtype)
    h0 = randn(B, D, seed=4).requires_grad_() if state else None
    ghT = randn(B, D, seed=5) if state else None
    h, st = x_b200.linear_recurrence(gate, x, b=b, B=B, h0=h0, kind=kind, return_state=True)
    outs, gs = ([h, st], [gh, ghT]) if state else ([h], [gh])
    got = (h, st, *torch.autograd.grad(outs, [gate, x] + ([h0] if state else []), gs))
    r = R.recurrence(kind, R.f64(gate), R.f64(x), bn, B, R.f64(h0) if state else None, R.f64(gh),
                     R.f64(ghT) if state else None)
    for name, t in zip(["h", "state", "dgate", "dx", "dh0"], got):
        R.check(t, *r[name], name)
    for name in ("h", "dx"):  # the bound is far below the values
        assert np.median(r[name][1]) < 0.1 * np.median(np.abs(r[name][0])), name
