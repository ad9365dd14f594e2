"""The event-sequence operators on the GPU against their float64 statements (tests/sequence_ref.py), at the sizes,
layouts and masks where they can go wrong, with tolerances that count the roundings."""
import numpy as np
import pytest
import torch

import x_b200
from tests import sequence_ref as R
from x_b200 import rng as RNG

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ------------------------------------------------------------------------------------------------ embedding
def lookup_inputs(N, V, D, dtype, seed, dist):
    g = gen(seed)
    if dist == "one":  # every event reads one row
        idx = torch.full((N,), V // 2, device=DEV)
    elif dist == "skew":
        idx = (torch.rand(N, generator=g, device=DEV) ** 4 * V).long().clamp_(max=max(V - 1, 0))
    else:
        idx = torch.randint(-2, V + 2, (N,), generator=g, device=DEV)  # some outside the table
    if N > 3:
        idx[N // 2], idx[N // 3] = -1, V
    return randn(V, D, seed=seed + 1, dtype=dtype), idx, randn(N, D, seed=seed + 2, dtype=dtype, scale=0.1)


@pytest.mark.parametrize("N,V,D,dist", [
    (0, 5, 8, "any"), (1, 1, 1, "one"), (5, 0, 4, "any"), (7, 3, 0, "any"), (33, 300, 64, "any"), (31, 1, 24, "one"),
    (2049, 33, 96, "any"), (2048, 1024, 7, "skew"), (4097, 1023, 33, "skew"), (5000, 1, 8, "one"),
    (6000, 2, 257, "any"), (20000, 43200, 32, "skew"), (3000, 1 << 21, 16, "any"), (70001, 300, 40, "skew"),
    (300000, 5, 8, "skew")])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding(N, V, D, dist, dtype):
    w, idx, g = lookup_inputs(N, V, D, dtype, N + V, dist)
    w.requires_grad_()
    out = x_b200.embedding(w, idx, 0.375)
    (gw,) = torch.autograd.grad(out, [w], g)
    fwd, bwd = R.embedding(R.f64(w), idx.cpu().numpy(), 0.375, R.f64(g))
    assert out.dtype == gw.dtype == dtype and out.shape == (N, D)
    R.check(out, *fwd, "out")
    R.check(gw, *bwd, "grad")
    out2 = x_b200.embedding(w, idx, 0.375)
    assert same_bits(out, out2) and same_bits(gw, torch.autograd.grad(out2, [w], g)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_layouts(dtype):
    """Index shapes and types, rows of a wider table, rows of a wider gradient, an expanded gradient."""
    w0, idx, _ = lookup_inputs(600, 50, 131, dtype, 3, "any")
    wide = w0.clone().requires_grad_()
    for lo, hi in ((0, 64), (1, 65), (3, 131), (8, 40)):
        w = wide[:, lo:hi]
        D = hi - lo
        out = x_b200.embedding(w, idx.view(20, 30).t().int(), 2.0)
        assert out.shape == (30, 20, D)
        order = idx.view(20, 30).t().reshape(-1).cpu().numpy()
        gbig = randn(600, 131 + 5, seed=9, dtype=dtype, scale=0.1)
        g = gbig[:, lo:hi].unflatten(0, (30, 20))
        (gw,) = torch.autograd.grad(out, [wide], g)
        fwd, bwd = R.embedding(R.f64(w), order, 2.0, R.f64(g).reshape(600, D))
        R.check(out.reshape(600, D), *fwd, "out")
        R.check(gw[:, lo:hi], *bwd, "grad")
        out = x_b200.embedding(w, idx)
        (gw,) = torch.autograd.grad(out.float().sum(), [wide])
        _, bwd = R.embedding(R.f64(w), idx.cpu().numpy(), 1.0, np.ones((600, D)))
        R.check(gw[:, lo:hi], *bwd, "grad of a sum")
    col = x_b200.embedding(w0.t().contiguous().t(), idx, 2.0)  # a column-major table
    R.check(col, *R.embedding(R.f64(w0), idx.cpu().numpy(), 2.0))
    row = x_b200.embedding(w0[7:8].expand(50, -1), idx, 2.0)  # one row for all
    R.check(row, *R.embedding(R.f64(w0[7:8].expand(50, -1)), idx.cpu().numpy(), 2.0))


def test_embedding_refuses():
    w, i = torch.zeros(4, 8, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    for bad in (lambda: x_b200.embedding(w, i.cpu()), lambda: x_b200.embedding(w, i.float()),
                lambda: x_b200.embedding(w.double(), i)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        x_b200.embedding(w[0], i)
    # not differentiable twice
    w.requires_grad_()
    (g,) = torch.autograd.grad(x_b200.embedding(w, i).sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("shape", [(0,), (1,), (3,), (4,), (5,), (1025,), (333, 77), (4096, 64), (2, 3, 5, 7)])
@pytest.mark.parametrize("p,residual", [(0.0, False), (0.1, True), (0.5, False), (0.999, True), (1.0, True), (1.0, False)])
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout(shape, p, residual, dtype):
    seed, call = 2**40 + 7, 2**33 + 5
    x = randn(*shape, seed=1, dtype=dtype).requires_grad_()
    r = randn(*shape, seed=2, dtype=dtype).requires_grad_() if residual else None
    g = randn(*shape, seed=3, dtype=dtype)
    out = x_b200.dropout(x, p, seed, call, residual=r)
    ref, bound = R.dropout(R.f64(x), p, seed, call, R.f64(r) if residual else None)
    R.check(out, ref, bound, "out")
    grads = torch.autograd.grad(out, [x] + ([r] if residual else []), g)
    ref, bound = R.dropout(R.f64(g), p, seed, call)
    R.check(grads[0], ref, bound, "grad")
    if residual:
        assert torch.equal(grads[1], g)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_mask_values_and_layouts(dtype):
    """The mask goes by the element's index in row-major order whatever the layout, and a dropped infinity or NaN
    leaves zero."""
    big = randn(200, 131, seed=4, dtype=dtype)
    keep = R.keep_mask((200, 130), 0.3, 11, 4)
    for x in (big[:, 1:], big[:, :130], torch.empty(130, 200, dtype=dtype, device=DEV).normal_(generator=gen(5)).t()):
        R.check(x_b200.dropout(x, 0.3, 11, 4), *R.dropout(R.f64(x), 0.3, 11, 4))
    flat = big.view(-1)[1:26001]  # not aligned to the vector width
    R.check(x_b200.dropout(flat, 0.3, 11, 4, residual=big.view(-1)[3:26003]),
            *R.dropout(R.f64(flat), 0.3, 11, 4, R.f64(big.view(-1)[3:26003])))
    x = torch.full((200, 130), float("inf"), dtype=dtype, device=DEV)
    x[::2] = float("nan")
    y = x_b200.dropout(x, 0.3, 11, 4).cpu()
    assert (y[torch.from_numpy(~keep)] == 0).all() and not torch.isfinite(y[torch.from_numpy(keep)]).any()
    ones = torch.ones(1 << 20, device=DEV)
    kept = (x_b200.dropout(ones, 0.3, 11, 5) != 0).float().mean().item()
    assert abs(kept - 0.7) < 6 * (0.21 / 2**20) ** 0.5  # six standard deviations
    assert not torch.equal(x_b200.dropout(ones, 0.3, 11, 5), x_b200.dropout(ones, 0.3, 12, 5))
    assert not torch.equal(x_b200.dropout(ones, 0.3, 11, 5), x_b200.dropout(ones, 0.3, 11, 6))
    d = RNG.DeviceDraws(11)
    assert torch.equal(x_b200.dropout(ones, 0.3, d.seed, d.next_call()), x_b200.dropout(ones, 0.3, 11, 0))


def test_dropout_refuses():
    x = torch.zeros(8, device=DEV)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            x_b200.dropout(x, p, 0)
    with pytest.raises(ValueError):
        x_b200.dropout(x, 0.1, 0, residual=x[:4])
    with pytest.raises(ValueError):
        x_b200.dropout(x, 0.1, 0, residual=x.half())
    with pytest.raises(ValueError):
        x_b200.dropout(x, 0.1, 0, call=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError):
        x_b200.dropout(x, 0.1, 0, call=torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError):
        x_b200.dropout(x.double(), 0.1, 0)


def test_dropout_draws_anew_in_a_captured_graph():
    x = randn(5000, seed=6).requires_grad_()
    g = randn(5000, seed=7)
    call = torch.zeros(1, dtype=torch.int64, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x_b200.dropout(x, 0.4, 3, call)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x_b200.dropout(x, 0.4, 3, call)
        (gx,) = torch.autograd.grad(y, [x], g)
        call.add_(1)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        R.check(y, *R.dropout(R.f64(x), 0.4, 3, step))
        R.check(gx, *R.dropout(R.f64(g), 0.4, 3, step))


# ------------------------------------------------------------------------------------------------ recurrence
def windows(N, B, seed, pads):
    """Packed windows of random lengths, some empty; with pads, rows of no window (-1 and B) between them."""
    rng = np.random.default_rng(seed)
    cut = np.sort(rng.integers(0, N + 1, B - 1)) if B > 1 else np.array([], int)
    b = np.searchsorted(cut, np.arange(N), side="right").astype(np.int64)
    if pads:
        for w in range(B):
            rows = np.nonzero(b == w)[0]
            if len(rows) > 2:
                b[rows[-(1 + rng.integers(0, min(3, len(rows) - 1))):]] = -1 if w % 2 else B
    return b


def run_recurrence(kind, gate, x, b, B, h0, gh, ghT):
    leaves = [gate, x] + ([h0] if h0 is not None else [])
    h, st = x_b200.linear_recurrence(gate, x, b=b, B=B, h0=h0, kind=kind, return_state=True)
    outs, gs = [h], [gh]
    if ghT is not None:
        outs, gs = outs + [st], gs + [ghT]
    return (h, st, *torch.autograd.grad(outs, leaves, gs))


def compare_recurrence(kind, gate, x, b, B, h0, gh, ghT, got):
    N = x.shape[0]
    bn = b.cpu().numpy() if b is not None else np.repeat(np.arange(B), N // B)
    f = lambda t: None if t is None else R.f64(t)  # noqa: E731
    with np.errstate(all="ignore"):
        r = R.recurrence(kind, f(gate), f(x), bn, B, f(h0), f(gh), f(ghT))
    for name, t in zip(["h", "state", "dgate", "dx", "dh0"], got):
        R.check(t, *r[name], name)


def gates(kind, N, D, dtype, seed):
    z = randn(N, D, seed=seed, scale=1.5)
    return (z + 1.0).to(dtype) if kind == "sigmoid" else (torch.sigmoid(z + 2.0) * torch.sign(z + 2.5)).to(dtype)


@pytest.mark.parametrize("N,B,D", [(1, 1, 1), (2, 1, 33), (31, 3, 2), (128, 1, 64), (129, 2, 100), (300, 7, 31),
                                   (1000, 40, 8), (1000, 1, 130), (4097, 5, 5), (3000, 3000, 6)])
@pytest.mark.parametrize("kind", ["sigmoid", "decay"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pads", [False, True])
def test_recurrence_packed(N, B, D, kind, dtype, pads):
    b = torch.from_numpy(windows(N, B, N + D, pads)).to(DEV)
    gate, x = gates(kind, N, D, dtype, 1), randn(N, D, seed=2, dtype=dtype)
    gh = randn(N, D, seed=3, dtype=dtype)
    if pads:  # what rows of no window hold reaches nothing
        out = (b < 0) | (b >= B)
        gate[out], x[out], gh[out] = float("nan"), float("inf"), float("nan")
    gate.requires_grad_(), x.requires_grad_()
    state = N % 2 == 0
    h0 = randn(B, D, seed=4).requires_grad_() if state else None
    ghT = randn(B, D, seed=5) if state else None
    got = run_recurrence(kind, gate, x, b, B, h0, gh, ghT)
    compare_recurrence(kind, gate, x, b, B, h0, gh, ghT, got)
    again = run_recurrence(kind, gate, x, b, B, h0, gh, ghT)
    assert all(same_bits(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("B,T,D", [(3, 1, 40), (64, 1, 256), (4, 250, 17), (1, 2048, 24), (5, 128, 64)])
@pytest.mark.parametrize("kind", ["sigmoid", "decay"])
@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_equal_windows(B, T, D, kind, dtype):
    N = B * T
    gate, x = gates(kind, N, D, dtype, 1).requires_grad_(), randn(N, D, seed=2, dtype=dtype).requires_grad_()
    h0, ghT = randn(B, D, seed=4).requires_grad_(), randn(B, D, seed=5)
    gh = randn(N, D, seed=3, dtype=dtype)
    got = run_recurrence(kind, gate, x, None, B, h0, gh, ghT)
    compare_recurrence(kind, gate, x, None, B, h0, gh, ghT, got)
    b = torch.arange(B, device=DEV).repeat_interleave(T)
    assert all(same_bits(p, q) for p, q in zip(got, run_recurrence(kind, gate, x, b, B, h0, gh, ghT)))


@pytest.mark.parametrize("kind", ["sigmoid", "decay"])
@pytest.mark.parametrize("N,D", [(40001, 3), (70000, 2)])
def test_recurrence_long(kind, N, D):
    """Long memories over many chunks: gates near one."""
    gate = randn(N, D, seed=1)
    gate = (gate + 6.0 if kind == "sigmoid" else 1.0 - 2.0 ** -9 * torch.rand(N, D, generator=gen(1), device=DEV))
    gate.requires_grad_()
    x, gh = randn(N, D, seed=2).requires_grad_(), randn(N, D, seed=3)
    b = torch.from_numpy(windows(N, 3, 7, False)).to(DEV)
    got = run_recurrence(kind, gate, x, b, 3, None, gh, None)
    compare_recurrence(kind, gate, x, b, 3, None, gh, None, got)


@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_layouts(dtype):
    """Column slices of one projection (aligned and not), a gate shared by all rows or columns, an expanded gradient."""
    N, D, B = 500, 24, 3
    b = torch.from_numpy(windows(N, B, 1, True)).to(DEV)
    for off in (0, 1, 8):
        proj = randn(N, 2 * D + 9, seed=off, dtype=dtype).requires_grad_()
        gate, x = proj[:, off:off + D], proj[:, off + D:off + 2 * D]
        gh = randn(N, D + 3, seed=3, dtype=dtype)[:, off % 3:off % 3 + D]
        h = x_b200.linear_recurrence(gate, x, b=b, B=B)
        (gp,) = torch.autograd.grad(h, [proj], gh)
        compare_recurrence("sigmoid", gate, x, b, B, None, gh, None,
                           (h, x_b200.linear_recurrence(gate, x, b=b, B=B, return_state=True)[1],
                            gp[:, off:off + D], gp[:, off + D:off + 2 * D]))
    x = randn(N, D, seed=8, dtype=dtype).requires_grad_()
    for shape in ((1, D), (N, 1), (1, 1)):
        small = gates("decay", *shape, dtype, 5).requires_grad_()
        gate = small.expand(N, D)
        h = x_b200.linear_recurrence(gate, x, b=b, B=B, kind="decay")
        gx, gs = torch.autograd.grad(h.float().sum(), [x, small])
        r = R.recurrence("decay", R.f64(gate), R.f64(x), b.cpu().numpy(), B, None, np.ones((N, D)))
        R.check(h, *r["h"])
        R.check(gx, *r["dx"])
        # torch sums the rounded gradients of the shared gate: each off by its tolerance, the sum by N D roundings
        # in fp32 and one to the gate's type
        axes = tuple(i for i, n in enumerate(shape) if n == 1)
        dg, bd = r["dgate"]
        each = R.tol(dg, bd, dtype)
        bound = each.sum(axes, keepdims=True) + N * D * R.U * (np.abs(dg) + each).sum(axes, keepdims=True)
        R.check(gs, dg.sum(axes, keepdims=True), bound)


def test_recurrence_values():
    """NaN and infinities stay in their window and column; a large gate on a zero state leaves it zero; h0 alone."""
    N, D = 600, 4
    b = torch.from_numpy(np.repeat([0, 1, 2], 200)).to(DEV)
    gate, x = gates("decay", N, D, torch.float32, 1), randn(N, D, seed=2)
    clean = x_b200.linear_recurrence(gate, x, b=b, B=3, kind="decay")
    x2 = x.clone()
    x2[250, 1], x2[300, 2] = float("nan"), float("inf")
    h = x_b200.linear_recurrence(gate, x2, b=b, B=3, kind="decay")
    mask = torch.zeros(N, D, dtype=torch.bool, device=DEV)
    mask[250:400, 1], mask[300:400, 2] = True, True
    assert same_bits(h[~mask], clean[~mask])
    assert not torch.isfinite(h[250:400, 1]).any()
    zero = x_b200.linear_recurrence(torch.full((N, D), 8.0, device=DEV), torch.zeros(N, D, device=DEV), kind="decay")
    assert (zero == 0).all()
    h0 = randn(3, D, seed=9)
    h, st = x_b200.linear_recurrence(gate[:0], x[:0], b=b[:0], B=3, h0=h0, return_state=True)
    assert h.shape == (0, D) and same_bits(st, h0)
    assert x_b200.linear_recurrence(gate[:, :0], x[:, :0], b=b, B=3).shape == (N, 0)
    empty = x[:0].clone().requires_grad_()
    h, st = x_b200.linear_recurrence(gate[:0], empty, b=b[:0], B=3, h0=h0.requires_grad_(), return_state=True)
    assert same_bits(torch.autograd.grad(st, [h0], x[:3])[0], x[:3])


@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_saturated_gates(dtype):
    """A gate of +inf (or far above) keeps the state, one of -inf (or far below) takes x, both to the bit; no NaN in the
    gradients."""
    N, D = 70, 8
    big = 200.0 if dtype == torch.float16 else 1e4
    gate = torch.empty(N, D, dtype=dtype, device=DEV)
    gate[0], gate[1:40], gate[40:] = -big, big, -float("inf")
    gate[5], gate[41] = float("inf"), -big
    gate.requires_grad_()
    x = randn(N, D, seed=1, dtype=dtype).requires_grad_()
    h = x_b200.linear_recurrence(gate, x)
    assert torch.equal(h[:40], x[:1].expand(40, D)) and torch.equal(h[40:], x[40:])
    gg, gx = torch.autograd.grad(h.float().sum(), [gate, x])
    assert torch.isfinite(gg).all() and torch.isfinite(gx).all()
    assert torch.equal(gx[40:], torch.ones_like(gx[40:])) and (gx[1:40] == 0).all()


@pytest.mark.parametrize("kind", ["sigmoid", "decay"])
def test_recurrence_step_by_step(kind):
    """A window read whole, in two parts and row by row, the state handed on, gives the same states up to rounding."""
    B, T, D = 3, 40, 70
    gate, x = gates(kind, B * T, D, torch.float32, 1), randn(B * T, D, seed=2)
    whole, end = x_b200.linear_recurrence(gate, x, B=B, kind=kind, return_state=True)
    r = R.recurrence(kind, R.f64(gate), R.f64(x), np.repeat(np.arange(B), T), B)
    g3, x3, st, rows = gate.view(B, T, D), x.view(B, T, D), None, []
    for t in range(T):
        h, st = x_b200.linear_recurrence(g3[:, t], x3[:, t], B=B, h0=st, kind=kind, return_state=True)
        rows.append(h)
    R.check(torch.stack(rows, 1).reshape(B * T, D), *r["h"])
    R.check(st, *r["state"])
    R.check(whole, *r["h"])
    R.check(end, *r["state"])


def test_recurrence_refuses():
    x = torch.zeros(6, 4, device=DEV)
    b = torch.zeros(6, dtype=torch.long, device=DEV)
    f = x_b200.linear_recurrence
    for bad in (lambda: f(x, x[:, :2]), lambda: f(x.half(), x), lambda: f(x, x, kind="gru"), lambda: f(x, x, B=4),
                lambda: f(x, x, B=0), lambda: f(x[0], x[0]), lambda: f(x, x, b=b[:3]),
                lambda: f(x, x, b=b, B=2, h0=x[:1]), lambda: f(x, x, b=b, B=-1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(x.double(), x.double()), lambda: f(x, x, b=b.int()), lambda: f(x, x, b=b.cpu()),
                lambda: f(x, x, h0=x[:1].half()), lambda: f(x.cpu(), x)):
        with pytest.raises(RuntimeError):
            bad()


# ------------------------------------------------------------------------------------------------ streams, graphs
def test_operators_on_another_stream_and_in_graphs():
    """On a side stream, and captured twice with replays in turn, the three operators give the bits of a plain call."""
    N, V, D, B = 9000, 700, 48, 4
    w, idx, g = lookup_inputs(N, V, D, torch.bfloat16, 1, "skew")
    gate = gates("sigmoid", N, D, torch.bfloat16, 3)
    b = torch.from_numpy(windows(N, B, 2, True)).to(DEV)
    h0 = randn(B, D, seed=5)
    leaves = [w.requires_grad_(), gate.requires_grad_(), h0.requires_grad_()]

    def step():
        x = x_b200.dropout(x_b200.embedding(w, idx, 1.5), 0.2, 5, 6)
        h, st = x_b200.linear_recurrence(gate, x, b=b, B=B, h0=h0, return_state=True)
        # detached: a capture may not meet a living eager graph of the same leaves
        return (h.detach(), st.detach(), *torch.autograd.grad([h, st], leaves, [g, st.detach()]))

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(same_bits(p, q) for p, q in zip(ref, other))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for _ in range(2):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(same_bits(p, q) for p, q in zip(ref, o))


def test_operators_from_two_threads():
    """Calls from two threads, each on its own stream, give the bits of calls one after the other."""
    import threading
    args = []
    for k in range(2):
        w, idx, g = lookup_inputs(20000, 900, 64, torch.float32, 40 + k, "skew")
        args.append((w.requires_grad_(), idx, g, gates("sigmoid", 20000, 64, torch.float32, 50 + k)))

    def step(w, idx, g, gate):
        h = x_b200.linear_recurrence(gate, x_b200.dropout(x_b200.embedding(w, idx), 0.3, 1, 2), B=4)
        return h.detach(), torch.autograd.grad(h, [w], g)[0]

    ref, out = [step(*a) for a in args], [[], []]
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                out[k].append(step(*args[k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(out[k]) == 5
        for o in out[k]:
            assert all(same_bits(p, q) for p, q in zip(ref[k], o))


# ------------------------------------------------------------------------------------------------ offsets past 32 bits
def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows, whose offsets do not fit 32 bits, against the float64 statements."""
    N, D, dtype = 35_000_000, 64, torch.bfloat16
    assert N * D > 2**31
    # dropout: elements near the end
    x = torch.zeros(N, D, dtype=dtype, device=DEV)
    tail = slice(N - 16, N)
    x[tail] = randn(16, D, seed=1, dtype=dtype)
    y = x_b200.dropout(x, 0.4, 9, 3)
    keep = (R.philox_words(16 * D, 9, 3, start=(N - 16) * D) >= np.uint64(np.floor(0.4 * 2.0**32 + 0.5))).reshape(16, D)
    ref = np.where(keep, R.f64(x[tail]) / 0.6, 0.0)
    R.check(y[tail], ref, 2 * R.U * np.abs(ref))
    del y
    # recurrence: a short last window behind one long one
    b = torch.zeros(N, dtype=torch.long, device=DEV)
    b[tail] = 1
    gate = torch.zeros(N, D, dtype=dtype, device=DEV)
    gate[tail] = gates("sigmoid", 16, D, dtype, 2)
    gate.requires_grad_(), x.requires_grad_()
    h, st = x_b200.linear_recurrence(gate, x, b=b, B=2, return_state=True)
    g_state = randn(2, D, seed=3)
    gg, gx = torch.autograd.grad(st, [gate, x], g_state)
    r = R.recurrence("sigmoid", R.f64(gate[tail]), R.f64(x[tail]), np.zeros(16, int), 1, None, np.zeros((16, D)),
                     R.f64(g_state[1:]))
    R.check(h[tail], *r["h"])
    R.check(st[1:], *r["state"])
    R.check(gg[tail], *r["dgate"])
    R.check(gx[tail], *r["dx"])
    del h, st, gate, gg, gx, b
    # lookup: the output's last rows, and their gradients (x as the incoming one)
    w = randn(3, D, seed=4, dtype=dtype).requires_grad_()
    idx = torch.full((N,), -1, device=DEV)
    idx[tail] = torch.arange(16, device=DEV) % 3
    out = x_b200.embedding(w, idx, 0.5)
    (gw,) = torch.autograd.grad(out, [w], x.detach())
    fwd, bwd = R.embedding(R.f64(w), idx[tail].cpu().numpy(), 0.5, R.f64(x[tail]))
    R.check(out[tail], *fwd)
    R.check(gw, *bwd)


# ------------------------------------------------------------------------------------------------ together
def test_event_sequence_model_under_the_objective():
    """Events looked up by pixel, dropped out, run through the recurrence; its end states give each window's motion,
    which AnchoredExact scores.  The gradients of both tables from the objective's gradient at the states are those of
    the float64 statements chained by hand."""
    from x_b200 import motion as Mo
    from x_b200 import synth
    from x_b200.objectives import AnchoredExact
    B, H, W, D, n = 2, 48, 60, 16, 3000
    ev = synth.textured_window(n, H, W, seed=3, batch=B, device=DEV)
    N = ev.n
    pix = (ev.xy[:, 1] * W + ev.xy[:, 0]).long()
    tx, tg = randn(H * W, D, seed=1).requires_grad_(), randn(H * W, D, seed=2).requires_grad_()
    head = randn(D, 2, seed=4, scale=0.5)
    draws = RNG.DeviceDraws(8)
    x = x_b200.dropout(x_b200.embedding(tx, pix), 0.25, draws.seed, draws.next_call())
    gate = x_b200.embedding(tg, pix)
    h, state = x_b200.linear_recurrence(gate, x, b=ev.b, B=B, return_state=True)
    coeff = (state @ head).view(B, 2, 1, 1).expand(B, 2, H, W)
    obj = AnchoredExact(h=1.0, n_anchors=None, seed=5)
    loss = obj(ev, Mo.PixelTrajectories(coeff, K=1))["loss"]
    gst, gx, gg = torch.autograd.grad(loss, [state, tx, tg])
    assert torch.isfinite(gst).all() and gst.abs().max() > 0
    # by hand: dropout scales x by 1 / 0.75 with three roundings (table, scale, product)
    keep = R.keep_mask((N, D), 0.25, 8, 0) / 0.75
    xs, gs = R.f64(tx)[pix.cpu().numpy()] * keep, R.f64(tg)[pix.cpu().numpy()]
    r = R.recurrence("sigmoid", gs, xs, ev.b.cpu().numpy(), B, None, np.zeros((N, D)), R.f64(gst), xerr=3.0)
    R.check(state, *r["state"], "state")
    for got, (val, bound), k in ((gx, r["dx"], keep), (gg, r["dgate"], 1.0)):
        val, bound = val * k, bound * k + 4 * R.U * np.abs(val * k)
        grad, err, mag, cnt = (np.zeros((H * W, c)) for c in (D, D, D, 1))
        for acc, v in ((grad, val), (err, bound), (mag, np.abs(val)), (cnt, np.ones((N, 1)))):
            np.add.at(acc, pix.cpu().numpy(), v)
        R.check(got, grad, err + (cnt + 1) * R.U * mag, "table")
