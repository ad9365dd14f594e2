"""Plain float64 statements of the event-sequence operators (x_b200/sequence.py), row by row, each with the largest
error that fp32 arithmetic on the same inputs can make.

U = 2^-24 is half a step of fp32, relative to the value.  A bound counts every rounding on the way to an element: a
sum of k terms in any order is off by at most k U times the sum of the magnitudes, a product by U, and an input that
carries a relative error r passes r times its magnitude on.  ``tol`` adds the one rounding of the output to its type."""
import numpy as np
import torch

U = 2.0 ** -24
# Below 2^-126 a rounding to fp32 is off by up to 2^-150 instead of U of the value.  No element of the tests takes a
# million (2^20) roundings, and no factor behind one exceeds one, so together these stay below 2^20 2^-150.
UNDERFLOW = 2.0 ** -130


def f64(t):
    return t.detach().cpu().double().numpy()


def tol(ref, bound, dtype):
    """Largest deviation of an output of ``dtype``: the fp32 value's bound, then one rounding (half a step of the
    value, or half the smallest subnormal)."""
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bound = bound + UNDERFLOW
    return bound + half * (np.abs(ref) + bound) + tiny


def check(got, ref, bound, what=""):
    g = f64(got)
    assert g.shape == ref.shape, (what, g.shape, ref.shape)
    lim = tol(ref, bound, got.dtype)
    # from half a step above the largest number on (half a step there is eps / 4 of it: fp16 65504 + 16), a value
    # rounds to infinity; where the bound reaches that border, either answer is right
    info = torch.finfo(got.dtype)
    border = info.max * (1 + info.eps / 4)
    inf = np.isinf(g) & (np.sign(g) == np.sign(ref)) & (np.abs(ref) + bound >= border)
    bad = ~((np.abs(np.where(inf, ref, g) - ref) <= lim) & (inf | (np.abs(ref) - bound <= border)))
    assert not bad.any(), (what, int(bad.sum()), np.abs(g - ref)[bad].max(), lim[bad].max(), np.argwhere(bad)[:3].tolist())


# ------------------------------------------------------------------------------------------------ embedding
def embedding(weight, idx, scale, g=None):
    """(out, bound), and with the incoming gradient (grad, bound)."""
    V, D = weight.shape
    ok = (idx >= 0) & (idx < V)
    out = np.zeros((len(idx), D))
    out[ok] = weight[idx[ok]] * scale
    if g is None:
        return out, U * np.abs(out)
    grad, mag, cnt = np.zeros((V, D)), np.zeros((V, D)), np.zeros((V, 1))
    np.add.at(grad, idx[ok], g[ok])
    np.add.at(mag, idx[ok], np.abs(g[ok]))
    np.add.at(cnt, idx[ok], 1.0)
    return (out, U * np.abs(out)), (grad * scale, (cnt + 1) * U * mag * abs(scale))


# ------------------------------------------------------------------------------------------------ dropout
def philox_words(n, seed, call, start=0):
    """Words start .. start + n - 1 of the dropout stream (start a multiple of 4): four per counter
    (i // 4, 2^31 + (i // 4 >> 32), call)."""
    u64, m = np.uint64, np.uint64(0xFFFFFFFF)
    q = np.arange((n + 3) // 4, dtype=np.uint64) + u64(start // 4)
    c = [q & m, (q >> u64(32)) | u64(1 << 31), np.full_like(q, call & 0xFFFFFFFF), np.full_like(q, call >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(b >> u64(32)) ^ c[1] ^ u64(k[0]), b & m, (a >> u64(32)) ^ c[3] ^ u64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n]


def keep_mask(shape, p, seed, call):
    return (philox_words(int(np.prod(shape)), seed, call) >= np.uint64(int(np.floor(p * 2.0 ** 32 + 0.5)))).reshape(shape)


def dropout(x, p, seed, call, residual=None):
    """The scale is rounded once, the product once, and the sum with the residual once."""
    v = np.where(keep_mask(x.shape, p, seed, call), x / (1.0 - p) if p < 1 else 0.0, 0.0)
    if residual is None:
        return v, 2 * U * np.abs(v)
    return v + residual, 2 * U * np.abs(v) + U * np.abs(v + residual)


# ------------------------------------------------------------------------------------------------ recurrence
def sigmoid_error(kind, zmax):
    """Relative error of a and 1 - a, in U.  sigmoid: exp(-|z|), at worst by __expf with 2 + 1.173 |z| ulp, then 1 + e, its
    reciprocal (1 ulp) and the product; an ulp is at most 2 U of the value."""
    return 2 * (2 + np.floor(1.173 * zmax)) + 1 + 2 + 1 if kind == "sigmoid" else 0.0


def recurrence(kind, gate, x, b, B, h0=None, gh=None, ghT=None, xerr=0.0, zmax=None):
    """h, state and, where gh is given, dgate, dx and dh0: a dict of (value, bound).

    Per row the bound takes the state's own, scaled by a, and c U of the magnitudes' recurrence, with c counting the
    coefficient's error and the roundings of a row (product of the chunk's map, product with 1 - a, multiply-add) twice
    over, since a state may reach a row through a chunk's map and through the replay.  xerr: relative error of x and
    gate's effect on the way in, in U."""
    N, D = x.shape
    if kind == "sigmoid":
        e = np.exp(-np.abs(gate))
        a, w = np.where(gate >= 0, 1 / (1 + e), e / (1 + e)), np.where(gate >= 0, e / (1 + e), 1 / (1 + e))
    else:
        a, w = gate, np.ones_like(gate)
    ok = (b >= 0) & (b < B)
    if zmax is None:
        zmax = np.abs(gate[ok]).max() if ok.any() and kind == "sigmoid" else 0.0
    c = 2 * (sigmoid_error(kind, zmax) + 4) + xerr
    first = np.array([n == 0 or b[n] != b[n - 1] for n in range(N)], bool)
    last = np.array([n + 1 == N or b[n + 1] != b[n] for n in range(N)], bool)
    start = np.zeros((B, D)) if h0 is None else h0
    h, H, E, prev, Hp, Ep = (np.zeros((N, D)) for _ in range(6))
    state, Estate = start.copy(), np.zeros((B, D))
    for n in range(N):
        if not ok[n]:
            continue
        if first[n]:
            prev[n], Hp[n] = start[b[n]], np.abs(start[b[n]])
        else:
            prev[n], Hp[n], Ep[n] = h[n - 1], H[n - 1], E[n - 1]
        h[n] = a[n] * prev[n] + w[n] * x[n]
        H[n] = np.abs(a[n]) * Hp[n] + w[n] * np.abs(x[n])
        E[n] = np.abs(a[n]) * Ep[n] + c * U * H[n]
        if last[n]:
            state[b[n]], Estate[b[n]] = h[n], E[n]
    out = {"h": (h, E), "state": (state, Estate)}
    if gh is None:
        return out
    gT = np.zeros((B, D)) if ghT is None else ghT
    g, G, Eg = (np.zeros((N, D)) for _ in range(3))
    dh0, Edh0 = gT.copy(), np.zeros((B, D))
    u = Um = Eu = None
    for n in range(N - 1, -1, -1):
        if not ok[n]:
            continue
        if last[n]:
            u, Um, Eu = gT[b[n]], np.abs(gT[b[n]]), np.zeros(D)
        g[n], G[n], Eg[n] = gh[n] + u, np.abs(gh[n]) + Um, Eu + c * U * (np.abs(gh[n]) + Um)
        u, Um, Eu = a[n] * g[n], np.abs(a[n]) * G[n], np.abs(a[n]) * (Eg[n] + c * U * G[n])
        if first[n]:
            dh0[b[n]], Edh0[b[n]] = u, Eu
    if kind == "sigmoid":
        q = a * w
        dgate = g * (prev - x) * q
        Ed = q * (Eg * (Hp + np.abs(x)) + G * Ep + 3 * c * U * G * (Hp + np.abs(x)))
        dx, Ex = g * w, w * (Eg + c * U * G)
    else:
        dgate, Ed = g * prev, Eg * Hp + G * Ep + c * U * G * Hp
        dx, Ex = g, Eg
    z = ~ok
    for m in (dgate, Ed, dx, Ex):
        m[z] = 0.0
    out.update(dgate=(dgate, Ed), dx=(dx, Ex), dh0=(dh0, Edh0))
    return out
