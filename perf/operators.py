"""The event-sequence operators, measured: table lookup of events, counter-based dropout, gated linear recurrence.

Each case runs one pass of one operator.  ``run`` computes it in elementary torch operations, or, where ``own`` is
true, through the public entry points of x_b200.  Sizes follow the benchmark configurations: 100k events on a
240x180 sensor, 1M on 640x480, windows of 2M, sweeps of 4M.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------ cases
def _embed(N, V, D, dtype, train):
    return {"op": "embedding", "N": N, "V": V, "D": D, "dtype": dtype, "train": train}


def _drop(N, D, dtype, p, residual, train):
    return {"op": "dropout", "N": N, "D": D, "dtype": dtype, "p": p, "residual": residual, "train": train}


def _rec(N, B, D, dtype, kind, packed, state, train):
    return {"op": "recurrence", "N": N, "B": B, "D": D, "dtype": dtype, "kind": kind, "packed": packed,
            "state": state, "train": train}


def listed():
    return [
        # a few events that just arrived, their pixels' feature rows read: latency
        {"name": "embed_step", **_embed(48, 640 * 480, 64, "bf16", False)},
        # the rows of a small window on a 240x180 sensor, trained
        {"name": "embed_100k", **_embed(100_000, 240 * 180, 32, "f32", True)},
        # one window on a 640x480 sensor, one learned row per pixel, trained
        {"name": "embed_1m", **_embed(1_000_000, 640 * 480, 64, "bf16", True)},
        # rows by polarity and time bin: a handful of rows that every event of the window shares
        {"name": "embed_bins_4m", **_embed(4_000_000, 33, 96, "f16", True)},
        # one odd-sized activation row: latency
        {"name": "drop_row", **_drop(1, 1025, "f32", 0.1, False, False)},
        # activations of one window, trained
        {"name": "drop_1m", **_drop(1_000_000, 64, "bf16", 0.1, False, True)},
        # a residual branch over a 2M-event window with an odd count, trained
        {"name": "drop_res_2m", **_drop(2_000_003, 48, "f32", 0.25, True, True)},
        # one new event in each of 64 windows, states kept between calls: latency
        {"name": "rec_step", **_rec(64, 64, 256, "bf16", "sigmoid", False, True, False)},
        # one small window of decaying traces, trained
        {"name": "rec_100k", **_rec(100_000, 1, 32, "f32", "decay", False, False, True)},
        # a batch of eight ragged windows packed one behind the other, with initial states, trained
        {"name": "rec_1m", **_rec(1_000_000, 8, 64, "bf16", "sigmoid", True, True, True)},
        # equal windows of 2048 tokens with wide features, trained
        {"name": "rec_wide", **_rec(16 * 2048, 16, 1024, "bf16", "sigmoid", False, False, True)},
        # one long window read through without training
        {"name": "rec_4m", **_rec(4_000_000, 1, 64, "f16", "sigmoid", False, False, False)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "dropout", "recurrence"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.7
    D = rng.choice([_log_int(rng, 1, 1024), 8 * _log_int(rng, 1, 64), rng.choice([32, 64, 128, 256])])
    cap = max(1, (64_000_000 if dtype == "f32" else 128_000_000) // D)
    N = _log_int(rng, 1, min(4_000_000, cap))
    if op == "embedding":
        return _embed(N, _log_int(rng, 1, min(640 * 480, cap)), D, dtype, train)
    if op == "dropout":
        return _drop(N, D, dtype, rng.choice([0.1, 0.25, 0.5, round(rng.uniform(0.0, 0.9), 3)]), rng.random() < 0.5,
                     train)
    packed = rng.random() < 0.5
    B = min(_log_int(rng, 1, 64), N)
    if not packed:
        N = N // B * B
    return _rec(N, B, D, dtype, rng.choice(["sigmoid", "decay"]), packed, rng.random() < 0.5, train)


# ------------------------------------------------------------------------------------------------ inputs
def _window_index(case, g):
    """Sorted window numbers of N packed events, ragged, with a few rows that belong to none (-1) at the end."""
    N, B = case["N"], case["B"]
    pad = min(N // 1000, 100)
    w = torch.rand(B, generator=g, device="cuda", dtype=torch.float64) + 0.1
    edges = (torch.cumsum(w, 0) / w.sum() * (N - pad)).round().long()
    b = torch.searchsorted(edges, torch.arange(N, device="cuda"), right=True)
    return torch.where(b < B, b, -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = DT[case["dtype"]], "cuda"
    N, D = case["N"], case["D"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).add_(shift).to(dtype)

    st = {"case": case}
    if case["op"] == "embedding":
        V = case["V"]
        # textured scenes: some rows are read far more often than others, and some events lie outside the image
        w = torch.randn(V, generator=g, device=dev).square_().add_(1e-4)
        cdf = torch.cumsum(w.double(), 0)
        u = torch.rand(N, generator=g, device=dev, dtype=torch.float64) * cdf[-1]
        idx = torch.searchsorted(cdf, u).clamp_(max=V - 1)
        idx[torch.rand(N, generator=g, device=dev) < 0.001] = -1
        st.update(weight=normal(V, D, scale=0.02), idx=idx, scale=math.sqrt(D))
        if case["train"]:
            st["weight"].requires_grad_()
            st["g"] = normal(N, D, scale=0.01)
    elif case["op"] == "dropout":
        st.update(x=normal(N, D), p=case["p"], seed=1000003 * seed + 17, call=seed % 1000)
        if case["residual"]:
            st["residual"] = normal(N, D)
        if case["train"]:
            st["x"].requires_grad_()
            if case["residual"]:
                st["residual"].requires_grad_()
            st["g"] = normal(N, D)
    else:
        B = case["B"]
        if case["kind"] == "sigmoid":
            gate = normal(N, D, scale=1.5, shift=2.0)
        else:
            # exp(-dt / tau): gaps between events, one time constant per channel, of 8 to 4096 mean gaps
            # (8 to 64 in 16 bits, which hold no longer ones)
            gap = torch.empty(N, 1, device=dev).exponential_(generator=g)
            span = math.log(512.0 if case["dtype"] == "f32" else 8.0)
            rate = torch.exp(-torch.rand(1, D, generator=g, device=dev) * span) / 8.0
            gate = torch.exp(-gap * rate).to(dt)
        st.update(gate=gate, x=normal(N, D), B=B)
        if case["packed"]:
            st["b"] = _window_index(case, g)
        if case["state"]:
            st["h0"] = normal(B, D, dtype=torch.float32)
        if case["train"]:
            for k in ("gate", "x", "h0"):
                if k in st:
                    st[k].requires_grad_()
            st["g"] = normal(N, D)
            if case["state"]:
                st["g_state"] = normal(B, D, dtype=torch.float32)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _embedding_plain(st):
    c, w, idx, s = st["case"], st["weight"].detach(), st["idx"], st["scale"]
    ok = (idx >= 0) & (idx < c["V"])
    safe = torch.where(ok, idx, 0)
    out = torch.where(ok[:, None], w[safe].float() * s, 0.0).to(w.dtype)
    if not c["train"]:
        return out
    acc = torch.float64 if c["N"] > 256 * c["V"] else torch.float32  # sums over many thousand rows
    gw = torch.zeros(c["V"] + 1, c["D"], dtype=acc, device=w.device)
    gw.index_add_(0, torch.where(ok, idx, c["V"]), st["g"].to(acc))
    return out, (gw[:-1] * s).to(w.dtype)


def _philox_keep(n, p, seed, call, device):
    """keep[i] for i < n: word i % 4 of Philox4x32-10 at counter (i // 4, 2^31 + (i // 4 >> 32), call) under the
    key seed, compared with p 2^32."""
    q = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = q & MASK32, (q >> 32) | 0x80000000
    c2, c3 = torch.full_like(q, call & MASK32), torch.full_like(q, call >> 32 & MASK32)
    k0, k1 = seed & MASK32, seed >> 32 & MASK32

    def mul(m, x):  # 32 x 32 -> high and low words, in halves that stay inside 63 bits
        lo = (x & 0xFFFF) * m
        hi = (x >> 16) * m + (lo >> 16)
        return hi >> 16, (hi & 0xFFFF) << 16 | lo & 0xFFFF

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = k0 + 0x9E3779B9 & MASK32, k1 + 0xBB67AE85 & MASK32
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n] >= int(math.floor(p * 2.0 ** 32 + 0.5))


def _dropout_plain(st):
    x, p = st["x"].detach(), st["p"]
    keep = _philox_keep(x.numel(), p, st["seed"], st["call"], x.device).view(x.shape)
    s = 1.0 / (1.0 - p)
    out = torch.where(keep, x.float() * s, 0.0)
    if "residual" in st:
        out = out + st["residual"].detach().float()
    out = out.to(x.dtype)
    if not st["case"]["train"]:
        return out
    gx = torch.where(keep, st["g"].float() * s, 0.0).to(x.dtype)
    return (out, gx, st["g"]) if "residual" in st else (out, gx)


def _scan_plain(a, x):
    """h_t = a_t h_(t-1) + x_t along the first axis, by doubling: after step k every row holds 2^k rows' map."""
    a, x = a.clone(), x.clone()
    d = 1
    while d < a.shape[0]:
        x[d:] = x[d:] + a[d:] * x[:-d]
        a[d:] = a[d:] * a[:-d]
        d *= 2
    return x


def _bounds(st):
    """Window of every row (-1: none) and the flags of a window's first and last rows."""
    c, dev = st["case"], st["x"].device
    b = st["b"] if "b" in st else torch.arange(c["N"], device=dev) // (c["N"] // c["B"])
    edge = torch.ones(1, dtype=torch.bool, device=dev)
    change = b[1:] != b[:-1]
    return b, torch.cat([edge, change]), torch.cat([change, edge])


def _recurrence_plain(st):
    c, x0 = st["case"], st["x"].detach()
    B, D, dev = c["B"], c["D"], x0.device
    b, first, last = _bounds(st)
    ok, safe = (b >= 0)[:, None], b.clamp(min=0)
    x, gate = x0.float(), st["gate"].detach().float()
    a, w = (torch.sigmoid(gate), torch.sigmoid(-gate)) if c["kind"] == "sigmoid" else (gate, None)
    u = x * w if w is not None else x
    h0 = st["h0"].detach() if "h0" in st else torch.zeros(B, D, device=dev)
    start = torch.where(first[:, None], h0[safe], 0.0)
    u = torch.where(ok, u + a * start, 0.0)
    h = _scan_plain(torch.where(ok & ~first[:, None], a, 0.0), u)
    out = [h.to(x0.dtype)]
    if c["state"]:
        hT = h0.clone()
        sel = last & (b >= 0)
        hT[b[sel]] = h[sel]
        out.append(hT)
    if not c["train"]:
        return tuple(out) if len(out) > 1 else out[0]
    g = st["g"].float()
    if c["state"]:
        g = g + torch.where(last[:, None], st["g_state"][safe], 0.0)
    # g_t = dL/dh_t + a_(t+1) g_(t+1) inside a window: the same scan from the end
    nxt = torch.zeros_like(a)
    nxt[:-1] = torch.where(last[:-1, None], 0.0, a[1:])
    g = _scan_plain(nxt.flip(0), torch.where(ok, g, 0.0).flip(0)).flip(0)
    prev = start.clone()
    prev[1:] = torch.where(first[1:, None], start[1:], h[:-1])
    if c["kind"] == "sigmoid":
        dgate, dx = g * (prev - x) * a * w, g * w
    else:
        dgate, dx = g * prev, g
    out += [torch.where(ok, dgate, 0.0).to(x0.dtype), torch.where(ok, dx, 0.0).to(x0.dtype)]
    if c["state"]:
        dh0 = st["g_state"].clone()
        sel = first & (b >= 0)
        dh0[b[sel]] = (a * g)[sel]
        out.append(dh0)
    return tuple(out)


# ------------------------------------------------------------------------------------------------ the library
def _run_own(st):
    import x_b200
    c = st["case"]
    if c["op"] == "embedding":
        out = x_b200.embedding(st["weight"], st["idx"], st["scale"])
        if not c["train"]:
            return out
        (gw,) = torch.autograd.grad(out, [st["weight"]], st["g"])
        return out.detach(), gw
    if c["op"] == "dropout":
        out = x_b200.dropout(st["x"], st["p"], st["seed"], st["call"], residual=st.get("residual"))
        if not c["train"]:
            return out
        leaves = [st["x"]] + ([st["residual"]] if c["residual"] else [])
        return (out.detach(), *torch.autograd.grad(out, leaves, st["g"]))
    out = x_b200.linear_recurrence(st["gate"], st["x"], b=st.get("b"), B=st["B"], h0=st.get("h0"), kind=c["kind"],
                                   return_state=c["state"])
    if not c["train"]:
        return out
    if c["state"]:
        grads = torch.autograd.grad(out, [st["gate"], st["x"], st["h0"]], [st["g"], st["g_state"]])
        return (out[0].detach(), out[1].detach(), *grads)
    return (out.detach(), *torch.autograd.grad(out, [st["gate"], st["x"]], st["g"]))


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"embedding": _embedding_plain, "dropout": _dropout_plain,
                "recurrence": _recurrence_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    s, N, D = SIZE[case["dtype"]], case["N"], case["D"]
    n = N * D
    if case["op"] == "embedding":
        V = case["V"]
        by, fl = 8 * N + min(N, V) * D * s + n * s, n
        if case["train"]:
            by, fl = by + n * s + V * D * s, fl + 2 * n
    elif case["op"] == "dropout":
        by, fl = n * s * (3 if case["residual"] else 2), n * (2 if case["residual"] else 1)
        if case["train"]:
            # the residual's gradient is the incoming gradient itself
            by, fl = by + 2 * n * s, fl + n
    else:
        by, fl = 3 * n * s, (6 if case["kind"] == "sigmoid" else 2) * n
        if case["packed"]:
            by += 8 * N
        if case["state"]:
            by += 8 * case["B"] * D
        if case["train"]:
            by, fl = by + 3 * n * s + (8 * case["B"] * D if case["state"] else 0), fl + 8 * n
    return {"bytes": by, "flops": fl}


# ------------------------------------------------------------------------------------------------ 64-bit values
def _exact_scan(a, x):
    """The recurrence row by row, in 64 bits: blocks of rows side by side, then the blocks joined in order."""
    N, D = a.shape
    L = max(1, int(math.isqrt(N)))
    K = (N + L - 1) // L
    fill = K * L - N
    if fill:
        a = torch.cat([a, a.new_zeros(fill, D)])
        x = torch.cat([x, x.new_zeros(fill, D)])
    a, x = a.view(K, L, D), x.view(K, L, D)
    h, P = torch.empty_like(x), torch.empty_like(a)
    hc, pc = torch.zeros_like(x[:, 0]), torch.ones_like(a[:, 0])
    for i in range(L):
        hc = torch.addcmul(x[:, i], a[:, i], hc)
        pc = pc * a[:, i]
        h[:, i], P[:, i] = hc, pc
    carry = torch.zeros_like(x[0, 0])
    carries = []
    for k in range(K):
        carries.append(carry)
        carry = torch.addcmul(h[k, -1], P[k, -1], carry)
    h.addcmul_(P, torch.stack(carries)[:, None, :])
    return h.view(K * L, D)[:N]


def _exact_keep(n, p, seed, call):
    u64, m = np.uint64, np.uint64(MASK32)
    q = np.arange((n + 3) // 4, dtype=np.uint64)
    x = [q & m, (q >> u64(32)) | u64(1 << 31), np.full_like(q, call & MASK32), np.full_like(q, call >> 32 & MASK32)]
    key = [seed & MASK32, seed >> 32 & MASK32]
    for _ in range(10):
        p0, p1 = x[0] * u64(0xD2511F53), x[2] * u64(0xCD9E8D57)
        x = [(p1 >> u64(32)) ^ x[1] ^ u64(key[0]), p1 & m, (p0 >> u64(32)) ^ x[3] ^ u64(key[1]), p0 & m]
        key = [(key[0] + 0x9E3779B9) & MASK32, (key[1] + 0xBB67AE85) & MASK32]
    words = np.empty((q.size, 4), dtype=np.uint32)
    for j in range(4):
        words[:, j] = x[j]
    return words.reshape(-1)[:n].astype(np.float64) >= np.floor(p * 2.0 ** 32 + 0.5)


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    with torch.no_grad():
        if case["op"] == "embedding":
            V = case["V"]
            table = torch.cat([st["weight"].to(f64) * st["scale"], torch.zeros(1, case["D"], dtype=f64, device="cuda")])
            row = torch.where((st["idx"] < 0) | (st["idx"] >= V), V, st["idx"])
            out = table.index_select(0, row)
            if not case["train"]:
                return out
            grad = torch.zeros_like(table).index_put_((row,), st["g"].to(f64), accumulate=True)
            return out, grad[:V] * st["scale"]
        if case["op"] == "dropout":
            x = st["x"].to(f64)
            keep = _exact_keep(x.numel(), case["p"], st["seed"], st["call"])
            m = torch.from_numpy(keep).to("cuda").view(x.shape).to(f64) / (1.0 - case["p"])
            out = x * m + (st["residual"].to(f64) if case["residual"] else 0.0)
            if not case["train"]:
                return out
            res = (out, st["g"].to(f64) * m)
            return res + (st["g"].to(f64),) if case["residual"] else res
        return _exact_recurrence(case, st)


def _exact_recurrence(case, st):
    f64 = torch.float64
    N, B, D = case["N"], case["B"], case["D"]
    b = st["b"] if "b" in st else torch.arange(B, device="cuda").repeat_interleave(N // B)
    x, z = st["x"].to(f64), st["gate"].to(f64)
    if case["kind"] == "sigmoid":
        a = 1.0 / (1.0 + torch.exp(-z))
        k = 1.0 / (1.0 + torch.exp(z))  # 1 - a without the cancellation
    else:
        a, k = z, torch.ones_like(z)
    # lengths and offsets of the windows; rows of no window stand behind the last one
    length = torch.bincount(b[b >= 0], minlength=B)
    end = torch.cumsum(length, 0)
    begin = end - length
    used = int(end[-1])
    full = length > 0
    h0 = st["h0"].to(f64) if case["state"] else torch.zeros(B, D, dtype=f64, device="cuda")
    u = k[:used] * x[:used]
    t0 = begin[full]
    u[t0] += a[t0] * h0[full]
    inner = a[:used].clone()
    inner[t0] = 0.0
    h = torch.zeros_like(x)
    h[:used] = _exact_scan(inner, u)
    res = [h]
    if case["state"]:
        hT = h0.clone()
        hT[full] = h[end[full] - 1]
        res.append(hT)
    if not case["train"]:
        return tuple(res) if len(res) > 1 else res[0]
    dh = st["g"][:used].to(f64)
    if case["state"]:
        dh[end[full] - 1] += st["g_state"].to(f64)[full]
    back = torch.zeros_like(inner)
    back[1:] = inner.flip(0)[:-1]
    g = torch.zeros_like(x)
    g[:used] = _exact_scan(back, dh.flip(0)).flip(0)
    before = torch.zeros_like(x)
    before[1:] = h[:-1]
    before[t0] = h0[full]
    if case["kind"] == "sigmoid":
        res += [g * (before - x) * a * k, g * k]
    else:
        res += [g * before, g]
    if case["state"]:
        d0 = st["g_state"].to(f64).clone()
        d0[full] = a[t0] * g[t0]
        res.append(d0)
    return tuple(res)
