"""Event-sequence operators: the front of a model whose input is the packed events themselves.

The objectives score a motion; a model that produces it from events needs, per event, a row of features
(:func:`embedding`), regularisation while it trains (:func:`dropout`) and a state that runs along each window's
events (:func:`linear_recurrence`).  All three work on the layout of the other ops of this package: one row per event,
windows packed one behind the other and sorted by (b, t), ``b`` (N,) int64.  The reference's ops have no counterpart.

float32, bfloat16 and float16; sums, states and products are held in float32 or more and every output is rounded once.  The
kernels run on the tensors' device and its current stream, allocate with torch and never synchronise, so calls can be
captured in CUDA graphs; a backward pass only while no eager autograd graph of the same leaves lives (torch ties a
leaf's gradient to the stream of its first graph, and the capture fails).  Results do not depend on the timing of a
run.  There is no CPU path, the gradients are not differentiable again, and forward-mode derivatives are refused.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

_MASK64 = 2**64 - 1
_INDEX_TYPES = (torch.int64, torch.int32, torch.int16, torch.uint8)
# The current device, and a device's current stream as an integer: a Stream object costs several microseconds to make.
# The public calls stand in where a torch build lacks the bindings.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: torch.cuda.current_stream(dev).cuda_stream)


# ------------------------------------------------------------------------------------------- arguments
# A small call is bound by the host, so the checks are made on integers, and what they refuse is put into words here.
def _device(what: str, first: str, t, **others) -> int:
    """The CUDA device that all the given tensors lie on (None is none)."""
    d = t.get_device()
    if d < 0:
        raise RuntimeError(f"x_b200.{what}: {first} must be a CUDA tensor (there is no CPU path)")
    for name, o in others.items():
        if o is not None and o.get_device() != d:
            if not o.is_cuda:
                raise RuntimeError(f"x_b200.{what}: {name} must be a CUDA tensor (there is no CPU path)")
            raise RuntimeError(f"x_b200.{what}: {name} lies on {o.device}, {first} on {t.device}")
    return d


def _dtype_code(what: str, name: str, t) -> int:
    code = L.DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"x_b200.{what}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rows(t):
    """(t, row stride) with neighbouring elements in each row of the 2-D tensor; a copy where they are not."""
    n, d = t.shape
    ld, one = t.stride()
    if d > 1 and one != 1:
        return t.contiguous(), d
    return t, ld if n > 1 else d


def _addr(t):
    return None if t is None else t.data_ptr()


def _tracked(*tensors) -> bool:
    """Does a derivative of any of the tensors (None is none) have to be tracked?  A forward-mode one as well: the autograd
    function refuses it, as it has no forward-mode formula, where the kernel alone would drop it."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside all dual levels; asking each tensor takes a microsecond
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


# ------------------------------------------------------------------------------------------- embedding
def _embedding_fwd(weight, idx, scale):
    dev = weight.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _embedding_fwd(weight, idx, scale)
    w, ldw = _rows(weight)
    V, D = w.shape
    out = w.new_empty((*idx.shape, D))
    L.check(L.load_library().atlb_embedding_fwd(L.DTYPES[w.dtype], w.data_ptr(), ldw, V, D, idx.data_ptr(), idx.numel(),
                                                scale, out.data_ptr(), _stream(dev)), "embedding")
    return out


def _embedding_bwd(g, idx, V, D, scale):
    dev = g.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _embedding_bwd(g, idx, V, D, scale)
    N, lib = idx.numel(), L.load_library()
    g, ldg = _rows(g if g.dim() == 2 else g.reshape(N, D))
    grad = g.new_empty((V, D))
    nb = lib.atlb_embedding_workspace_bytes(N, V, D)
    ws = L.workspace(nb, g.device)
    L.check(lib.atlb_embedding_bwd(L.DTYPES[g.dtype], g.data_ptr(), ldg, idx.data_ptr(), N, V, D, scale, grad.data_ptr(),
                                   ws.data_ptr(), nb, _stream(dev)), "embedding_bwd")
    return grad


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, idx, scale):
        ctx.save_for_backward(idx)
        ctx.meta = (*weight.shape, scale)
        return _embedding_fwd(weight, idx, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (idx,) = ctx.saved_tensors
        return _embedding_bwd(g, idx, *ctx.meta), None, None


def embedding(weight: torch.Tensor, idx: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """Rows of a table, scaled: ``scale * weight[idx]``, of shape ``idx.shape + (D,)``.

    weight (V, D) float32, bfloat16 or float16; idx integers of any shape.  An index outside [0, V) reads a row of
    zeros and gives no gradient, as :func:`x_b200.gather` does outside the image: events that left the sensor and
    padding (-1) need no mask.  The gradient of ``weight`` is summed over the events of each row without atomics, in an
    order that depends on the sizes and ``idx`` alone (float32 within chunks of events, float64 across them); rows that
    no event reads get zeros."""
    _device("embedding", "weight", weight, idx=idx)
    if weight.dim() != 2:
        raise ValueError(f"x_b200.embedding: weight must be (V, D), got {tuple(weight.shape)}")
    _dtype_code("embedding", "weight", weight)
    if idx.dtype not in _INDEX_TYPES:
        raise RuntimeError(f"x_b200.embedding: idx must be int64, int32, int16 or uint8, got {idx.dtype}")
    idx = idx.long().contiguous()
    if _tracked(weight):
        return _Embedding.apply(weight, idx, float(scale))
    return _embedding_fwd(weight, idx, float(scale))


# ------------------------------------------------------------------------------------------- dropout
def _dropout_run(x, residual, p, seed, call):
    """call: an integer, or a device tensor."""
    dev = x.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _dropout_run(x, residual, p, seed, call)
    x = x.contiguous()
    out = torch.empty_like(x)
    call, call_dev = (call, None) if isinstance(call, int) else (0, call.data_ptr())
    L.check(L.load_library().atlb_dropout(L.DTYPES[x.dtype], x.data_ptr(), _addr(residual), x.numel(), p, seed, call,
                                          call_dev, out.data_ptr(), _stream(dev)), "dropout")
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, call):
        ctx.meta = (p, seed, call if isinstance(call, int) else None)
        if not isinstance(call, int):
            ctx.save_for_backward(call)
        return _dropout_run(x, residual, p, seed, call)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        p, seed, call = ctx.meta
        if call is None:
            (call,) = ctx.saved_tensors
        gx = _dropout_run(g, None, p, seed, call) if ctx.needs_input_grad[0] else None
        return gx, g if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, call=0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """Dropout from the counter-based generator of :mod:`x_b200.rng`: each element of x is kept with probability
    1 - p and scaled by 1 / (1 - p), or becomes 0 whatever it held.  With ``residual`` (shape and dtype of x) the
    result is ``residual + dropout(x)``, rounded once.

    The mask is a function of (seed, call) and the element's index and is never stored: the backward pass draws it
    again.  Give every place and step that drops its own (seed, call), for instance
    ``dropout(x, p, draws.seed, draws.next_call())`` with a :class:`x_b200.rng.DeviceDraws`; the same pair gives the
    same mask, and so does every replay of a CUDA graph that captured an integer ``call``.  ``call`` may be a one-element
    int64 tensor on x's device instead, read when the kernel runs: a captured graph that adds to it after its backward
    pass drops anew on every replay."""
    dev = _device("dropout", "x", x, residual=residual)
    _dtype_code("dropout", "x", x)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"x_b200.dropout: p = {p} lies outside [0, 1]")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"x_b200.dropout: residual is {tuple(residual.shape)} {residual.dtype}, "
                             f"x {tuple(x.shape)} {x.dtype}")
        residual = residual.contiguous()
    if torch.is_tensor(call):
        if call.numel() != 1 or call.dtype != torch.int64 or call.get_device() != dev:
            raise ValueError("x_b200.dropout: call must be an integer or a one-element int64 tensor on x's device")
    else:
        call = int(call) & _MASK64
    seed = int(seed) & _MASK64
    if _tracked(x, residual):
        return _Dropout.apply(x, residual, float(p), seed, call)
    return _dropout_run(x, residual, float(p), seed, call)


# ------------------------------------------------------------------------------------------- recurrence
def _recurrence_fwd(gate, x, b, B, h0, kind, want_state, save):
    dev = x.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _recurrence_fwd(gate, x, b, B, h0, kind, want_state, save)
    gate, ldgate = _rows(gate)
    x, ldx = _rows(x)
    N, D = x.shape
    lib = L.load_library()
    h = x.new_empty((N, D))
    hT = x.new_empty((B, D), dtype=torch.float32) if want_state else None
    saved = L.workspace(lib.atlb_recurrence_saved_bytes(N, D), x.device) if save else None
    nb = lib.atlb_recurrence_workspace_bytes(N, D)
    ws = L.workspace(nb, x.device)
    L.check(lib.atlb_recurrence_fwd(L.DTYPES[x.dtype], kind, gate.data_ptr(), ldgate, x.data_ptr(), ldx, _addr(b), N, B, D,
                                    _addr(h0), h.data_ptr(), _addr(hT), _addr(saved), ws.data_ptr(), nb, _stream(dev)),
            "linear_recurrence")
    return h, hT, saved


def _recurrence_bwd(gate, x, b, B, h0, kind, saved, gh, ghT):
    dev = x.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _recurrence_bwd(gate, x, b, B, h0, kind, saved, gh, ghT)
    gate, ldgate = _rows(gate)
    x, ldx = _rows(x)
    gh, ldgh = _rows(torch.zeros_like(x) if gh is None else gh)
    ghT = None if ghT is None else ghT.contiguous()
    N, D = x.shape
    lib = L.load_library()
    ggate, gx = x.new_empty((N, D)), x.new_empty((N, D))
    gh0 = x.new_empty((B, D), dtype=torch.float32) if h0 is not None else None
    nb = lib.atlb_recurrence_workspace_bytes(N, D)
    ws = L.workspace(nb, x.device)
    L.check(lib.atlb_recurrence_bwd(L.DTYPES[x.dtype], kind, gate.data_ptr(), ldgate, x.data_ptr(), ldx, _addr(b), N, B, D,
                                    _addr(h0), saved.data_ptr(), gh.data_ptr(), ldgh, _addr(ghT), ggate.data_ptr(),
                                    gx.data_ptr(), _addr(gh0), ws.data_ptr(), nb, _stream(dev)), "linear_recurrence_bwd")
    return ggate, gx, gh0


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, b, B, h0, kind, want_state):
        h, hT, saved = _recurrence_fwd(gate, x, b, B, h0, kind, want_state, True)
        ctx.save_for_backward(gate, x, b, h0, saved)
        ctx.meta = (B, kind)
        ctx.set_materialize_grads(False)
        return h, hT

    @staticmethod
    @once_differentiable
    def backward(ctx, gh, ghT):
        gate, x, b, h0, saved = ctx.saved_tensors
        B, kind = ctx.meta
        ggate, gx, gh0 = _recurrence_bwd(gate, x, b, B, h0, kind, saved, gh, ghT)
        return ggate, gx, None, None, gh0, None, None


def linear_recurrence(gate: torch.Tensor, x: torch.Tensor, b: torch.Tensor | None = None, B: int = 1,
                      h0: torch.Tensor | None = None, kind: str = "sigmoid", return_state: bool = False):
    """A state per column that runs along the rows of each window:

        kind="sigmoid"  h_t = a_t h_(t-1) + (1 - a_t) x_t,  a_t = sigmoid(gate_t), zero below 2^-126
        kind="decay"    h_t = gate_t h_(t-1) + x_t          (exp(-dt / tau): decaying event traces)

    gate, x (N, D), one dtype; slices of a wider projection are taken as they are.  ``b`` (N,) int64 is the window of
    each row in [0, B), the rows of a window contiguous, as in events sorted by (b, t) (not checked: every run of equal
    ``b`` starts from h0, and which run's state is returned is open); rows with any other value (padding, -1) get h = 0
    and no gradient, and what they hold reaches nothing.  Without ``b`` the rows are B equal
    windows: a (B, T, D) batch is ``flatten(0, 1)``.  ``h0`` (B, D) float32 is the state before each window's first
    row (default zero).  Returns h (N, D), or (h, state) with ``return_state``: state (B, D) float32 after each
    window's last row (h0 where a window has none), to be given as the next call's ``h0``; one row per window is one
    step.  Differentiable in gate, x and h0, through h and state."""
    _device("linear_recurrence", "x", x, gate=gate, b=b, h0=h0)
    _dtype_code("linear_recurrence", "x", x)
    if x.dim() != 2 or gate.shape != x.shape or gate.dtype != x.dtype:
        raise ValueError(f"x_b200.linear_recurrence: gate and x must be (N, D) of one dtype, got "
                         f"{tuple(gate.shape)} {gate.dtype} and {tuple(x.shape)} {x.dtype}")
    code = L.REC_KINDS.get(kind)
    if code is None:
        raise ValueError(f"x_b200.linear_recurrence: unknown kind {kind!r}")
    N, D = x.shape
    B = int(B)
    if B < 0 or (b is None and (B < 1 or N % B)):
        raise ValueError(f"x_b200.linear_recurrence: {N} rows do not make {B} equal windows")
    if b is not None:
        if b.dtype != torch.int64:
            raise RuntimeError(f"x_b200.linear_recurrence: b must be int64, got {b.dtype}")
        if b.shape != (N,):
            raise ValueError(f"x_b200.linear_recurrence: b must be ({N},), got {tuple(b.shape)}")
        b = b.contiguous()
    if h0 is not None:
        if h0.dtype != torch.float32:
            raise RuntimeError(f"x_b200.linear_recurrence: h0 must be float32, got {h0.dtype}")
        if h0.shape != (B, D):
            raise ValueError(f"x_b200.linear_recurrence: h0 must be ({B}, {D}), got {tuple(h0.shape)}")
        h0 = h0.contiguous()
    if _tracked(gate, x, h0):
        h, state = _Recurrence.apply(gate, x, b, B, h0, code, return_state)
    else:
        h, state, _ = _recurrence_fwd(gate, x, b, B, h0, code, return_state, False)
    return (h, state) if return_state else h
