"""The event-sequence operators without a GPU: refusals of the wrappers and of the C entry points, and the float64
statements that the GPU tests compare with (their gradients against central differences, their random words against
the oracle's generator)."""
import ctypes
import os

import numpy as np
import pytest
import torch

import x_b200
from oracle import oracle as O
from tests import sequence_ref as R
from x_b200 import _lib

P = ctypes.c_void_p(256)  # never read: every call below is refused before any device work


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        x_b200.embedding(x, torch.zeros(3, dtype=torch.long))
    with pytest.raises(RuntimeError, match="CUDA"):
        x_b200.dropout(x, 0.1, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        x_b200.linear_recurrence(x, x)


@pytest.mark.parametrize("name,args,status,msg", [
    ("atlb_embedding_fwd", (3, P, 4, 4, 4, P, 2, 1.0, P, None), _lib.ATLB_ERR_ARG, b"dtype"),
    ("atlb_embedding_fwd", (0, None, 4, 4, 4, P, 2, 1.0, P, None), _lib.ATLB_ERR_ARG, b"NULL"),
    ("atlb_embedding_fwd", (0, P, -1, 4, 4, P, 2, 1.0, P, None), _lib.ATLB_ERR_ARG, b"negative"),
    ("atlb_embedding_fwd", (0, P, 4, 2**31, 4, P, 2, 1.0, P, None), _lib.ATLB_ERR_OVERFLOW, b"rows"),
    ("atlb_embedding_fwd", (0, P, 4, 4, 2**21, P, 2, 1.0, P, None), _lib.ATLB_ERR_OVERFLOW, b"columns"),
    ("atlb_embedding_fwd", (0, P, 2**31, 4, 4, P, 2, 1.0, P, None), _lib.ATLB_ERR_OVERFLOW, b"stride"),
    ("atlb_embedding_bwd", (0, P, 4, P, 2**31 - 1, 4, 4, 1.0, P, P, 16, None), _lib.ATLB_ERR_OVERFLOW, b"rows"),
    ("atlb_embedding_bwd", (0, P, 4, P, 2, 4, 4, 1.0, P, P, 16, None), _lib.ATLB_ERR_WORKSPACE, b"workspace"),
    ("atlb_embedding_bwd", (0, P, 4, P, 2**31, 4, 4, 1.0, P, P, 16, None), _lib.ATLB_ERR_OVERFLOW, b"rows"),
    ("atlb_dropout", (0, P, None, 4, 1.5, 0, 0, None, P, None), _lib.ATLB_ERR_ARG, b"p ="),
    ("atlb_dropout", (0, P, None, 4, float("nan"), 0, 0, None, P, None), _lib.ATLB_ERR_ARG, b"p ="),
    ("atlb_dropout", (0, P, None, -4, 0.5, 0, 0, None, P, None), _lib.ATLB_ERR_ARG, b"negative"),
    ("atlb_dropout", (0, P, None, 4, 0.5, 0, 0, None, None, None), _lib.ATLB_ERR_ARG, b"NULL"),
    ("atlb_recurrence_fwd", (0, 2, P, 4, P, 4, None, 4, 1, 4, None, P, None, None, P, 1 << 20, None),
     _lib.ATLB_ERR_ARG, b"kind"),
    ("atlb_recurrence_fwd", (0, 0, P, 4, P, 4, None, 5, 2, 4, None, P, None, None, P, 1 << 20, None),
     _lib.ATLB_ERR_ARG, b"equal windows"),
    ("atlb_recurrence_fwd", (0, 0, P, 4, P, 4, None, 4, 2, 4, None, P, None, None, P, 8, None),
     _lib.ATLB_ERR_WORKSPACE, b"workspace"),
    ("atlb_recurrence_bwd", (0, 0, P, 4, P, 4, None, 4, 2, 4, None, None, P, 4, None, P, P, None, P, 1 << 20, None),
     _lib.ATLB_ERR_ARG, b"saved"),
])
def test_c_entries_refuse_before_device_work(name, args, status, msg):
    lib = _lib.load_library()
    assert getattr(lib, name)(*args) == status
    assert msg in lib.atlb_last_error()


def test_workspace_queries_grow_with_the_sizes():
    lib = _lib.load_library()
    assert lib.atlb_embedding_workspace_bytes(0, 0, 0) > 0
    assert lib.atlb_embedding_workspace_bytes(10**6, 307200, 64) > 4 * 4 * 10**6
    assert lib.atlb_recurrence_workspace_bytes(10**6, 64) > lib.atlb_recurrence_workspace_bytes(10**5, 64)
    assert lib.atlb_recurrence_saved_bytes(1, 7) >= 28


@pytest.mark.parametrize("seed,call", [(0, 0), (2**40 + 3, 2**33 + 5)])
def test_words_are_the_oracles_generator(seed, call):
    w = R.philox_words(10, seed, call)
    for q in range(3):
        ref = O.philox4x32_10([q, 2**31, call & 0xFFFFFFFF, call >> 32], [seed & 0xFFFFFFFF, seed >> 32])
        assert w[4 * q:4 * q + 4].tolist() == ref.tolist()[:len(w[4 * q:4 * q + 4])]


@pytest.mark.parametrize("kind", ["sigmoid", "decay"])
def test_recurrence_gradients_against_differences(kind):
    """Central differences of the float64 statement: the truncation error is about step^2, the rounding error about
    2^-52 / step, so a step of 1e-5 leaves both below 1e-8 for values of order one."""
    rng = np.random.default_rng(5)
    N, D, B = 14, 2, 4
    b = np.array([0] * 5 + [-1] + [1] * 1 + [3] * 6 + [-1])  # window 2 is empty
    gate, x = rng.normal(size=(N, D)) * 0.7, rng.normal(size=(N, D))
    h0, gh, ghT = rng.normal(size=(B, D)), rng.normal(size=(N, D)), rng.normal(size=(B, D))
    r = R.recurrence(kind, gate, x, b, B, h0, gh, ghT)

    def loss(gate, x, h0):
        q = R.recurrence(kind, gate, x, b, B, h0)
        return (q["h"][0] * gh).sum() + (q["state"][0] * ghT).sum()

    args = [gate, x, h0]
    for k, name in enumerate(["dgate", "dx", "dh0"]):
        num = np.zeros_like(args[k])
        for i in np.ndindex(num.shape):
            lo, hi = [a.copy() for a in args], [a.copy() for a in args]
            lo[k][i] -= 1e-5
            hi[k][i] += 1e-5
            num[i] = (loss(*hi) - loss(*lo)) / 2e-5
        np.testing.assert_allclose(r[name][0], num, rtol=0, atol=1e-7)


def test_embedding_gradient_against_differences():
    rng = np.random.default_rng(6)
    w, idx, g = rng.normal(size=(4, 3)), np.array([1, -1, 1, 3, 4, 0, 1]), rng.normal(size=(7, 3))
    _, (grad, _) = R.embedding(w, idx, 1.5, g)
    for i in np.ndindex(w.shape):
        d = np.zeros_like(w)
        d[i] = 0.5  # linear in w: any step gives the gradient
        num = ((R.embedding(w + d, idx, 1.5)[0] - R.embedding(w - d, idx, 1.5)[0]) * g).sum()
        assert abs(num - grad[i]) < 1e-12


def test_import_without_cuda_bindings():
    """A torch built without CUDA has none of the private bindings; the package imports, and a call says what is missing."""
    import subprocess
    import sys
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "import x_b200\n"
            "try:\n"
            "    x_b200.embedding(torch.zeros(4, 8), torch.zeros(3, dtype=torch.long))\n"
            "except RuntimeError as e:\n"
            "    assert 'CUDA tensor' in str(e)\n"
            "else:\n"
            "    raise SystemExit('no error')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(__file__)))
    assert r.returncode == 0, r.stderr
