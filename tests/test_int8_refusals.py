"""What the 8-bit rows and products refuse: the launchers' own checks, and those of their Python faces (which run here on CPU tensors,
behind the check that tensors are on a GPU)."""

import ctypes

import pytest
import torch

from ullm_b200.csrc import launchers, ops
from ullm_b200.csrc.build import build, load_native

PYTHON_ROWS, PYTHON_VECTOR = ops._rows, ops._vector

BAD_DTYPE, BAD_SIZE = 1, 2


@pytest.fixture(scope="module")
def lib():
    dll = ctypes.CDLL(build())
    kinds = {"P": ctypes.c_void_p, "I": ctypes.c_int, "F": ctypes.c_float, "LL": ctypes.c_longlong}
    for name in ("ullm_quantize_rows_int8", "ullm_act_mul_int8", "ullm_add_rmsnorm_int8", "ullm_linear_int8"):
        getattr(dll, name).argtypes = [kinds[t] for t in launchers.LAUNCHERS[name]]
        getattr(dll, name).restype = ctypes.c_int
    return dll


def test_launchers(lib):
    for dtype, rows, cols, xs, os, want in ((0, 4, 0, 8, 8, BAD_SIZE), (0, -1, 8, 8, 8, BAD_SIZE), (0, 4, 8, 7, 8, BAD_SIZE),
                                            (0, 4, 8, 8, 7, BAD_SIZE), (3, 4, 8, 8, 8, BAD_DTYPE), (0, 4, 1 << 29, 1 << 29, 1 << 29, BAD_SIZE),
                                            (1, 0, 8, 8, 8, 0)):
        assert lib.ullm_quantize_rows_int8(dtype, None, xs, None, os, None, rows, cols, None, None) == want
    assert lib.ullm_act_mul_int8(1, 2, None, None, 8, None, 4, 8, None, None) == BAD_SIZE  # an activation that does not exist
    assert lib.ullm_act_mul_int8(1, 0, None, None, 7, None, 4, 8, None, None) == BAD_SIZE
    assert lib.ullm_add_rmsnorm_int8(5, None, None, None, None, 8, None, 4, 8, 1e-6, None, None) == BAD_DTYPE
    assert lib.ullm_add_rmsnorm_int8(1, None, None, None, None, 4, None, 4, 8, 1e-6, None, None) == BAD_SIZE
    for dtype, M, N, k, xs, ws, want in ((0, 4, 8, 0, 16, 16, BAD_SIZE), (0, 4, 8, 131072, 131072, 131072, BAD_SIZE),
                                         (0, 4, 0, 16, 16, 16, BAD_SIZE), (0, (1 << 30) + 1, 8, 16, 16, 16, BAD_SIZE), (0, 4, (1 << 30) + 1, 16, 16, 16, BAD_SIZE), (0, -1, 8, 16, 16, 16, BAD_SIZE), (0, 4, 8, 16, 15, 16, BAD_SIZE),
                                         (0, 4, 8, 16, 16, 8, BAD_SIZE), (7, 4, 8, 16, 16, 16, BAD_DTYPE), (1, 0, 8, 16, 16, 16, 0)):
        assert lib.ullm_linear_int8(dtype, None, xs, None, None, ws, None, None, None, M, N, k, None, None) == want


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def face(monkeypatch):
    """The Python faces with their checks as Python writes them, on CPU tensors, in front of a library that records what reaches it."""
    monkeypatch.setattr(ops, "_here", lambda t: True)
    monkeypatch.setattr(ops, "_at_once", None)
    monkeypatch.setattr(ops, "_rows", PYTHON_ROWS)
    monkeypatch.setattr(ops, "_vector", PYTHON_VECTOR)
    monkeypatch.setattr(ops, "_ptr", lambda t: t)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    k = object.__new__(ops.Kernels)
    k.skip_groups, k.timer, k.launches, k.status, k.lib, k.device_index = frozenset(), None, 0, None, Recorder(), -1
    return k


def refused(face, call, match="do not fit"):
    with pytest.raises(ops.KernelError, match=match if not torch.cuda.is_available() else None):
        call()
    assert face.lib.calls == []


def test_rows(face):
    x, q, s = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    for call in (lambda: face.quantize_rows_int8(x.double(), q, s),
                 lambda: face.quantize_rows_int8(x, q.short(), s),
                 lambda: face.quantize_rows_int8(x, q, s[:2]),
                 lambda: face.quantize_rows_int8(x, q, s.double()),
                 lambda: face.quantize_rows_int8(x, q, torch.zeros(6)[::2]),
                 lambda: face.quantize_rows_int8(x, q[:, :7], s),
                 lambda: face.quantize_rows_int8(torch.zeros(8, 3).t(), q, s),
                 lambda: face.quantize_rows_int8(torch.zeros(1, 8).expand(3, 8), q, s),
                 lambda: face.quantize_rows_int8(x, torch.zeros(8, 3, dtype=torch.int8).t(), s),
                 lambda: face.quantize_rows_int8(x, torch.zeros(1, 8, dtype=torch.int8).expand(3, 8), s),
                 lambda: face.quantize_rows_int8(x[0], q, s),
                 lambda: face.act_mul_int8(torch.zeros(3, 15), q, s),
                 lambda: face.act_mul_int8(x, q, s),
                 lambda: face.act_mul_int8(torch.zeros(3, 20)[:, :16], q, s),
                 lambda: face.add_rmsnorm_int8(x, x[:2].clone(), torch.ones(8), 1e-6, q, s),
                 lambda: face.add_rmsnorm_int8(x, x.half(), torch.ones(8), 1e-6, q, s),
                 lambda: face.add_rmsnorm_int8(x, torch.zeros(3, 9)[:, :8], torch.ones(8), 1e-6, q, s),
                 lambda: face.add_rmsnorm_int8(torch.zeros(3, 9)[:, :8], None, torch.ones(8), 1e-6, q, s),
                 lambda: face.add_rmsnorm_int8(x, None, torch.ones(4), 1e-6, q, s),
                 lambda: face.add_rmsnorm_int8(x, None, torch.ones(8).half(), 1e-6, q, s)):
        refused(face, call)
    assert face.quantize_rows_int8(torch.zeros(3, 12)[:, :8], face.int8_rows(3, 8, "cpu"), s) is not None
    (name, args), = face.lib.calls
    assert name == "ullm_quantize_rows_int8" and args[0] == 0 and args[2] == 12 and args[4] == 16 and args[6:8] == (3, 8)


def test_products(face):
    x, w = torch.zeros(3, 32, dtype=torch.int8), torch.zeros(5, 32, dtype=torch.int8)
    xs, ws, out = torch.zeros(3), torch.zeros(5), torch.zeros(3, 5)
    for call in (lambda: face.linear_int8(x.float(), xs, w, ws, out),
                 lambda: face.linear_int8(x, xs, w.to(torch.uint8), ws, out),
                 lambda: face.linear_int8(x[:, :16], xs, w, ws, out),
                 lambda: face.linear_int8(x, xs[:2], w, ws, out),
                 lambda: face.linear_int8(x, xs, w, ws[:1], out),
                 lambda: face.linear_int8(x, xs, w, ws, out.t().contiguous()),
                 lambda: face.linear_int8(x, xs, w, ws, out.double()),
                 lambda: face.linear_int8(x, xs, w, ws, torch.zeros(3, 8)[:, :5]),
                 lambda: face.linear_int8(x, xs, w, ws, out, torch.zeros(5).half()),
                 lambda: face.linear_int8(x, xs, w, ws, out, torch.zeros(4)),
                 lambda: face.linear_int8(x, xs, torch.zeros(32, 5, dtype=torch.int8).t(), ws, out),
                 lambda: face.linear_int8(x, xs, w[0], ws, out)):
        refused(face, call)
    big = torch.zeros(1, 131072, dtype=torch.int8)
    face.device_index = 1  # (the tensors are not where the kernels were set up)
    refused(face, lambda: face.linear_int8(x, xs, w, ws, out))
    face.device_index = -1
    refused(face, lambda: face.linear_int8(big, xs[:1], big, ws[:1], out[:1, :1].contiguous()), "131,071")
    assert face.linear_int8(x, xs, w, ws, out) is out
    assert face.linear_int8(x[1:2], xs[1:2], w, ws, out[1:2]) is not None
    assert face.lib.calls[0][1][2] == 32 and face.lib.calls[0][1][-5:-2] == (3, 5, 32) and face.lib.calls[1][1][2] == 32


def test_tensors_elsewhere():
    """On the CPU, with the checks as they are: the message says where the tensor is."""
    x, q, s = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    k = object.__new__(ops.Kernels)
    k.skip_groups, k.timer, k.device_index, k.lib, k.status = frozenset(), None, 0, Recorder(), s
    with pytest.raises(ops.KernelError):
        k.quantize_rows_int8(x, q, s)
    native = load_native()
    launcher = native.bind("ullm_quantize_rows_int8", 1)
    for args in ((launcher, x, q, s, s), (launcher, x, q, s), (launcher, None, q, s, s), (launcher, x, q, s, None)):
        assert native.quantize_rows_int8(*args) is None
    assert native.rows(q, torch.int8, 3, 8) == -1 and native.vector(s, torch.float32, 3) is False
