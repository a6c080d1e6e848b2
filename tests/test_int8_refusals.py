"""What the 8-bit rows and products refuse: the launchers' own checks, and those of their Python faces (which run here on CPU tensors,
behind the check that tensors are on a GPU)."""

import ctypes

import pytest
import torch

from ullm_b200.csrc import launchers, ops
from ullm_b200.csrc.build import build

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
        assert lib.ullm_quantize_rows_int8(dtype, None, xs, None, os, None, rows, cols, None) == want
    assert lib.ullm_act_mul_int8(1, 2, None, None, 8, None, 4, 8, None) == BAD_SIZE  # an activation that does not exist
    assert lib.ullm_act_mul_int8(1, 0, None, None, 7, None, 4, 8, None) == BAD_SIZE
    assert lib.ullm_add_rmsnorm_int8(5, None, None, None, None, 8, None, 4, 8, 1e-6, None) == BAD_DTYPE
    assert lib.ullm_add_rmsnorm_int8(1, None, None, None, None, 4, None, 4, 8, 1e-6, None) == BAD_SIZE
    for dtype, M, N, k, xs, ws, want in ((0, 4, 8, 0, 16, 16, BAD_SIZE), (0, 4, 8, 131072, 131072, 131072, BAD_SIZE),
                                         (0, 4, 0, 16, 16, 16, BAD_SIZE), (0, -1, 8, 16, 16, 16, BAD_SIZE), (0, 4, 8, 16, 15, 16, BAD_SIZE),
                                         (0, 4, 8, 16, 16, 8, BAD_SIZE), (7, 4, 8, 16, 16, 16, BAD_DTYPE), (1, 0, 8, 16, 16, 16, 0)):
        assert lib.ullm_linear_int8(dtype, None, xs, None, None, ws, None, None, None, M, N, k, None, None) == want


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def face(monkeypatch):
    def need(t, name, dtype=None, contiguous=True):
        if dtype is not None and t.dtype != dtype:
            raise ops.KernelError(f"{name} has dtype {t.dtype}, expected {dtype}")
        if contiguous and not t.is_contiguous():
            raise ops.KernelError(f"{name} must be contiguous")

    monkeypatch.setattr(ops, "_need", need)
    monkeypatch.setattr(ops, "_ptr", lambda t: t)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_on_current_device", lambda *a: None)
    k = object.__new__(ops.Kernels)
    k.skip_groups, k.timer, k.launches, k.status, k.lib = frozenset(), None, 0, None, Recorder()
    return k


def refused(face, match, call):
    with pytest.raises(ops.KernelError, match=match):
        call()
    assert face.lib.calls == []


def test_rows(face):
    x, q, s = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    refused(face, "rows of torch.float64", lambda: face.quantize_rows_int8(x.double(), q, s))
    refused(face, "out has dtype", lambda: face.quantize_rows_int8(x, q.short(), s))
    refused(face, "scales", lambda: face.quantize_rows_int8(x, q, s[:2]))
    refused(face, "scales has dtype", lambda: face.quantize_rows_int8(x, q, s.double()))
    refused(face, "3 rows of 8", lambda: face.quantize_rows_int8(x, q[:, :7], s))
    refused(face, "3 rows of 0", lambda: face.quantize_rows_int8(x[:, :0], q[:, :0], s))
    refused(face, "side by side", lambda: face.quantize_rows_int8(torch.zeros(8, 3).t(), q, s))
    refused(face, "rows overlap", lambda: face.quantize_rows_int8(torch.zeros(1, 8).expand(3, 8), q, s))
    refused(face, "side by side", lambda: face.quantize_rows_int8(x, torch.zeros(8, 3, dtype=torch.int8).t(), s))
    refused(face, "shape", lambda: face.quantize_rows_int8(x[0], q, s))
    refused(face, "gate_up", lambda: face.act_mul_int8(torch.zeros(3, 15), q, s))
    refused(face, "3 rows of 4", lambda: face.act_mul_int8(x, q, s))
    refused(face, "contiguous", lambda: face.act_mul_int8(torch.zeros(3, 20)[:, :16], q, s))
    w = torch.ones(8)
    refused(face, "residual shape", lambda: face.add_rmsnorm_int8(x, x[:2].clone(), w, 1e-6, q, s))
    refused(face, "residual has dtype", lambda: face.add_rmsnorm_int8(x, x.half(), w, 1e-6, q, s))
    refused(face, "weight", lambda: face.add_rmsnorm_int8(x, None, w[:4], 1e-6, q, s))
    face.quantize_rows_int8(torch.zeros(3, 12)[:, :8], face.int8_rows(3, 8, "cpu"), s)
    (name, args), = face.lib.calls
    assert name == "ullm_quantize_rows_int8" and args[0] == 0 and args[2] == 12 and args[4] == 16 and args[6:8] == (3, 8)


def test_products(face):
    x, w = torch.zeros(3, 32, dtype=torch.int8), torch.zeros(5, 32, dtype=torch.int8)
    xs, ws, out = torch.zeros(3), torch.zeros(5), torch.zeros(3, 5)
    refused(face, "x has dtype", lambda: face.linear_int8(x.float(), xs, w, ws, out))
    refused(face, "weight has dtype", lambda: face.linear_int8(x, xs, w.to(torch.uint8), ws, out))
    refused(face, "linear_int8: x", lambda: face.linear_int8(x[:, :16], xs, w, ws, out))
    refused(face, "linear_int8: x", lambda: face.linear_int8(x, xs[:2], w, ws, out))
    refused(face, "linear_int8: x", lambda: face.linear_int8(x, xs, w, ws[:1], out))
    refused(face, "linear_int8: x", lambda: face.linear_int8(x, xs, w, ws, out.t().contiguous()))
    refused(face, "linear_int8: x", lambda: face.linear_int8(x, xs, w, ws, out.double()))
    refused(face, "contiguous", lambda: face.linear_int8(x, xs, w, ws, torch.zeros(3, 8)[:, :5]))
    refused(face, "bias has dtype", lambda: face.linear_int8(x, xs, w, ws, out, torch.zeros(5).half()))
    refused(face, "bias", lambda: face.linear_int8(x, xs, w, ws, out, torch.zeros(4)))
    refused(face, "side by side", lambda: face.linear_int8(x, xs, torch.zeros(32, 5, dtype=torch.int8).t(), ws, out))
    big = torch.zeros(1, 131072, dtype=torch.int8)
    refused(face, "131,071", lambda: face.linear_int8(big, xs[:1], big, ws[:1], out[:1, :1].contiguous()))
    refused(face, "k=0", lambda: face.linear_int8(x[:, :0], xs, w[:, :0], ws, out))
    assert face.linear_int8(x, xs, w, ws, out) is out
    assert face.lib.calls[0][1][2] == 32 and face.lib.calls[0][1][-5:-2] == (3, 5, 32)
