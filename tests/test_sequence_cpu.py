"""The recurrence along a sequence and the products grouped by expert without
a GPU: every shape check runs before any CUDA call, so refused calls return
DS_INVALID_ARGUMENT with a message on a CPU-only host."""
import ctypes

import numpy as np
import pytest

import sequence_ref as ref


@pytest.fixture(scope="module")
def L():
    import importlib
    importlib.import_module("build").build()
    from ds_b200 import _lib
    return _lib


R = ctypes.byref
WS = ctypes.c_void_p(0x40000000)
BIG = 1 << 40


class Bufs:
    """Descriptors at made-up, disjoint device addresses."""

    def __init__(self, L):
        self.L, self.next, self.keep = L, 0x100000000, []

    def __call__(self, *shape, ptr=None):
        if ptr is None:
            ptr, self.next = self.next, self.next + 0x10000000
        b, d = self.L.make_buffer(ptr, shape)
        self.keep.append((b, d))
        return b


def refused(L, name, args, match):
    st = getattr(L.lib(), name)(*args)
    msg = L.last_error()
    assert st == L.DS_INVALID_ARGUMENT, (st, msg)
    assert match in msg, msg


def test_recurrence_refusals(L):
    b = Bufs(L)
    x, y, z, h0 = b(2, 5, 3), b(2, 5, 3), b(2, 5, 3), b(2, 3)
    f = "ds_linear_recurrence_f64"

    def call(a=x, bb=y, h=h0, out=z, ws=WS, n=BIG):
        return (R(a), R(bb), R(h) if h else None, R(out), ws, n, None)

    refused(L, f, call(bb=b(2, 5, 4)), "same shape")
    refused(L, f, call(out=b(2, 5, 4)), "output shape")
    refused(L, f, call(h=b(2, 5)), "h0 must be")
    refused(L, f, call(h=b(3)), "h0 must be")
    refused(L, f, call(a=b(3), bb=b(3), out=b(3)), "[..., T, D]")
    refused(L, f, call(a=b(2, 5, 3, ptr=0)), "null")
    refused(L, f, call(bb=b(2, 5, 3, ptr=0x100000004)), "aligned")
    refused(L, f, call(out=x), "h overlaps a")
    refused(L, f, call(out=b(2, 5, 3, ptr=y.data + 8)), "h overlaps b")
    refused(L, f, call(out=b(2, 5, 3, ptr=h0.data + 40)), "h overlaps h0")
    refused(L, f, call(a=b(-1, 5, 3)), "invalid buffer")
    huge = (1 << 31, 1 << 31, 4)
    refused(L, f, call(a=b(*huge), bb=b(*huge), out=b(*huge)), "too large")
    refused(L, "ds_linear_recurrence_packed", call(), "last dim == 2")
    p = b(5, 3, 2)
    refused(L, "ds_linear_recurrence_packed",
            call(a=b(5, 3, 2, ptr=0x100000004), bb=p, h=None, out=p), "aligned")


def test_recurrence_gradient_refusals(L):
    b = Bufs(L)
    a, h, g, h0 = b(2, 5, 3), b(2, 5, 3), b(2, 5, 3), b(2, 3)
    ga, gb, g0 = b(2, 5, 3), b(2, 5, 3), b(2, 3)
    f = "ds_linear_recurrence_vjp_f32"

    def call(a=a, h=h, g=g, h0=h0, ga=ga, gb=gb, g0=g0):
        return (R(a), R(h), R(g), R(h0) if h0 else None, R(ga), R(gb), R(g0), WS, BIG, None)

    refused(L, f, call(h=b(2, 4, 3)), "same shape")
    refused(L, f, call(g0=b(3, 2)), "output shape")
    refused(L, f, call(ga=b(2, 5, 2)), "output shape")
    refused(L, f, call(h0=b(2, 4)), "h0 must be")
    refused(L, f, call(gb=g), "grad_b overlaps grad_h")
    refused(L, f, call(ga=gb), "grad_b overlaps grad_a")
    refused(L, f, call(g0=h0), "grad_h0 overlaps h0")


def test_ragged_refusals(L):
    b = Bufs(L)
    x, w, s, o = b(8, 4), b(3, 4, 6), b(3), b(8, 6)
    f = "ds_ragged_dot_f64"

    def call(x=x, w=w, s=s, c=1, o=o, ws=WS, n=BIG):
        return (R(x), R(w), R(s), c, R(o), ws, n, None)

    refused(L, f, call(c=0), "rhs_contracting")
    refused(L, f, call(c=2), "contracting dimensions")
    refused(L, f, call(x=b(8, 4, 1)), "[M, K]")
    refused(L, f, call(w=b(4, 6)), "[G, K, N]")
    refused(L, f, call(s=b(4)), "[G]")
    refused(L, f, call(s=b(3, 1)), "[G]")
    refused(L, f, call(o=b(8, 4)), "output shape")
    refused(L, f, call(o=b(8, 6, ptr=w.data)), "overlaps rhs")
    refused(L, f, call(o=b(8, 6, ptr=x.data + 8)), "overlaps lhs")
    refused(L, f, call(ws=None, n=0), "workspace")
    refused(L, f, call(ws=ctypes.c_void_p(0x40000010)), "workspace")
    refused(L, f, call(s=b(3, ptr=0)), "null")
    refused(L, f, call(x=b(0, 4), w=b(70000, 4, 6), s=b(70000), o=b(0, 6)), "65535 groups")
    refused(L, f, call(x=b(1 << 31, 0), w=b(3, 0, 6), o=b(1 << 31, 6)), "2^31")
    refused(L, "ds_ragged_dot", (R(x), R(b(8, 3)), R(w), R(w), R(s), 1, R(o), R(b(8, 6)), WS, BIG,
                                 None), "same shape")
    refused(L, "ds_ragged_dot", (R(x), R(x), R(w), R(w), R(s), 1, R(o), R(o), WS, BIG, None),
            "out_lo overlaps out_hi")


def test_ragged_contract_refusals(L):
    b = Bufs(L)
    x, y, s, o = b(8, 4), b(8, 6), b(3), b(3, 4, 6)
    f = "ds_ragged_dot_contract_f64"

    def call(x=x, y=y, s=s, o=o, ws=WS, n=BIG):
        return (R(x), R(y), R(s), R(o), ws, n, None)

    refused(L, f, call(y=b(7, 6)), "contracting dimensions")
    refused(L, f, call(x=b(8)), "[M, K]")
    refused(L, f, call(s=b(3, 1)), "[G]")
    refused(L, f, call(o=b(3, 6, 4)), "output shape")
    refused(L, f, call(o=b(3, 4, 6, ptr=y.data)), "overlaps rhs")
    refused(L, f, call(n=0), "workspace")
    refused(L, "ds_ragged_dot_contract",
            (R(x), R(x), R(y), R(b(8, 5)), R(s), R(o), R(b(3, 4, 6)), WS, BIG, None), "same shape")


def test_workspace_queries(L):
    """0 where the call would be refused, and no error left behind."""
    b = Bufs(L)
    lib = L.lib()
    q = lib.ds_linear_recurrence_workspace_size
    assert q(R(b(3)), L.DS_FUSED_F64) == 0
    assert q(R(b(2, 5, 3)), 9) == 0
    assert q(R(b(1 << 31, 1 << 31, 4)), L.DS_FUSED_F64) == 0
    assert lib.ds_ragged_dot_workspace_size(R(b(8, 4)), R(b(3, 5, 6)), 1) == 0
    assert lib.ds_ragged_dot_workspace_size(R(b(8, 4)), R(b(3, 4, 6)), 1) > 0
    assert lib.ds_ragged_dot_contract_workspace_size(R(b(8, 4)), R(b(8, 6)), R(b(3))) > 0


def test_targets_are_registered_and_check_their_operands():
    import torch
    from ds_b200 import ffi, ops
    assert set(ffi.SEQUENCE_TARGETS) <= set(ffi.registered_targets())
    x = torch.zeros((2, 5, 3), dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.ds_linear_recurrence_f64(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.ds_ragged_dot_contract_f64(x[0], x[0], torch.zeros(2, dtype=torch.int32))
    assert ops._state_shape((2, 5, 3)) == (2, 3) and ops._state_shape((5, 3)) == (3,)
    assert ops._state_shape((2, 5, 3, 2), packed=True) == (2, 3, 2)


def test_host_loops_agree_with_each_other():
    """The oracle's gradient is the derivative of the oracle's recurrence
    (central differences, exact for a multilinear function up to rounding)."""
    rng = np.random.default_rng(0)
    a, b, w = (rng.standard_normal((1, 9, 2)) for _ in range(3))
    h0 = rng.standard_normal((1, 2))
    h = ref.recurrence(a, b, h0)[0].astype(np.float64)
    grads, _ = ref.recurrence_vjp(a, h, w, h0)
    for which in range(3):
        for at in np.ndindex((a, b, h0)[which].shape):
            v = [[x.copy() for x in (a, b, h0)] for _ in range(2)]
            v[0][which][at] += 2.0 ** -8
            v[1][which][at] -= 2.0 ** -8
            f = [float(np.sum(ref.recurrence(*q)[0] * w)) for q in v]
            d = (f[0] - f[1]) * 2.0 ** 7
            # the loss's values are below 1000 here: 2^-53 of them over 2^-7
            assert abs(d - float(grads[which][at])) <= 1000 * 2.0 ** -44


def test_adapters_have_a_handler_for_every_new_target():
    """ds_b200_ffi.cc, read as text: one XLA-FFI handler per target."""
    import os
    import re
    from conftest import ROOT
    from ds_b200 import ffi
    text = open(os.path.join(ROOT, "ds-experiment_b200", "adapters", "ds_b200_ffi.cc")).read()
    symbols = set(re.findall(r"XLA_FFI_DEFINE_HANDLER_SYMBOL\((\w+),", text))
    for name in re.findall(r"^DS_RECURRENCE_HANDLERS\((\w+),", text, re.M):
        symbols |= {f"DsLinearRecurrence{name}", f"DsLinearRecurrenceVjp{name}"}
    for target in ffi.SEQUENCE_TARGETS:
        assert "".join(p[:1].upper() + p[1:] for p in target.split("_")) in symbols, target


def test_threads_have_workspaces_of_their_own(monkeypatch):
    import threading
    import torch
    from ds_b200 import ffi
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ffi, "_workspaces", {})
    got = []
    here = ffi._workspace(100, torch.device("cpu"), 7)
    t = threading.Thread(target=lambda: got.append(ffi._workspace(100, torch.device("cpu"), 7)))
    t.start()
    t.join()
    assert got[0] is not here and ffi._workspace(100, torch.device("cpu"), 7) is here


def test_no_groups_ask_for_no_planes(L):
    """A product of batch size without groups is zeros: no tensor-core product, whose
    planes would take hundreds of megabytes."""
    b = Bufs(L)
    q = L.lib().ds_ragged_dot_workspace_size
    for contracting, w in ((1, b(0, 1024, 1024)), (2, b(0, 1024, 1024))):
        assert 0 < q(R(b(8192, 1024)), R(w), contracting) <= 1 << 20
    assert 0 < L.lib().ds_ragged_dot_contract_workspace_size(
        R(b(8192, 1024)), R(b(8192, 1024)), R(b(0))) <= 1 << 20


def test_ragged_algorithms(L):
    """The entry points that take an algorithm refuse what the others do and unknown
    algorithms; f64 sums need no planes."""
    b = Bufs(L)
    lib = L.lib()
    x, w, s, o = b(8, 4), b(3, 4, 6), b(3), b(8, 6)
    f = "ds_ragged_dot_algorithm_f64"
    refused(L, f, (R(x), R(w), R(s), 1, 7, R(o), WS, BIG, None), "unknown algorithm")
    refused(L, f, (R(x), R(w), R(s), 2, 1, R(o), WS, BIG, None), "contracting dimensions")
    refused(L, f, (R(x), R(w), R(s), 1, 1, R(x), WS, BIG, None), "output shape")
    refused(L, f, (R(x), R(w), R(s), 1, 1, R(o), None, 0, None), "workspace")
    refused(L, "ds_ragged_dot_algorithm",
            (R(x), R(x), R(w), R(w), R(s), 1, -1, R(o), R(b(8, 6)), WS, BIG, None), "unknown")
    y, oc = b(8, 6), b(3, 4, 6)
    f = "ds_ragged_dot_contract_algorithm_f64"
    refused(L, f, (R(x), R(y), R(s), 2, R(oc), WS, BIG, None), "unknown algorithm")
    refused(L, f, (R(x), R(y), R(s), 1, R(b(3, 6, 4)), WS, BIG, None), "output shape")
    refused(L, "ds_ragged_dot_contract_algorithm",
            (R(x), R(x), R(y), R(y), R(s), 9, R(oc), R(b(3, 4, 6)), WS, BIG, None), "unknown")
    q = lib.ds_ragged_dot_algorithm_workspace_size
    big = (R(b(8192, 2048)), R(b(8, 2048, 2048)), 1)
    assert q(*big, L.DS_DOT_TENSOR_INT8) == lib.ds_ragged_dot_workspace_size(*big) > 1 << 28
    assert 0 < q(*big, L.DS_DOT_CUDA_CORE) <= 1 << 20
    assert q(*big, 5) == 0
    q = lib.ds_ragged_dot_contract_algorithm_workspace_size
    big = (R(b(8192, 2048)), R(b(8192, 2048)), R(b(8)))
    assert q(*big, L.DS_DOT_TENSOR_INT8) == lib.ds_ragged_dot_contract_workspace_size(*big) > 1 << 28
    assert 0 < q(*big, L.DS_DOT_CUDA_CORE) <= 1 << 20
    assert q(*big, 5) == 0


def test_workspaces_end_with_their_thread(monkeypatch):
    import threading
    import torch
    from ds_b200 import ffi
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ffi, "_workspaces", {})
    here = ffi._workspace(100, torch.device("cpu"), 7)

    def work():
        for stream in (7, 8):
            ffi._workspace(100, torch.device("cpu"), stream)
        assert len(ffi._workspaces) == 3

    for _ in range(3):
        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert list(ffi._workspaces) == [(None, 7, threading.get_ident())]
    assert ffi._workspace(100, torch.device("cpu"), 7) is here
