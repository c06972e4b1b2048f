"""The grouped products' algorithms on the GPU.  Sums in f64 (algorithm="cuda_core", and
groups too small for the tensor cores under either) are held to the f64 bound alone:
a sum of K terms by fused multiply-adds, up to 16 parts and 4 accumulators taking
turns makes at most K + 20 roundings of 2^-53 (1.01 for their higher orders) of the
terms' magnitudes."""
import numpy as np
import pytest
import torch

import sequence_ref as ref
from gpu_util import cu
from test_ragged_gpu import CASES, IDS, LARGE, LARGE_IDS, Reached, make, on_gpu, pair, sz

pytestmark = pytest.mark.gpu


class FewGroups:
    """The calls inside did not run the tensor-core product."""

    def __enter__(self):
        from ds_b200 import _lib
        _lib.profile_enable(True)
        _lib.profile_reset()

    def __exit__(self, *exc):
        from ds_b200 import _lib
        n = _lib.profile_read("ozaki_gemm")[1]
        _lib.profile_enable(False)
        if exc[0] is None:
            assert n == 0, "the tensor-core product ran"


def f64_bound(a, b, c, pairs=False, sums=1):
    """Of `sums` sums in f64 (the kernel's, and torch's where it is the oracle)."""
    bound = sums * 1.01 * (a.shape[1] + 20) * ref.U * (a.abs() @ b.abs())
    return bound * 1.0001 + (c.abs() * 2.0 ** -48 + 2.0 ** -150 if pairs else 0.0)


def exact(a, b):
    """a @ b in long double on the host, of f64 tensors."""
    c = a.cpu().numpy().astype(ref.LONG) @ b.cpu().numpy().astype(ref.LONG)
    return torch.from_numpy(c.astype(np.float64)).cuda()


def within(got, want, bound):
    assert bool(((got - want).abs() <= bound + want.abs() * ref.U).all())


def both(hi, lo):
    return hi.double() + lo.double()


@pytest.mark.parametrize("algorithm", ["tensor", "cuda_core"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_small_groups_sum_in_f64(case, algorithm):
    from ds_b200 import ops
    M, K, N, sizes = case
    x, w, y, _ = make(case, 30)
    x, w, y, s = cu(x), cu(w), cu(y), sz(sizes)
    wt = w.transpose(1, 2).contiguous()
    kw = {"algorithm": algorithm}
    with FewGroups():
        out = ops.ds_ragged_dot_f64(x, w, s, **kw)
        outt = ops.ds_ragged_dot_f64(x, wt, s, rhs_contracting=2, **kw)
        p = both(*ops.ds_ragged_dot(*pair(x), *pair(w), s, **kw))
        pt = both(*ops.ds_ragged_dot(*pair(x), *pair(wt), s, rhs_contracting=2, **kw))
        outc = ops.ds_ragged_dot_contract_f64(x, y, s, **kw)
        pc = both(*ops.ds_ragged_dot_contract(*pair(x), *pair(y), s, **kw))
    xp, wp, yp = (both(*pair(t)) for t in (x, w, y))
    for g, b, e in ref.spans(sizes, M):
        if e == b:
            continue
        for a, m, got, pairs in ((x[b:e], w[g], (out[b:e], outt[b:e]), False),
                                 (xp[b:e], wp[g], (p[b:e], pt[b:e]), True),
                                 (x[b:e].T, y[b:e], (outc[g],), False),
                                 (xp[b:e].T, yp[b:e], (pc[g],), True)):
            want = exact(a, m)
            for v in got:
                within(v, want, f64_bound(a, m, want, pairs))


@pytest.mark.parametrize("case", LARGE + [(33041, 70, 90, [33000, 0, 41])],
                         ids=LARGE_IDS + ["windows"])
def test_large_groups_sum_in_f64_when_asked(case):
    """Against torch's f64 sums, whose error the bound takes once more."""
    from ds_b200 import ops
    M, K, N, sizes = case
    x, w, y = on_gpu(M, K, seed=1), on_gpu(len(sizes), K, N, seed=2), on_gpu(M, N, seed=3)
    s, kw = sz(sizes), {"algorithm": "cuda_core"}
    wt = w.transpose(1, 2).contiguous()
    with FewGroups():
        out = ops.ds_ragged_dot_f64(x, w, s, **kw)
        outt = ops.ds_ragged_dot_f64(x, wt, s, rhs_contracting=2, **kw)
        p = both(*ops.ds_ragged_dot(*pair(x), *pair(w), s, **kw))
        outc = ops.ds_ragged_dot_contract_f64(x, y, s, **kw)
        pc = both(*ops.ds_ragged_dot_contract(*pair(x), *pair(y), s, **kw))
    xp, wp, yp = (both(*pair(t)) for t in (x, w, y))
    end = 0
    for g, b, e in ref.spans(sizes, M):
        end = e
        if e == b:
            assert not outc[g].any() and not pc[g].any()
            continue
        for a, m, got, pairs in ((x[b:e], w[g], (out[b:e], outt[b:e]), False),
                                 (xp[b:e], wp[g], (p[b:e],), True),
                                 (x[b:e].T, y[b:e], (outc[g],), False),
                                 (xp[b:e].T, yp[b:e], (pc[g],), True)):
            want = a @ m
            for v in got:
                within(v, want, f64_bound(a, m, want, pairs, sums=2))
    assert not out[end:].any() and not outt[end:].any() and not p[end:].any()


def test_rows_with_an_outlier():
    """One entry of each row 2^30 above the rest, which meets a small weight: f64 sums
    keep their bound, the tensor-core product its own, 2^-24 of each output."""
    from ds_b200 import ops
    M, K, N, sizes = 4100, 700, 1000, [1500, 0, 2000, 300]
    x, w, s = on_gpu(M, K, seed=4), on_gpu(4, K, N, seed=5), sz(sizes)
    x[:, 11] = 2.0 ** 30
    w[:, 11] *= 2.0 ** -40
    with FewGroups():
        f64 = ops.ds_ragged_dot_f64(x, w, s, algorithm="cuda_core")
    with Reached():
        tensor = ops.ds_ragged_dot_f64(x, w, s)
    for g, b, e in ref.spans(sizes, M):
        if e > b:
            want = x[b:e] @ w[g]
            bound = f64_bound(x[b:e], w[g], want, sums=2)
            within(f64[b:e], want, bound)
            within(tensor[b:e], want, bound + 2.0 ** -24 * want.abs())


def test_algorithms_take_turns():
    """Calls of one shape keep their algorithm, eagerly, into a given result, through
    the registry and in graphs."""
    from ds_b200 import _lib, ffi, ops
    M, K, N, sizes = LARGE[1]
    x, w, y = on_gpu(M, K, seed=6), on_gpu(len(sizes), K, N, seed=7), on_gpu(M, N, seed=8)
    s = sz(sizes)
    calls = [lambda **kw: ops.ds_ragged_dot_f64(x, w, s, **kw),
             lambda **kw: ops.ds_ragged_dot_contract_f64(x, y, s, **kw)]
    for call, target in zip(calls, ("ds_ragged_dot_f64", "ds_ragged_dot_contract_f64")):
        t, c = call(), call(algorithm="cuda_core")
        assert not torch.equal(t, c)
        for _ in range(3):
            assert torch.equal(call(algorithm="tensor"), t)
            assert torch.equal(call(algorithm="cuda_core"), c)
        out = torch.empty_like(c)
        assert torch.equal(call(algorithm="cuda_core", out=out), c) and torch.equal(out, c)
        spec = ffi.ShapeDtypeStruct(c.shape, torch.float64)
        args = (x, w, s) if target == "ds_ragged_dot_f64" else (x, y, s)
        assert torch.equal(ffi.ffi_call(target, spec)(*args, algorithm=_lib.DS_DOT_CUDA_CORE), c)
        assert torch.equal(ffi.ffi_call(target, spec)(*args), t)
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        outs = []
        for g, algorithm in zip(graphs, ("tensor", "cuda_core")):
            with torch.cuda.graph(g):
                outs.append(call(algorithm=algorithm))
        for _ in range(2):
            for g in graphs:
                g.replay()
            assert torch.equal(outs[0], t) and torch.equal(outs[1], c)
    with pytest.raises(KeyError):
        calls[0](algorithm="f16")


def test_ds_tensors_choose():
    from ds_b200 import ops
    from ds_b200.dstensor import DSTensor
    M, K, N, sizes = LARGE[1]
    x, w, s = on_gpu(M, K, seed=9), on_gpu(len(sizes), K, N, seed=10), sz(sizes)
    X, W = DSTensor.from_f64(x), DSTensor.from_f64(w)
    for algorithm in ("tensor", "cuda_core"):
        want = ops.ds_from_f64(ops.ds_ragged_dot_f64(X.to_f64(), W.to_f64(), s,
                                                     algorithm=algorithm))
        assert torch.equal(X.ragged_matmul(W, s, algorithm=algorithm).packed, want)
    assert torch.equal(X.ragged_matmul(W, s).packed, X.ragged_matmul(W, s, "tensor").packed)
