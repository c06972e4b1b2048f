"""The linear recurrence along a sequence and its gradient on the GPU, against
the step-by-step loop on the host (tests/sequence_ref.py, with the bounds)."""
import numpy as np
import pytest
import torch

import sequence_ref as ref
from gpu_util import cu, host, misaligned

pytestmark = pytest.mark.gpu

KINDS = ["f64", "f32", "packed"]
SHAPES = [(1, 1, 1), (2, 1, 7), (1, 2, 1), (3, 5, 2), (1, 31, 3), (2, 33, 64), (1, 64, 65),
          (1, 1000, 1), (2, 513, 4), (1, 4097, 5), (2, 257, 250), (1, 2500, 17), (70, 9, 33),
          (5, 65, 130), (1, 20000, 3), (1, 9000, 70)]


def forward(kind):
    from ds_b200 import ops
    return getattr(ops, f"ds_linear_recurrence_{kind}")


def vjp(kind):
    from ds_b200 import ops
    return getattr(ops, f"ds_linear_recurrence_vjp_{kind}")


def inputs(shape, seed, kind, resets=True):
    """Gates near one, some exactly zero and some negative; ordinary values."""
    rng = np.random.default_rng(seed)
    B, T, D = shape
    a = 1.0 / (1.0 + np.exp(-2.0 - 1.5 * rng.standard_normal(shape)))
    if resets:
        a *= (rng.random((B, T, 1)) > 0.03) * np.where(rng.random(shape) < 0.1, -1.0, 1.0)
    b, gh = rng.standard_normal(shape), rng.standard_normal(shape)
    h0 = rng.standard_normal((B, D))
    return [ref.as_type(x, kind) for x in (a, b, gh, h0)]


def val(t, kind):
    x = host(t)
    return ref.value_of(x) if kind == "packed" else x.astype(np.float64)


def check(got, want, bound, what=""):
    err = np.abs(got.astype(ref.LONG) - want)
    assert np.all(err <= bound), f"{what}: {float(np.max(err / np.maximum(bound, 1e-300)))} bounds"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(shape, kind):
    (a, av), (b, bv), _, (h0, h0v) = inputs(shape, 1, kind)
    for start in (None, h0):
        want, mag = ref.recurrence(av, bv, None if start is None else h0v)
        got = val(forward(kind)(cu(a), cu(b), None if start is None else cu(h0)), kind)
        check(got, want, ref.recurrence_bound(mag, kind, want.astype(np.float64)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradient(shape, kind):
    (a, av), (b, bv), (g, gv), (h0, h0v) = inputs(shape, 2, kind)
    h, hv = ref.as_type(ref.recurrence(av, bv, h0v)[0].astype(np.float64), kind)
    for start in (None, h0):
        want, mag = ref.recurrence_vjp(av, hv, gv, None if start is None else h0v)
        got = vjp(kind)(cu(a), cu(h), cu(g), None if start is None else cu(h0))
        bounds = ref.vjp_bounds([w.astype(np.float64) for w in want], mag, kind, shape[1])
        for x, w, e, name in zip(got, want, bounds, ("grad_a", "grad_b", "grad_h0")):
            check(val(x, kind), w, e, name)


def test_gradient_against_differences():
    """The recurrence is linear in b and h0 and multilinear in a: a central
    difference in one coefficient is exact up to rounding (2^-53 of the
    values over the step 2^-10, a few hundred of them summed)."""
    (a, _), (b, _), (w, _), (h0, _) = inputs((2, 40, 3), 5, "f64")
    f, g = forward("f64"), vjp("f64")
    h = f(cu(a), cu(b), cu(h0))
    grads = [host(x) for x in g(cu(a), h, cu(w), cu(h0))]

    def loss(a, b, h0):
        return float(np.sum(host(f(cu(a), cu(b), cu(h0))) * w))

    rng = np.random.default_rng(0)
    step = 2.0 ** -10
    size = float(np.sum(np.abs(host(h)) * np.abs(w)))
    for which in range(3):
        for _ in range(6):
            at = tuple(rng.integers(0, n) for n in (a, b, h0)[which].shape)
            lo, hi = [x.copy() for x in (a, b, h0)], [x.copy() for x in (a, b, h0)]
            lo[which][at] -= step
            hi[which][at] += step
            d = (loss(*hi) - loss(*lo)) / (2 * step)
            assert abs(d - grads[which][at]) <= 1000 * 2.0 ** -53 * size / step


def test_leading_dimensions():
    """[T, D] and [2, 3, T, D] are one and six sequences."""
    (a, _), (b, _), (g, _), (h0, _) = inputs((6, 21, 10), 3, "f64")
    f = forward("f64")
    want = host(f(cu(a), cu(b), cu(h0)))
    got = f(cu(a.reshape(2, 3, 21, 10)), cu(b.reshape(2, 3, 21, 10)), cu(h0.reshape(2, 3, 10)))
    assert np.array_equal(host(got).reshape(6, 21, 10), want)
    assert np.array_equal(host(f(cu(a[0]), cu(b[0]), cu(h0[0]))), want[0])
    ga, gb, g0 = vjp("f64")(cu(a[0]), cu(want[0]), cu(g[0]), cu(h0[0]))
    assert ga.shape == (21, 10) and g0.shape == (10,)
    pa, pb, ph = (cu(ref.pair_of(x)) for x in (a[0], b[0], h0[0]))
    assert forward("packed")(pa, pb, ph).shape == (21, 10, 2)
    assert vjp("packed")(pa, pb, pb, ph)[2].shape == (10, 2)


@pytest.mark.parametrize("shape", [(0, 4, 3), (2, 0, 3), (2, 4, 0)], ids=str)
def test_empty(shape):
    z = torch.empty(shape, dtype=torch.float64, device="cuda")
    h0 = torch.ones((shape[0], shape[2]), dtype=torch.float64, device="cuda")
    assert forward("f64")(z, z.clone(), h0).shape == shape
    ga, gb, g0 = vjp("f64")(z, z.clone(), z.clone(), h0)
    assert ga.shape == gb.shape == shape
    assert torch.equal(g0, torch.zeros_like(h0))  # no step reads the state


@pytest.mark.parametrize("shape", [(2, 300, 9), (1, 5000, 3), (1, 3000, 80)], ids=str)
def test_non_finite_stays_in_its_sequence(shape):
    """A NaN or infinity makes its own channel non-finite from its step on, and
    nothing else; the finite entries keep their bounds."""
    (a, _), (b, _), _, (h0, _) = inputs(shape, 4, "f64")
    rng = np.random.default_rng(9)
    for bad in (np.nan, np.inf, -np.inf):
        for x in (a, b):
            x[rng.integers(shape[0]), rng.integers(shape[1]), rng.integers(shape[2])] = bad
    h0[0, 0] = np.inf
    want, mag = ref.recurrence(a, b, h0)
    got = host(forward("f64")(cu(a), cu(b), cu(h0)))
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine)
    assert fine.any() and not fine.all()
    bound = ref.recurrence_bound(mag, "f64", np.where(fine, want, 0).astype(np.float64))
    assert np.all(np.abs(got[fine] - want[fine]) <= bound[fine])


def test_products_that_overflow_meet_a_zero_state():
    """Coefficients whose product overflows, with nothing to multiply: the
    state stays zero as in the loop, then takes the values that follow."""
    T = 3000
    a = np.full((1, T, 2), 1e30)
    b = np.zeros((1, T, 2))
    a[:, 2000:] = 0.5
    b[:, 2000:] = 1.0
    b[0, :, 1] = 0.0
    want, mag = ref.recurrence(a, b)
    got = host(forward("f64")(cu(a), cu(b)))
    check(got, want, ref.recurrence_bound(mag, "f64", want.astype(np.float64)))
    g = np.zeros((1, T, 2))
    g[0, :500, 0] = 1.0
    a2 = a[:, ::-1].copy()
    (ga, gb, g0), mags = ref.recurrence_vjp(a2, b, g)
    got = vjp("f64")(cu(a2), cu(b), cu(g))
    check(host(got[1]), gb, ref.vjp_bounds([gb.astype(np.float64)], [mags[1]], "f64", T)[0])


def test_long_decays_underflow_to_nothing():
    """Small coefficients: the old state vanishes, nothing turns NaN."""
    shape = (1, 4000, 6)
    (_, _), (b, _), _, (h0, _) = inputs(shape, 6, "f64")
    a = np.full(shape, 2.0 ** -40)
    want, mag = ref.recurrence(a, b, h0)
    got = host(forward("f64")(cu(a), cu(b), cu(h0)))
    check(got, want, ref.recurrence_bound(mag, "f64", want.astype(np.float64)))


def test_steps_equal_the_whole():
    """Serving one token at a time: T calls of one step, each from the state
    before, follow the recurrence (each step one FMA: bit for bit the loop)."""
    (a, _), (b, _), _, (h0, _) = inputs((3, 20, 17), 7, "f64")
    f = forward("f64")
    state = cu(h0)
    for t in range(20):
        at, bt = a[:, t:t + 1], b[:, t:t + 1]
        step = f(cu(at), cu(bt), state)
        wide = at[:, 0].astype(ref.LONG) * host(state) + bt[:, 0]
        assert np.all(np.abs(host(step)[:, 0] - wide) <= 2.0 ** -52 * np.abs(wide) + 1e-300)
        state = step[:, 0].contiguous()
    want, mag = ref.recurrence(a, b, h0)
    check(host(state), want[:, -1], ref.recurrence_bound(mag, "f64", want.astype(np.float64))[:, -1])


@pytest.mark.parametrize("kind", KINDS)
def test_views_off_the_vector_boundary_and_guards(kind):
    """Operands one row into their storage; results inside a larger buffer
    whose other values stay as they were."""
    shape = (1, 701, 5)
    (a, _), (b, _), (g, _), (h0, _) = inputs(shape, 8, kind)
    f = forward(kind)
    want = host(f(cu(a), cu(b), cu(h0)))
    flat = [x.reshape((-1,) + x.shape[3:]) for x in (a, b)]
    ma, mb = (misaligned(x).reshape(a.shape) for x in flat)
    n = want.size
    buf = torch.full((n + 64,), 7.0, dtype=torch.float64 if kind == "f64" else torch.float32,
                     device="cuda")
    out = buf[32:32 + n].view(want.shape)
    assert f(ma, mb, cu(h0), out=out) is out
    assert np.array_equal(host(out), want)
    edge = host(buf)
    assert np.all(edge[:32] == 7.0) and np.all(edge[32 + n:] == 7.0)
    res = vjp(kind)(ma, cu(want), cu(g), cu(h0))
    again = vjp(kind)(cu(a), cu(want), cu(g), cu(h0))
    assert all(torch.equal(x, y) for x, y in zip(res, again))


def test_results_repeat_bit_for_bit():
    (a, _), (b, _), (g, _), (h0, _) = inputs((2, 6000, 40), 10, "f64")
    ta, tb, tg, th = cu(a), cu(b), cu(g), cu(h0)
    h = forward("f64")(ta, tb, th)
    first = vjp("f64")(ta, h, tg, th)
    for _ in range(5):
        assert torch.equal(forward("f64")(ta, tb, th), h)
        assert all(torch.equal(x, y) for x, y in zip(vjp("f64")(ta, h, tg, th), first))


def test_streams_and_graphs():
    """On a side stream; captured twice (each graph with scratch of its own)
    and replayed with other inputs, interleaved with eager calls."""
    shape = (2, 5000, 24)
    (a, _), (b, _), (g, _), (h0, _) = inputs(shape, 11, "f64")
    f, v = forward("f64"), vjp("f64")
    ta, tb, tg, th = cu(a), cu(b), cu(g), cu(h0)
    want = f(ta, tb, th)
    grads = v(ta, want, tg, th)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = f(ta, tb, th)
        others = v(ta, other, tg, th)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want) and all(torch.equal(x, y) for x, y in zip(grads, others))
    sa, sb = ta.clone(), tb.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = f(sa, sb, th)
    with torch.cuda.graph(g2):
        o2 = v(sa, want, tg, th)
    for scale in (1.0, 0.5, -1.0):
        sb.copy_(tb * scale)
        sa.copy_(ta * abs(scale))
        g2.replay()
        g1.replay()
        eager = f(sa, sb, th)
        assert torch.equal(o1, eager)
        assert all(torch.equal(x, y) for x, y in zip(o2, v(sa, want, tg, th)))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device():
    (a, _), (b, _), _, (h0, _) = inputs((2, 3000, 8), 12, "f64")
    want = host(forward("f64")(cu(a), cu(b), cu(h0)))
    got = forward("f64")(*(torch.from_numpy(x).to("cuda:1") for x in (a, b, h0)))
    assert np.array_equal(got.cpu().numpy(), want)


def test_threads_on_one_stream():
    """Two host threads launch on one stream in any order: their calls do not
    meet in a workspace."""
    from concurrent.futures import ThreadPoolExecutor
    from ds_b200 import ops
    values = [inputs((1, 5000, 12), 20 + i, "f64") for i in range(2)]
    seqs = [(cu(v[0][0]), cu(v[1][0])) for v in values]
    rng = np.random.default_rng(5)
    rows = [cu(rng.standard_normal((9, 1024))) for _ in range(2)]
    W = cu(rng.standard_normal((4, 1024, 96)))
    s = torch.tensor([2, 0, 3, 1], dtype=torch.int32, device="cuda")

    def run(i):
        return (ops.ds_linear_recurrence_f64(*seqs[i]), ops.ds_ragged_dot_f64(rows[i], W, s))
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(2) as pool:
        for i, got in enumerate(pool.map(lambda i: [run(i) for _ in range(100)], range(2))):
            for g in got:
                assert all(torch.equal(x, y) for x, y in zip(g, want[i]))


def test_ds_tensors_keep_their_pairs():
    """DSTensor's recurrence and grouped product are the packed and f64 targets on
    its pairs; a pending expression enters as its pairs."""
    from ds_b200 import ops
    from ds_b200.dstensor import DSTensor
    (a, _), (b, _), _, (h0, _) = inputs((2, 40, 6), 13, "f64")
    A, B, H = (DSTensor.from_f64(cu(x)) for x in (a, b, h0))
    h = A.linear_recurrence(B * 2.0, H)
    want = ops.ds_linear_recurrence_packed(A.packed, (B * 2.0).packed, H.packed)
    assert torch.equal(h.packed, want) and h.shape == (2, 40, 6)
    assert torch.equal(A.linear_recurrence(B).packed,
                       ops.ds_linear_recurrence_packed(A.packed, B.packed))
    w = np.random.default_rng(0).standard_normal((3, 6, 5))
    s = torch.tensor([10, 0, 30], dtype=torch.int32, device="cuda")
    W, X = DSTensor.from_f64(cu(w)), DSTensor.from_f64(cu(a[0]))
    got = X.ragged_matmul(W, s)
    want = ops.ds_from_f64(ops.ds_ragged_dot_f64(X.to_f64(), W.to_f64(), s))
    assert torch.equal(got.packed, want)
    with pytest.raises(TypeError, match="DSTensor"):
        A.linear_recurrence(cu(b))
    with pytest.raises(TypeError, match="DSTensor"):
        X.ragged_matmul(cu(w), s)


def test_calls_through_the_registry():
    """ffi_call by target name gives what ops gives, with and without h0."""
    from ds_b200 import ffi, ops
    (a, _), (b, _), (g, _), (h0, _) = inputs((2, 70, 6), 14, "f64")
    ta, tb, tg, th = cu(a), cu(b), cu(g), cu(h0)
    spec = ffi.ShapeDtypeStruct(ta.shape, torch.float64)
    state = ffi.ShapeDtypeStruct(th.shape, torch.float64)
    h = ops.ds_linear_recurrence_f64(ta, tb, th)
    for _ in range(2):
        assert torch.equal(ffi.ffi_call("ds_linear_recurrence_f64", spec)(ta, tb, th), h)
    assert torch.equal(ffi.ffi_call("ds_linear_recurrence_f64", spec)(ta, tb, None),
                       ops.ds_linear_recurrence_f64(ta, tb))
    got = ffi.ffi_call("ds_linear_recurrence_vjp_f64", (spec, spec, state))(ta, h, tg, th)
    want = ops.ds_linear_recurrence_vjp_f64(ta, h, tg, th)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    with pytest.raises(ValueError, match="output shape"):
        ffi.ffi_call("ds_linear_recurrence_f64", state)(ta, tb, th)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ffi.ffi_call("ds_linear_recurrence_f64", spec)(ta, None, th)


def test_refusals_on_device():
    f = forward("f64")
    x = torch.zeros((2, 8, 4), dtype=torch.float64, device="cuda")
    with pytest.raises(TypeError, match="float64"):
        f(x, x.float())
    with pytest.raises(ValueError, match="contiguous"):
        f(x.transpose(1, 2), x)
    with pytest.raises(ValueError, match="same shape"):
        f(x, x[:1])
    with pytest.raises(ValueError, match="h0"):
        f(x, x, torch.zeros((2, 8), dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="overlaps"):
        f(x, x, out=x)
    with pytest.raises(ValueError, match=r"\[..., T, D\]"):
        f(x[0, 0], x[0, 0])
    buf = torch.zeros(2 * 8 * 4 * 2 + 1, device="cuda")
    odd = buf[1:].view(2, 8, 4, 2)
    with pytest.raises(ValueError, match="aligned"):
        forward("packed")(odd, odd)
