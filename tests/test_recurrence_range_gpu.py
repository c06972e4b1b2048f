"""The linear recurrence and its gradient where products of coefficients leave
the f64 range and no state does, against the step-by-step loop in long double
(tests/sequence_ref.py, with the bounds): every state lies within 2^-950 and 2^950,
so the loop in f64 rounds each step by 2^-53 of it and nothing else."""
import numpy as np
import pytest

import sequence_ref as ref
from gpu_util import cu, host

pytestmark = pytest.mark.gpu

KINDS = ["f64", "f32", "packed"]
# chunks of a block's own, and chunks shared out (a few, some and many channels)
SHAPES = [(1, 64, 1), (2, 513, 4), (1, 5000, 3), (1, 9000, 70), (3, 700, 33), (2, 1500, 1024),
          (2, 600, 8192)]


def forward(kind):
    from ds_b200 import ops
    return getattr(ops, f"ds_linear_recurrence_{kind}")


def vjp(kind):
    from ds_b200 import ops
    return getattr(ops, f"ds_linear_recurrence_vjp_{kind}")


def val(t, kind):
    x = host(t)
    return ref.value_of(x) if kind == "packed" else x.astype(np.float64)


def power(rng, e):
    """Random signs and mantissas at the exponents e."""
    m = rng.uniform(1.0, 2.0, e.shape) * np.where(rng.random(e.shape) < 0.5, -1.0, 1.0)
    return np.ldexp(m, e.astype(np.int64))


def walk(shape, kind, seed, resets=0.0):
    """(a, b, h0): a state that starts at h0 and is multiplied by coefficients of up
    to 2^800 (f32 and pairs: 2^100), whose exponents wander up and down
    between -900 and 900; where it starts again (a share `resets` of the steps) a = 0
    and b is the new state."""
    rng = np.random.default_rng(seed)
    B, T, D = shape
    step, wide = (800, 900) if kind == "f64" else (100, 900)
    start = 300 if kind == "f64" else 60
    h0 = power(rng, rng.integers(-start, start + 1, (B, D)))
    state, up = h0.copy(), rng.random((B, D)) < 0.5
    a, b = np.empty(shape), np.zeros(shape)
    for t in range(T):
        e = np.frexp(state)[1]
        d = rng.integers(0, step + 1, (B, D))
        up ^= np.abs(np.where(up, e + d, e - d)) > wide - 4
        d = np.where(np.abs(np.where(up, e + d, e - d)) > wide - 4, d // 2, d)
        a[:, t] = power(rng, np.where(up, d, -d))
        again = rng.random((B, D)) < resets
        a[:, t][again] = 0.0
        b[:, t][again] = power(rng, rng.integers(-start, start + 1, (B, D)))[again]
        state = a[:, t] * state + b[:, t]
    return [ref.as_type(x, kind) for x in (a, b, h0)]


def bursts(shape, kind, seed):
    """Ordinary gates and values; now and then a channel starts again from a tiny
    value, grows by more than the range, and starts again from an ordinary one."""
    rng = np.random.default_rng(seed)
    B, T, D = shape
    a = 1.0 / (1.0 + np.exp(-2.0 - 1.5 * rng.standard_normal(shape)))
    b = rng.standard_normal(shape)
    big = [0.0, 2.0 ** 900, 2.0 ** 900] if kind == "f64" else \
        [0.0] + [2.0 ** -120] * 6 + [2.0 ** 120] * 9
    first = 2.0 ** (-990 if kind == "f64" else -126)
    for i in range(B):
        for c in range(D):
            for t in rng.integers(0, T, max(1, T // 200)):
                n = min(len(big), T - t)
                a[i, t:t + n, c], b[i, t:t + n, c] = big[:n], 0.0
                b[i, t, c] = first
                if t + n < T:
                    a[i, t + n, c] = 0.0
    return [ref.as_type(x, kind) for x in (a, b, rng.standard_normal((B, D)))]


def check(got, want, bound, kind, what=""):
    """Where the result's type holds the value."""
    seen = np.abs(want) < 2.0 ** (960 if kind == "f64" else 100)
    assert seen.all() or kind != "f64"
    err = np.abs(got[seen].astype(ref.LONG) - want[seen])
    assert np.all(np.isfinite(got[seen])), what
    assert np.all(err <= bound[seen]), \
        f"{what}: {float(np.max(err / np.maximum(bound[seen], 1e-300)))} bounds"


def forward_case(a, b, h0, kind):
    want, mag = ref.recurrence(a[1], b[1], h0[1])
    got = val(forward(kind)(cu(a[0]), cu(b[0]), cu(h0[0])), kind)
    check(got, want, ref.recurrence_bound(mag, kind, want.astype(np.float64)), kind)


def gradient_case(a, b, h0, kind):
    """The forward case backwards in time: g_{T-1} = h0 to begin with, the
    coefficients and values in reverse."""
    shape = a[1].shape
    turned = [np.concatenate([np.zeros_like(x[0][:, :1]), x[0][:, ::-1]], axis=1)
              for x in (a, b)]
    if kind == "packed":
        turned[0][:, 0, :, 0] = 1.0
    else:
        turned[0][:, 0] = 1.0
    # grad_h at the last step is h0, before it (reversed) b; a_{t+1} pairs with step t
    g = np.concatenate([turned[1][:, 1:], h0[0][:, None]], axis=1)
    av, gv = (ref.value_of(x) if kind == "packed" else x.astype(np.float64)
              for x in (turned[0], g))
    rng = np.random.default_rng(3)
    h = ref.as_type(rng.uniform(0.5, 1.0, av.shape), kind)
    s = ref.as_type(rng.uniform(0.5, 1.0, (shape[0], shape[2])), kind)
    want, mag = ref.recurrence_vjp(av, h[1], gv, s[1])
    got = vjp(kind)(cu(turned[0]), cu(h[0]), cu(np.ascontiguousarray(g)), cu(s[0]))
    bounds = ref.vjp_bounds([w.astype(np.float64) for w in want], mag, kind, av.shape[1])
    for x, w, e, name in zip(got, want, bounds, ("grad_a", "grad_b", "grad_h0")):
        check(val(x, kind), w, e, kind, name)


def test_a_reset_after_an_overflowing_product():
    """The shortest case: states 1e-100, 1e100, 1, then a half each step plus one."""
    T = 64
    a, b = np.full((1, T, 1), 0.5), np.ones((1, T, 1))
    a[0, :3, 0], b[0, :3, 0] = (1e200, 1e200, 0.0), (0.0, 0.0, 1.0)
    h0 = np.full((1, 1), 1e-300)
    cases = [(x, x) for x in (a, b, h0)]
    forward_case(*cases, "f64")
    gradient_case(*cases, "f64")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_bursts_between_resets(shape, kind):
    forward_case(*bursts(shape, kind, 1), kind)
    gradient_case(*bursts(shape, kind, 2), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_states_that_wander_over_the_range(shape, kind):
    """Products overflow and underflow in every chunk, with resets and without."""
    for seed, resets in ((3, 0.0), (4, 0.02)):
        forward_case(*walk(shape, kind, seed, resets), kind)
        gradient_case(*walk(shape, kind, seed + 10, resets), kind)


@pytest.mark.parametrize("shape", [(1, 5000, 64), (2, 700, 8192)], ids=str)
def test_other_channels_keep_their_bits(shape):
    """A channel whose products leave the range changes no bit of the others, and
    results repeat."""
    rng = np.random.default_rng(5)
    a = 1.0 / (1.0 + np.exp(-2.0 - 1.5 * rng.standard_normal(shape)))
    b, h0 = rng.standard_normal(shape), rng.standard_normal((shape[0], shape[2]))
    f = forward("f64")
    plain = host(f(cu(a), cu(b), cu(h0)))
    wa, wb, wh = (x[0] for x in walk((1, shape[1], 1), "f64", 6, 0.01))
    a[0, :, 5], b[0, :, 5], h0[0, 5] = wa[0, :, 0], wb[0, :, 0], wh[0, 0]
    got = host(f(cu(a), cu(b), cu(h0)))
    other = np.ones(shape, bool)
    other[0, :, 5] = False
    assert np.array_equal(got[other], plain[other])
    for _ in range(5):
        assert np.array_equal(host(f(cu(a), cu(b), cu(h0))), got)
