"""Products grouped by expert and the contraction over each group on the GPU,
against the host's products (tests/sequence_ref.py, with the bounds)."""
import numpy as np
import pytest
import torch

import sequence_ref as ref
from gpu_util import cu, host

pytestmark = pytest.mark.gpu

# (M, K, N, group sizes)
CASES = [
    (1, 1, 1, [1]),
    (5, 3, 2, [2, 0, 3]),
    (7, 1, 9, [0, 0, 7, 0]),
    (16, 33, 65, [1] * 12 + [4]),
    (9, 64, 130, [3, 2]),                  # rows behind the last group
    (40, 20, 17, [-3, 10, 0, 50]),         # a negative size; a group past row M
    (130, 77, 66, [64, 65, 1]),
    (300, 129, 255, [0, 299, 0, 1]),
    (700, 256, 260, [300, 8, 129, 257]),
    (1030, 300, 515, [600, 17, 0, 400]),
    (64, 513, 40, [17, 16, 15, 8, 8]),
    (520, 128, 512, [520]),
    (600, 140, 300, [150, 0, 0, 450]),
]
IDS = [f"{m}x{k}x{n}/{len(s)}" for m, k, n, s in CASES]
# a graph of G groups replayed with these sizes
SIZES = [[300, 8, 129, 257], [0, 0, 0, 700], [175] * 4, [1, 2, 3, 4], [0] * 4, [700, 1, -1, 9]]


def sz(sizes):
    return torch.tensor(sizes, dtype=torch.int32, device="cuda")


def make(case, seed=0):
    M, K, N, sizes = case
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((M, K)), rng.standard_normal((len(sizes), K, N)),
            rng.standard_normal((M, N)), sizes)


def check(got, want, bound, what=""):
    err = np.abs(got - want)
    assert np.all(err <= bound), f"{what}: {float(np.max(err / np.maximum(bound, 1e-300)))} bounds"


def split(x):
    p = ref.pair_of(x)
    return cu(p[..., 0]), cu(p[..., 1]), ref.value_of(p)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_products(case):
    from ds_b200 import ops
    x, w, _, sizes = make(case)
    want, bound = ref.ragged_dot(x, w, sizes)
    check(host(ops.ds_ragged_dot_f64(cu(x), cu(w), sz(sizes))), want, bound, "plain")
    wt = np.ascontiguousarray(w.transpose(0, 2, 1))
    check(host(ops.ds_ragged_dot_f64(cu(x), cu(wt), sz(sizes), rhs_contracting=2)), want, bound,
          "transposed")


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_products_of_pairs(case):
    from ds_b200 import ops
    x, w, _, sizes = make(case, 1)
    xh, xl, xv = split(x)
    wh, wl, wv = split(w)
    want, bound = ref.ragged_dot(xv, wv, sizes, "pair")
    hi, lo = ops.ds_ragged_dot(xh, xl, wh, wl, sz(sizes))
    check(ref.value_of(host(torch.stack([hi, lo], -1))), want, bound)
    wth, wtl, _ = split(np.ascontiguousarray(w.transpose(0, 2, 1)))
    hi, lo = ops.ds_ragged_dot(xh, xl, wth, wtl, sz(sizes), rhs_contracting=2)
    check(ref.value_of(host(torch.stack([hi, lo], -1))), want, bound)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_contraction(case):
    from ds_b200 import ops
    x, _, y, sizes = make(case, 2)
    want, bound = ref.ragged_contract(x, y, sizes)
    check(host(ops.ds_ragged_dot_contract_f64(cu(x), cu(y), sz(sizes))), want, bound)
    xh, xl, xv = split(x)
    yh, yl, yv = split(y)
    want, bound = ref.ragged_contract(xv, yv, sizes, "pair")
    hi, lo = ops.ds_ragged_dot_contract(xh, xl, yh, yl, sz(sizes))
    check(ref.value_of(host(torch.stack([hi, lo], -1))), want, bound)


@pytest.mark.parametrize("M,K,G", [(4096, 24, 32), (4160, 24, 32), (900, 40, 33), (9000, 12, 1300),
                                   (70, 700, 5), (40, 1030, 40)])
def test_tiles_of_every_kind(M, K, G):
    """Groups of 0 to 200 rows, so that tails of every size stand behind the full
    tiles; as many groups and tiles as a block plans for itself, one more, and
    more than a pass of the planning kernel takes; contractions in several parts."""
    from ds_b200 import ops
    rng = np.random.default_rng(M + G)
    sizes = rng.integers(0, max(2, min(200, 2 * M // G)), G).tolist()
    x, w, y, _ = make((M, K, 30, sizes), 3)
    want, bound = ref.ragged_dot(x, w, sizes)
    check(host(ops.ds_ragged_dot_f64(cu(x), cu(w), sz(sizes))), want, bound)
    want, bound = ref.ragged_contract(x, y, sizes)
    check(host(ops.ds_ragged_dot_contract_f64(cu(x), cu(y), sz(sizes))), want, bound)


@pytest.mark.parametrize("M,K,N,G", [(0, 4, 5, 3), (6, 0, 5, 3), (6, 4, 0, 3), (6, 4, 5, 0)])
def test_empty(M, K, N, G):
    """No rows, columns or groups: nothing; no contraction or no group: zeros."""
    from ds_b200 import ops
    x = torch.ones((M, K), dtype=torch.float64, device="cuda")
    w = torch.ones((G, K, N), dtype=torch.float64, device="cuda")
    y = torch.ones((M, N), dtype=torch.float64, device="cuda")
    s = sz([2] * G)
    out = ops.ds_ragged_dot_f64(x, w, s)
    assert out.shape == (M, N) and not out.any()
    out = ops.ds_ragged_dot_contract_f64(x, y, s)
    assert out.shape == (G, K, N)
    if M == 0:
        assert not out.any()


@pytest.mark.parametrize("sizes", [[200, 0, 300, 100], [40, 500, 20, 30]], ids=str)
def test_non_finite_stays_in_its_group(sizes):
    """NaN and infinities in a row, in a matrix, in unused rows and in an
    unused matrix reach the outputs that read them and no others."""
    from ds_b200 import ops
    M, K, N = 620, 130, 258
    x, w, y, sizes = make((M, K, N, sizes), 3)
    used = sum(sizes)
    ends = np.cumsum(sizes)
    want, bound = ref.ragged_dot(x, w, sizes)
    wantc, boundc = ref.ragged_contract(x, y, sizes)
    bad = np.zeros((M, N), bool)
    badc = np.zeros((len(sizes), K, N), bool)
    x[used:], y[used:] = np.nan, np.inf      # behind the last group: not read
    if sizes[1] == 0:
        w[1] = np.nan                        # nobody's matrix
    x[3, 7] = np.nan
    bad[3] = True
    badc[0, 7] = True
    w[2, 5, 11] = np.inf
    bad[ends[1]:ends[2], 11] = True
    y[ends[2] + 1, 20] = -np.inf
    badc[3, :, 20] = True
    with np.errstate(invalid="ignore"):
        got = host(ops.ds_ragged_dot_f64(cu(x), cu(w), sz(sizes)))
        gotc = host(ops.ds_ragged_dot_contract_f64(cu(x), cu(y), sz(sizes)))
        assert np.array_equal(~np.isfinite(got), bad)
        assert np.array_equal(~np.isfinite(gotc), badc)
        assert np.all(np.abs(got - want)[~bad] <= bound[~bad])
        assert np.all(np.abs(gotc - wantc)[~badc] <= boundc[~badc])
    assert not got[used:].any()


def test_wide_range_within_rows():
    """Values spread over 60 binades inside rows and columns, large entries
    facing zeros: every output stays within the f64 sums' bound of its own
    terms or 2^-24 of the result (the certificate of the tensor-core path,
    whose uncertified outputs are summed again)."""
    from ds_b200 import ops
    rng = np.random.default_rng(4)
    M, K, N, sizes = 600, 200, 260, [300, 280, 20]
    x = rng.standard_normal((M, K)) * 2.0 ** rng.integers(-60, 1, (M, K))
    w = rng.standard_normal((3, K, N)) * 2.0 ** rng.integers(-60, 1, (3, K, N))
    x[:, 0], w[:, 0] = 2.0 ** 40, 0.0
    y = rng.standard_normal((M, N)) * 2.0 ** rng.integers(-60, 1, (M, N))
    for got, (want, _), terms in (
            (ops.ds_ragged_dot_f64(cu(x), cu(w), sz(sizes)), ref.ragged_dot(x, w, sizes),
             ref.ragged_dot(np.abs(x), np.abs(w), sizes)[0]),
            (ops.ds_ragged_dot_contract_f64(cu(x), cu(y), sz(sizes)),
             ref.ragged_contract(x, y, sizes),
             ref.ragged_contract(np.abs(x), np.abs(y), sizes)[0])):
        bound = (600 + 2) * 2 * ref.U * terms + 2.0 ** -24 * np.abs(want)
        check(host(got), want, bound)


def test_results_repeat_and_guards():
    """The same bits every time; nothing outside the result is written, the
    rows behind the last group become zeros."""
    from ds_b200 import ops
    x, w, y, sizes = make((700, 256, 260, [300, 8, 129, 150]), 5)
    tx, tw, ty, s = cu(x), cu(w), cu(y), sz(sizes)
    for call, shape in ((lambda out: ops.ds_ragged_dot_f64(tx, tw, s, out=out), (700, 260)),
                        (lambda out: ops.ds_ragged_dot_contract_f64(tx, ty, s, out=out),
                         (4, 256, 260))):
        n = int(np.prod(shape))
        buf = torch.full((n + 64,), 7.0, dtype=torch.float64, device="cuda")
        out = buf[32:32 + n].view(shape)
        assert call(out) is out
        first = host(out).copy()
        edge = host(buf)
        assert np.all(edge[:32] == 7.0) and np.all(edge[32 + n:] == 7.0)
        if len(shape) == 2:
            assert not first[587:].any() and first[586].any()
        for _ in range(4):
            out.fill_(float("nan"))
            call(out)
            assert np.array_equal(host(out), first)


def test_unaligned_views():
    """Operands whose rows start off the 16-byte boundary."""
    from ds_b200 import ops
    case = (300, 129, 255, [10, 280, 3])
    x, w, y, sizes = make(case, 6)

    def off(v):
        t = torch.empty(v.size + 1, dtype=torch.float64, device="cuda")
        t[1:] = cu(v).flatten()
        return t[1:].view(v.shape)

    a = ops.ds_ragged_dot_f64(cu(x), cu(w), sz(sizes))
    assert torch.equal(ops.ds_ragged_dot_f64(off(x), off(w), sz(sizes)), a)
    c = ops.ds_ragged_dot_contract_f64(cu(x), cu(y), sz(sizes))
    assert torch.equal(ops.ds_ragged_dot_contract_f64(off(x), off(y), sz(sizes)), c)


def test_graph_replayed_with_other_sizes():
    """Sizes are read on the device: one captured graph serves every split of
    the rows; a second graph and eager calls beside it do not disturb it."""
    from ds_b200 import ops
    x, w, y, _ = make((700, 256, 260, SIZES[0]), 7)
    tx, tw, ty, s = cu(x), cu(w), cu(y), sz(SIZES[0])
    ops.ds_ragged_dot_f64(tx, tw, s)
    ops.ds_ragged_dot_contract_f64(tx, ty, s)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ops.ds_ragged_dot_f64(tx, tw, s)
    with torch.cuda.graph(g2):
        o2 = ops.ds_ragged_dot_contract_f64(tx, ty, s)
    for sizes in SIZES:
        s.copy_(sz(sizes))
        g1.replay()
        g2.replay()
        assert torch.equal(o1, ops.ds_ragged_dot_f64(tx, tw, s))
        assert torch.equal(o2, ops.ds_ragged_dot_contract_f64(tx, ty, s))
        check(host(o1), *ref.ragged_dot(x, w, sizes))
        check(host(o2), *ref.ragged_contract(x, y, sizes))


def test_side_stream():
    from ds_b200 import ops
    x, w, _, sizes = make((700, 256, 260, [300, 8, 129, 257]), 8)
    tx, tw, s = cu(x), cu(w), sz(sizes)
    want = ops.ds_ragged_dot_f64(tx, tw, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.ds_ragged_dot_f64(tx, tw, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


# ---- calls whose large groups take the tensor-core product ---------------------------
# Compared on the GPU with torch's f64 products; the bounds are sequence_ref's.

LARGE = [
    (2100, 1001, 1103, [900, 0, 127, 128, 645, 257]),  # odd sizes, both kinds of groups
    (4100, 1000, 900, [1500, -5, 2000]),               # rows behind the last group
    (3000, 900, 1030, [40, 2900, 100]),                # a group past row M
]
LARGE_IDS = [f"{m}x{k}x{n}/{len(s)}" for m, k, n, s in LARGE]


def on_gpu(*shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64, device="cuda")


def expect(a, b, pairs=False):
    """a @ b and sequence_ref's bound, with torch's own f64 sums (their error is
    the f64 term once more)."""
    K = a.shape[1]
    c, terms = a @ b, a.abs() @ b.abs()
    chunks = -(-K // 32768)
    P = min(50, int((110.2 - 2 - np.log2(min(K, 32768))) // 2))
    if chunks > 1:
        P = int((110.2 - 2 - 15) // 2)
    unit = 4.0 * a.abs().amax(1)[:, None] * b.abs().amax(0)[None, :] * 2.0 ** -P
    f64 = (K + 2) * 2 * ref.U * terms
    bound = f64 + torch.maximum(f64, (K + 2.0 ** (35 - P) * chunks) * unit +
                                (2 + chunks) * ref.U * c.abs())
    return c, bound + (c.abs() * 2.0 ** -48 + 2.0 ** -150 if pairs else 0.0)


def within(got, want, bound):
    assert bool(((got - want).abs() <= bound).all())


class Reached:
    """The calls inside ran the tensor-core product."""

    def __enter__(self):
        from ds_b200 import _lib
        _lib.profile_enable(True)
        _lib.profile_reset()

    def __exit__(self, *exc):
        from ds_b200 import _lib
        n = _lib.profile_read("ozaki_gemm")[1]
        _lib.profile_enable(False)
        if exc[0] is None:
            assert n > 0, "the tensor-core product did not run"


def pair(x):
    hi = x.float()
    return hi, (x - hi.double()).float()


@pytest.mark.parametrize("case", LARGE, ids=LARGE_IDS)
@pytest.mark.parametrize("contracting", [1, 2])
def test_large_products(case, contracting):
    from ds_b200 import ops
    M, K, N, sizes = case
    x, w = on_gpu(M, K, seed=1), on_gpu(len(sizes), K, N, seed=2)
    wt = w if contracting == 1 else w.transpose(1, 2).contiguous()
    s = sz(sizes)
    with Reached():
        out = ops.ds_ragged_dot_f64(x, wt, s, rhs_contracting=contracting)
        hi, lo = ops.ds_ragged_dot(*pair(x), *pair(wt), s, rhs_contracting=contracting)
    end = 0
    for g, b, e in ref.spans(sizes, M):
        if e > b:
            within(out[b:e], *expect(x[b:e], w[g]))
            xp, wp = (sum(v.double() for v in pair(t)) for t in (x[b:e], w[g]))
            within(hi[b:e].double() + lo[b:e].double(), *expect(xp, wp, pairs=True))
        end = e
    assert not out[end:].any() and not hi[end:].any() and not lo[end:].any()
    assert torch.equal(out, ops.ds_ragged_dot_f64(x, wt, s, rhs_contracting=contracting))


@pytest.mark.parametrize("case", [(4100, 1000, 900, [1500, -5, 2000]),
                                  (5000, 901, 1103, [255, 2000, 0, 256, 1700, 30])],
                         ids=["even", "odd"])
def test_large_contraction(case):
    from ds_b200 import ops
    M, K, N, sizes = case
    x, y, s = on_gpu(M, K, seed=3), on_gpu(M, N, seed=4), sz(sizes)
    with Reached():
        out = ops.ds_ragged_dot_contract_f64(x, y, s)
        hi, lo = ops.ds_ragged_dot_contract(*pair(x), *pair(y), s)
    for g, b, e in ref.spans(sizes, M):
        if e > b:
            within(out[g], *expect(x[b:e].T, y[b:e]))
            xp, yp = (sum(v.double() for v in pair(t)) for t in (x[b:e], y[b:e]))
            within(hi[g].double() + lo[g].double(), *expect(xp.T, yp, pairs=True))
        else:
            assert not out[g].any() and not hi[g].any() and not lo[g].any()
    assert torch.equal(out, ops.ds_ragged_dot_contract_f64(x, y, s))


def test_large_views_off_the_boundary_and_guards():
    """Operands one value into their storage, results inside a larger buffer."""
    from ds_b200 import ops
    M, K, N, sizes = LARGE[0]
    x, w, s = on_gpu(M, K, seed=5), on_gpu(len(sizes), K, N, seed=6), sz(sizes)

    def off(t):
        v = torch.empty(t.numel() + 1, dtype=torch.float64, device="cuda")
        v[1:] = t.flatten()
        return v[1:].view(t.shape)

    want = ops.ds_ragged_dot_f64(x, w, s)
    buf = torch.full((M * N + 65,), 7.0, dtype=torch.float64, device="cuda")
    out = buf[33:33 + M * N].view(M, N)
    ops.ds_ragged_dot_f64(off(x), off(w), s, out=out)
    assert torch.equal(out, want)
    assert bool((buf[:33] == 7.0).all()) and bool((buf[33 + M * N:] == 7.0).all())
    M, K, N, sizes = 4100, 1000, 901, [1500, 0, 2000]
    x, y, s = on_gpu(M, K, seed=7), on_gpu(M, N, seed=8), sz(sizes)
    want = ops.ds_ragged_dot_contract_f64(x, y, s)
    n = want.numel()
    buf = torch.full((n + 65,), 7.0, dtype=torch.float64, device="cuda")
    out = buf[33:33 + n].view(want.shape)
    with Reached():
        ops.ds_ragged_dot_contract_f64(off(x), off(y), s, out=out)
    assert torch.equal(out, want)
    assert bool((buf[:33] == 7.0).all()) and bool((buf[33 + n:] == 7.0).all())


def test_large_non_finite_stays_in_its_group():
    from ds_b200 import ops
    M, K, N, sizes = 4100, 1000, 900, [1500, 0, 2000, 300]
    x, w, y = on_gpu(M, K, seed=9), on_gpu(4, K, N, seed=10), on_gpu(M, N, seed=11)
    s = sz(sizes)
    bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    badc = torch.zeros((4, K, N), dtype=torch.bool, device="cuda")
    want, wantc = (f(*v, s) for f, v in ((ops.ds_ragged_dot_f64, (x, w)),
                                         (ops.ds_ragged_dot_contract_f64, (x, y))))
    w[1] = float("nan")                     # nobody's matrix
    x[3800:], y[3800:] = float("nan"), float("inf")  # behind the last group
    x[3, 7] = float("nan")
    bad[3], badc[0, 7] = True, True
    w[2, 5, 11] = float("inf")
    bad[1500:3500, 11] = True
    y[3600, 20] = -float("inf")
    badc[3, :, 20] = True
    with Reached():
        got, gotc = ops.ds_ragged_dot_f64(x, w, s), ops.ds_ragged_dot_contract_f64(x, y, s)
    assert torch.equal(~got.isfinite(), bad)
    assert torch.equal(~gotc.isfinite(), badc)
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(gotc[~badc], wantc[~badc])
    assert not got[3800:].any()


def test_large_zero_rows_columns_and_wide_range():
    """Rows and columns of zeros give exact zeros; with values over 60 binades
    and large entries facing zeros most outputs fail the certificate and are
    summed again: each stays within 2^-24 of itself or the f64 sums' bound."""
    from ds_b200 import ops
    M, K, N, sizes = 4100, 700, 1000, [1500, 0, 2000, 300]
    g = torch.Generator(device="cuda")
    g.manual_seed(12)

    def spread(t):
        e = torch.randint(-60, 1, t.shape, generator=g, device="cuda")
        return t * torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), e)

    x, w, y = spread(on_gpu(M, K, seed=13)), spread(on_gpu(4, K, N, seed=14)), \
        spread(on_gpu(M, N, seed=15))
    x[:, 0], w[:, 0] = 2.0 ** 40, 0.0
    x[5], w[2, :, 9], y[:1500, 4] = 0.0, 0.0, 0.0
    s = sz(sizes)
    with Reached():
        out, outc = ops.ds_ragged_dot_f64(x, w, s), ops.ds_ragged_dot_contract_f64(x, y, s)
    assert not out[5].any() and not out[1500:3500, 9].any() and not outc[0, :, 4].any()
    for i, b, e in ref.spans(sizes, M):
        for got, p, q in ((out[b:e], x[b:e], w[i]), (outc[i], x[b:e].T, y[b:e])):
            if e > b:
                terms = p.abs() @ q.abs()
                within(got, p @ q, (p.shape[1] + 2) * 4 * ref.U * terms + 2.0 ** -24 * got.abs())


def test_large_scales_beyond_the_range():
    """Rows times 2^-800 and columns times 2^-200: their scale exponents together
    leave the f64 range, the results (about 2^-1000) do not, and scaling by powers
    of two changes no bit of them."""
    from ds_b200 import ops
    M, K, N, sizes = 4100, 700, 1000, [1500, 0, 2000, 300]
    x, w, y = on_gpu(M, K, seed=30), on_gpu(4, K, N, seed=31), on_gpu(M, N, seed=32)
    s = sz(sizes)

    def scale(n, e):
        return torch.where(torch.arange(n, device="cuda") % 3 == 0, 2.0 ** e, 1.0).double()
    rows, feats, cols = scale(M, -800), scale(K, -800), scale(N, -200)
    cases = (
        (lambda a, b: ops.ds_ragged_dot_f64(a, b, s), x, w, rows[:, None], cols,
         rows[:, None] * cols),
        (lambda a, b: ops.ds_ragged_dot_f64(a, b.transpose(1, 2).contiguous(), s,
                                            rhs_contracting=2), x, w, rows[:, None], cols,
         rows[:, None] * cols),
        (lambda a, b: ops.ds_ragged_dot_contract_f64(a, b, s), x, y, feats, cols,
         feats[:, None] * cols))
    for f, a, b, sa, sb, want in cases:
        with Reached():
            base, got = f(a, b), f(a * sa, b * sb)
        far = base.abs() > 2.0 ** -20  # those below may become subnormal
        assert torch.equal(got[far], (base * want)[far]) and bool(far.any())
        assert bool(((got - base * want).abs() <= 2.0 ** -1073).all())


def test_large_subnormal_rows():
    """Rows and matrices whose every value is subnormal, with nothing in its high
    word, keep all their bits: integers times the smallest f64."""
    from ds_b200 import ops
    M, K, N, sizes = 4100, 700, 1000, [1500, 0, 2000, 300]
    g = torch.Generator(device="cuda")
    g.manual_seed(40)

    def ints(*shape):
        return torch.randint(-2 ** 20, 2 ** 20, shape, generator=g, device="cuda").double()
    x, w, s = ints(M, K), ints(4, K, N), sz(sizes)
    tiny, back = 2.0 ** -1074, 2.0 ** 500
    with Reached():
        base = ops.ds_ragged_dot_f64(x, w, s)
        rows = ops.ds_ragged_dot_f64(x * tiny, w * back, s)
        wt = (w * tiny).transpose(1, 2).contiguous()
        cols = ops.ds_ragged_dot_f64(x * back, wt, s, rhs_contracting=2)
    assert torch.equal(rows, base * 2.0 ** -574) and torch.equal(cols, rows) and bool(base.any())


def test_large_graph_replayed_with_other_sizes():
    """One captured graph for every split of the rows: groups change kind."""
    from ds_b200 import ops
    M, K, N = 4100, 1000, 900
    x, w, y = on_gpu(M, K, seed=16), on_gpu(4, K, N, seed=17), on_gpu(M, N, seed=18)
    s = sz([1500, 0, 2000, 300])
    ops.ds_ragged_dot_f64(x, w, s)
    ops.ds_ragged_dot_contract_f64(x, y, s)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ops.ds_ragged_dot_f64(x, w, s)
    with torch.cuda.graph(g2):
        o2 = ops.ds_ragged_dot_contract_f64(x, y, s)
    for sizes in ([1500, 0, 2000, 300], [0, 0, 0, 4100], [1, 127, 128, 129], [0] * 4,
                  [255, 256, 257, 3000], [4100, 5, 5, -1]):
        s.copy_(sz(sizes))
        g2.replay()
        g1.replay()
        assert torch.equal(o1, ops.ds_ragged_dot_f64(x, w, s))
        assert torch.equal(o2, ops.ds_ragged_dot_contract_f64(x, y, s))
        end = 0
        for i, b, e in ref.spans(sizes, M):
            if e > b:
                within(o1[b:e], *expect(x[b:e], w[i]))
                within(o2[i], *expect(x[b:e].T, y[b:e]))
            else:
                assert not o2[i].any()
            end = e
        assert not o1[end:].any()


def test_long_contractions():
    """Contractions above 32768, which the tensor-core product takes in chunks."""
    from ds_b200 import ops
    n = 33000 + 41
    x, w = on_gpu(700, n, seed=19), on_gpu(3, n, 300, seed=20)
    wt = w.transpose(1, 2).contiguous()
    out = ops.ds_ragged_dot_f64(x, w, sz([400, 40, 250]))
    outt = ops.ds_ragged_dot_f64(x, wt, sz([400, 40, 250]), rhs_contracting=2)
    for g, b, e in ref.spans([400, 40, 250], 700):
        within(out[b:e], *expect(x[b:e], w[g]))
        within(outt[b:e], *expect(x[b:e], w[g]))
    assert not out[690:].any()
    x, w = on_gpu(1100, n, seed=23), on_gpu(2, n, 500, seed=24)
    wt = w.transpose(1, 2).contiguous()
    with Reached():
        out = ops.ds_ragged_dot_f64(x, w, sz([600, 490]))
    with Reached():
        outt = ops.ds_ragged_dot_f64(x, wt, sz([600, 490]), rhs_contracting=2)
    for g, b, e in ref.spans([600, 490], 1100):
        within(out[b:e], *expect(x[b:e], w[g]))
        within(outt[b:e], *expect(x[b:e], w[g]))
    assert not out[1090:].any()
    x, y = on_gpu(n, 300, seed=21), on_gpu(n, 400, seed=22)
    for sizes in ([n - 3, 3], [100, 32700, 241], [0, 32768, 0, 273], [32500, 541],
                  [32768 - 100, 100, 273]):
        with Reached():
            out = ops.ds_ragged_dot_contract_f64(x, y, sz(sizes))
            hi, lo = ops.ds_ragged_dot_contract(*pair(x), *pair(y), sz(sizes))
        xp, yp = (sum(v.double() for v in pair(t)) for t in (x, y))
        for g, b, e in ref.spans(sizes, n):
            if e > b:
                within(out[g], *expect(x[b:e].T, y[b:e]))
                want, bound = expect(xp[b:e].T, yp[b:e], pairs=True)
                # the pairs of two chunks are rounded twice
                within(hi[g].double() + lo[g].double(), want, bound + want.abs() * 2.0 ** -47)
            else:
                assert not out[g].any() and not hi[g].any()


def test_gradients_are_the_adjoint():
    """<grad, f(x, w)> is linear in x and in w: moving x (w) by d changes it by
    <grad_x, d> (<grad_w, d>), to the rounding of the sums (their bound: 2000
    roundings of the magnitudes' sum)."""
    from ds_b200 import ops
    x, w, g, sizes = make((300, 129, 255, [10, 200, 60]), 10)
    tx, tw, tg, s = cu(x), cu(w), cu(g), sz(sizes)
    gx = host(ops.ds_ragged_dot_f64(tg, tw, s, rhs_contracting=2))
    gw = host(ops.ds_ragged_dot_contract_f64(tx, tg, s))
    rng = np.random.default_rng(1)
    for grad, base, call in ((gx, x, lambda v: ops.ds_ragged_dot_f64(cu(v), tw, s)),
                             (gw, w, lambda v: ops.ds_ragged_dot_f64(tx, cu(v), s))):
        d = rng.standard_normal(base.shape)
        change = float(np.sum(g * (host(call(base + d)) - host(call(base)))))
        size = float(np.sum(np.abs(g) * (np.abs(host(call(base + d))) + np.abs(host(call(base))))))
        assert abs(change - float(np.sum(grad * d))) <= 2000 * ref.U * 2 * size


def test_refusals_on_device():
    from ds_b200 import ops
    x = torch.zeros((8, 4), dtype=torch.float64, device="cuda")
    w = torch.zeros((2, 4, 6), dtype=torch.float64, device="cuda")
    s = sz([4, 4])
    with pytest.raises(TypeError, match="int32"):
        ops.ds_ragged_dot_f64(x, w, s.long())
    with pytest.raises(ValueError, match="contracting"):
        ops.ds_ragged_dot_f64(x, w, s, rhs_contracting=2)
    with pytest.raises(ValueError, match="rhs_contracting"):
        ops.ds_ragged_dot_f64(x, w, s, rhs_contracting=0)
    with pytest.raises(ValueError, match=r"\[G\]"):
        ops.ds_ragged_dot_f64(x, w, sz([8]))
    with pytest.raises(ValueError, match="contiguous"):
        ops.ds_ragged_dot_f64(x, w.transpose(1, 2), s)
    with pytest.raises(ValueError, match="CUDA"):
        ops.ds_ragged_dot_f64(x, w, s.cpu())
    with pytest.raises(ValueError, match="overlaps"):
        ops.ds_ragged_dot_f64(x, torch.zeros((2, 4, 4), dtype=torch.float64, device="cuda"), s,
                              out=x)
    with pytest.raises(ValueError, match="contracting"):
        ops.ds_ragged_dot_contract_f64(x, x[:4], s)


def test_recurrent_experts_layer():
    """The operators as a layer of recurrent experts uses them, forward and
    backward, against autograd of the same layer in torch f64: tokens sorted by
    expert, projected by their expert, put back in time order, run through the
    recurrence, and projected again.  Both sides sum in f64 or better; the
    bound is 2^-30 of each gradient's largest entry."""
    from ds_b200 import ops
    rng = np.random.default_rng(12)
    B, T, D, E, G = 2, 150, 40, 64, 5
    M = B * T
    expert = torch.from_numpy(rng.integers(0, G, M)).cuda()
    order = torch.argsort(expert, stable=True)
    back = torch.argsort(order)
    s = torch.bincount(expert, minlength=G).to(torch.int32)
    x, w1 = cu(rng.standard_normal((M, D))), cu(rng.standard_normal((G, D, E)) / 6)
    w2 = cu(rng.standard_normal((G, E, D)) / 8)
    gate = cu(1 / (1 + np.exp(-2 - rng.standard_normal((B, T, E)))))
    h0, gy = cu(rng.standard_normal((B, E))), cu(rng.standard_normal((M, D)))

    xs = x[order]
    p = ops.ds_ragged_dot_f64(xs, w1, s)
    b = p[back].view(B, T, E)
    h = ops.ds_linear_recurrence_f64(gate, b, h0)
    hs = h.view(M, E)[order]
    y = ops.ds_ragged_dot_f64(hs, w2, s)
    # backward of sum(y gy)
    gw2 = ops.ds_ragged_dot_contract_f64(hs, gy, s)
    gh = ops.ds_ragged_dot_f64(gy, w2, s, rhs_contracting=2)[back].view(B, T, E)
    ggate, gb, gh0 = ops.ds_linear_recurrence_vjp_f64(gate, h, gh, h0)
    gp = gb.view(M, E)[order]
    gw1 = ops.ds_ragged_dot_contract_f64(xs, gp, s)
    gx = ops.ds_ragged_dot_f64(gp, w1, s, rhs_contracting=2)[back]

    leaves = [v.cpu().requires_grad_() for v in (x, w1, w2, gate, h0)]
    lx, lw1, lw2, lg, lh0 = leaves
    e = expert.cpu()
    pb = torch.einsum("md,mde->me", lx, lw1[e]).view(B, T, E)
    state, hist = lh0, []
    for t in range(T):
        state = lg[:, t] * state + pb[:, t]
        hist.append(state)
    yy = torch.einsum("me,med->md", torch.stack(hist, 1).view(M, E), lw2[e])
    (yy[order.cpu()] * gy.cpu()).sum().backward()
    for got, want in ((y[back], yy), (gx, lx.grad), (gw1, lw1.grad), (gw2, lw2.grad),
                      (ggate, lg.grad), (gh0, lh0.grad)):
        got, want = got.cpu(), want.detach()
        assert float((got - want).abs().max()) <= 2.0 ** -30 * float(want.abs().max())


@pytest.mark.parametrize("M,K,N", [(2048, 1024, 1024), (8192, 1024, 1024)])
def test_no_groups_at_batch_size(M, K, N):
    """Zeros, as of a few rows, for f64 and pairs and either layout."""
    from ds_b200 import ops
    x, s = on_gpu(M, K, seed=50), sz([])
    for contracting, shape in ((1, (0, K, N)), (2, (0, N, K))):
        w = torch.empty(shape, dtype=torch.float64, device="cuda")
        out = torch.full((M, N), float("nan"), dtype=torch.float64, device="cuda")
        ops.ds_ragged_dot_f64(x, w, s, rhs_contracting=contracting, out=out)
        assert not out.any()
        hi, lo = ops.ds_ragged_dot(*pair(x), w.float(), w.float(), s, rhs_contracting=contracting)
        assert hi.shape == lo.shape == (M, N) and not hi.any() and not lo.any()
    assert ops.ds_ragged_dot_contract_f64(x, on_gpu(M, N, seed=51), s).shape == (0, K, N)
