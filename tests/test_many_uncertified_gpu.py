"""Tensor-core products with more than 2^31 outputs, none of which the certificate
accepts: every row of the left operand has a large entry that meets zeros.  The
list of outputs to recompute holds 2^20, so all are recomputed; the products of two
integers below 2^10 are exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NEED = 70 << 30  # bytes on the device


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < NEED:
        pytest.skip("needs 70 GB of device memory")
    yield
    torch.cuda.empty_cache()


def ints(n, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(1, 1000, (n,), generator=g, device="cuda").double()


def same_as_outer(got, r, s):
    """got == r s^T, a few rows at a time."""
    for i in range(0, got.shape[0], 4096):
        if not torch.equal(got[i:i + 4096], r[i:i + 4096, None] * s):
            return False
    return True


def test_grouped_product():
    from ds_b200 import _lib, ops
    M, K, N, G = 66000, 256, 32768, 4
    assert M * N > 2 ** 31
    r, s = ints(M, 1), ints(G * N, 2).view(G, N)
    x = torch.zeros((M, K), dtype=torch.float64, device="cuda")
    w = torch.zeros((G, K, N), dtype=torch.float64, device="cuda")
    x[:, 0], x[:, 1], w[:, 1] = 2.0 ** 40, r, s
    sizes = [20000, 16000, 20000, 10000]
    out = torch.full((M, N), float("nan"), dtype=torch.float64, device="cuda")
    _lib.profile_enable(True)
    _lib.profile_reset()
    ops.ds_ragged_dot_f64(x, w, torch.tensor(sizes, dtype=torch.int32, device="cuda"), out=out)
    reached = _lib.profile_read("ozaki_gemm")[1]
    _lib.profile_enable(False)
    assert reached > 0
    for g, e in enumerate(np.cumsum(sizes)):
        b = int(e) - sizes[g]
        assert same_as_outer(out[b:int(e)], r[b:int(e)], s[g])


def test_contraction():
    from ds_b200 import _lib, ops
    K, N, sizes = 20000, 18000, [300, 256, 280, 260, 256, 270]
    M, G = sum(sizes), len(sizes)
    assert G * K * N > 2 ** 31
    r, s = ints(G * K, 3).view(G, K), ints(G * N, 4).view(G, N)
    x = torch.zeros((M, K), dtype=torch.float64, device="cuda")
    y = torch.zeros((M, N), dtype=torch.float64, device="cuda")
    starts = np.cumsum(sizes) - sizes
    for g, b in enumerate(starts):
        x[int(b)], x[int(b) + 1], y[int(b) + 1] = 2.0 ** 40, r[g], s[g]
    out = torch.full((G, K, N), float("nan"), dtype=torch.float64, device="cuda")
    _lib.profile_enable(True)
    _lib.profile_reset()
    ops.ds_ragged_dot_contract_f64(x, y, torch.tensor(sizes, dtype=torch.int32, device="cuda"),
                                   out=out)
    reached = _lib.profile_read("ozaki_gemm")[1]
    _lib.profile_enable(False)
    assert reached > 0
    for g in range(G):
        assert same_as_outer(out[g], r[g], s[g])


def test_dot_general():
    from ds_b200 import ops
    M, K, N = 66000, 256, 32768
    r, s = ints(M, 5), ints(N, 6)
    x = torch.zeros((M, K), dtype=torch.float64, device="cuda")
    w = torch.zeros((K, N), dtype=torch.float64, device="cuda")
    x[:, 0], x[:, 1], w[1] = 2.0 ** 40, r, s
    stale = torch.full((M, N), float("nan"), dtype=torch.float64, device="cuda")
    del stale  # its memory is the result's
    assert same_as_outer(ops.ds_matmul_f64(x, w), r, s)
