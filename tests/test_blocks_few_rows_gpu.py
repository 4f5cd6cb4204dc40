"""Products of up to 16 rows with k contiguous and 16-byte loads possible, which run on a kernel of their own: operands inside larger
buffers, and values and scales that are not finite."""
import numpy as np
import pytest

from gorgonia_b200 import _lib
from gorgonia_b200._lib import lib
from gorgonia_b200.engine import _BLOCK, _F8
from tests import blocks_util as bu
from tests.test_blocks_gpu import check, multiply, operands

pytestmark = pytest.mark.gpu

SIZES = [(1, 130, 16), (3, 17, 272), (8, 100, 1040), (9, 33, 144), (16, 70, 528)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("off,pad", [(0, 16), (16, 48), (32, 112)])
@pytest.mark.parametrize("av,bv", [(True, False), (False, True)])
def test_rows_inside_larger_buffers(fresh, M, N, K, off, pad, av, bv):
    """NaN lies before, between and behind the rows, and must neither be read nor written over."""
    e = fresh
    a, b = operands(31, M, N, K, False, True, av, bv)

    def padded(q):
        wide = np.full((q.shape[0], K + pad), 0x7f, np.uint8)
        wide[:, :K] = q
        return e.tensor(np.concatenate([np.full(off, 0x7f, np.uint8), wide.reshape(-1), np.full(64, 0x7f, np.uint8)]))
    qa, qb, sa, sb = padded(a[0]), padded(b[0]), e.tensor(a[1]), e.tensor(b[1])
    ldc = N + 3
    c = e.tensor(np.full(M * ldc + 5, 7.0, np.float32))
    rc = lib.b200_gemm_blocks(e.h, _lib.F32, 0, 1, M, N, K, qa.ptr + off, _F8[a[2]], _BLOCK[a[3]][0], K + pad, sa.ptr, qb.ptr + off,
                              _F8[b[2]], _BLOCK[b[3]][0], K + pad, sb.ptr, c.ptr + 4, ldc, None)
    assert rc == 0, lib.b200_last_error(e.h)
    got = c.numpy()
    assert got[0] == 7.0 and np.all(got[1 + M * ldc:] == 7.0)
    got = got[1:1 + M * ldc].reshape(M, ldc)
    check(got[:, :N], a, b, K, False, True)
    assert np.all(got[:, N:] == 7.0)


@np.errstate(invalid="ignore")
def by_blocks(a, b, K):
    """The product as it is defined, block by block: the sum of a block's products times its two scales. (An infinite scale
    makes a sum infinite, where value by value it would make Inf - Inf of one whose terms differ in sign.)"""
    (qa, sa, fa, ba), (qb, sb, fb, bb) = a, b
    va, vb = bu.f8_values(fa)[qa], bu.f8_values(fb)[qb]
    wa, wb = (np.repeat(s.astype(np.float64), 128, 0)[:len(v)] if block == "tile" else s.astype(np.float64)
              for s, v, block in ((sa, va, ba), (sb, vb, bb)))
    c = np.zeros((len(va), len(vb)))
    for k in range(-(-K // 128)):
        c += va[:, k * 128:(k + 1) * 128] @ vb[:, k * 128:(k + 1) * 128].T * (wa[:, k][:, None] * wb[:, k][None])
    return c


@pytest.mark.parametrize("M", [2, 7, 13])
@pytest.mark.parametrize("bv", [False, True])
def test_values_and_scales_that_are_not_finite(fresh, M, bv):
    """A NaN spoils its row or column and nothing else, from a value as from a scale; scales of zero, negative ones and infinite
    ones are taken as they are."""
    e = fresh
    N, K = 200, 400
    a, b = operands(32, M, N, K, False, True, True, bv, "e5m2", "e5m2")
    a[0][0, 385] = 0x7f                       # NaN, in the last and partial block
    b[0][7, 100] = 0x7c                       # Inf
    b[0][150, 0] = 0xfc                       # -Inf
    a[1][1, 0], a[1][1, 1] = -3.0, 0.0
    if bv:
        b[1][20, 3], b[1][21, 0] = np.nan, np.inf
    if M > 7:
        a[1][12, 2] = np.inf
    with np.errstate(invalid="ignore"):
        size = bu.matmul(a, b, False, True)[1]
    want = by_blocks(a, b, K)
    got = multiply(e, a, b, M, N, False, True)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[0]).all()
    inf = np.isinf(want)
    assert inf.any() and np.array_equal(got[inf], want[inf])
    fine = np.isfinite(want)
    assert fine.any() and (np.abs(got[fine] - want[fine]) <= bu.matmul_bound(size, K)[fine]).all()
