"""Products of 8-bit matrices whose scales' product leaves float32's range where the result does not.

A block's sum is 0 or lies between 2^-32 (the least E5M2 value squared) and 2^39, a scale between 2^-149 and 2^128. Every kernel
has to give what the definition gives: an exact 0 stays one, and a result that float32 holds is not lost on the way."""
import numpy as np
import pytest

from gorgonia_b200 import Engine
from tests import blocks_util as bu
from tests.test_blocks_gpu import multiply, upload

pytestmark = pytest.mark.gpu

# (M, N, K, transA, transB, rows or columns have their own scales): few rows on the kernel for these, then with the operands
# exchanged, tiles of every width, shared k ranges, pairs of CTAs
KERNELS = [(3, 70, 256, False, True, False), (12, 70, 272, False, True, True), (3, 70, 300, False, True, True), (24, 200, 260, False, True, False),
           (24, 200, 260, False, False, True), (60, 300, 260, False, True, True), (130, 150, 300, False, True, False),
           (130, 150, 300, True, False, True), (600, 520, 384, True, False, True), (256, 256, 4096, True, False, True),
           (300, 300, 4096, False, True, False), (5000, 2048, 300, False, True, False), (5000, 2048, 300, True, False, True)]


def powers(r, shape, lo, hi):
    """Numbers that are no powers of two, their exponents even between lo and hi, of either sign."""
    e = r.integers(lo, hi, shape, endpoint=True)
    m = np.ldexp(r.uniform(1, 2, shape), e).astype(np.float32)   # subnormal below 2^-126
    return np.where(r.random(shape) < 0.5, -m, m)


def operands(seed, M, N, K, ta, tb, each, fa, fb, a_exp, b_exp, zeros=0.0, tiny=False):
    r = np.random.Generator(np.random.Philox(seed))
    out = []
    for (rows, cols, k_down, fmt, (lo, hi), own) in ((*((K, M) if ta else (M, K)), ta, fa, a_exp, True), (*((N, K) if tb else (K, N)), not tb, fb, b_exp, each)):
        block = ("col" if k_down else "row") if own else "tile"
        v, _ = bu.quantize(r.standard_normal((rows, cols)).astype(np.float32), fmt, block)
        if tiny:     # the format's least values
            v = r.integers(-3, 4, v.shape) * np.abs(bu.f8_values(fmt)[1])
        if zeros:
            gone = r.random(cols if k_down else rows) < zeros
            v[(slice(None), gone) if k_down else (gone, slice(None))] = 0.0
        br, bc = bu.BLOCKS[block]
        out.append((bu.to_bytes(v, fmt), powers(r, (-(-rows // br), -(-cols // bc)), lo, hi), fmt, block))
    return out


def compare(got, a, b, K, ta, tb, least):
    """Where the sum of the terms' magnitudes stays inside float32 (so that no partial sum can leave it), the usual bound and half of
    the least subnormal for each of the additions; exact zeros everywhere."""
    want, size = bu.matmul(a, b, ta, tb)
    inside = size < 2.0 ** 127
    assert inside.mean() >= least
    assert np.all(got[size == 0] == 0)
    lim = bu.matmul_bound(size, K) + 2 * -(-K // 128) * 2.0 ** -150
    err = np.abs(got.astype(np.float64) - want)
    assert (err[inside] <= lim[inside]).all(), (np.isnan(got).sum(), np.argwhere(inside & ~(err <= lim))[:5])


# exponents of A's and B's scales, the share of zero rows, tiny values, and how much of the result is inside the range
RANGES = {"both large": ((70, 70), (66, 66), 0.3, False, 0.2), "both large, tiny values": ((65, 66), (63, 64), 0.1, True, 0.9),
          "large and small": ((100, 110), (-110, -100), 0.0, False, 1.0), "both small": ((-80, -76), (-80, -76), 0.0, False, 1.0),
          "subnormal": ((-149, -127), (20, 40), 0.0, False, 1.0), "any": ((-149, 127), (-149, 127), 0.1, False, 0.05)}


@pytest.mark.parametrize("fa,fb", [("e4m3", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("name", list(RANGES))
@pytest.mark.parametrize("M,N,K,ta,tb,each", KERNELS)
def test_products_of_scales_out_of_range(fresh, M, N, K, ta, tb, each, name, fa, fb):
    a_exp, b_exp, zeros, tiny, least = RANGES[name]
    if name == "any" and K > 300:
        pytest.skip("a sum over many such blocks leaves the range itself")
    a, b = operands(M + K, M, N, K, ta, tb, each, fa, fb, a_exp, b_exp, zeros, tiny)
    compare(multiply(fresh, a, b, M, N, ta, tb), a, b, K, ta, tb, least)


@pytest.mark.parametrize("name", ["both large", "both large, tiny values", "both small", "any"])
def test_out_of_range_on_cuda_cores(name):
    """An arena without room for the copy of an operand."""
    a_exp, b_exp, zeros, tiny, least = RANGES[name]
    M, N, K = 130, 150, 275
    a, b = operands(5, M, N, K, False, True, True, "e5m2", "e5m2", a_exp, b_exp, zeros, tiny)
    e = Engine(0, 8 << 20)
    try:
        ta, tb, c = upload(e, a), upload(e, b), e.empty((M, N))
        while e.arena_stats()["largest_free"] >= 256:
            e.Get(e.arena_stats()["largest_free"])
        e.MatMulBlocks(ta, tb, c, transB=True)
        compare(c.numpy(), a, b, K, False, True, least)
    finally:
        e.Close()


@pytest.mark.parametrize("M", [4, 40, 200])
@pytest.mark.parametrize("block", ["row", "tile"])
def test_finite_matrices_of_large_values(fresh, M, block):
    """Through the quantiser: values of 1e22 that never meet another one in the sum, and rows of zeros beside them."""
    e = fresh
    N, K = 96, 256
    x, w = np.zeros((M, K), np.float32), np.zeros((N, K), np.float32)
    x[::2, 0] = 1e22
    w[::2, 1] = 1e22
    w[1::4, 200] = 2.0
    x[1, 200] = 3.0
    qx, qw, c = e.empty_blocks(x.shape, "row"), e.empty_blocks(w.shape, block), e.empty((M, N))
    e.QuantizeBlocks(e.tensor(x), qx)
    e.QuantizeBlocks(e.tensor(w), qw)
    e.MatMulBlocks(qx, qw, c, transB=True)
    assert np.array_equal(c.numpy(), x.astype(np.float64) @ w.T.astype(np.float64))


@pytest.mark.parametrize("each", [False, True])
def test_far_neighbours_change_nothing(each):
    """Without shared k ranges a row's bits depend on no other row, nor on how many there are, also where rows beside it take
    scales that need care."""
    e = Engine(0, 256 << 20, streamk=False)
    try:
        M, N, K = 300, 520, 640
        a, b = operands(6, M, N, K, False, True, each, "e4m3", "e5m2", (-20, 20), (-70, -66))
        plain = multiply(e, a, b, M, N, False, True)
        far = (a[0], a[1].copy(), a[2], a[3])
        far[1][5::7] = np.float32(2.0 ** -100)
        mixed = multiply(e, far, b, M, N, False, True)
        keep = np.ones(M, bool)
        keep[5::7] = False
        assert np.array_equal(mixed[keep].view(np.uint32), plain[keep].view(np.uint32))
        for m in (6, 40, 130):
            part = (far[0][:m].copy(), far[1][:m].copy(), far[2], far[3])
            assert np.array_equal(multiply(e, part, b, m, N, False, True).view(np.uint32), mixed[:m].view(np.uint32))
    finally:
        e.Close()
