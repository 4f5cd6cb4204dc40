"""8-bit matrices with a scale for each block of 128: rounding to them, and their products.

Rounding has one right answer, which is compared bit for bit. Products are held to the bound that
blocks_util.matmul_bound derives."""
import ctypes as C
import threading

import numpy as np
import pytest

from gorgonia_b200 import BlockTensor, Engine, _lib
from gorgonia_b200._lib import lib
from gorgonia_b200.engine import _BLOCK, _F8, from_bf16, to_bf16
from tests import blocks_util as bu
from tests import util
from tests.util import assert_bits_equal

pytestmark = pytest.mark.gpu


# ---- rounding ------------------------------------------------------------------------------------

def awkward(seed, shape):
    """Values over the whole float32 range: blocks of zeros, of subnormals, of the largest numbers, exact ties."""
    x = util.normal(seed, shape)
    r = util.rng(seed + 1)
    x *= np.exp2(r.integers(-8, 9, shape)).astype(np.float32)
    flat = x.reshape(-1)
    n = flat.size
    kind = np.repeat(r.integers(0, 8, n // 128 + 1), 128)[:n]
    flat[kind == 0] = 0.0
    flat[kind == 1] *= np.float32(1e-42)
    with np.errstate(over="ignore"):
        flat[kind == 2] = np.clip(flat[kind == 2] * np.float32(1e37), -3.4e38, 3.4e38)
    tie = kind == 3  # halfway between two neighbours
    flat[tie] = np.round(flat[tie] * 16) / 16
    flat[kind == 4] = np.sign(flat[kind == 4]) * 448
    return x


def bf16_of(x):
    return from_bf16(to_bf16(x))


def same_bytes(got, want_values, fmt):
    """Equal values, NaN for NaN, zeros with their sign."""
    v = bu.f8_values(fmt)[got]
    assert np.array_equal(v, want_values, equal_nan=True)
    fine = ~np.isnan(want_values)
    assert np.array_equal(np.signbit(v[fine]), np.signbit(want_values[fine]))


QUANT_SHAPES = [(1, 1), (1, 128), (1, 5000), (3, 127), (5, 129), (128, 128), (129, 257), (300, 1), (200, 1000), (257, 384)]


@pytest.mark.parametrize("block", ["row", "col", "tile"])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shape", QUANT_SHAPES)
def test_quantize(fresh, shape, bf16, fmt, block):
    e = fresh
    x = awkward(sum(shape), shape)
    if bf16:
        x = bf16_of(x)
        x[~np.isfinite(x)] = 3e38
        x = bf16_of(x)
    q = e.empty_blocks(shape, block, fmt)
    e.QuantizeBlocks(e.tensor_bf16(x) if bf16 else e.tensor(x), q)
    want, scales = bu.quantize(x, fmt, block)
    assert np.array_equal(q.scales.numpy().astype(np.float64), scales)
    same_bytes(q.q.numpy(), want, fmt)


@pytest.mark.parametrize("block", ["row", "col", "tile"])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_keeps_what_is_not_finite(fresh, fmt, block):
    e = fresh
    x = util.normal(5, (130, 300))
    x[0, 0], x[1, 130], x[129, 299], x[7, 256:] = np.nan, np.inf, -np.inf, np.nan
    q = e.empty_blocks(x.shape, block, fmt)
    e.QuantizeBlocks(e.tensor(x), q)
    want, scales = bu.quantize(x, fmt, block)
    assert np.array_equal(q.scales.numpy().astype(np.float64), scales)
    same_bytes(q.q.numpy(), want, fmt)


@pytest.mark.parametrize("block", ["row", "col", "tile"])
@pytest.mark.parametrize("off,ldx,ldq", [(0, 320, 320), (1, 301, 307), (3, 300, 304), (8, 304, 300)])
@pytest.mark.parametrize("bf16", [False, True])
def test_quantize_leading_dimensions(fresh, bf16, off, ldx, ldq, block):
    """Rows further apart than they are long, from any element on; what lies between them stays as it was."""
    e = fresh
    rows, cols = 140, 300
    x = util.normal(6, rows * ldx + off)
    if bf16:
        x = bf16_of(x)
    tx = e.tensor_bf16(x) if bf16 else e.tensor(x)
    tq = e.tensor(np.full(rows * ldq + off, 0xAB, np.uint8))
    ts = e.empty(BlockTensor.scale_shape((rows, cols), block))
    rc = lib.b200_quantize_blocks(e.h, _lib.BF16 if bf16 else _lib.F32, _lib.E4M3, _BLOCK[block][0],
                                  tx.ptr + off * tx.dtype.itemsize, ldx, rows, cols, tq.ptr + off, ldq, ts.ptr)
    assert rc == 0, lib.b200_last_error(e.h)
    want, scales = bu.quantize(x[off:].reshape(rows, ldx)[:, :cols], "e4m3", block)
    assert np.array_equal(ts.numpy().astype(np.float64), scales)
    got = tq.numpy()
    assert np.all(got[:off] == 0xAB)
    got = got[off:].reshape(rows, ldq)
    same_bytes(got[:, :cols], want, "e4m3")
    assert np.all(got[:, cols:] == 0xAB)


def test_quantize_empty_and_refusals(fresh):
    e = fresh
    x, q, s = e.tensor(np.ones(300, np.float32)), e.empty(300, np.uint8), e.empty(8)

    def call(dtype=_lib.F32, qtype=_lib.E4M3, block=0, xp=x.ptr, ldx=100, rows=2, cols=100, qp=q.ptr, ldq=100, sp=s.ptr):
        return lib.b200_quantize_blocks(e.h, dtype, qtype, block, xp, ldx, rows, cols, qp, ldq, sp)
    assert call() == 0
    assert call(rows=0, xp=None) == 0 and call(cols=0, qp=None) == 0
    for bad in (dict(dtype=_lib.F64), dict(dtype=7), dict(qtype=_lib.F32), dict(qtype=5), dict(block=3), dict(block=-1),
                dict(rows=-1), dict(cols=-1), dict(ldx=99), dict(ldq=99), dict(xp=None), dict(qp=None), dict(sp=None),
                dict(xp=x.ptr + 2), dict(sp=s.ptr + 1)):
        assert call(**bad) == _lib.ERR_INVALID, bad


# ---- products ------------------------------------------------------------------------------------

def upload(e, o):
    q, s, fmt, block = o
    return BlockTensor(e.tensor(q), e.tensor(s), fmt, block)


def operands(seed, M, N, K, ta, tb, av=True, bv=False, af="e4m3", bf="e4m3"):
    """av, bv: a scale for each row of 128 k, else for each 128 x 128 tile."""
    sa, sb = ((K, M) if ta else (M, K)), ((N, K) if tb else (K, N))
    ab = ("col" if ta else "row") if av else "tile"
    bb = ("row" if tb else "col") if bv else "tile"
    return (bu.random_blocks(seed, sa, af, ab) + (af, ab)), (bu.random_blocks(seed + 1, sb, bf, bb) + (bf, bb))


def check(got, a, b, K, ta, tb, bf16=False):
    want, size = bu.matmul(a, b, ta, tb)
    lim = bu.matmul_bound(size, K, 2.0 ** -7 if bf16 else 0.0, want)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= lim).all(), (np.argwhere(err > lim)[:5], (err / np.maximum(lim, 1e-300)).max())


def multiply(e, a, b, M, N, ta, tb, bf16=False, **kw):
    if bf16:
        c = e.empty((M, N), np.uint16).set(np.full((M, N), 0x7fc0, np.uint16))
        c.is_bf16 = True
        e.MatMulBlocks(upload(e, a), upload(e, b), c, transA=ta, transB=tb, **kw)
        return from_bf16(c.numpy())
    c = e.empty((M, N)).set(np.full((M, N), np.nan, np.float32))
    e.MatMulBlocks(upload(e, a), upload(e, b), c, transA=ta, transB=tb, **kw)
    return c.numpy()


SIZES = [(1, 1, 1), (1, 128, 128), (1, 300, 257), (5, 64, 128), (17, 40, 384), (33, 130, 500), (128, 128, 128), (129, 257, 640),
         (64, 1000, 272), (200, 625, 1152), (256, 512, 130), (300, 16, 2048), (130, 3, 129)]


@pytest.mark.parametrize("av,bv", [(True, False), (True, True), (False, False), (False, True)])
@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, True), (True, False)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_matmul(fresh, M, N, K, ta, tb, av, bv):
    e = fresh
    a, b = operands(M + N + K, M, N, K, ta, tb, av, bv)
    check(multiply(e, a, b, M, N, ta, tb), a, b, K, ta, tb)


@pytest.mark.parametrize("M,N,K", [(1, 512, 4096), (3, 4096, 1024), (16, 640, 3000), (40, 2000, 1536), (64, 1024, 2048),
                                   (100, 384, 8192), (512, 512, 512), (1000, 1000, 1000), (2048, 1024, 384), (1, 20000, 256),
                                   (2500, 2600, 300)])
@pytest.mark.parametrize("layout", ["forward", "kept", "dw"])
def test_matmul_larger(fresh, M, N, K, layout):
    """A layer's product with weights stored (out, in) and (in, out), and the gradient of the weights."""
    e = fresh
    ta, tb, bv = {"forward": (False, True, False), "kept": (False, False, False), "dw": (True, False, True)}[layout]
    a, b = operands(M + K, M, N, K, ta, tb, True, bv, bf="e5m2" if layout == "dw" else "e4m3")
    bf16 = layout != "dw"
    check(multiply(e, a, b, M, N, ta, tb, bf16), a, b, K, ta, tb, bf16)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 17, 48), (3, 33, 128), (8, 200, 1040), (8, 16, 8192), (9, 40, 256), (12, 200, 512),
                                   (16, 48, 144), (16, 4096, 1024), (11, 1000, 2064)])
@pytest.mark.parametrize("av,bv", [(True, False), (True, True), (False, False)])
@pytest.mark.parametrize("af,bf", [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
def test_matmul_few_rows(fresh, M, N, K, av, bv, af, bf):
    """The tokens of a few sequences: weights (out, in), k a multiple of 16, one and two column tiles; bias of either
    kind, activation, both types of the result, addition to it."""
    e = fresh
    a, b = operands(M + N, M, N, K, False, True, av, bv, af, bf)
    got = multiply(e, a, b, M, N, False, True)
    check(got, a, b, K, False, True)
    check(multiply(e, a, b, M, N, False, True, True), a, b, K, False, True, True)
    want, size = bu.matmul(a, b, False, True)
    for kind, n in (("col", N), ("row", M)):
        bias = util.normal(20, n) * np.float32(np.abs(want).mean())
        c = e.tensor(np.ones((M, N), np.float32))
        e.MatMulBlocks(upload(e, a), upload(e, b), c, transB=True, bias=e.tensor(bias), bias_kind=kind, act="rectify", incr=True)
        t = (got + (bias if kind == "col" else bias[:, None])).astype(np.float32)
        assert_bits_equal(c.numpy(), np.float32(1) + np.where(t >= 0, t, np.float32(0)))


@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, False)])
@pytest.mark.parametrize("af,bf", [("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
def test_matmul_formats(fresh, af, bf, ta, tb):
    e = fresh
    M, N, K = 150, 200, 400
    a, b = operands(8, M, N, K, ta, tb, True, ta, af, bf)
    check(multiply(e, a, b, M, N, ta, tb), a, b, K, ta, tb)


@pytest.mark.parametrize("M,N,K", [(4, 96, 260), (70, 130, 200), (600, 520, 384)])
@pytest.mark.parametrize("kind", ["col", "row"])
@pytest.mark.parametrize("act", [None, "rectify", "leaky"])
def test_matmul_epilogue(fresh, M, N, K, kind, act):
    """Bias and activation, alone and added to what C holds."""
    e = fresh
    a, b = operands(9, M, N, K, False, False)
    want, size = bu.matmul(a, b, False, False)
    bias = util.normal(10, N if kind == "col" else M) * np.float32(np.abs(want).mean())
    want = want + (bias if kind == "col" else bias[:, None])
    old = util.normal(11, (M, N)) * np.float32(np.abs(want).mean())
    lim = bu.matmul_bound(size, K) + np.abs(want) * 3 * 2.0 ** -24   # the bias, the activation's product and sum
    if act:
        want = np.where(want >= 0, want, want * (0.0 if act == "rectify" else 0.25))
    got = multiply(e, a, b, M, N, False, False, bias=e.tensor(bias), bias_kind=kind, act=act, alpha=0.25)
    assert (np.abs(got - want) <= lim).all()
    c = e.tensor(old)
    e.MatMulBlocks(upload(e, a), upload(e, b), c, bias=e.tensor(bias), bias_kind=kind, act=act, alpha=0.25, incr=True)
    assert_bits_equal(c.numpy(), old + got)


@pytest.mark.parametrize("M,N,K", [(3, 130, 300), (200, 150, 260)])
@pytest.mark.parametrize("off,pad", [(0, 4), (1, 16), (0, 1), (16, 16), (5, 3)])
@pytest.mark.parametrize("ta,tb", [(False, True), (False, False), (True, False)])
def test_matmul_leading_dimensions(fresh, M, N, K, off, pad, ta, tb):
    """Operands and results from any byte on, with rows further apart than they are long."""
    e = fresh
    a, b = operands(12, M, N, K, ta, tb)

    def padded(q):
        wide = np.full((q.shape[0], q.shape[1] + pad), 0x5A, np.uint8)
        wide[:, :q.shape[1]] = q
        return e.tensor(np.concatenate([np.full(off, 0x33, np.uint8), wide.reshape(-1)])), wide.shape[1]
    (qa, lda), (qb, ldb) = padded(a[0]), padded(b[0])
    sa, sb = e.tensor(a[1]), e.tensor(b[1])
    ldc = N + pad
    c = e.tensor(np.full(M * ldc + off, 7.0, np.float32))
    rc = lib.b200_gemm_blocks(e.h, _lib.F32, int(ta), int(tb), M, N, K, qa.ptr + off, _F8[a[2]], _BLOCK[a[3]][0], lda, sa.ptr,
                              qb.ptr + off, _F8[b[2]], _BLOCK[b[3]][0], ldb, sb.ptr, c.ptr + 4 * off, ldc, None)
    assert rc == 0, lib.b200_last_error(e.h)
    got = c.numpy()
    assert np.all(got[:off] == 7.0)
    got = got[off:].reshape(M, ldc)
    check(got[:, :N], a, b, K, ta, tb)
    assert np.all(got[:, N:] == 7.0)


def test_matmul_empty_sum(fresh):
    e = fresh
    bias = util.normal(13, 40)
    c = e.tensor(np.full((30, 40), np.nan, np.float32))
    ep = _lib.Epilogue()
    ep.bias_kind, ep.bias = _lib.BIAS_COL, e.tensor(bias).ptr
    rc = lib.b200_gemm_blocks(e.h, _lib.F32, 0, 1, 30, 40, 0, None, _lib.E4M3, 0, 0, None, None, _lib.E4M3, 2, 0, None, c.ptr, 40,
                              C.byref(ep))
    assert rc == 0, lib.b200_last_error(e.h)
    assert_bits_equal(c.numpy(), np.broadcast_to(bias, (30, 40)).copy())


def test_matrices_without_rows_or_columns(fresh):
    """Through the tensors' own calls: nothing to round, nothing to multiply, or nothing to sum."""
    e = fresh
    none, wide = e.empty_blocks((0, 256)), e.empty_blocks((40, 256), "tile")
    assert none.scales.shape == (0, 2)
    e.QuantizeBlocks(e.empty((0, 256)), none)
    e.QuantizeBlocks(e.tensor(np.ones((40, 256), np.float32)), wide)
    e.MatMulBlocks(none, wide, e.empty((0, 40)), transB=True)
    a, b = e.empty_blocks((30, 0)), e.empty_blocks((0, 40), "tile")
    c = e.tensor(np.full((30, 40), 5.0, np.float32))
    e.MatMulBlocks(a, b, c, incr=True)
    assert np.all(c.numpy() == 5.0)
    e.MatMulBlocks(a, b, c)
    assert np.all(c.numpy() == 0.0)


@pytest.mark.parametrize("M", [2, 150])
def test_matmul_values_that_are_not_finite(fresh, M):
    """A NaN spoils its row (column) of the result and nothing else, from a value as from a scale; infinities of
    E5M2 likewise; scales of zero, negative ones and ones far apart are just numbers."""
    e = fresh
    N, K = 200, 390
    a, b = operands(14, M, N, K, False, True, af="e5m2", bf="e5m2")
    a[0][0, 385] = 0x7f                      # NaN
    b[0][7, 100] = 0x7c                      # Inf
    a[1][1, 0], a[1][1, 1] = -3.0, 0.0
    b[1][1, 2] = np.float32(1e-30)
    want, size = bu.matmul(a, b, False, True)
    got = multiply(e, a, b, M, N, False, True)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[0]).all()
    inf = np.isinf(want)
    assert inf.any() and np.array_equal(got[inf], want[inf])
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= bu.matmul_bound(size, K)[fine]).all()


@pytest.mark.parametrize("M,N,K,ta,tb", [(1, 4096, 2048, False, True), (24, 768, 4096, False, True), (300, 300, 4096, False, False),
                                         (256, 256, 8192, True, False), (1000, 625, 1152, False, False)])
def test_matmul_repeats_to_the_bit(fresh, M, N, K, ta, tb):
    """Eagerly, recorded, replayed, and on an engine that works on other things in between."""
    e = fresh
    a, b = operands(15, M, N, K, ta, tb, True, ta)
    ta_, tb_ = upload(e, a), upload(e, b)
    c = e.empty((M, N))
    first = e.MatMulBlocks(ta_, tb_, c, transA=ta, transB=tb).numpy()
    for _ in range(5):
        c.set(np.zeros((M, N), np.float32))
        assert_bits_equal(e.MatMulBlocks(ta_, tb_, c, transA=ta, transB=tb).numpy(), first)
    tapes, outs = [], []
    for _ in range(2):      # two tapes that take scratch from the same arena
        outs.append(e.empty((M, N)))
        e.tape_begin()
        e.MatMulBlocks(ta_, tb_, outs[-1], transA=ta, transB=tb)
        tapes.append(e.tape_end())
    filler = e.tensor(np.full(1 << 20, 3.0, np.float32))
    for _ in range(3):
        for t in tapes:
            e.tape_launch(t)
    for o in outs:
        assert_bits_equal(o.numpy(), first)
    assert np.all(filler.numpy() == 3.0)
    for t in tapes:
        e.tape_destroy(t)


@pytest.mark.parametrize("M,N,K", [(5000, 2048, 300), (4500, 2100, 4096)])
@pytest.mark.parametrize("ta,tb,bv", [(False, True, False), (False, False, False), (True, False, True)])
def test_matmul_pairs_of_ctas(fresh, M, N, K, ta, tb, bv):
    """Large products run on pairs of CTAs, the second with the k ranges of its last tiles shared out: right, and
    the same bits as on single CTAs where nothing is shared."""
    e = fresh
    a, b = operands(19, M, N, K, ta, tb, True, bv)
    check(multiply(e, a, b, M, N, ta, tb), a, b, K, ta, tb)
    got = []
    for pairs in (True, False):
        one = Engine(0, 256 << 20, streamk=False, pairs=pairs)
        try:
            got.append(multiply(one, a, b, M, N, ta, tb))
        finally:
            one.Close()
    assert_bits_equal(got[0], got[1])


def test_matmul_order_does_not_depend_on_the_batch():
    """Without shared k ranges a row of the result has the same bits in a batch of any size."""
    e = Engine(0, 256 << 20, streamk=False)
    try:
        a, b = operands(16, 300, 520, 2048, False, True)
        whole = multiply(e, a, b, 300, 520, False, True)
        for m in (1, 7, 64, 130):
            part = (a[0][:m].copy(), a[1][:m].copy(), a[2], a[3])
            assert_bits_equal(multiply(e, part, b, m, 520, False, True), whole[:m])
    finally:
        e.Close()


def test_matmul_in_a_full_arena():
    """Without room for scratch the product is made all the same."""
    e = Engine(0, 8 << 20)
    try:
        M, N, K = 130, 150, 1111
        a, b = operands(17, M, N, K, False, True)
        ta, tb, c = upload(e, a), upload(e, b), e.empty((M, N))
        held = []
        while e.arena_stats()["largest_free"] >= 256:
            held.append(e.Get(e.arena_stats()["largest_free"]))
        e.MatMulBlocks(ta, tb, c, transB=True)
        check(c.numpy(), a, b, K, False, True)
    finally:
        e.Close()


def test_two_engines_at_once(fresh):
    """Two threads, each with an engine (a stream) of its own."""
    a, b = operands(18, 200, 300, 3000, False, True)
    want = multiply(fresh, a, b, 200, 300, False, True)
    wrong = []

    def work():
        e = Engine(0, 256 << 20)
        try:
            ta, tb, c = upload(e, a), upload(e, b), e.empty((200, 300))
            for _ in range(20):
                e.MatMulBlocks(ta, tb, c, transB=True)
                if not np.array_equal(c.numpy(), want):
                    wrong.append(1)
        finally:
            e.Close()
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_matmul_refusals(fresh):
    e = fresh
    q, s, c = e.empty(1 << 16, np.uint8), e.empty(1 << 12), e.empty(1 << 14)

    def call(ct=_lib.F32, ta=0, tb=1, M=8, N=8, K=256, A=q.ptr, at=_lib.E4M3, ab=0, lda=256, sa=s.ptr, B=q.ptr, bt=_lib.E4M3, bb=2,
             ldb=256, sb=s.ptr, cp=c.ptr, ldc=8, ep=None):
        return lib.b200_gemm_blocks(e.h, ct, ta, tb, M, N, K, A, at, ab, lda, sa, B, bt, bb, ldb, sb, cp, ldc, ep)

    def epi(**kw):
        x = _lib.Epilogue()
        for k, v in kw.items():
            setattr(x, k, v)
        return C.byref(x)
    q.set(np.zeros(1 << 16, np.uint8))
    assert call() == 0 and call(M=0, cp=None) == 0 and call(N=0) == 0
    for bad in (dict(ct=_lib.F64), dict(at=_lib.F32), dict(bt=9), dict(ab=1), dict(bb=1), dict(ab=3), dict(ta=1, ab=0),
                dict(tb=0, bb=0), dict(M=-1), dict(K=-1), dict(N=1 << 31, ldc=1 << 31), dict(cp=None), dict(A=None), dict(sb=None),
                dict(lda=255), dict(ldb=255), dict(ldc=7), dict(cp=c.ptr + 2), dict(sa=s.ptr + 2),
                dict(ep=epi(bias_kind=3)), dict(ep=epi(act=3)), dict(ep=epi(bias_kind=1)),
                dict(ep=epi(accumulate=1), ct=_lib.BF16)):
        assert call(**bad) == _lib.ERR_INVALID, bad
    flag = e.tensor(np.zeros(1, np.int32))
    with e.only_if(flag.ptr):
        assert call() == _lib.ERR_STATE
    assert call() == 0
