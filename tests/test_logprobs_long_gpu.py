"""Long rows, held to the sums that really run: a thread adds some dozen to some hundred terms, and a head or tail of a row that
got lost, or a rounding in the wrong place, shows.

The bound. A block of 256 threads takes a row, or a cluster of up to 8 blocks of 512 where rows are few, so a thread adds `terms` values,
some one by one and some after its maximum has risen; u = 2^-24. A term e^d, d = x - m, is off by 3 |d| u (the difference, its product
with log2 e, that constant) and by 4 u (the hardware's power of two, 2^-22). A sum of n positive terms is off by n u of
itself at most. Each rise of the maximum, at most one for each group of loads and each of the 32 + 16 + 8 that are
joined, multiplies by another such power: 7 u and 3 |d| u, the |d| of all rises together at most the spread of the row's values. So s
is off by `rel` of itself, ln s by rel, lse by half a step more, and logp = (x - m) - ln s by two. H = ln s - t / s: t carries the same
errors on terms |d| e^d, E|d| of s in all, and half a step for each d that a rise adds, at most the spread in all."""
import numpy as np
import pytest

from gorgonia_b200.engine import from_bf16, to_bf16
from tests import blocks_util as bu
from tests import util

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def threads_of(rows, vocab, dtype):
    """Threads that share a row: the launch's rule."""
    nvec = vocab // (8 if dtype == "bf16" else 4)

    def block(most):
        nt = 32
        while nt < most and nt * 16 < nvec:
            nt *= 2
        return nt
    nt, cl = block(512), 1
    while cl < 8 and rows * cl < 148 and nvec // (2 * cl) >= 2 * nt:
        cl *= 2
    return (block(256) if cl == 1 else nt), cl


def bounds(x, want, dtype):
    rows, vocab = x.shape
    nt, cl = threads_of(rows, vocab, dtype)
    terms = -(-vocab // (nt * cl)) + 2 * 8          # and a vector's rest at either end
    rises = terms / 4 + 3
    m = x.max(axis=1)
    d = x - m[:, None]
    p = np.exp(d)
    s = p.sum(axis=1)
    mean = (p * -d).sum(axis=1) / s                 # E|d|
    spread = m - x.min(axis=1)
    rel = U * (terms + 5 + 16 + 8 + 4 + 3 * mean + 7 * rises + 3 * spread)
    lse = rel + U * (2 * np.abs(want["lse"]) + 4 * np.log(s))
    ent = rel * (1 + 2 * mean) + U * (spread + 8 * (mean + np.log(s) + 1))
    return lse, ent


def put(e, x, dtype):
    return e.tensor_bf16(x.astype(np.float32)) if dtype == "bf16" else e.tensor(x.astype(np.float32))


def rounded(x, dtype):
    x = x.astype(np.float32)
    return (from_bf16(to_bf16(x)) if dtype == "bf16" else x).astype(np.float64)


def run(e, x, t, dtype, top=3):
    rows = len(x)
    o = [e.empty(rows) for _ in range(3)]
    tl, ti = e.empty((rows, top)), e.empty((rows, top), np.int64)
    e.TokenLogProbs(put(e, x, dtype), e.tensor(t), o[0], o[1], o[2], tl, ti)
    return dict(zip(("logp", "entropy", "lse"), (v.numpy().astype(np.float64) for v in o))), tl.numpy(), ti.numpy()


def compare(e, x, t, dtype):
    got, tl, ti = run(e, x, t, dtype)
    want = bu.logprobs(x, t, 3)
    lim, lim_h = bounds(x, want, dtype)
    for name, bound in (("lse", lim), ("entropy", lim_h), ("logp", lim + 2 * U * np.abs(want["logp"]))):
        err = np.abs(got[name] - want[name])
        assert (err <= bound).all(), (name, (err / bound).max(), err.max())
    assert np.array_equal(ti, want["top_index"])
    assert (np.abs(tl - want["top_logp"]) <= lim[:, None] + 2 * U * np.abs(want["top_logp"])).all()
    return got, lim


SHAPES = [(1, 131072), (2, 200003), (12, 32000), (80, 50001), (200, 32000), (160, 128257)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_even_rows(fresh, rows, vocab, dtype):
    x = rounded(util.normal(rows + vocab, (rows, vocab)) * np.float32(2.5), dtype)
    compare(fresh, x, util.rng(1).integers(0, vocab, rows), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_the_mass_lies_at_the_ends(fresh, rows, vocab, dtype):
    """Each row's weight is on one of its first or last nine values, on each of them in some row."""
    x = rounded(util.normal(rows + vocab, (rows, vocab)) * np.float32(0.5), dtype)
    at = np.array([(i if i < 9 else vocab - 18 + i) for i in np.arange(rows) * (1 if rows >= 18 else 7) % 18])
    # as much weight there as the rest has together, so that either's loss halves the sum
    x[np.arange(rows), at] = rounded(np.full(rows, np.log(vocab) + 0.125), dtype)
    got, lim = compare(fresh, x, at, dtype)
    assert lim.max() < 0.01 and np.all(np.abs(got["logp"] - np.log(0.5)) < 0.1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_first_and_last_value_counts(fresh, dtype):
    """Rows that begin at any place of 16 bytes (their length is odd): without each of the ends' values the sum is another."""
    rows, vocab = 36, 30011
    x = np.full((rows, vocab), -20.0)
    for r in range(rows):
        x[r, r if r < 18 else vocab - 36 + r] = 5.0     # e^25 times each of the others, 30010 of which make e^10.3
    x = rounded(x, dtype)
    got, _ = compare(fresh, x, np.full(rows, vocab // 2), dtype)
    assert np.all(np.abs(got["lse"] - 5.0) < 1e-5)
