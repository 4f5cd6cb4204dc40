"""Log probabilities of given tokens with entropy and alternatives, and their gradient; and the 8-bit head of a model
from its activations to the gradients of its weights."""
import numpy as np
import pytest

from gorgonia_b200 import B200Error, _lib
from gorgonia_b200._lib import lib
from gorgonia_b200.engine import from_bf16, to_bf16
from tests import blocks_util as bu
from tests import util
from tests.util import assert_bits_equal

pytestmark = pytest.mark.gpu
INF = np.inf


def logits(seed, rows, vocab, dtype, masked=0.0, scale=3.0):
    """(values as float64, engine's host array) with some -Inf; bf16 values hold many ties."""
    x = util.normal(seed, (rows, vocab)).astype(np.float64) * scale
    if masked:
        x[util.rng(seed + 1).random((rows, vocab)) < masked] = -INF
    if dtype == "bf16":
        return from_bf16(to_bf16(x.astype(np.float32))).astype(np.float64)
    return x.astype(np.float32).astype(np.float64) if dtype == "f32" else x


def put(e, x, dtype):
    return e.tensor_bf16(x.astype(np.float32)) if dtype == "bf16" else e.tensor(x.astype(stat(dtype)))


def stat(dtype):
    return np.float64 if dtype == "f64" else np.float32


def unit(dtype):
    return 2.0 ** -53 if dtype == "f64" else 2.0 ** -24


def forward(e, tx, targets, top, dtype):
    rows = tx.shape[0]
    s = stat(dtype)
    o = {k: e.empty(rows, s).set(np.full(rows, 123, s)) for k in ("lse", "entropy", "logp")}
    tl, ti = (e.empty((rows, top), s), e.empty((rows, top), np.int64)) if top else (None, None)
    e.TokenLogProbs(tx, e.tensor(targets), o["logp"], o["entropy"], o["lse"], tl, ti)
    r = {k: t.numpy() for k, t in o.items()}
    if top:
        r["top_logp"], r["top_index"] = tl.numpy(), ti.numpy()
    return r


def close(got, want, lim):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    special = ~np.isfinite(want)
    assert np.array_equal(got[special], want[special], equal_nan=True)
    err = np.abs(got[~special] - want[~special])
    lim = np.broadcast_to(lim, got.shape)[~special]
    assert (err <= lim).all(), ((err / lim).max(), err.max())


@np.errstate(over="ignore")
def compare(got, x, targets, top, dtype):
    want = bu.logprobs(x, targets, top)
    lse = np.where(np.isfinite(want["lse"]), want["lse"], 0.0)
    lim, lim_h = bu.stat_bound(x, lse, unit(dtype))
    close(got["lse"], want["lse"], lim)
    close(got["entropy"], want["entropy"], lim_h)
    logp = np.where(np.isfinite(want["logp"]), np.abs(want["logp"]), 0.0)
    close(got["logp"], want["logp"], lim + 2 * logp * unit(dtype))
    if top:
        assert np.array_equal(got["top_index"], want["top_index"])
        tl = np.where(np.isfinite(want["top_logp"]), np.abs(want["top_logp"]), 0.0)
        close(got["top_logp"], want["top_logp"], lim[:, None] + 2 * tl * unit(dtype))
    return want


SHAPES = [(1, 1, 1), (3, 2, 2), (256, 10, 3), (5, 31, 31), (7, 33, 32), (2, 129, 20), (65, 1000, 5), (3, 1023, 32), (4, 4096, 8), (2, 4099, 1),
          (300, 2048, 4), (9, 32000, 20), (1, 50001, 32), (2, 131072, 20), (1, 200003, 5), (160, 9000, 32), (40, 17000, 10)]


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("masked", [0.0, 0.4])
@pytest.mark.parametrize("rows,vocab,top", SHAPES)
def test_logprobs(fresh, rows, vocab, top, masked, dtype):
    e = fresh
    x = logits(rows + vocab, rows, vocab, dtype, masked)
    t = util.rng(vocab).integers(0, vocab, rows)
    t[::7] = -1
    compare(forward(e, put(e, x, dtype), t, top, dtype), x, t, top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("vocab", [40, 700, 5000, 70000])
def test_rows_that_masks_and_values_leave_odd(fresh, vocab, dtype):
    e = fresh
    top = 20
    x = logits(3, 14, vocab, dtype)
    low = float(np.float32(-3.3895314e38)) if dtype != "f64" else -1.7e308   # bf16's lowest value
    x[0] = -INF                                    # a mask that leaves nothing
    x[1] = -INF
    x[1, vocab - 1] = 2.0                          # ... that leaves one token
    x[2] = low                                     # the type's lowest value instead
    x[3] = low
    x[3, [5, 7, 11]] = [1.0, 3.0, 1.0]
    x[4] = 1.5                                     # all the same
    x[5, 17] = np.nan
    x[6, 3] = INF
    x[7, [3, 20]] = [-INF, np.nan]
    x[8] = np.where(np.arange(vocab) % 2, 0.0, -0.0)   # zeros of both signs are equal
    x[9] = np.sort(x[9])
    x[10] = np.sort(x[10])[::-1]
    x[11] = -INF
    x[11, vocab // 2:vocab // 2 + 30] = 1.0        # ties across few tokens, fewer than any share of the row
    x[12] = np.arange(vocab) // 16                 # ascending runs of ties
    if dtype == "bf16":
        x[12] = x[12] % 256
    x[13] = 0.0
    x[13, ::3] = 60.0
    t = np.arange(14) % vocab
    t[1], t[3] = vocab - 1, 7
    compare(forward(e, put(e, x, dtype), t, top, dtype), x, t, top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["up", "down", "clustered"])
def test_alternatives_of_sorted_rows(fresh, dtype, order):
    """The best tokens side by side, or all in one stride: no share of the row holds its fair part of them."""
    e = fresh
    rows, vocab, top = 3, 60000, 32
    x = np.sort(logits(4, rows, vocab, dtype), axis=1)
    if order == "down":
        x = x[:, ::-1].copy()
    if order == "clustered":
        x[:, :] = np.sin(np.arange(vocab) / 997.0)[None]
        x[:, 1024:21504] += 5.0
        x[1, 3::512] += 9.0
        x = from_bf16(to_bf16(x.astype(np.float32))).astype(np.float64) if dtype == "bf16" else x.astype(np.float32).astype(np.float64)
    t = np.array([0, vocab - 1, 30000])
    compare(forward(e, put(e, x, dtype), t, top, dtype), x, t, top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
def test_what_is_asked_for_does_not_change_the_rest(fresh, dtype):
    e = fresh
    rows, vocab = 6, 3000
    x = logits(8, rows, vocab, dtype)
    tx, t = put(e, x, dtype), util.rng(1).integers(0, vocab, rows)
    all_ = forward(e, tx, t, 9, dtype)
    s = stat(dtype)
    ent = e.empty(rows, s)
    e.TokenLogProbs(tx, None, None, entropy=ent)
    assert_bits_equal(ent.numpy(), all_["entropy"])
    tl, ti = e.empty((rows, 4), s), e.empty((rows, 4), np.int64)
    e.TokenLogProbs(tx, None, None, top_logp=tl, top_index=ti)
    assert_bits_equal(tl.numpy(), np.ascontiguousarray(all_["top_logp"][:, :4]))
    assert np.array_equal(ti.numpy(), all_["top_index"][:, :4])
    lp = e.empty(rows, s)
    e.TokenLogProbs(tx, e.tensor(t), lp)
    assert_bits_equal(lp.numpy(), all_["logp"])


@pytest.mark.parametrize("dtype,code,es", [("f32", _lib.F32, 4), ("f64", _lib.F64, 8), ("bf16", _lib.BF16, 2)])
@pytest.mark.parametrize("rows,vocab,ld,off", [(5, 1000, 1003, 1), (3, 40000, 40008, 3), (9, 17, 40, 5), (2, 33333, 33333, 0)])
def test_leading_dimensions(fresh, rows, vocab, ld, off, dtype, code, es):
    """Rows from any element on; behind the last one, and between them, nothing is read or written."""
    e = fresh
    x = logits(9, rows, vocab, dtype)
    wide = np.full(off + rows * ld + 8, np.nan)
    for r in range(rows):
        wide[off + r * ld:off + r * ld + vocab] = x[r]
    tx, s = put(e, wide, dtype), stat(dtype)
    t = util.rng(2).integers(0, vocab, rows)
    tt = e.tensor(t)
    o = [e.empty(rows, s) for _ in range(3)]
    rc = lib.b200_token_logprobs(e.h, code, tx.ptr + off * es, ld, rows, vocab, tt.ptr, o[0].ptr, o[1].ptr, o[2].ptr, 0, None, None)
    assert rc == 0, lib.b200_last_error(e.h)
    compare({"logp": o[0].numpy(), "entropy": o[1].numpy(), "lse": o[2].numpy()}, x, t, 0, dtype)
    g = e.tensor(np.ones(rows, s))
    before = tx.numpy().copy()
    for dst in (None, tx):     # a buffer of its own, then in place
        d = e.tensor(np.full(wide.size, 7, before.dtype)) if dst is None else dst
        rc = lib.b200_token_logprobs_bwd(e.h, code, tx.ptr + off * es, ld, rows, vocab, tt.ptr, o[2].ptr, o[1].ptr, g.ptr, g.ptr,
                                         d.ptr + off * es, ld)
        assert rc == 0, lib.b200_last_error(e.h)
        got = d.numpy()
        inside = np.zeros(wide.size, bool)
        for r in range(rows):
            inside[off + r * ld:off + r * ld + vocab] = True
        if dst is None:
            own = got[inside]
            assert np.all(got[~inside] == 7)
            assert_bits_equal(tx.numpy(), before)
        else:
            assert_bits_equal(got[inside], own)
            assert_bits_equal(got[~inside], before[~inside])


def diff_bound(x, f, targets, g, h, want, dtype):
    """p = e^(x - lse) carries a relative error of (|x - lse| (3 units: the difference, its product with log2 e, the constant) +
    8 units) and what the difference's own rounding adds; the entropy's term a few more on |p (ln p + H)|; the result one
    rounding to its type."""
    u = unit(dtype)
    lse, ent = f["lse"].astype(np.float64)[:, None], f["entropy"].astype(np.float64)[:, None]
    with np.errstate(invalid="ignore"):
        lp = np.where(np.isfinite(x), x - lse, 0.0)
        p = np.where(np.isfinite(x), np.exp(np.where(np.isfinite(x), x - lse, 0.0)), 0.0)
    rel = (3 * np.abs(lp) + 8) * u
    on = ((targets >= 0) & (targets < x.shape[1]))[:, None]
    err = np.abs(g)[:, None] * on * (p * (rel + 2 * u) + u)
    if h is not None:
        err += np.abs(h)[:, None] * p * ((np.abs(lp + ent)) * (rel + 4 * u) + (np.abs(lp) + np.abs(ent)) * 2 * u)
    out = 2.0 ** -8 if dtype == "bf16" else u
    tiny = 2.0 ** -120 if dtype != "f64" else 2.0 ** -1000   # an exponential that has left the normal range may be 0
    return err + 2 * u * np.abs(want) + out * (np.abs(want) + err) + tiny


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("with_entropy", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (256, 10), (3, 33), (65, 1000), (4, 4099), (9, 32000), (1, 131072), (2, 50001), (300, 640)])
def test_gradient(fresh, rows, vocab, with_entropy, dtype):
    e = fresh
    x = logits(rows + vocab, rows, vocab, dtype, 0.2 if vocab > 10 else 0.0)
    t = util.rng(vocab).integers(0, vocab, rows)
    if rows > 2:
        x[1] = -INF                 # no token left
        t[2] = -1
    tx = put(e, x, dtype)
    f = forward(e, tx, t, 0, dtype)
    s = stat(dtype)
    g, h = util.normal(21, rows).astype(s), (util.normal(22, rows).astype(s) if with_entropy else None)
    if rows > 4:
        g[3] = 0
        g[4], h = -1, h
    want = bu.logprobs_diff(x, t, f["lse"].astype(np.float64), f["entropy"].astype(np.float64), g, h)
    dx = e.empty((rows, vocab), np.uint16 if dtype == "bf16" else s)
    if dtype == "bf16":
        dx.is_bf16 = True
    up = {k: e.tensor(f[k]) for k in ("lse", "entropy")}
    e.TokenLogProbsDiff(tx, e.tensor(t), up["lse"], up["entropy"], e.tensor(g), dx, grad_entropy=None if h is None else e.tensor(h))
    got = from_bf16(dx.numpy()) if dtype == "bf16" else dx.numpy()
    close(got, want, diff_bound(x, f, t, g, h, want, dtype))


def test_gradient_against_differences(fresh):
    """The gradient of the forward call's own outputs, by central differences in float64."""
    e = fresh
    rows, vocab = 4, 37
    x = logits(31, rows, vocab, "f64", scale=1.0)
    t = np.array([3, 36, -1, 0])
    g, h = util.normal(32, rows, np.float64), util.normal(33, rows, np.float64)

    def value(y):
        f = forward(e, e.tensor(y), t, 0, "f64")
        return f["logp"] * g + f["entropy"] * h
    f = forward(e, e.tensor(x), t, 0, "f64")
    dx = e.empty(x.shape, np.float64)
    e.TokenLogProbsDiff(e.tensor(x), e.tensor(t), e.tensor(f["lse"]), e.tensor(f["entropy"]), e.tensor(g), dx, grad_entropy=e.tensor(h))
    got, step = dx.numpy(), 1e-5
    for v in range(vocab):
        up, down = x.copy(), x.copy()
        up[:, v] += step
        down[:, v] -= step
        slope = (value(up) - value(down)) / (2 * step)
        # third derivatives are of order |g| + |h| ln V here: step^2 of them, and rounding 1e-16 * 10 / step
        assert (np.abs(slope - got[:, v]) <= 1e-9 * (1 + np.abs(g) + np.abs(h))).all()


def test_rows_without_gradient_need_no_logits(fresh):
    """Padding: no token, no entropy gradient. Such rows may hold anything and get zeros."""
    e = fresh
    x = logits(41, 6, 5000, "f32")
    x[2] = np.nan
    x[4, 9] = INF
    t = np.array([1, 2, -1, 4, -1, 5])
    f = forward(e, put(e, x, "f32"), t, 0, "f32")
    g, h = np.ones(6, np.float32), np.array([1, 1, 0, 1, 0, 0], np.float32)
    dx = e.empty(x.shape)
    e.TokenLogProbsDiff(put(e, x, "f32"), e.tensor(t), e.tensor(f["lse"]), e.tensor(f["entropy"]), e.tensor(g), dx, grad_entropy=e.tensor(h))
    got = dx.numpy()
    assert np.all(got[[2, 4]] == 0)
    want = bu.logprobs_diff(x, t, f["lse"].astype(np.float64), f["entropy"].astype(np.float64), g, h)
    close(got, want, diff_bound(x, {k: np.nan_to_num(v) for k, v in f.items()}, t, g, h, want, "f32"))


@pytest.mark.parametrize("vocab", [50, 20000])
def test_tokens_outside_the_vocabulary(fresh, vocab):
    """They are not read with; the row says NaN and the next call that waits reports it, once."""
    e = fresh
    x = logits(51, 4, vocab, "f32")
    tx = e.tensor(x.astype(np.float32))
    logp, lse = e.empty(4), e.empty(4)
    for bad in (vocab, -2, 1 << 40, -(1 << 62)):
        t = e.tensor(np.array([0, bad, -1, vocab - 1]))
        e.TokenLogProbs(tx, t, logp, lse=lse)
        with pytest.raises(B200Error, match="outside the vocabulary") as err:
            e.Signal()
        assert err.value.code == _lib.ERR_INVALID
        e.Signal()
        got = logp.numpy()
        assert np.isnan(got[1]) and got[2] == 0 and np.isfinite(got[[0, 3]]).all()
        dx = e.empty(x.shape)
        e.TokenLogProbsDiff(tx, t, lse, None, e.tensor(np.ones(4, np.float32)), dx)
        with pytest.raises(B200Error, match="outside the vocabulary"):
            dx.numpy()
        assert np.all(dx.numpy()[1:3] == 0)
    good = e.tensor(np.array([0, 1, -1, 2]))
    swap = e.tensor(np.array([0, 1, -1, 2]))
    e.TokenLogProbs(tx, good, logp)
    e.Signal()
    e.tape_begin()
    e.TokenLogProbs(tx, swap, logp)
    tape = e.tape_end()
    e.tape_launch(tape)
    e.Signal()
    swap.set(np.array([0, vocab, -1, 2]))
    e.tape_launch(tape)
    with pytest.raises(B200Error, match="outside the vocabulary"):
        e.Signal()
    swap.set(np.array([0, 3, -1, 2]))
    e.tape_launch(tape)
    e.Signal()
    e.tape_destroy(tape)


def test_no_rows(fresh):
    e = fresh
    x, t, s = e.empty((0, 50)), e.empty((0,), np.int64), e.empty((0,))
    e.TokenLogProbs(x, t, s, s, s, e.empty((0, 4)), e.empty((0, 4), np.int64))
    e.TokenLogProbsDiff(x, t, s, s, s, x, grad_entropy=s)


@pytest.mark.parametrize("rows,vocab,top,dtype", [(2, 100000, 20, "bf16"), (300, 3000, 5, "f32"), (64, 10, 2, "f64")])
def test_repeats_to_the_bit(fresh, rows, vocab, top, dtype):
    e = fresh
    x = logits(61, rows, vocab, dtype)
    tx, t = put(e, x, dtype), util.rng(5).integers(0, vocab, rows)
    first = forward(e, tx, t, top, dtype)
    s = stat(dtype)
    tt, lp, ent, lse = e.tensor(t), e.empty(rows, s), e.empty(rows, s), e.empty(rows, s)
    tl, ti = e.empty((rows, top), s), e.empty((rows, top), np.int64)
    e.tape_begin()
    e.TokenLogProbs(tx, tt, lp, ent, lse, tl, ti)
    tape = e.tape_end()
    for _ in range(3):
        for o in (lp, ent, lse, tl):
            o.set(np.zeros(o.shape, s))
        e.tape_launch(tape)
        for k, o in (("logp", lp), ("entropy", ent), ("lse", lse), ("top_logp", tl)):
            assert_bits_equal(o.numpy(), first[k])
        assert np.array_equal(ti.numpy(), first["top_index"])
    e.tape_destroy(tape)


def test_refusals(fresh):
    e = fresh
    x, i, s = e.tensor(np.zeros(400, np.float32)), e.tensor(np.zeros(64, np.int64)), e.empty(64)

    def fwd(dt=0, xp=x.ptr, ld=100, rows=4, vocab=100, t=i.ptr, lp=s.ptr, ent=s.ptr, lse=s.ptr, top=0, tl=None, ti=None):
        return lib.b200_token_logprobs(e.h, dt, xp, ld, rows, vocab, t, lp, ent, lse, top, tl, ti)

    def bwd(dt=0, xp=x.ptr, ld=100, rows=4, vocab=100, t=i.ptr, lse=s.ptr, ent=None, g=s.ptr, h=None, dx=x.ptr, lddx=100):
        return lib.b200_token_logprobs_bwd(e.h, dt, xp, ld, rows, vocab, t, lse, ent, g, h, dx, lddx)
    assert fwd() == 0 and fwd(rows=0, xp=None) == 0 and bwd() == 0 and bwd(rows=0, xp=None) == 0
    assert fwd(t=None, lp=None) == 0 and fwd(lse=None, ent=None) == 0
    for bad in (dict(dt=3), dict(dt=9), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 30) + 1, ld=1 << 31), dict(ld=99), dict(xp=None), dict(t=None), dict(lp=None),
                dict(top=33, tl=s.ptr, ti=i.ptr), dict(top=-1), dict(top=5, vocab=4, tl=s.ptr, ti=i.ptr), dict(top=2), dict(top=2, tl=s.ptr),
                dict(tl=s.ptr), dict(xp=x.ptr + 2), dict(t=i.ptr + 4), dict(lse=s.ptr + 2)):
        assert fwd(**bad) == _lib.ERR_INVALID, bad
    for bad in (dict(dt=4), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(lddx=99), dict(xp=None), dict(t=None), dict(lse=None),
                dict(g=None), dict(dx=None), dict(h=s.ptr), dict(lddx=101), dict(dx=x.ptr + 1), dict(g=s.ptr + 2)):
        assert bwd(**bad) == _lib.ERR_INVALID, bad
    flag = e.tensor(np.zeros(1, np.int32))
    with e.only_if(flag.ptr):
        assert fwd() == _lib.ERR_STATE and bwd() == _lib.ERR_STATE


# ---- the head as a whole -----------------------------------------------------------------------------

@pytest.mark.parametrize("recorded", [False, True])
def test_head_forward_and_backward(fresh, recorded):
    """Activations and weights to 8 bits, logits, the tokens' log probabilities, and back to the gradients of both: the
    calls of a training step one after the other, against the same steps in 64 bits on the same 8-bit values."""
    e = fresh
    rows, width, vocab = 130, 200, 500
    x, w = util.normal(71, (rows, width)), util.normal(72, (width, vocab), scale=0.1)
    t = util.rng(73).integers(0, vocab, rows)
    t[-9:] = -1                                    # the padded end of the batch
    tx, tw, tt = e.tensor(x), e.tensor(w), e.tensor(t)
    xr, xc = e.empty_blocks(x.shape, "row"), e.empty_blocks(x.shape, "col")
    wt = e.empty_blocks(w.shape, "tile")
    z, dz, dx, dw = e.empty((rows, vocab)), e.empty((rows, vocab)), e.empty(x.shape), e.tensor(np.zeros_like(w))
    zr, zc = e.empty_blocks((rows, vocab), "row", "e5m2"), e.empty_blocks((rows, vocab), "col", "e5m2")
    lp, ent, lse = e.empty(rows), e.empty(rows), e.empty(rows)
    tl, ti = e.empty((rows, 3)), e.empty((rows, 3), np.int64)
    g, h = e.tensor(np.full(rows, -1.0 / rows, np.float32)), e.tensor(np.where(t >= 0, -0.01, 0).astype(np.float32))

    def step():
        e.QuantizeBlocks(tx, xr)
        e.QuantizeBlocks(tx, xc)
        e.QuantizeBlocks(tw, wt)
        e.MatMulBlocks(xr, wt, z)
        e.TokenLogProbs(z, tt, lp, ent, lse, tl, ti)
        e.TokenLogProbsDiff(z, tt, lse, ent, g, dz, grad_entropy=h)
        e.QuantizeBlocks(dz, zr)
        e.QuantizeBlocks(dz, zc)
        e.MatMulBlocks(zr, wt, dx, transB=True)
        e.MatMulBlocks(xc, zc, dw, transA=True)
    step()
    if recorded:
        e.tape_begin()
        step()
        tape = e.tape_end()
        for o in (z, dz, dx, dw):
            o.set(np.zeros(o.shape, np.float32))
        e.tape_launch(tape)

    def host(b):
        return b.q.numpy(), b.scales.numpy(), b.format, b.block
    want_z, size = bu.matmul(host(xr), host(wt), False, False)
    zv = z.numpy()
    assert (np.abs(zv - want_z) <= bu.matmul_bound(size, width)).all()
    f = {"lse": lse.numpy(), "entropy": ent.numpy(), "logp": lp.numpy(), "top_logp": tl.numpy(), "top_index": ti.numpy()}
    compare(f, zv.astype(np.float64), t, 3, "f32")
    gv, hv = g.numpy(), h.numpy()
    want_dz = bu.logprobs_diff(zv, t, f["lse"].astype(np.float64), f["entropy"].astype(np.float64), gv, hv)
    dzv = dz.numpy()
    close(dzv, want_dz, diff_bound(zv.astype(np.float64), f, t, gv, hv, want_dz, "f32"))
    assert np.all(dzv[-9:] == 0)
    for b, block in ((zr, "row"), (zc, "col")):
        q, s = bu.quantize(dzv, "e5m2", block)
        assert np.array_equal(bu.f8_values("e5m2")[b.q.numpy()], q) and np.array_equal(b.scales.numpy(), s)
    want, size = bu.matmul(host(zr), host(wt), False, True)
    assert (np.abs(dx.numpy() - want) <= bu.matmul_bound(size, vocab)).all()
    want, size = bu.matmul(host(xc), host(zc), True, False)
    assert (np.abs(dw.numpy() - want) <= bu.matmul_bound(size, rows)).all()
    # and the gradient that comes out is the loss's: against 64 bits without any rounding to 8, to the 8-bit formats'
    # half steps (2^-4 of x and w, 2^-3 of the gradient), which average out over a sum
    exact_z = x.astype(np.float64) @ w
    f64 = bu.logprobs(exact_z, t)
    d64 = bu.logprobs_diff(exact_z, t, f64["lse"], f64["entropy"], gv, hv)
    for got, true in ((dx.numpy(), d64 @ w.T), (dw.numpy(), x.T.astype(np.float64) @ d64)):
        assert np.linalg.norm(got - true) <= (2 * 2.0 ** -4 + 2.0 ** -3) * np.linalg.norm(true)
    if recorded:
        e.tape_destroy(tape)
