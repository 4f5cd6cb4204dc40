"""64-bit definitions of the 8-bit block operators and of the token log probabilities, in numpy."""
import numpy as np

BLOCKS = {"row": (1, 128), "col": (128, 1), "tile": (128, 128)}
F8 = {"e4m3": (3, 7, 448.0), "e5m2": (2, 15, 57344.0)}  # mantissa bits, exponent bias, largest value


def f8_values(fmt):
    """What each of the 256 bytes stands for."""
    bits, bias, _ = F8[fmt]
    b = np.arange(256)
    man, ex = b & ((1 << bits) - 1), (b & 0x7f) >> bits
    v = np.where(ex == 0, man * 2.0 ** (1 - bias - bits), (1 + man * 2.0 ** -bits) * 2.0 ** (ex - bias).astype(float))
    if fmt == "e4m3":
        v[(b & 0x7f) == 0x7f] = np.nan
    else:
        v[ex == 31] = np.where(man[ex == 31] == 0, np.inf, np.nan)
    return np.where(b >= 128, -v, v)


def spread(scales, shape, block):
    br, bc = BLOCKS[block]
    return np.repeat(np.repeat(scales.astype(np.float64), br, 0)[:shape[0]], bc, 1)[:, :shape[1]]


def quantize(x, fmt, block):
    """(values, scales) of the float32 matrix x, as float64."""
    bits, bias, most = F8[fmt]
    rows, cols = x.shape
    br, bc = BLOCKS[block]
    x = x.astype(np.float64)
    rb, cb = -(-rows // br), -(-cols // bc)
    scales = np.ones((rb, cb))
    for i in range(rb):
        for j in range(cb):
            b = x[i * br:(i + 1) * br, j * bc:(j + 1) * bc]
            b = np.abs(b[np.isfinite(b)])
            amax = b.max() if b.size else 0.0
            if amax > 0:
                e = -126
                while amax / 2.0 ** e > most:
                    e += 1
                scales[i, j] = 2.0 ** e
    with np.errstate(invalid="ignore"):
        v = x / spread(scales, x.shape, block)
        mag = np.abs(np.where(np.isfinite(v), v, 0.0))
        ex = np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -60))), 1 - bias)
        step = 2.0 ** (ex - bits)
        q = np.rint(v / step) * step
    if fmt == "e4m3":
        q[np.isinf(v)] = np.nan
    return q, scales


def to_bytes(values, fmt):
    """The bytes of values that the format holds."""
    table = f8_values(fmt)
    order = np.argsort(table[:128][np.isfinite(table[:128])])
    fin = table[:128][np.isfinite(table[:128])][order]
    mag = np.abs(values)
    idx = np.searchsorted(fin, mag)
    assert np.array_equal(fin[idx], mag)
    return (order[idx] | np.where(np.signbit(values), 0x80, 0)).astype(np.uint8)


def random_blocks(seed, shape, fmt, block, spread_exp=3):
    """(bytes, scales) with values over the whole format and scales that are no powers of two."""
    r = np.random.Generator(np.random.Philox(seed))
    v, _ = quantize(r.standard_normal(shape).astype(np.float32), fmt, block)
    br, bc = BLOCKS[block]
    s = np.exp(r.uniform(-spread_exp, spread_exp, (-(-shape[0] // br), -(-shape[1] // bc)))).astype(np.float32)
    return to_bytes(v, fmt), s


def matmul(a, b, ta, tb):
    """op(a) op(b) in 64 bits and the sum of the magnitudes of its terms; a, b = (bytes, scales, fmt, block)."""
    def wide(o, t):
        q, s, fmt, block = o
        w = f8_values(fmt)[q] * spread(s, q.shape, block)
        return w.T if t else w
    wa, wb = wide(a, ta), wide(b, tb)
    return wa @ wb, np.abs(wa) @ np.abs(wb)


def matmul_bound(size, K, out_eps=0.0, value=0.0):
    """Error bound of a product whose terms' magnitudes sum to `size`. A block of 128 products (exact in fp32)
    is summed in fp32 by an adder that may cut off instead of rounding: at most 2^-23 of the running magnitude for
    each term. A block's sum is multiplied by its two scales (three roundings of 2^-24 with their product) and added to at
    most ceil(K / 128) others, in shares at most twice that many additions of 2^-24. Rounding the result
    to its own type adds half a step."""
    blocks = -(-K // 128)
    return size * (128 * 2.0 ** -23 + (3 + 2 * blocks) * 2.0 ** -24) + out_eps / 2 * np.abs(value)


def logprobs(x, targets=None, top=0):
    """The definition of token log probabilities in 64 bits: dict of lse, entropy, logp, top_logp, top_index."""
    x = x.astype(np.float64)
    rows, vocab = x.shape
    out = {k: np.empty(rows) for k in ("lse", "entropy", "logp")}
    out["top_index"] = np.empty((rows, top), np.int64)
    out["top_logp"] = np.empty((rows, top))
    for r in range(rows):
        v = x[r]
        wild = np.isnan(v).any() or (v == np.inf).any()
        some = v > -np.inf
        if wild:
            lse = ent = np.nan
        elif not some.any():
            lse, ent = -np.inf, 0.0
        else:
            m = v[some].max()
            log_s = np.log(np.exp(v[some] - m).sum())
            lse = m + log_s
            d = v[some] - m
            p = np.exp(d - log_s)
            ent = -(p * np.where(p > 0, d - log_s, 0.0)).sum()

        def lp(i):
            return np.nan if wild else (-np.inf if v[i] == -np.inf else (v[i] - m) - log_s)
        out["lse"][r], out["entropy"][r] = lse, ent
        if targets is not None:
            t = targets[r]
            out["logp"][r] = 0.0 if t == -1 else (lp(t) if 0 <= t < vocab else np.nan)
        key = np.where(np.isnan(v), np.inf, v)
        order = np.lexsort((np.arange(vocab), -key, ~np.isnan(v)))[:top]
        out["top_index"][r] = order
        out["top_logp"][r] = [lp(i) for i in order]
    return out


def logprobs_diff(x, targets, lse, entropy, g, h):
    x = x.astype(np.float64)
    rows, vocab = x.shape
    dx = np.zeros((rows, vocab))
    for r in range(rows):
        gr = g[r] if 0 <= targets[r] < vocab else 0.0
        hr = 0.0 if h is None else h[r]
        if (gr == 0 and hr == 0) or lse[r] == -np.inf:
            continue
        lp = x[r] - lse[r]
        p = np.exp(lp)
        dx[r] = -gr * p
        if hr:
            with np.errstate(invalid="ignore"):
                dx[r] -= np.where(p == 0, 0.0, hr * p * (lp + entropy[r]))
        if 0 <= targets[r] < vocab:
            dx[r, targets[r]] += gr
    return dx


def stat_bound(x, lse, unit):
    """Error bound of lse, entropy and log probabilities; unit = half a step of the type they are computed in.
    A term e^d, d = x - m, is off by (2 |d| + 8) units (the product d log2 e and its constant, the exponential); weighted by
    p the |d| average at most ln V. A thread adds at most V / 32 terms one after the other, and their partial sums are
    joined in at most 16 steps. The entropy's second sum is of terms e^d d, |d| at most ln V on average."""
    vocab = x.shape[1]
    ln = np.log(vocab) + 1
    terms = (2 * ln + 8 + vocab / 32 + 16) * unit
    return terms + 2 * np.abs(lse) * unit, 3 * (1 + ln) * terms
