"""Rounding to 8 bits of matrices with more rows than one launch's grid has blocks for."""
import numpy as np
import pytest

from tests import blocks_util as bu

pytestmark = pytest.mark.gpu

PIECE = 65535 * 128     # rows of a grid


@pytest.mark.parametrize("block", ["row", "col", "tile"])
@pytest.mark.parametrize("cols,bf16", [(1, False), (8, True)])
def test_quantize_many_rows(fresh, cols, bf16, block):
    e = fresh
    rows = 2 * PIECE + 300
    x = np.resize(np.random.Generator(np.random.Philox(7)).standard_normal((10007, cols)).astype(np.float32), (rows, cols))
    tx = e.tensor_bf16(x) if bf16 else e.tensor(x)
    q = e.empty_blocks(x.shape, block)
    q.q.set(np.full(x.shape, 0x7f, np.uint8))
    q.scales.set(np.zeros(q.scales.shape, np.float32))
    e.QuantizeBlocks(tx, q)
    got, scales = q.q.numpy(), q.scales.numpy()
    if bf16:
        from gorgonia_b200.engine import from_bf16
        x = from_bf16(tx.numpy())
    for first in (0, PIECE - 256, 2 * PIECE - 256, rows - 300 - 128):
        assert first % 128 == 0
        part = x[first:first + 428]
        want, s = bu.quantize(part, "e4m3", block)
        n = len(part) if first + len(part) == rows else len(part) // 128 * 128     # whole blocks, or the last ones
        assert np.array_equal(bu.f8_values("e4m3")[got[first:first + n]], want[:n])
        at, count = (first, n) if block == "row" else (first // 128, -(-n // 128))
        assert np.array_equal(scales[at:at + count].astype(np.float64), s[:count])
    assert np.all((got & 0x7f) != 0x7f) and np.all(scales > 0)
