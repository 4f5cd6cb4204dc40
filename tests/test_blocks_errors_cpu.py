"""Arguments of the 8-bit and token calls that have the wrong number of dimensions: refused with the library's own error."""
import numpy as np
import pytest

from gorgonia_b200 import B200Error, Engine, Tensor, _lib


@pytest.fixture()
def e():
    """An engine without a device."""
    x = Engine.__new__(Engine)
    x.h = None
    return x


def tensor(e, shape, dtype=np.float32):
    return Tensor(e, 4096, shape, dtype, owned=False)


def refused(text, call, *args, code=_lib.ERR_INVALID, **kw):
    with pytest.raises(B200Error, match=text) as err:
        call(*args, **kw)
    assert err.value.code == code


@pytest.mark.parametrize("shape", [(4, 3, 50), (50,), ()])
def test_logits_are_a_matrix(e, shape):
    """Logits of a batch of sequences are reshaped first; a row alone is (1, vocab)."""
    x, rows = tensor(e, shape), 12
    s, t = tensor(e, (rows,)), tensor(e, (rows,), np.int64)
    refused("TokenLogProbs: the logits are a matrix", e.TokenLogProbs, x, t, s)
    refused("TokenLogProbsDiff: the logits are a matrix", e.TokenLogProbsDiff, x, t, s, s, s, x)
