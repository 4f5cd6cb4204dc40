"""Arguments of the 8-bit and token calls that have the wrong number of dimensions or an unknown name: refused with the
library's own error, before anything is taken from the arena."""
import numpy as np
import pytest

from gorgonia_b200 import B200Error, Engine, Tensor, _lib


@pytest.fixture()
def e():
    """An engine without a device that counts what is taken from its arena and given back."""
    x = Engine.__new__(Engine)
    x.h = None
    x.held = []
    x.room = 10

    def get(nbytes):
        if len(x.held) == x.room:
            raise B200Error(_lib.ERR_OOM, "full")
        x.held.append(4096 * (len(x.held) + 1))
        return x.held[-1]
    x.Get = get
    x.Put = lambda ptr, nbytes=0: x.held.remove(ptr)
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


@pytest.mark.parametrize("shape", [(4, 3, 50), (50,), (4, -1), ()])
def test_block_matrices_have_two_dimensions(e, shape):
    refused("two dimensions", e.empty_blocks, shape)
    assert not e.held


def test_unknown_blocks_and_formats(e):
    refused("block 'diagonal' is not one of", e.empty_blocks, (4, 50), "diagonal")
    refused("format 'e3m4' is not one of", e.empty_blocks, (4, 50), "row", "e3m4")
    assert not e.held


def test_no_room_for_the_scales(e):
    """What has been taken for the values goes back."""
    e.room = 1
    refused("full", e.empty_blocks, (4, 50), code=_lib.ERR_OOM)
    assert not e.held
