"""A gather's index out of range is reported by the next call that waits, whatever other gathers have run since."""
import numpy as np
import pytest

from gorgonia_b200 import B200Error, _lib

pytestmark = pytest.mark.gpu


def reported(call):
    with pytest.raises(B200Error, match="gather") as err:
        call()
    assert err.value.code == _lib.ERR_INVALID


@pytest.fixture()
def parts(fresh):
    e = fresh
    ids = [e.tensor(np.array([0, 2, 1])) for _ in range(2)]
    return e, e.tensor(np.arange(24, dtype=np.float32).reshape(3, 8)), ids, [e.empty((3, 8)) for _ in range(2)]


@pytest.mark.parametrize("bad", [0, 1])
def test_two_gathers_in_a_tape(parts, bad):
    e, table, ids, out = parts
    e.tape_begin()
    for i, o in zip(ids, out):
        e.ByIndices(table, i, o)
    tape = e.tape_end()
    e.tape_launch(tape)
    e.Signal()
    ids[bad].set(np.array([0, 3, 1]))
    e.tape_launch(tape)
    reported(e.Signal)
    e.Signal()
    ids[bad].set(np.array([1, 1, 1]))
    e.tape_launch(tape)
    e.Signal()
    assert np.array_equal(out[bad].numpy(), table.numpy()[[1, 1, 1]])
    e.tape_destroy(tape)


def test_a_good_gather_after_a_bad_tape(parts):
    """Nothing has waited in between: the eager call is the one that does, and reports it; its own rows are there."""
    e, table, ids, out = parts
    e.tape_begin()
    e.ByIndices(table, ids[0], out[0])
    tape = e.tape_end()
    ids[0].set(np.array([0, -1, 1]))
    e.tape_launch(tape)
    reported(lambda: e.ByIndices(table, ids[1], out[1]))
    e.Signal()
    assert np.array_equal(out[1].numpy(), table.numpy()[[0, 2, 1]])
    e.ByIndices(table, ids[1], out[1])
    e.tape_destroy(tape)


def test_a_bad_tape_replayed_again_with_good_indices(parts):
    e, table, ids, out = parts
    good = e.tensor(np.array([2, 1, 0]))
    ids[0].set(np.array([0, 7, 1]))
    e.tape_begin()
    e.ByIndices(table, ids[0], out[0])
    tape = e.tape_end()
    e.tape_begin()
    e.ByIndices(table, good, out[1])
    other = e.tape_end()
    e.tape_launch(tape)
    e.tape_launch(other)
    reported(e.Signal)
    e.Signal()
    e.tape_launch(other)
    e.Signal()
    for t in (tape, other):
        e.tape_destroy(t)


def test_a_bad_eager_gather_is_reported_once(parts):
    e, table, ids, out = parts
    ids[0].set(np.array([0, 3, 1]))
    reported(lambda: e.ByIndices(table, ids[0], out[0]))
    e.Signal()
    e.tape_begin()
    e.ByIndices(table, ids[1], out[1])
    tape = e.tape_end()
    e.tape_launch(tape)
    e.Signal()
    e.ByIndices(table, ids[1], out[1])
    e.tape_destroy(tape)
