"""Errors that are found on the device are reported one to a call, none lost for another: a target outside the vocabulary beside a
gather's index out of range, or beside a wait that ran out."""
import numpy as np
import pytest

from gorgonia_b200 import B200Error, _lib

pytestmark = pytest.mark.gpu


def reported(e, text, code=_lib.ERR_INVALID):
    with pytest.raises(B200Error, match=text) as err:
        e.Signal()
    assert err.value.code == code


@pytest.fixture()
def head(fresh):
    """An engine, a call of TokenLogProbs with a target outside its vocabulary, and the targets' tensor."""
    e = fresh
    x, logp = e.tensor(np.zeros((4, 50), np.float32)), e.empty(4)
    t = e.tensor(np.array([0, 50, -1, 3]))
    return e, (lambda: e.TokenLogProbs(x, t, logp)), t


def test_bad_token_beside_a_bad_gather_of_a_tape(head):
    """The same id looked up in the embeddings and asked for in the logits."""
    e, score, t = head
    table, rows = e.tensor(np.ones((50, 8), np.float32)), e.empty((4, 8))
    ids = e.tensor(np.array([0, 50, 1, 3]))
    e.tape_begin()
    e.ByIndices(table, ids, rows)
    score()
    tape = e.tape_end()
    for _ in range(2):
        e.tape_launch(tape)
        reported(e, "gather")
        reported(e, "outside the vocabulary")
        e.Signal()
    t.set(np.array([0, 1, -1, 3]))
    e.tape_launch(tape)
    reported(e, "gather")
    e.Signal()
    ids.set(np.array([0, 1, 2, 3]))
    e.tape_launch(tape)
    e.Signal()
    e.tape_destroy(tape)


def test_bad_token_beside_a_bad_eager_gather(head):
    """The gather's call waits and reports what it finds first; the next call that waits reports the other."""
    e, score, _ = head
    table, rows = e.tensor(np.ones((50, 8), np.float32)), e.empty((4, 8))
    ids, good = e.tensor(np.array([0, 50, 1, 3])), e.tensor(np.array([0, 1, 1, 3]))
    score()
    found = []
    for call in (lambda: e.ByIndices(table, ids, rows), e.Signal):
        with pytest.raises(B200Error) as err:
            call()
        assert err.value.code == _lib.ERR_INVALID
        found.append("vocabulary" if "vocabulary" in str(err.value) else "gather")
    assert sorted(found) == ["gather", "vocabulary"]
    e.Signal()
    e.ByIndices(table, good, rows)


def test_bad_token_beside_a_wait_that_ran_out(head):
    e, score, _ = head
    score()
    _lib.check(_lib.lib.b200_selftest_wait(e.h, 50), e.h)
    reported(e, "wait", _lib.ERR_TIMEOUT)
    reported(e, "outside the vocabulary")
    e.Signal()


def test_all_three(head):
    e, score, _ = head
    table, rows = e.tensor(np.ones((50, 8), np.float32)), e.empty((4, 8))
    ids = e.tensor(np.array([0, 50, 1, 3]))
    e.tape_begin()
    e.ByIndices(table, ids, rows)
    score()
    tape = e.tape_end()
    e.tape_launch(tape)
    _lib.check(_lib.lib.b200_selftest_wait(e.h, 50), e.h)
    reported(e, "wait", _lib.ERR_TIMEOUT)
    reported(e, "gather")
    reported(e, "outside the vocabulary")
    e.Signal()
    e.tape_destroy(tape)
