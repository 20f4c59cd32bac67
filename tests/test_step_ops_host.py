"""The Python side of the step operators and of the model's controls, without
a GPU: what crosses the C boundary and when.  The C library's calls are stood in for."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_model_sessions import q2


class _Model:
    """A Model without a device: set_controls and its callback only."""

    def __new__(cls, vocab):
        m = q2()
        M = m.Model.__new__(m.Model)
        M.h, M.cfg, M._callbacks, M._keep = C.c_void_p(), dict(vocab=vocab), {}, {}
        M.kept = []

        class Lib:
            @staticmethod
            def qw2_set_controls(h, session, c):
                M.kept.append(c)
                return 0

        M.L = Lib
        return M


def mask_of(M, session, ids, gen_from, n_words):
    """(the callback's status, the words it filled in), as the engine calls it."""
    words = np.full(n_words, 0xFFFFFFFF, np.uint32)
    tokens = (C.c_int * max(1, len(ids)))(*ids)
    rc = M._callbacks[session](None, session, tokens, len(ids), gen_from, words.ctypes.data_as(C.POINTER(C.c_uint32)), n_words)
    return rc, words


@pytest.mark.parametrize("form", ["bool", "every second bool", "uint32", "every second word"])
@pytest.mark.parametrize("vocab", [1, 33, 1000, 8193, 32000, 151936])
def test_mask_callback_hands_over_every_word(vocab, form):
    M = _Model(vocab)
    rng = np.random.default_rng(vocab)
    words = -(-vocab // 32)
    given = []

    def mask(session, ids, gen_from):
        if "bool" in form:
            a = rng.random(vocab * (2 if "second" in form else 1)) < 0.5
        else:
            a = rng.integers(0, 1 << 32, words * (2 if "second" in form else 1), dtype=np.uint32)
        a = a[::2] if "second" in form else a
        given.append(np.array(a))
        return a

    M.set_controls(3, mask=mask)
    for i in range(20):
        rc, got = mask_of(M, 3, [1, 2, 3], 2, words)
        assert rc == 1
        want = given[-1]
        if "bool" in form:
            bits = np.unpackbits(got.view(np.uint8), bitorder="little")
            assert np.array_equal(bits[:vocab].astype(bool), want) and not bits[vocab:].any()
        else:
            assert np.array_equal(got, want)


@pytest.mark.filterwarnings("error::pytest.PytestUnraisableExceptionWarning")
@pytest.mark.parametrize("error", [RuntimeError, KeyboardInterrupt, SystemExit, GeneratorExit])
def test_mask_callback_that_raises_fails_its_request(error):
    """Whatever it raises: a status of 0 would choose without the mask."""
    M = _Model(1000)

    def mask(session, ids, gen_from):
        raise error

    M.set_controls(0, mask=mask)
    assert mask_of(M, 0, [5], 0, 32)[0] < 0


@pytest.mark.parametrize("answer", [np.ones(999, bool), np.ones((1, 1000), bool), np.ones(32, np.int64), np.ones(31, np.uint32)])
def test_mask_callback_with_an_unfit_answer_fails_its_request(answer):
    M = _Model(1000)
    M.set_controls(0, mask=lambda session, ids, gen_from: answer)
    assert mask_of(M, 0, [5], 0, 32)[0] < 0
