"""The device model on 4-bit weights (qw2_quantize_weights) and with controls
on its choices (qw2_set_controls).

Weights that 4 bits hold exactly (whole multiples of a power of two, each
group's largest 7) make the 4-bit and the fp16 model the same function up to
the order of the fp32 sums.  Such a difference can move a projection's result
by one fp16 step (2^-10 of it, the truncating rounding); with 4 projections in
each of 2 layers and the head, and each moving the norms behind it at most
twice as far, logits differ by at most 2 * 9 * 2^-10 of their norm.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_model_sessions import SMALL, need_gpu, prompt, q2
from test_step_ops import plain_logits

FAR = 2 * 9 * 2.0**-10


def exact_weights(seed):
    """Every matrix k / 128 with whole |k| <= 7, a 7 in each run of 32 inputs."""
    rng = np.random.default_rng(seed)
    for name, shape, init in q2().tensor_specs(SMALL):
        if len(shape) == 2:
            a = np.clip(np.rint(rng.standard_normal(shape) * 2.5), -7, 7)
            a[:, ::32] = np.where(rng.random(a[:, ::32].shape) < 0.5, 7, -7)
            yield name, (a / 128).astype(np.float32)
        elif init == "ones":
            yield name, (1 + 0.1 * rng.standard_normal(shape)).astype(np.float32)
        else:
            yield name, (rng.standard_normal(shape) * 0.02).astype(np.float32)


def build(seed=3, sessions=8):
    M = q2().Model(0, SMALL, max_sessions=sessions)
    for name, a in exact_weights(seed):
        M.set_tensor(name, a)
    return M


def near(a, b):
    return np.linalg.norm(a - b) <= FAR * np.linalg.norm(b)


@pytest.fixture(scope="module")
def plain_model():
    need_gpu()
    M = build()
    yield M
    M.close()


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros", [(32, False), (64, False), (128, False)])
def test_4bit_model_is_the_fp16_model_on_exact_weights(plain_model, group, zeros):
    need_gpu()
    P, M = plain_model, build()
    before = M.weight_bytes()
    M.quantize_weights(group, zeros)
    assert M.weight_bytes() < before * (0.27 + 2 / group / 2)
    for n in (1, 5, 40, 130):  # one token, a chunk through one pass and several
        ids = prompt(n, 50 + n)
        sp, sm = P.create_session(), M.create_session()
        a, _ = P.forward_session(sp, ids)
        b, am = M.forward_session(sm, ids)
        assert near(b, a) and am == int(np.argmax(b))
        for t in prompt(4, n):
            a, _ = P.forward_session(sp, [t])
            b, am = M.forward_session(sm, [t])
            assert near(b, a) and am == int(np.argmax(b))
        P.destroy_session(sp)
        M.destroy_session(sm)
    # several sessions decoding together
    sids = [M.create_session() for _ in range(4)]
    reqs = [dict(session=s, input_ids=prompt(7 + 9 * i, 80 + i), max_new_tokens=6) for i, s in enumerate(sids)]
    for (ids, res), r in zip(M.generate_batch(reqs), reqs):
        assert res["status"] == 0 and len(ids) == 6
        s = P.create_session()
        logits, _ = P.forward_session(s, r["input_ids"])
        for t in ids:
            assert logits[t] >= logits.max() - 2 * FAR * np.linalg.norm(logits)
            logits, _ = P.forward_session(s, [t])
        P.destroy_session(s)
    M.close()


@pytest.mark.gpu
def test_4bit_model_with_zero_points_runs_near(plain_model):
    """Zero points round these weights (a group's range over 15 is no power of two): the same choice of scale as
    w4_quantize makes, so the logits stay near the fp16 model's."""
    need_gpu()
    M = build()
    M.quantize_weights(32, True)
    ids = prompt(20, 4)
    s = plain_model.create_session()
    a, _ = plain_model.forward_session(s, ids)
    plain_model.destroy_session(s)
    b, _ = M.forward(ids)
    assert np.all(np.isfinite(b))
    # a code is off by at most half a step of 14 / 15 / 128 in weights of rms 3 / 128: 8 % per projection
    assert np.linalg.norm(b - a) < 0.5 * np.linalg.norm(a)
    M.close()


@pytest.mark.gpu
def test_4bit_model_refusals():
    need_gpu()
    m = q2()
    M = build(sessions=2)
    for group in (0, 16, 48, 256):
        with pytest.raises(m.KVError):
            M.quantize_weights(group)
    a, _ = M.forward(prompt(3, 1))
    M.set_exact(True)
    with pytest.raises(m.KVError):
        M.quantize_weights(128)
    M.set_exact(False)
    M.quantize_weights(128)
    for call in (lambda: M.quantize_weights(128), lambda: M.set_exact(True),
                 lambda: M.set_tensor("model.layers.0.mlp.up_proj.weight", np.zeros((512, 256), np.float32)),
                 lambda: M.set_tensor("model.embed_tokens.weight", np.zeros((1000, 256), np.float32))):
        with pytest.raises(m.KVError):
            call()
    M.set_tensor("model.norm.weight", np.ones(256, np.float32))  # vectors stay open
    M.forward(prompt(3, 1))
    M.close()
    M = m.Model(0, SMALL)
    with pytest.raises(m.KVError):
        M.quantize_weights(128)  # no tensors yet
    M.close()


def choice(logits, history, gen_from, rep=1.0, pres=0.0, freq=0.0, bias=(), allowed=None):
    y, _ = plain_logits(logits.astype(np.float64), history, gen_from, float(np.float32(rep)), float(np.float32(pres)),
                        float(np.float32(freq)), [(t, float(np.float32(b))) for t, b in bias], allowed)
    return int(np.argmax(y)) if np.any(np.isfinite(y)) else -1


@pytest.mark.gpu
def test_controls_choose_as_their_definition_says(plain_model):
    need_gpu()
    M = plain_model
    s = M.create_session()
    allowed = np.random.default_rng(2).random(SMALL["vocab"]) < 0.6
    bias = {5: 0.25, 700: -0.5, 31: 0.125}
    kw = dict(repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=0.25)
    M.set_controls(s, bias=bias, allowed=allowed, **kw)
    history = prompt(12, 9)
    logits, am = M.forward_session(s, history)
    gen = len(history)
    for _ in range(12):
        assert am == choice(logits, history, gen, 1.25, 0.5, 0.25, bias.items(), allowed)
        history = history + [am]
        logits, am = M.forward_session(s, [am])
    # a longer forward: what it brings is prompt again
    more = prompt(6, 10)
    history, gen = history + more, len(history) + 6
    logits, am = M.forward_session(s, more)
    assert am == choice(logits, history, gen, 1.25, 0.5, 0.25, bias.items(), allowed)
    M.clear_controls(s)
    logits, am = M.forward_session(s, [1])
    assert am == int(np.argmax(logits))
    M.destroy_session(s)


@pytest.mark.gpu
def test_controls_in_a_batch_and_grammar_callback(plain_model):
    """Requests with and without controls in one batch: the plain ones are as without; a grammar that ends, ends its
    request; a failing callback fails its request alone."""
    need_gpu()
    M = plain_model
    V = SMALL["vocab"]
    a, b, c, d = (M.create_session() for _ in range(4))
    alone, _ = M.generate_session(a, prompt(10, 20), 8)
    M.destroy_session(a)
    a = M.create_session()
    seen = []

    def grammar(session, ids, gen_from):
        seen.append((session, len(ids), gen_from))
        ok = np.zeros(V, bool)
        n = len(ids) - gen_from
        if n < 4:
            ok[n::7] = True  # the n-th id is n modulo 7
        return ok

    def broken(session, ids, gen_from):
        raise RuntimeError("no grammar")

    M.set_controls(b, mask=grammar)
    M.set_controls(c, frequency_penalty=0.75, repetition_penalty=1.1)
    M.set_controls(d, mask=broken)
    got = M.generate_batch([dict(session=a, input_ids=prompt(10, 20), max_new_tokens=8),
                            dict(session=b, input_ids=prompt(14, 21), max_new_tokens=8),
                            dict(session=c, input_ids=prompt(5, 22), max_new_tokens=8),
                            dict(session=d, input_ids=prompt(5, 23), max_new_tokens=8)])
    ids, res = got[0]
    assert res["status"] == 0 and len(ids) == 8
    replay = M.create_session()
    logits, _ = M.forward_session(replay, prompt(10, 20))
    for t in ids:
        assert logits[t] >= logits.max() - 2 * FAR * np.linalg.norm(logits)
        logits, _ = M.forward_session(replay, [t])
    M.destroy_session(replay)
    ids, res = got[1]
    assert [t % 7 for t in ids] == [0, 1, 2, 3] and res["hit_stop"] == 1 and res["status"] == 0
    assert seen == [(b, 14 + i, 14) for i in range(5)]
    ids, res = got[2]
    assert res["status"] == 0 and len(ids) == 8
    assert got[3][1]["status"] != 0 and got[3][0] == []
    for s in (a, b, c, d):
        M.destroy_session(s)
    # through the async calls, with the session's controls gone after its destruction
    s = M.create_session()
    job = M.submit(s, prompt(10, 20), 8)
    ids, res = M.wait(job)
    assert res["status"] == 0 and ids == alone
    M.set_controls(s, mask=lambda session, h, g: np.arange(V) == 42)
    ids, res = M.wait(M.submit(s, prompt(3, 1), 3))
    assert ids == [42, 42, 42]
    M.destroy_session(s)


@pytest.mark.gpu
def test_controls_refusals(plain_model):
    need_gpu()
    M, err = plain_model, q2().KVError
    s = M.create_session()
    for kw in (dict(repetition_penalty=0.0), dict(repetition_penalty=float("nan")), dict(presence_penalty=float("inf"))):
        with pytest.raises(err):
            M.set_controls(s, **kw)
    with pytest.raises(ValueError):
        M.set_controls(s, allowed=np.ones(5, bool))
    with pytest.raises(err):
        M.set_controls(99)
    M.set_controls(s, allowed=np.zeros(SMALL["vocab"], bool))
    logits, am = M.forward_session(s, prompt(4, 2))
    assert am == -1 and np.all(np.isfinite(logits))
    ids, res = M.generate_session(s, prompt(4, 2), 5)
    assert ids == [] and res["hit_stop"] == 1
    M.destroy_session(s)
