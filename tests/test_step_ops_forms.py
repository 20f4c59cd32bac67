"""More forms of the step operators on a GPU: calls on several streams, operand
rows at the borders between the kernels, special values in each of them,
waits that run out.  Tolerances are those of test_step_ops.py."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from test_model_sessions import SMALL, prompt, q2
from test_step_ops import dbl, fill, half_step, need_gpu, plain_quantize, random_matrix, sum_tol  # noqa: F401


def near_linear(kv, w, ref, x, out, group, yd):
    """out = x W^T within test_step_ops.py's bound."""
    want = dbl(x) @ ref.T
    tol = sum_tol(dbl(x), ref, group) + 2.0**-23 * np.abs(want)
    tol = tol + half_step(np.abs(want) + tol, yd)
    assert np.all(np.abs(dbl(out) - want) <= tol), np.max(np.abs(dbl(out) - want) / tol)


# --------------------------------------------- rows at the borders between the kernels
@pytest.mark.gpu
@pytest.mark.parametrize("n,k,group", [(96, 4096, 32), (200, 4100, 128), (1500, 640, 64)])
@pytest.mark.parametrize("xd", ["f32", "bf16"])
def test_linear_from_few_to_many_rows(kv, n, k, group, xd):
    """Every count of rows from 1 to 24, and around a tile of columns: with the scratch that the planner asks for,
    where the parts of five fp32 rows go to the tensor-memory form, and without any."""
    need_gpu()
    rng = np.random.default_rng(k)
    w, ref = random_matrix(kv, rng, n, k, group, True)
    for m in (*range(1, 25), 41, 43, 64, 65, 85, 86):
        x, out = fill(rng, (m, k), xd), torch.empty(m, n, device="cuda")
        kv.w4_linear(w, x, out)
        near_linear(kv, w, ref, x, out, group, "f32")
        out.fill_(0)
        kv.call("w4_linear", w._at, x.data_ptr(), kv.STEP_F32 if xd == "f32" else kv.STEP_BF16, m, k, None, None, 0,
                out.data_ptr(), kv.STEP_F32, n, None, torch.cuda.current_stream().cuda_stream)
        near_linear(kv, w, ref, x, out, group, "f32")
    assert kv.step_ops_status() == kv.KV_OK


# ------------------------------------------------------------------ streams
@pytest.mark.gpu
@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("xd,offset", [("f32", 0), ("f16", 1)])
def test_calls_on_two_streams_at_once(kv, op, xd, offset):
    """Different rows on two streams at once, both through scratch: each result is the one that its rows have alone."""
    need_gpu()
    rng = np.random.default_rng(41)
    m, n, k = 64, 1536, 8960
    w, _ = random_matrix(kv, rng, n, k, 128, False)
    xs = [fill(rng, (m, k + 8), xd)[:, offset:offset + k] for _ in range(2)]

    def go(x, out, stream=None):
        if op == "linear":
            kv.w4_linear(w, x, out, stream=stream)
        else:
            kv.w4_gated(w, w, x, out, stream=stream)

    alone = [torch.empty(m, n, device="cuda") for _ in xs]
    for x, out in zip(xs, alone):
        go(x, out)
        torch.cuda.synchronize()
    assert not torch.equal(*alone)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [[torch.empty(m, n, device="cuda") for _ in xs] for _ in range(12)]
    torch.cuda.synchronize()
    for a, b in outs:
        go(xs[0], a)
        go(xs[1], b, s)
    for a, b in outs[:2]:  # an address in place of a stream object
        go(xs[1], b, s.cuda_stream)
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, alone[0]) and torch.equal(b, alone[1])


@pytest.mark.gpu
def test_results_on_another_stream_leave_pending_work_alone(kv):
    """Quantising and reading back on another stream while the current one still has work on a tensor that was freed."""
    need_gpu()
    rng = np.random.default_rng(42)
    w = fill(rng, (512, 1024), "f16")
    want = kv.w4_quantize(w, 32, zero_points=True)
    values = want.dequantize()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        ones = [torch.ones(size, dtype=torch.uint8, device="cuda")
                for size in (want.codes.nbytes, want.scales.nbytes, want.zeros.nbytes, values.nbytes)]
        s.wait_stream(torch.cuda.current_stream())
        torch.cuda._sleep(20_000_000)  # the sums come ten milliseconds later
        sums = [t.sum(dtype=torch.int64) for t in ones]
        sizes = [t.numel() for t in ones]
        del ones
        got = kv.w4_quantize(w, 32, zero_points=True, stream=s)
        read = got.dequantize(stream=s)
        torch.cuda.synchronize()
        assert [int(t) for t in sums] == sizes
        assert torch.equal(got.codes, want.codes) and torch.equal(read, values)


# ---------------------------------------------------------- after an error
@pytest.mark.gpu
def test_a_refused_call_leaves_no_error_behind(kv):
    """A device that is not there and memory that is not there are reported once, by the call that asked for them."""
    need_gpu()
    w = fill(np.random.default_rng(1), (64, 64), "f16")
    m = kv.w4_quantize(w, 32)
    values = m.dequantize()

    def fine():
        assert torch.equal(kv.w4_quantize(w, 32).codes, m.codes) and torch.equal(m.dequantize(), values)

    with pytest.raises(kv.KVError):
        kv.step_ops_status(999)
    fine()
    far = kv._W4Matrix(999, 64, 64, 32, m.codes.data_ptr(), m.scales.data_ptr(), None)
    out = torch.empty(2, 64, device="cuda")
    for name, args in (("w4_quantize", (w.data_ptr(), 0, 64)), ("w4_dequantize", (values.data_ptr(), 64)),
                       ("w4_linear", (w.data_ptr(), 0, 2, 64, None, None, 0, out.data_ptr(), 2, 64, None))):
        with pytest.raises(kv.KVError):
            kv.call(name, C.addressof(far), *args, None)
        fine()
    cfg = dict(q2().QWEN2_1_5B, hidden=4096, q_heads=32, kv_heads=32, vocab=2**30, layers=1)  # 8 TB of embedding
    with pytest.raises(kv.KVError):
        q2().Model(0, cfg)
    fine()


# ------------------------------------------------------- waits that run out
@pytest.fixture
def no_waiting(kv):
    """Launches give up wherever something is not ready, from its call on; the default limit afterwards."""
    yield lambda: kv.step_ops_wait_limit(0)
    kv.step_ops_wait_limit()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,xd", [(20, 200, 4096, "f16"), (100, 200, 4096, "bf16"), (300, 200, 4096, "f16"),
                                      (70, 20000, 260, "f16"), (60, 500, 700, "f32")])
@pytest.mark.parametrize("group", [32, 128])
def test_a_wait_that_runs_out_is_reported(kv, no_waiting, m, n, k, xd, group):
    """By step_ops_status, once; the device works on and the next call is right."""
    need_gpu()
    rng = np.random.default_rng(m + n)
    w, ref = random_matrix(kv, rng, n, k, group, True)
    x, out = fill(rng, (m, k), xd), torch.empty(m, n, device="cuda")
    assert kv.step_ops_status() == kv.KV_OK
    for op in (lambda: kv.w4_linear(w, x, out), lambda: kv.w4_gated(w, w, x, out)):
        no_waiting()
        op()
        assert kv.step_ops_status() == kv.KV_ERR_TIMEOUT
        assert kv.step_ops_status() == kv.KV_OK
        kv.step_ops_wait_limit()
        kv.w4_linear(w, x, out)
        near_linear(kv, w, ref, x, out, group, "f32")
        assert kv.step_ops_status() == kv.KV_OK


@pytest.fixture(scope="module")
def model4():
    """The small model on 4-bit weights."""
    need_gpu()
    M = q2().Model(0, SMALL, max_sessions=8)
    for name, a in q2().synth_weights(SMALL, seed=21):
        M.set_tensor(name, a)
    M.quantize_weights(64)
    yield M
    M.close()


@pytest.mark.gpu
def test_a_forwards_wait_that_runs_out_fails_the_forward(kv, no_waiting, model4):
    """KV_ERR_TIMEOUT from the model's own call, nothing for step_ops_status to find; other sessions go on."""
    need_gpu()
    M = model4
    a, b = M.create_session(), M.create_session()
    M.forward_session(a, prompt(20, 1))
    want, pick = M.forward_session(b, prompt(130, 2))
    M.destroy_session(b)
    b = M.create_session()
    no_waiting()
    with pytest.raises(q2().KVError) as e:
        M.forward_session(b, prompt(130, 2))
    assert e.value.status == kv.KV_ERR_TIMEOUT
    with pytest.raises(q2().KVError) as e:
        M.generate_session(b, prompt(130, 3), 3)
    assert e.value.status == kv.KV_ERR_TIMEOUT
    kv.step_ops_wait_limit()
    assert kv.step_ops_status() == kv.KV_OK
    M.destroy_session(b)
    b = M.create_session()
    got, again = M.forward_session(b, prompt(130, 2))
    assert np.array_equal(got, want) and again == pick
    logits, _ = M.forward_session(a, [3])
    assert np.all(np.isfinite(logits))
    for s in (a, b):
        M.destroy_session(s)


@pytest.mark.gpu
def test_a_failed_forwards_ids_stay_in_the_history(kv, no_waiting, model4):
    """The history that controls see is the ids in the cache, those of a forward that failed on the way included."""
    need_gpu()
    M, seen = model4, []
    s = M.create_session()
    M.set_controls(s, mask=lambda session, ids, gen_from: seen.append((list(ids), gen_from)))
    first = prompt(130, 5)
    no_waiting()
    with pytest.raises(q2().KVError):
        M.forward_session(s, first)
    kv.step_ops_wait_limit()
    M.forward_session(s, [9])
    assert seen == [(first + [9], 130)]
    M.destroy_session(s)
