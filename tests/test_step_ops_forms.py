"""More forms of the step operators on a GPU: calls on several streams, operand
rows at the borders between the kernels, special values in each of them,
waits that run out.  Tolerances are those of test_step_ops.py."""
from __future__ import annotations

import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from test_model_sessions import SMALL, prompt, q2
from test_step_ops import dbl, fill, flat, half_step, logits_inputs, mask_words, need_gpu, plain_logits, random_matrix, sum_tol


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


# ---------------------------------------------------------- special values
@pytest.mark.gpu
@pytest.mark.parametrize("xd", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k,group", [(20, 100, 4100, 32), (100, 70, 700, 64), (300, 40, 333, 128)])
def test_non_finite_rows_among_many(kv, m, n, k, group, xd):
    """Infinity, NaN and large values in rows of the tensor-memory form and of the copies that it reads: every column
    tile; a row's value stays in its row, and what it makes of the row is what the products say."""
    need_gpu()
    rng = np.random.default_rng(m)
    w, ref = random_matrix(kv, rng, n, k, group, True)
    x = fill(rng, (m, k), xd)
    rows = [0, m // 3, m // 2, m - 1]
    top = min(torch.finfo(x.dtype).max, 1e34)
    for row, value in zip(rows, (float("inf"), float("-inf"), float("nan"), top)):
        x[row, (7 * row + k - 1) % k] = value
    out = torch.empty(m, n, device="cuda")
    kv.w4_linear(w, x, out)
    got, want = dbl(out), (x.cpu().double() @ torch.from_numpy(ref).T).numpy()
    for row in rows[:3]:
        assert np.array_equal(np.isnan(got[row]), np.isnan(want[row]))
        f = ~np.isnan(want[row])
        assert np.array_equal(got[row][f], want[row][f])
    others = np.setdiff1d(np.arange(m), rows[:3])
    y = dbl(x)[others]
    tol = sum_tol(y, ref, group) + 2.0**-23 * np.abs(want[others])
    assert np.all(np.abs(got[others] - want[others]) <= tol)
    gate = torch.empty(m, n, device="cuda")
    kv.w4_gated(w, w, x, gate)
    assert np.all(np.isfinite(dbl(gate)[np.setdiff1d(np.arange(m), rows)]))


@pytest.mark.gpu
@pytest.mark.parametrize("m,xd,yd", [(300, "f16", "f16"), (64, "f32", "bf16"), (30, "bf16", "f32")])
def test_many_rows_in_place(kv, m, xd, yd):
    """The residual is out itself, rows apart, and out's rows start anywhere."""
    need_gpu()
    rng = np.random.default_rng(m)
    n, k = 333, 4104
    w, ref = random_matrix(kv, rng, n, k, 64, False)
    x, wide = fill(rng, (m, k), xd), fill(rng, (m, n + 9), yd)
    before = wide.clone()
    out = wide[:, 5:5 + n]
    kv.w4_linear(w, x, out, residual=out)
    res = dbl(before[:, 5:5 + n])
    want = dbl(x) @ ref.T + res
    tol = sum_tol(dbl(x), ref, 64) + 2.0**-22 * np.abs(want) + 2.0**-23 * np.abs(res)
    tol = tol + half_step(np.abs(want) + tol, yd)
    assert np.all(np.abs(dbl(out) - want) <= tol)
    assert torch.equal(wide[:, :5], before[:, :5]) and torch.equal(wide[:, 5 + n:], before[:, 5 + n:])


# ------------------------------------------------------------- offsets past 32 bits
@pytest.mark.gpu
def test_a_matrix_past_32_bits(kv):
    """600000 x 8192: the codes pass 2^31 bytes and the values 2^32 elements.  Its last rows give what they give alone."""
    need_gpu()
    n, k, group = 600000, 8192, 64
    gen = torch.Generator(device="cuda").manual_seed(4)
    w = torch.empty(n, k, dtype=torch.float16, device="cuda").normal_(std=0.02, generator=gen)
    big = kv.w4_quantize(w, group, zero_points=True)
    spans = (0, 299984, n - 48)
    small = [kv.w4_quantize(w[a:a + 48].clone(), group, zero_points=True) for a in spans]
    del w
    rng = np.random.default_rng(5)
    for m, xd in ((1, "f32"), (7, "bf16"), (48, "f16")):
        x = fill(rng, (m, k), xd)
        out = torch.empty(m, n, device="cuda")
        kv.w4_linear(big, x, out)
        for a, s in zip(spans, small):
            near_linear(kv, s, dbl(s.dequantize()), x, out[:, a:a + 48], group, "f32")
    values = big.dequantize()
    for a, s in zip(spans, small):
        assert torch.equal(values[a:a + 48], s.dequantize())


@pytest.mark.gpu
def test_rows_further_apart_than_32_bits(kv):
    """Rows of x, out, residual and logits more than 2^31 elements from the first."""
    need_gpu()
    rng = np.random.default_rng(6)
    far = 2**31 // 32 + 8
    room = torch.empty(34 * far, dtype=torch.float16, device="cuda")
    w, ref = random_matrix(kv, rng, 40, 264, 32, False)
    for m in (3, 34):  # both forms
        x = torch.as_strided(room, (m, 264), (far * (33 // (m - 1)), 1))
        x.copy_(fill(rng, (m, 264), "f16"))
        out = torch.as_strided(room, (m, 40), (far * (33 // (m - 1)), 1), 512)
        out.zero_()
        kv.w4_linear(w, x, out, residual=out)
        near_linear(kv, w, ref, x, out, 32, "f16")
    logits = torch.as_strided(room, (34, 1000), (far, 1), 2048)
    logits.copy_(fill(rng, (34, 1000), "f16"))
    near, pick, want = torch.empty(34, 1000, dtype=torch.float16, device="cuda"), *(
        torch.empty(34, dtype=torch.int32, device="cuda") for _ in range(2))
    kw = dict(hist=torch.arange(34, dtype=torch.int32, device="cuda"), hist_off=torch.arange(35, dtype=torch.int32, device="cuda"),
              presence=torch.ones(34, device="cuda"))
    kv.logits_adjust(logits.contiguous(), near, pick=want, **kw)
    kv.logits_adjust(logits, logits, pick=pick, **kw)
    assert torch.equal(logits, near) and torch.equal(pick, want)


# --------------------------------------------------------------------- logits
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,hist,bias", [(3, 50257, 900, 40), (1, 160001, 300, 20), (20, 160001, 40, 5), (2, 700, 60, 70000)])
def test_logits_into_rows_aligned_otherwise(kv, dtype, rows, vocab, hist, bias):
    """out off the 16-byte boundaries that logits stands on, and rows of odd length: bit for bit what aligned rows give."""
    need_gpu()
    rng = np.random.default_rng(vocab + rows)
    x, hs, bs, gen, rep, pres, freq, ok = logits_inputs(rng, rows, vocab, dtype, hist, bias, True)
    args = dict(mask=mask_words(ok), gen_from=torch.tensor(gen, dtype=torch.int32, device="cuda"))
    args["hist"], args["hist_off"] = flat(hs)
    args["bias_ids"], args["bias_off"] = flat(bs, lambda v: v[0])
    args["bias"], _ = flat(bs, lambda v: v[1], torch.float32)
    for name, v in (("repetition", rep), ("presence", pres), ("frequency", freq)):
        args[name] = torch.from_numpy(v).cuda()
    want, pick = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
    kv.logits_adjust(x, want, pick=pick, **args)
    for a, b in ((0, 1), (1, 0), (3, 3), (5, 2)):  # elements before the rows of logits and of out
        src = torch.full((rows, vocab + 7), 9.0, dtype=x.dtype, device="cuda")
        dst = torch.full((rows, vocab + 8), 9.0, dtype=x.dtype, device="cuda")
        src[:, a:a + vocab] = x
        got = torch.empty_like(pick)
        kv.logits_adjust(src[:, a:a + vocab], dst[:, b:b + vocab], pick=got, **args)
        assert torch.equal(dst[:, b:b + vocab], want) and torch.equal(got, pick)
        assert torch.all(dst[:, :b] == 9.0) and torch.all(dst[:, b + vocab:] == 9.0)


@pytest.mark.gpu
def test_controls_in_the_reference_order_forward():
    """qw2_set_exact: the same controls on the logits of that forward."""
    need_gpu()
    M = q2().Model(0, SMALL, max_sessions=2)
    for name, a in q2().synth_weights(SMALL, seed=22):
        M.set_tensor(name, a)
    M.set_exact(True)
    s = M.create_session()
    M.set_controls(s, repetition_penalty=1.5, presence_penalty=0.25, frequency_penalty=0.5, bias={3: 1.0, 17: -2.0})
    history = prompt(9, 4)
    logits, am = M.forward_session(s, history)
    for _ in range(6):
        y, _ = plain_logits(logits.astype(np.float64), history, 9, 1.5, 0.25, 0.5, [(3, 1.0), (17, -2.0)], None)
        assert am == int(np.argmax(y))
        history = history + [am]
        logits, am = M.forward_session(s, [am])
    M.close()


FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np, torch
from conftest import load_pkg
from test_step_ops import fill, random_matrix
kv = load_pkg()
kv.load()
rng = np.random.default_rng(3)
w, _ = random_matrix(kv, rng, 300, 1000, 32, True)
calls = []
for m, xd in ((1, "f32"), (300, "f32"), (300, "f16"), (20, "bf16")):
    x, out = fill(rng, (m, 1000), xd), torch.zeros(m, 300, device="cuda")
    calls.append((lambda x=x, out=out: kv.w4_linear(w, x, out), out))
    out = torch.zeros(m, 300, device="cuda")
    calls.append((lambda x=x, out=out: kv.w4_gated(w, w, x, out), out))
logits, out = fill(rng, (3, 5000), "f32"), torch.zeros(3, 5000, device="cuda")
calls.append((lambda: kv.logits_adjust(logits, out, presence=torch.ones(3, device="cuda")), out))
half, values = fill(rng, (64, 200), "f16"), torch.zeros(64, 200, device="cuda")
calls.append((lambda: kv.w4_quantize(half, 64).dequantize(out=values), values))
got = []
for f, out in calls:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    graph.replay()
    torch.cuda.synchronize()
    got.append((graph, out.clone()))
    out.zero_()
for (f, out), (graph, was) in zip(calls, got):
    f()
    torch.cuda.synchronize()
    assert out.abs().sum() > 0 and torch.equal(out, was)
# two graphs and an eager call at once, the default stream by its address
s = torch.cuda.Stream()
for _ in range(3):
    for (f, out), (graph, was) in zip(calls, got):
        graph.replay()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got[2][0].replay()
    got[4][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, was) for (f, out), (graph, was) in zip(calls, got))
x, out = fill(rng, (64, 1000), "f32"), [torch.zeros(64, 300, device="cuda") for _ in range(2)]
kv.w4_linear(w, x, out[0])
kv.w4_linear(w, x, out[1], stream=0)
assert torch.equal(kv.w4_quantize(half, 64, stream=0).dequantize(stream=0), values)
torch.cuda.synchronize()
assert torch.equal(*out)
print("fine")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_are_captured():
    """Every operator's first call of a process inside a capture, graphs replayed side by side, the default stream
    given by its address."""
    need_gpu()
    r = subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(os.path.abspath(__file__))], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr
