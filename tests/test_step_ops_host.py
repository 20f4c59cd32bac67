"""The Python side of the step operators and of the model's controls, without
a GPU: what crosses the C boundary and when.  The C library's calls are stood in for."""
from __future__ import annotations

import ctypes as C
import os
import re

import numpy as np
import pytest

from conftest import PKG_DIR
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


# ------------------------------------------------------------- memory of calls on a stream
class Tensor:
    """What the wrappers ask of a contiguous 2-D device tensor; `home`: the stream it was allocated for."""

    def __init__(self, shape, dtype, home=None):
        import torch
        self.shape, self.dtype, self.home = tuple(shape), dtype, home
        self.device, self.used = torch.device("cuda", 0), set()
        self.nbytes = int(np.prod(self.shape)) * dtype.itemsize

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 0x100000

    def record_stream(self, s):
        self.used.add(s.cuda_stream)


class Stream:
    def __init__(self, address):
        self.cuda_stream = address


HERE, SIDE = 0xC0, 0x51DE  # the current stream, another one


@pytest.fixture
def streams(kv, monkeypatch):
    """torch's allocations and the library's calls, recorded: {"made": tensors, "calls": (name, arguments)}."""
    import torch
    log, now = dict(made=[], calls=[]), [HERE]

    class On:
        def __init__(self, s):
            self.s = s

        def __enter__(self):
            self.before, now[0] = now[0], self.s.cuda_stream

        def __exit__(self, *a):
            now[0] = self.before

    def empty(*shape, dtype=None, device=None):
        shape = shape[0] if isinstance(shape[0], tuple) else shape
        log["made"].append(Tensor(shape, dtype, now[0]))
        return log["made"][-1]

    class Lib:
        def __getattr__(self, name):
            real = getattr(lib, name)
            if name in ("w4_linear", "w4_gated", "w4_quantize", "w4_dequantize", "kvp_gather", "kvp_gather_i8"):
                return lambda *a: log["calls"].append((name, a)) or 0
            return real

    lib = kv.load()
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "stream", On)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream(now[0]))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda a, device=None: Stream(a))
    monkeypatch.setattr(kv, "_raw_stream", lambda d: now[0])
    monkeypatch.setattr(kv, "_lib", Lib())
    return log


def w4_of(kv, n, k, group):
    import torch
    m = kv.W4.__new__(kv.W4)
    m._hold(Tensor((1,), torch.int32), Tensor((1,), torch.float16), None, n, k, group, 0)
    return m


@pytest.mark.parametrize("stream", [None, Stream(SIDE), SIDE], ids=["current", "object", "address"])
def test_memory_of_a_call_belongs_to_its_stream(kv, streams, stream):
    """Scratch, quantised arrays and values read back are allocated for the stream that writes them: a block of the
    current stream's may still be read or written by that stream's pending work, which another stream does not wait for."""
    import torch
    w, at = w4_of(kv, 64, 512, 64), HERE if stream is None else SIDE
    x, out = Tensor((64, 512), torch.float32), Tensor((64, 64), torch.float32)
    kv.w4_linear(w, x, out, stream=stream)
    kv.w4_gated(w, w, x, out, stream=stream)
    assert [t.home for t in streams["made"]] == [at, at]  # scratch of both
    m = kv.w4_quantize(Tensor((64, 512), torch.float16), 64, zero_points=True, stream=stream)
    y = w.dequantize(stream=stream)
    assert all(t.home == at for t in (m.codes, m.scales, m.zeros, y))
    # what is handed to the caller may be used on the current stream too, and freed there
    assert all(t.home == HERE or HERE in t.used for t in (m.codes, m.scales, m.zeros, y))
    assert [name for name, _ in streams["calls"]] == ["w4_linear", "w4_gated", "w4_quantize", "w4_dequantize"]
    assert all(a[-1] == at for _, a in streams["calls"])


@pytest.mark.parametrize("stream", [None, Stream(SIDE), SIDE], ids=["current", "object", "address"])
def test_gathered_rows_belong_to_the_calls_stream(kv, streams, stream):
    at = HERE if stream is None else SIDE
    P = kv.Pool.__new__(kv.Pool)
    P.h, P.device, P.kv_dim, P.cur_pos = None, 0, 256, lambda seq: 40
    rows = [*P.gather(0, 0, stream=stream), *P.gather_i8(0, 0, stream=stream)]
    P.h = None
    assert all(t.home == at and (at == HERE or HERE in t.used) for t in rows)
    assert [(name, a[-1]) for name, a in streams["calls"]] == [("kvp_gather", at), ("kvp_gather_i8", at)]


# (n, k, group): few tiles of long rows, where few operand rows take the tcgen05 form; short rows; many tiles
SCRATCH = [(1536, 8960, 128), (1536, 8960, 32), (100, 4000, 64), (100, 4096, 32), (2048, 1536, 128), (8960, 1536, 32),
           (40000, 1536, 128), (40000, 5000, 64), (33, 257, 64)]


@pytest.mark.parametrize("n,k,group", SCRATCH)
@pytest.mark.parametrize("xd", ["f32", "f16"])
def test_scratch_is_what_the_call_asks_for(kv, streams, n, k, group, xd):
    """w4_linear and w4_gated hand over scratch where w4_work_bytes says that rows of x go through it, of that size at
    least, and none where it says 0: 1 to 48 rows, and many; 16-bit rows that TMA can address never need any."""
    import torch
    w, size = w4_of(kv, n, k, group), C.c_size_t()
    dtype, code = (torch.float32, kv.STEP_F32) if xd == "f32" else (torch.float16, kv.STEP_F16)
    some = 0
    for m in (*range(1, 49), 100, 1000):
        for gated in (0, 1):
            kv.call("w4_work_bytes", n, k, group, code, m, gated, C.byref(size))
            x, out = Tensor((m, k), dtype), Tensor((m, n), torch.float32)
            for misaligned in (0, 2):
                if misaligned and xd == "f32":
                    continue
                x.data_ptr = lambda: 0x100000 + misaligned
                want = 0 if xd == "f16" and k % 8 == 0 and not misaligned else size.value
                streams["made"].clear()
                if gated:
                    kv.w4_gated(w, w, x, out)
                else:
                    kv.w4_linear(w, x, out)
                work = streams["calls"][-1][1][-2]
                made = [t.nbytes for t in streams["made"]]
                assert (work is not None) == (want > 0) == (len(made) == 1), (m, gated)
                assert sum(made) >= want, (m, gated)
                some += want > 0
    assert some


def test_register_splits_are_changed_by_whole_warpgroups():
    """setmaxnreg in w4_tc_kernel: one change per warpgroup and split, on conditions that do not part its four warps
    (warp 7 issues, 4 to 6 copy: one warpgroup), and no more registers asked for than the launch brings."""
    with open(os.path.join(PKG_DIR, "csrc", "w4_tc_kernel.cu")) as f:
        src = f.read()
    kernel = src[src.index("    w4_tc_kernel("):src.index("// x as TMA sees it")]
    changes = [(m.group(1), m.start()) for m in re.finditer(r"regs_(?:up|down)<([^>]*)>\(\)", kernel)]
    assert [c for c, _ in changes] == ["kRegs[0]", "kRegs[1]", "kRegs[2]", "kLaunchRegs", "kLaunchRegs"]
    # the roles of warps 4 to 7 part inside their warpgroup's branch, after its change
    branch = [kernel.index("if (warp < 4) {"), kernel.index("} else if (warp < 8) {"), kernel.index("} else if (warp == kMmaWarp) {")]
    assert branch[0] < changes[0][1] < branch[1] < changes[1][1] < branch[2] < changes[2][1]
    threads = int(re.search(r"kThreads = 16 \* (\d+)", src).group(1)) * 16
    a, b, c = (int(v) for v in re.search(r"kRegs\[3\] = \{(\d+), (\d+), (\d+)\}", src).groups())
    assert threads == 512 and 128 * (a + b + 2 * c) <= 65536 // threads * threads


def brute(a, rows_a, width_a, b, rows_b, width_b, pitch):
    one = {a + i * pitch + k for i in range(rows_a) for k in range(width_a)}
    return any(b + j * pitch + k in one for j in range(rows_b) for k in range(width_b))


def test_columns_of_one_buffer_do_not_overlap(kv):
    """x, out and residual, logits and out with the same distance between rows: refused where they share a byte, and
    only there (what is accepted gets as far as the device, which is not there)."""
    rng = np.random.default_rng(0)
    A = 0x100000
    codes = kv._W4Matrix(999, 3, 4, 32, 0x900000, 0x900000, None)
    seen = set()

    def outcome(fn, *args):
        with pytest.raises(kv.KVError) as e:
            kv.call(fn, *args, None)
        assert "overlap" in str(e.value) or "no CUDA device 999" in str(e.value), str(e.value)
        return "overlap" in str(e.value)

    for _ in range(3000):
        m, ld = int(rng.integers(1, 5)), int(rng.integers(4, 14))  # rows of 2-byte elements: 4 of x, 3 of out
        at, res = A + 2 * int(rng.integers(-40, 41)), A + 2 * int(rng.integers(-40, 41))
        # x of another pitch far away, so that only residual and out may meet
        got = (outcome("w4_linear", C.addressof(codes), A, 0, m, ld, None, None, 0, at, 0, ld, None),
               outcome("w4_linear", C.addressof(codes), 0x500000, 0, m, 4, None, res, ld, at, 0, ld, None),
               outcome("logits_adjust", C.byref(kv._LogitsCall(device=999, rows=m, vocab=3, dtype=0, logits=A, ld_logits=ld,
                                                               out=at, ld_out=ld))))
        want = (brute(A, m, 8, at, m, 6, 2 * ld), res != at and brute(res, m, 6, at, m, 6, 2 * ld),
                A != at and brute(A, m, 6, at, m, 6, 2 * ld))
        assert got == want, (m, ld, at - A, res - A)
        seen.update(enumerate(got))
    assert len(seen) == 6


@pytest.mark.parametrize("stream", [Stream(HERE), HERE], ids=["object", "address"])
def test_the_current_stream_by_name_is_the_current_stream(kv, streams, monkeypatch, stream):
    import torch

    def never(s):
        raise AssertionError("a change of stream for the current one")

    monkeypatch.setattr(torch.cuda, "stream", never)
    w = w4_of(kv, 64, 512, 64)
    kv.w4_linear(w, Tensor((64, 512), torch.float32), Tensor((64, 64), torch.float32), stream=stream)
    assert [t.home for t in streams["made"]] == [HERE]
