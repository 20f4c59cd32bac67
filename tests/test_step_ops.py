"""The operators of a decode step around the attention (include/step_ops.h):
products with 4-bit weights, the gated block on them, bringing a matrix to 4
bits, and penalties / biases / masks on logits with the greedy choice.

Tolerances, derived: within a group the tensor core adds at most 8 blocks of
16 products (each product exact) with at most 2^-22 of the sum of magnitudes
lost per block; groups, warps, CTAs and the parts of an fp32 x are then at
most Q + 64 fp32 additions and one multiplication each; an fp32 x loses at
most 2^-24 of itself in its third part.  So a result is off by at most
(32 + 2 Q + 64 + 2) 2^-24 of A = sum |x| |w|, then by half a step of its type.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
PLACE = (0, 4, 1, 5, 2, 6, 3, 7)


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


# ---------------------------------------------------------------- plain forms
def pack(codes, scales, zero):
    """numpy [n][k] codes, [n][Q] scales (fp16) and zero points -> the three arrays, by the layout's definition."""
    n, k = codes.shape
    q = scales.shape[1]
    t, s = -(-n // 16), -(-k // 128)
    full = np.full((t * 16, s * 128), 3, np.uint32)
    full[:n, :k] = codes
    out = np.zeros((t, s, 2, 32, 4), np.uint32)
    sc = np.full((t, q, 8, 2), np.nan, np.float16)  # padding may hold anything
    zz = np.full((t, q, 8, 2), 255, np.uint8)
    for h in range(2):
        for g in range(8):
            r = full[h * 8 + g::16].reshape(t, s, 4, 4, 8)  # tile, span, j, c, i
            for i, p in enumerate(PLACE):
                for c in range(4):
                    out[:, :, h, 4 * g + c, :] |= r[:, :, :, c, i] << np.uint32(4 * p)
            rows = scales[h * 8 + g::16]
            sc[:rows.shape[0], :, g, h] = rows
            zz[:rows.shape[0], :, g, h] = zero[h * 8 + g::16]
    return out.view(np.int32), sc, zz


def random_matrix(kv, rng, n, k, group, zeros):
    """(W4, its float64 values)."""
    q = -(-k // group)
    codes = rng.integers(0, 16, (n, k)).astype(np.uint32)
    scales = (rng.random((n, q)) * 0.02 + 0.001).astype(np.float16)
    zero = rng.integers(0, 16, (n, q)).astype(np.uint8) if zeros else np.full((n, q), 8, np.uint8)
    c, s, z = pack(codes, scales, zero)
    w = kv.W4(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), torch.from_numpy(z).cuda() if zeros else None, n, k,
              group)
    grp = np.arange(k) // group
    return w, (codes.astype(np.float64) - zero.astype(np.float64)[:, grp]) * scales.astype(np.float64)[:, grp]


def fill(rng, shape, dtype):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DT[dtype]).cuda()


def dbl(t):
    return t.detach().cpu().double().numpy()


def sum_tol(x, w, group):
    q = -(-w.shape[1] // group)
    return (98 + 2 * q) * 2.0**-24 * (np.abs(x) @ np.abs(w).T)


def half_step(y, dtype):
    fi = torch.finfo(DT[dtype])
    return np.abs(y) * fi.eps / 2 + fi.smallest_normal * fi.eps


# (m, n, k, group, zeros, x, y): one to many rows around the tile and pass edges, odd n and k, one span and less, many spans
LINEAR = [
    (1, 1, 1, 32, False, "f32", "f32"),
    (1, 16, 128, 128, False, "f16", "f32"),
    (2, 17, 129, 32, True, "f32", "f32"),
    (3, 33, 95, 64, True, "bf16", "bf16"),
    (5, 2048, 1536, 128, False, "f32", "f32"),
    (8, 100, 1000, 128, True, "f16", "f16"),
    (9, 1536, 8960, 64, False, "f16", "f32"),
    (11, 257, 8191, 32, True, "bf16", "f32"),
    (17, 300, 513, 128, False, "bf16", "bf16"),
    (22, 40, 384, 64, True, "f32", "f16"),
    (32, 515, 1536, 32, True, "f16", "f16"),
    (33, 64, 256, 128, False, "f32", "bf16"),
    (64, 130, 700, 64, True, "f16", "f32"),
    (65, 48, 2000, 128, True, "bf16", "f32"),
    (130, 1000, 260, 32, False, "f32", "f32"),
    (257, 200, 1536, 128, False, "f16", "f16"),
    (1, 20000, 640, 128, True, "f16", "f32"),
    (4, 64, 40000, 128, False, "f32", "f32"),
    (60, 32, 30000, 64, True, "bf16", "f32"),
    # few tiles: their spans over a cluster; long rows: x staged in turns
    (1, 100, 8200, 64, True, "f16", "f32"),
    (2, 17, 20000, 32, True, "bf16", "bf16"),
    (8, 2400, 12000, 64, True, "f16", "f32"),
    # many rows: short and unaligned ones, columns that fill a tile and one more, several tiles, fp32 in parts
    (100, 20, 1, 32, True, "f16", "f32"),
    (200, 64, 8, 128, False, "bf16", "f16"),
    (90, 33, 40, 32, True, "f32", "f32"),
    (128, 1153, 264, 64, False, "f16", "f32"),
    (129, 129, 4100, 128, True, "bf16", "bf16"),
    (256, 16, 127, 32, False, "f16", "f16"),
    (600, 272, 1537, 64, True, "f32", "bf16"),
    (41, 20000, 200, 128, False, "f16", "f16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "-".join(map(str, c)))
def test_linear(kv, case):
    need_gpu()
    m, n, k, group, zeros, xd, yd = case
    rng = np.random.default_rng(m * 1000003 + n * 101 + k)
    w, ref = random_matrix(kv, rng, n, k, group, zeros)
    x = fill(rng, (m, k), xd)
    bias, res = fill(rng, (n,), "f32"), fill(rng, (m, n), yd)
    y = dbl(x) @ ref.T
    for b, r in ((None, None), (bias, None), (None, res), (bias, res)):
        buf = torch.full((m * n + 64,), 77.0, dtype=DT[yd], device="cuda")
        out = buf[32:32 + m * n].view(m, n)
        kv.w4_linear(w, x, out, bias=b, residual=r)
        want = y + (dbl(b) if b is not None else 0) + (dbl(r) if r is not None else 0)
        mag = np.abs(dbl(b) if b is not None else 0) + np.abs(dbl(r) if r is not None else 0)
        tol = sum_tol(dbl(x), ref, group) + 2.0**-23 * (np.abs(y) + mag)
        tol = tol + half_step(np.abs(want) + tol, yd)
        assert np.all(np.abs(dbl(out) - want) <= tol), np.max(np.abs(dbl(out) - want) / tol)
        assert torch.all(buf[:32] == 77.0) and torch.all(buf[32 + m * n:] == 77.0)
    assert kv.step_ops_status() == kv.KV_OK


GATED = [
    (1, 1, 1, 32, False, "f32", "f32"),
    (1, 8960, 1536, 128, False, "f32", "f16"),
    (2, 31, 130, 64, True, "f16", "f32"),
    (7, 500, 999, 32, True, "bf16", "bf16"),
    (11, 64, 2048, 128, True, "f32", "f32"),
    (32, 260, 1536, 32, True, "f16", "f16"),
    (33, 48, 300, 128, False, "bf16", "f32"),
    (100, 130, 640, 64, False, "f16", "f16"),
    (300, 96, 520, 128, True, "bf16", "bf16"),
    (1, 40, 9000, 128, False, "f32", "f32"),
    (4, 2400, 12500, 128, True, "bf16", "f32"),
    (70, 65, 2000, 32, True, "f32", "f32"),
    (257, 700, 129, 64, False, "f16", "f32"),
    (86, 1, 300, 128, True, "f32", "f16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", GATED, ids=lambda c: "-".join(map(str, c)))
def test_gated(kv, case):
    need_gpu()
    m, n, k, group, zeros, xd, yd = case
    rng = np.random.default_rng(m * 1000003 + n * 101 + k + 1)
    wg, rg = random_matrix(kv, rng, n, k, group, zeros)
    wu, ru = random_matrix(kv, rng, n, k, group, zeros)
    x = fill(rng, (m, k), xd)
    out = torch.empty(m, n, dtype=DT[yd], device="cuda")
    kv.w4_gated(wg, wu, x, out)
    g, u = dbl(x) @ rg.T, dbl(x) @ ru.T
    tg, tu = sum_tol(dbl(x), rg, group), sum_tol(dbl(x), ru, group)
    with np.errstate(over="ignore"):
        s = g / (1 + np.exp(-g))
    want = s * u
    # |silu'| <= 1.1; exp, the sum, the quotient and the product: at most 8 roundings
    tol = 1.1 * tg * np.abs(u) + np.abs(s) * tu + 1.1 * tg * tu + 8 * 2.0**-24 * (np.abs(want) + np.abs(u) * tg)
    tol = tol + half_step(np.abs(want) + tol, yd)
    if yd == "f16":
        inside = np.abs(want) + tol < 65504
        assert np.all(np.isinf(dbl(out)[np.abs(want) - tol > 65520]))
    else:
        inside = np.ones_like(want, bool)
    err = np.abs(dbl(out) - want)
    assert np.all(err[inside] <= tol[inside]), np.max(err[inside] / tol[inside])


@pytest.mark.gpu
@pytest.mark.parametrize("xd,yd", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_linear_strided_rows(kv, xd, yd, offset):
    """Rows apart, off their 16-byte alignment, out and residual inside wider buffers; residual is out."""
    need_gpu()
    rng = np.random.default_rng(5 + offset)
    m, n, k = 6, 50, 200
    w, ref = random_matrix(kv, rng, n, k, 64, True)
    big = fill(rng, (m, k + 37), xd)
    x = big[:, offset:offset + k]
    wide = fill(rng, (m, n + 11), yd)
    before = wide.clone()
    out = wide[:, 3:3 + n]
    want = dbl(x) @ ref.T + dbl(before[:, 3:3 + n])
    kv.w4_linear(w, x, out, residual=out)
    tol = sum_tol(dbl(x), ref, 64) + 2.0**-22 * np.abs(want) + 2.0**-23 * np.abs(dbl(before[:, 3:3 + n]))
    tol = tol + half_step(np.abs(want) + tol, yd)
    assert np.all(np.abs(dbl(out) - want) <= tol)
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 3 + n:], before[:, 3 + n:])


@pytest.mark.gpu
@pytest.mark.parametrize("xd", ["f16", "f32"])
def test_linear_many_rows_without_scratch(kv, xd):
    """A C caller without scratch: rows that would go through it take the other form."""
    need_gpu()
    rng = np.random.default_rng(77)
    m, n, k = 100, 60, 333
    w, ref = random_matrix(kv, rng, n, k, 64, True)
    x = fill(rng, (m, k), xd)
    out = torch.empty(m, n, device="cuda")
    kv.call("w4_linear", w._at, x.data_ptr(), kv.STEP_F32 if xd == "f32" else kv.STEP_F16, m, k, None, None, 0, out.data_ptr(),
            kv.STEP_F32, n, None, torch.cuda.current_stream().cuda_stream)
    want = dbl(x) @ ref.T
    tol = sum_tol(dbl(x), ref, 64) + 2.0**-23 * np.abs(want)
    assert np.all(np.abs(dbl(out) - want) <= tol)


@pytest.mark.gpu
def test_linear_no_rows_and_non_finite(kv):
    need_gpu()
    rng = np.random.default_rng(8)
    w, ref = random_matrix(kv, rng, 40, 160, 32, False)
    kv.w4_linear(w, torch.empty(0, 160, device="cuda"), torch.empty(0, 40, device="cuda"))
    kv.w4_gated(w, w, torch.empty(0, 160, device="cuda"), torch.empty(0, 40, device="cuda"))
    for xd in DT:
        x = fill(rng, (9, 160), xd)
        x[2, 7], x[4, 100], x[5, 3] = math.inf, math.nan, min(torch.finfo(DT[xd]).max, 1e34)
        out = torch.empty(9, 40, device="cuda")
        kv.w4_linear(w, x, out)
        want = (x.cpu().double() @ torch.from_numpy(ref).T).numpy()
        got = dbl(out)
        fine = np.array([0, 1, 3, 6, 7, 8])
        assert np.all(np.isfinite(got[fine]))  # a row's infinity stays in its row
        assert np.array_equal(np.isnan(got[2]), np.isnan(want[2]))
        assert np.array_equal(got[2][~np.isnan(want[2])], want[2][~np.isnan(want[2])])
        assert np.all(np.isnan(got[4]))
        big = np.abs(want[5]) < 3e38
        assert np.allclose(got[5][big], want[5][big], rtol=1e-4)


@pytest.mark.gpu
def test_linear_repeats_on_streams_and_in_graphs(kv):
    """The same call twice gives the same bits, on another stream too, and in a captured graph."""
    need_gpu()
    rng = np.random.default_rng(9)
    w, _ = random_matrix(kv, rng, 1536, 8960, 128, False)
    x = fill(rng, (4, 8960), "f32")
    a, b, c = (torch.empty(4, 1536, device="cuda") for _ in range(3))
    kv.w4_linear(w, x, a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    kv.w4_linear(w, x, b, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    # many fp32 rows, through scratch, on both streams at once
    y = fill(rng, (64, 8960), "f32")
    one, two = torch.empty(64, 1536, device="cuda"), torch.empty(64, 1536, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        kv.w4_linear(w, y, one)
        kv.w4_linear(w, y, two, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(one, two)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.w4_linear(w, x, c)
        kv.w4_gated(w, w, x, b)
        kv.w4_linear(w, y, two)
        kv.logits_adjust(two, two, frequency=torch.ones(64, device="cuda"))
    x.mul_(2)
    y.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, 2 * a) and torch.equal(two, 2 * one)  # every step scales exactly by 2


# ------------------------------------------------------------------- quantise
def plain_quantize(w, group, zeros):
    """float64 values, from the definition."""
    n, k = w.shape
    out = np.zeros((n, k))
    for a in range(0, k, group):
        p = w[:, a:a + group]
        if zeros:
            lo, hi = np.minimum(p.min(1), 0), np.maximum(p.max(1), 0)
            s = ((hi - lo) / 15).astype(np.float16).astype(np.float64)[:, None]
            with np.errstate(all="ignore"):
                z = np.clip(np.rint(-lo[:, None] / s), 0, 15)
                q = np.clip(np.rint(p / s) + z, 0, 15) - z
        else:
            s = (np.abs(p).max(1) / 7).astype(np.float16).astype(np.float64)[:, None]
            with np.errstate(all="ignore"):
                q = np.clip(np.rint(p / s), -8, 7)
        out[:, a:a + group] = np.where(s > 0, np.where(s > 0, q, 0) * s, 0)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,group,zeros,dtype", [
    (1, 1, 32, False, "f16"), (16, 128, 128, True, "bf16"), (17, 130, 64, False, "f16"), (100, 1530, 32, True, "bf16"),
    (257, 1536, 128, False, "bf16"), (48, 513, 128, True, "f16"), (31, 96, 64, True, "f16"), (33, 1001, 32, False, "f16")])
def test_quantize(kv, n, k, group, zeros, dtype):
    need_gpu()
    rng = np.random.default_rng(n + k)
    w = fill(rng, (n, k + 5), dtype) * 0.03
    w[n // 2, :70] = 0
    w[0, -1 - 5] = 1.5  # a group with one large weight
    w[n - 1, : k // 2] = w[n - 1, : k // 2].abs()  # one-sided groups
    for off in (0, 1):
        part = w[:, off:off + k]
        m = kv.w4_quantize(part, group, zero_points=zeros)
        want = plain_quantize(dbl(part), group, zeros)
        wide = torch.full((n, k + 3), 5.0, device="cuda")
        m.dequantize(out=wide[:, 1:1 + k])
        # a code times a scale is exact in fp32; a quotient of two 11-bit values cannot be
        # nearer to a border than fp32 resolves, so the codes are those of the definition
        assert np.array_equal(dbl(wide[:, 1:1 + k]), want)
        assert torch.all(wide[:, 0] == 5.0) and torch.all(wide[:, 1 + k:] == 5.0)
        assert torch.equal(m.dequantize(), wide[:, 1:1 + k])


# --------------------------------------------------------------------- logits
def plain_logits(x, hist, gen_from, rep, pres, freq, bias, mask):
    """float64 of one row (x float64), and a bound on the fp32 steps' error."""
    x, mag = x.copy(), np.abs(x)
    v = x.shape[0]
    met = sorted({t for t in hist if 0 <= t < v})
    for t in met:
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
        mag[t] = max(mag[t], abs(x[t]))
    new = {}
    for t in hist[gen_from:]:
        if 0 <= t < v:
            new[t] = new.get(t, 0) + 1
    for t, c in new.items():
        x[t] -= freq * c + pres
        mag[t] += abs(freq * c) + abs(pres)
    last = {t: b for t, b in bias if 0 <= t < v}
    for t, b in last.items():
        x[t] += b
        mag[t] += abs(b)
    if mask is not None:
        x = np.where(mask, x, -np.inf)
    return x, 6 * 2.0**-24 * mag


LOGITS = [
    # rows, vocab, dtype, hist, bias, mask
    (1, 1, "f32", 3, 2, True),
    (1, 31, "f32", 0, 0, False),
    (3, 33, "bf16", 40, 7, True),
    (2, 1000, "f16", 500, 20, True),
    (4, 8193, "f32", 3000, 100, False),
    (5, 50257, "f32", 700, 0, True),
    (2, 151936, "f32", 512, 64, True),
    (1, 128257, "bf16", 20000, 300, True),
    (3, 200001, "f16", 10, 0, False),
    (70, 257, "f32", 33, 5, True),
    (18, 160001, "bf16", 50, 3, True),   # more tokens than a CTA notes at a time
    (1, 320000, "f32", 2000, 10, True),
    (2, 300, "f32", 7, 40000, False),    # more bias entries than 16 bits number
]


def logits_inputs(rng, rows, vocab, dtype, hist, bias, mask):
    x = (fill(rng, (rows, vocab), dtype) * 3)
    hs = [rng.integers(-2, vocab + 2, int(rng.integers(0, hist + 1))).tolist() for _ in range(rows)]
    hs = [[t if rng.random() < 0.5 else t % 7 for t in h] for h in hs]  # some ids often
    bs = [[(int(rng.integers(-1, vocab + 1)), float(np.float32(rng.standard_normal() * 3))) for _ in range(bias)] for _ in range(rows)]
    for b in bs:
        if len(b) > 2:
            b[-1] = (b[0][0], 2.5)  # the same id twice
    gen = [int(rng.integers(0, len(h) + 2)) for h in hs]
    rep, pres, freq = (rng.random(rows).astype(np.float32) + o for o in (np.float32(1), np.float32(-0.3), np.float32(0)))
    ok = rng.random((rows, vocab)) < 0.5 if mask else None
    if mask and rows > 2:
        ok[1] = False
    return x, hs, bs, gen, rep, pres, freq, ok


def mask_words(ok):
    rows, vocab = ok.shape
    bits = np.ones((rows, -(-vocab // 32) * 32), bool)  # bits behind the vocabulary may be set
    bits[:, :vocab] = ok
    w = (bits.reshape(rows, -1, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)
    return torch.from_numpy(w.view(np.int32)).cuda()


def flat(lists, of=lambda v: v, dtype=torch.int32):
    off = torch.tensor(np.cumsum([0] + [len(v) for v in lists]), dtype=torch.int32, device="cuda")
    return torch.tensor([of(v) for vs in lists for v in vs], dtype=dtype, device="cuda"), off


@pytest.mark.gpu
@pytest.mark.parametrize("case", LOGITS, ids=lambda c: "-".join(map(str, c)))
def test_logits(kv, case):
    need_gpu()
    rows, vocab, dtype, hist, bias, mask = case
    rng = np.random.default_rng(rows * 7 + vocab)
    x, hs, bs, gen, rep, pres, freq, ok = logits_inputs(rng, *case)
    args = {}
    if hist:
        args["hist"], args["hist_off"] = flat(hs)
        args["gen_from"] = torch.tensor(gen, dtype=torch.int32, device="cuda")
    if bias:
        args["bias_ids"], args["bias_off"] = flat(bs, lambda v: v[0])
        args["bias"], _ = flat(bs, lambda v: v[1], torch.float32)
    if mask:
        args["mask"] = mask_words(ok)
    for name, v in (("repetition", rep), ("presence", pres), ("frequency", freq)):
        args[name] = torch.from_numpy(v).cuda()
    out, pick = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
    kv.logits_adjust(x, out, pick=pick, **args)
    got, chosen = dbl(out), pick.cpu().tolist()
    full = torch.empty(rows, vocab, device="cuda")
    kv.logits_adjust(x.float(), full, **args)  # the fp32 values that the choice is made on
    exact32 = full.cpu().numpy()
    for r in range(rows):
        want, tol = plain_logits(dbl(x[r]), hs[r] if hist else [], gen[r], float(rep[r]), float(pres[r]), float(freq[r]),
                                 bs[r], ok[r] if mask else None)
        f = np.isfinite(want)
        assert np.array_equal(f, np.isfinite(got[r]))
        assert np.array_equal(want[~f], got[r][~f])
        t32 = tol + np.abs(want) * 2.0**-24
        assert np.all(np.abs(exact32[r][f] - want[f]) <= t32[f])
        assert np.all(np.abs(got[r][f] - want[f]) <= (t32 + half_step(np.abs(want) + t32, dtype))[f])
        best = int(np.argmax(exact32[r])) if np.any(np.isfinite(exact32[r])) else -1
        assert chosen[r] == best
    same = x.clone()
    again = torch.empty_like(pick)
    kv.logits_adjust(same, same, pick=again, **args)  # in place
    assert torch.equal(same, out) and torch.equal(again, pick)


@pytest.mark.gpu
def test_logits_special_values(kv):
    """NaN, infinities, ties and lowest values, masked and not; rows wider apart than long; nothing set."""
    need_gpu()
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    rows = [[1.0, 2.0, 2.0, nan], [nan, nan, nan, nan], [-inf, -inf, -inf, -inf], [low, low, low, low], [inf, 3.0, inf, 1.0],
            [nan, -5.0, -0.0, 0.0], [9.0, 8.0, 7.0, 6.0], [nan, inf, 1.0, 2.0]]
    buf = torch.full((8, 9), 4.0, device="cuda")
    buf[:, 2:6] = torch.tensor(rows, device="cuda")
    x, wide = buf[:, 2:6], torch.full((8, 7), 11.0, device="cuda")
    pick = torch.empty(8, dtype=torch.int32, device="cuda")
    kv.logits_adjust(x, wide[:, :4], pick=pick)
    assert pick.tolist() == [1, -1, -1, -1, 0, 2, 0, 1]
    assert torch.equal(wide[:, :4].nan_to_num(77.0), x.nan_to_num(77.0)) and torch.all(wide[:, 4:] == 11.0)
    mask = torch.tensor([[w] for w in (0b1001, 0b1111, 0b1111, 0b1111, 0b1010, 0b0011, 0b0000, 0b1100)], dtype=torch.int32, device="cuda")
    kv.logits_adjust(x, wide[:, :4], pick=pick, mask=mask)
    assert pick.tolist() == [0, -1, -1, -1, 1, 1, -1, 3]
    assert torch.all(torch.isneginf(wide[6, :4])) and torch.isneginf(wide[7, 0]) and torch.isneginf(wide[7, 1])


@pytest.mark.gpu
def test_logits_offsets_are_held_within_the_lists(kv):
    """Offsets beyond a list, negative or falling ones read nothing outside it."""
    need_gpu()
    x = torch.zeros(4, 64, device="cuda")
    hist = torch.arange(10, dtype=torch.int32, device="cuda")
    off = torch.tensor([-5, 3, 1, 9, 1 << 30], dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    kv.logits_adjust(x, out, hist=hist, hist_off=off, presence=torch.ones(4, device="cuda"))
    want = torch.zeros(4, 64)
    want[0, 0:3] = -1   # [0, 3)
    want[2, 1:9] = -1   # [1, 9)
    want[3, 9:10] = -1  # [9, 10)
    assert torch.equal(out.cpu(), want)


# --------------------------------------------------------- together, as a step
@pytest.mark.gpu
def test_step_of_operators(kv):
    """q/k/v projection, cached attention, output projection, gated block, head and choice of a two-layer step,
    in one stream, from quantised weights, against the same in 64 bits."""
    need_gpu()
    rng = np.random.default_rng(31)
    H, IS, V, B, L = 256, 512, 1000, 3, 2
    lens = [0, 20, 45]
    P = kv.Pool(0, L, 64, num_q_heads=2, num_kv_heads=1, max_seqs=4, max_seq_len=128)
    ids = []
    for n in lens:
        s = P.seq_alloc()
        P.reserve(s, n + 1)
        for layer in range(L):
            if n:
                rows = [torch.from_numpy((rng.standard_normal((n, 128)) * 0.5).astype(np.float16).view(np.int16)).cuda() for _ in range(2)]
                P.import_rows(layer, s, 0, *rows)
        P.set_cur_pos(s, n)
        ids.append(s)

    def weight(n, k):
        m = kv.w4_quantize(fill(rng, (n, k), "f16") * 0.05, 64, zero_points=True)
        return m, dbl(m.dequantize())

    hidden = fill(rng, (B, H), "f32")
    x = dbl(hidden)
    P.plan(ids)
    for layer in range(L):
        (wqkv, rqkv), (wo, ro), (wg, rg), (wu, ru), (wd, rd) = (weight(n, k) for n, k in (
            (H + 256, H), (H, H), (IS, H), (IS, H), (H, IS)))
        qkv = torch.empty(B, H + 256, device="cuda")
        kv.w4_linear(wqkv, hidden, qkv)
        q, k, v = (t.contiguous() for t in qkv.split((H, 128, 128), 1))
        attn = torch.empty(B, H, device="cuda")
        P.decode_layer(layer, q, k, v, attn)
        kv.w4_linear(wo, attn, hidden, residual=hidden)
        act, nxt = torch.empty(B, IS, device="cuda"), torch.empty(B, H, device="cuda")
        kv.w4_gated(wg, wu, hidden, act)
        kv.w4_linear(wd, act, nxt, residual=hidden)
        # the same in 64 bits around the attention's own output
        assert np.allclose(dbl(qkv), x @ rqkv.T, rtol=0, atol=1e-5 * np.abs(x @ rqkv.T).max())
        x = x + dbl(attn) @ ro.T
        g, u = x @ rg.T, x @ ru.T
        x = x + (g / (1 + np.exp(-g)) * u) @ rd.T
        assert np.allclose(dbl(nxt), x, rtol=0, atol=1e-5 * np.abs(x).max())
        hidden, x = nxt, dbl(nxt)
    P.commit()
    head, rhead = weight(V, H)
    logits, pick = torch.empty(B, V, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    kv.w4_linear(head, hidden, logits)
    hist, off = flat([[1, 2, 3], [], [7, 7]])
    raw = logits.clone()
    kv.logits_adjust(logits, logits, pick=pick, hist=hist, hist_off=off, frequency=torch.full((B,), 0.5, device="cuda"))
    y = x @ rhead.T
    assert np.allclose(dbl(raw), y, rtol=0, atol=1e-5 * np.abs(y).max())
    y = dbl(raw)
    y[0, [1, 2, 3]] -= 0.5
    y[2, 7] -= 1.0
    assert pick.tolist() == y.argmax(1).tolist()
    P.close()


# ------------------------------------------------------------------- refusals
_matrices = []


def matrix(kv, n=32, k=64, group=32, device=0, codes=0x1000, scales=0x1000, zeros=None):
    _matrices.append(kv._W4Matrix(device, n, k, group, codes, scales, zeros))
    return C.addressof(_matrices[-1])


def refused(kv, fn, *args):
    with pytest.raises(kv.KVError) as e:
        kv.call(fn, *args)
    assert e.value.status in (kv.KV_ERR_INVAL, kv.KV_ERR_RANGE)
    return str(e.value)


def test_linear_refusals(kv):
    A, B = 0x100000, 0x900000
    ok = dict(w=matrix(kv), x=A, xd=0, m=4, ldx=64, bias=None, res=None, ldr=0, out=B, od=2, ldo=32, work=None)

    def go(**kw):
        return refused(kv, "w4_linear", *{**ok, **kw}.values(), None)

    go(w=None)
    go(w=matrix(kv, n=0))
    go(w=matrix(kv, k=-1))
    assert "groups" in go(w=matrix(kv, group=48))
    go(w=matrix(kv, device=-1))
    go(w=matrix(kv, codes=None))
    go(w=matrix(kv, codes=0x1008))
    go(w=matrix(kv, scales=0x1002))
    go(w=matrix(kv, zeros=0x1001))
    go(xd=3)
    go(od=-1)
    go(m=-1)
    go(m=1 << 21)
    go(ldx=63)
    go(ldo=31)
    go(x=None)
    go(out=None)
    go(x=A + 1)
    go(out=B + 2)
    go(bias=B + 1)
    assert "overlaps x" in go(out=A + 64)
    go(res=A, ldr=31)
    assert "without being out" in go(res=B + 4, ldr=32)
    assert "without being out" in go(res=B, ldr=33)
    go(work=A + 8)
    assert "scratch overlaps" in go(xd=2, m=100, work=A + 16)
    assert "scratch overlaps" in go(xd=2, m=100, work=B - 16)
    g = dict(gate=matrix(kv), up=matrix(kv), x=A, xd=0, m=4, ldx=64, out=B, od=2, ldo=32, work=None)
    for up in (None, matrix(kv, n=33), matrix(kv, k=65), matrix(kv, group=64), matrix(kv, device=1), matrix(kv, zeros=0x1000)):
        refused(kv, "w4_gated", *{**g, "up": up}.values(), None)
    m = C.addressof(_matrices[0])
    refused(kv, "w4_quantize", m, A, 2, 64, None)
    refused(kv, "w4_quantize", m, A, 0, 63, None)
    refused(kv, "w4_quantize", m, A + 1, 0, 64, None)
    refused(kv, "w4_dequantize", m, None, 64, None)
    refused(kv, "w4_dequantize", m, A, 63, None)


def test_no_rows_need_no_device(kv):
    kv.call("w4_linear", matrix(kv), None, 0, 0, 64, None, None, 0, None, 2, 32, None, None)
    kv.call("w4_gated", matrix(kv), matrix(kv), None, 0, 0, 64, None, 2, 32, None, None)
    kv.call("logits_adjust", C.byref(kv._LogitsCall(device=0, rows=0, vocab=5, dtype=2)), None)


def test_work_bytes(kv):
    n = C.c_size_t()
    for m, k, dtype, some in ((1, 100, 2, False), (300, 100, 2, True), (300, 100, 0, True), (300, 101, 1, True), (1, 9000, 1, False)):
        kv.call("w4_work_bytes", 64, k, 64, dtype, m, 0, C.byref(n))
        assert n.value == ((3 if dtype == 2 else 1) * m * -(-k // 8) * 16 if some else 0)
    refused(kv, "w4_work_bytes", 64, 64, 64, 5, 1, 0, C.byref(n))
    refused(kv, "w4_work_bytes", 64, 64, 65, 2, 1, 0, C.byref(n))
    refused(kv, "w4_work_bytes", 64, 64, 64, 2, -1, 0, C.byref(n))
    refused(kv, "w4_work_bytes", 64, 64, 64, 2, 1, 0, None)


def test_w4_sizes(kv):
    for n, k, group in ((1, 1, 32), (16, 128, 128), (17, 129, 64), (2048, 1536, 128), (31, 97, 32)):
        s = [C.c_size_t() for _ in range(3)]
        kv.call("w4_sizes", n, k, group, *[C.byref(v) for v in s])
        t, sp, q = -(-n // 16), -(-k // 128), -(-k // group)
        assert [v.value for v in s] == [t * sp * 1024, t * q * 32, t * q * 16]
    refused(kv, "w4_sizes", 4, 4, 16, None, None, None)


def test_logits_refusals(kv):
    A, B = 0x100000, 0x900000
    ok = dict(device=0, rows=2, vocab=100, dtype=2, logits=A, ld_logits=100, out=B, ld_out=100)

    def go(**kw):
        return refused(kv, "logits_adjust", C.byref(kv._LogitsCall(**{**ok, **kw})), None)

    refused(kv, "logits_adjust", None, None)
    go(rows=-1)
    go(rows=65536)
    go(vocab=0)
    go(dtype=7)
    go(logits=None)
    go(out=None)
    go(out=B + 2)
    go(ld_logits=99)
    go(ld_out=99)
    assert "overlaps" in go(out=A + 400)
    assert "overlaps" in go(out=A, ld_out=101)
    go(hist=A)
    go(hist=A, hist_off=A, hist_n=-1)
    go(bias_ids=A, bias_off=A)
    go(bias_ids=A, bias=A)
    go(mask=A, ld_mask=3)
    go(pick=A + 2)
    go(device=-1)


@pytest.mark.gpu
def test_python_refusals(kv):
    need_gpu()
    rng = np.random.default_rng(3)
    w, _ = random_matrix(kv, rng, 32, 64, 32, False)
    x, out = torch.zeros(2, 64, device="cuda"), torch.zeros(2, 32, device="cuda")
    bad = [
        lambda: kv.w4_linear(w, x.cpu(), out),
        lambda: kv.w4_linear(w, x[:, :60], out),
        lambda: kv.w4_linear(w, x, out[:1]),
        lambda: kv.w4_linear(w, x.double(), out),
        lambda: kv.w4_linear(w, torch.zeros(64, 2, device="cuda").t(), out),
        lambda: kv.w4_linear(w, x, out, bias=torch.zeros(31, device="cuda")),
        lambda: kv.w4_linear(w, x, out, bias=torch.zeros(32, device="cuda", dtype=torch.float16)),
        lambda: kv.w4_linear(w, x, out, residual=out.half()),
        lambda: kv.w4_linear(w, x[:1].expand(2, 64), out),
        lambda: kv.w4_gated(w, w, x, x),
        lambda: kv.w4_quantize(x.float()),
        lambda: kv.w4_quantize(x.half(), group=48),
        lambda: kv.W4(w.codes[:1], w.scales, None, 32, 64, 32),
        lambda: kv.W4(w.codes, w.scales.float(), None, 32, 64, 32),
        lambda: kv.logits_adjust(x, out),
        lambda: kv.logits_adjust(x, x.clone(), pick=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: kv.logits_adjust(x, x.clone(), hist=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: kv.logits_adjust(x, x.clone(), mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
        lambda: kv.logits_adjust(x, x.clone(), repetition=torch.ones(1, device="cuda")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, kv.KVError)):
            f()
            pytest.fail(f"call {i} was accepted")
