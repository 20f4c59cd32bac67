"""The operators of a 4-bit decode step, as they are measured.

Four operators that stand around the cached attention of a decode step:

  linear    y = x W^T (+ bias) (+ residual), W in 4 bits with a scale (and a zero point) for each group of 32, 64 or 128 inputs
  gated     y = silu(x Wg^T) * (x Wu^T): both projections of a gated feed-forward block, activation and product
  logits    penalties for tokens met before, biases and a grammar mask on rows of logits, and the greedy choice of each row
  quantize  a matrix brought to 4 bits and read back as the values that its codes stand for

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's entry points.

4-bit layout.  The rows are taken 16 at a time (tiles), the inputs 128 at a time (spans).  codes is int32 [tile][span][2][32][4]:
element [t][s][h][4 g + c][j] holds row 16 t + 8 h + g and the inputs 128 s + 32 j + 8 c + i, i = 0..7, input i in the four bits
from 4 * (0, 4, 1, 5, 2, 6, 3, 7)[i].  scales is fp16 [tile][group][8][2] and zeros (where there are zero points) uint8 of the same
shape: element [t][q][g][h] is row 16 t + 8 h + g, inputs of group q.  A weight is (code - zero) * scale; zero is 8 where there are none.
What the padding of the last tile and span holds does not matter.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PLACE = (0, 4, 1, 5, 2, 6, 3, 7)  # where the inputs 0..7 of a 32-bit word stand in it, in units of four bits


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One token through the stacked q/k/v projection of a 1536-wide layer: fp32 activations as the layer loop keeps them, with
        # its bias.  The smallest call of a step; latency counts.
        dict(name="qkv one token", op="linear", m=1, n=2048, k=1536, group=128, zeros=False, x="f32", y="f32", bias=True, residual=False),
        # One token's logits over the 151936-word vocabulary: the largest matrix of a step, bound by its bytes.
        dict(name="head one token", op="linear", m=1, n=151936, k=1536, group=128, zeros=False, x="f16", y="f32", bias=False, residual=False),
        # Eleven sessions through a down projection of odd sizes with zero points, added to the residual stream.
        dict(name="down odd", op="linear", m=11, n=1531, k=8900, group=64, zeros=True, x="bf16", y="bf16", bias=False, residual=True),
        # A prompt chunk of 256 tokens through the down projection.
        dict(name="down prompt", op="linear", m=256, n=1536, k=8960, group=128, zeros=False, x="f16", y="f32", bias=False, residual=True),
        # The gated block of one token.
        dict(name="gated one token", op="gated", m=1, n=8960, k=1536, group=128, zeros=False, x="f32", y="f16"),
        # The gated block of 32 sessions decoding together, small groups.
        dict(name="gated 32 sessions", op="gated", m=32, n=8960, k=1536, group=32, zeros=True, x="f16", y="f16"),
        # The gated block of a 512-token prompt.
        dict(name="gated prompt", op="gated", m=512, n=8960, k=1536, group=128, zeros=False, x="bf16", y="bf16"),
        # One session chooses its next token: penalties over a full 512-token history.
        dict(name="choice one row", op="logits", rows=1, vocab=151936, dtype="f32", hist=512, bias=0, mask=False),
        # 32 sessions with biases and a grammar mask each; one mask leaves its row empty.
        dict(name="choice 32 rows", op="logits", rows=32, vocab=151936, dtype="f32", hist=512, bias=64, mask=True),
        # 61 sessions with long histories (to 32768 tokens), an odd vocabulary, 16-bit logits.
        dict(name="choice long", op="logits", rows=61, vocab=128257, dtype="bf16", hist=32768, bias=300, mask=True),
        # A down projection brought to 4 bits at load time.
        dict(name="quantize down", op="quantize", n=1536, k=8960, group=128, zeros=False, dtype="f16"),
        # Gate and up rows of odd sizes, small groups with zero points, from bf16.
        dict(name="quantize odd", op="quantize", n=17919, k=1530, group=32, zeros=True, dtype="bf16"),
    ]


MOST_FLOPS, MOST_BYTES = 28e9, 180e6


def _log(rng, a, b):
    """A whole number of [a, b], its logarithm spread evenly."""
    return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def _size(rng, a, b):
    """The same, brought to a multiple of 64 every other time: matrices are round more often than not."""
    n = _log(rng, a, b)
    return n if rng.random() < 0.5 else min(b, -(-n // 64) * 64)


def draw(rng):
    op = rng.choice(("linear", "linear", "gated", "gated", "logits", "logits", "quantize"))
    group, zeros = rng.choice((32, 64, 128, 128)), rng.random() < 0.5
    x, y = rng.choice((("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f16")))
    if op == "linear":
        c = dict(op=op, m=_log(rng, 1, 512), n=_size(rng, 64, 40000), k=_size(rng, 64, 9000), group=group, zeros=zeros, x=x, y=y,
                 bias=rng.random() < 0.4, residual=rng.random() < 0.4)
    elif op == "gated":
        c = dict(op=op, m=_log(rng, 1, 512), n=_size(rng, 64, 12000), k=_size(rng, 64, 4000), group=group, zeros=zeros, x=x, y=y)
    elif op == "logits":
        c = dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 1000, 160000), dtype=rng.choice(("f32", "f32", "f16", "bf16")),
                 hist=_log(rng, 1, 32768), bias=rng.choice((0, 0, 5, 64, 300)), mask=rng.random() < 0.6)
    else:
        c = dict(op=op, n=_size(rng, 64, 18000), k=_size(rng, 64, 9000), group=group, zeros=zeros, dtype=rng.choice(("f16", "bf16")))
    while work(c)["flops"] > MOST_FLOPS or work(c)["bytes"] > MOST_BYTES:
        big = max((v, q) for q, v in c.items() if q in ("m", "n", "k", "rows", "vocab"))[1]
        c[big] = max(1, c[big] * 2 // 3)
    return c


def work(case):
    c = case
    esize = lambda t: 4 if t == "f32" else 2  # noqa: E731
    if c["op"] in ("linear", "gated"):
        mats = 2 if c["op"] == "gated" else 1
        groups = -(-c["k"] // c["group"])
        b = mats * c["n"] * (c["k"] / 2 + groups * (3 if c["zeros"] else 2))
        b += c["m"] * (c["k"] * esize(c["x"]) + c["n"] * esize(c["y"]))
        if c.get("bias"):
            b += 4 * c["n"]
        if c.get("residual"):
            b += c["m"] * c["n"] * esize(c["y"])
        return {"bytes": b, "flops": 2.0 * mats * c["m"] * c["n"] * c["k"]}
    if c["op"] == "logits":
        cells = c["rows"] * c["vocab"]
        # the histories' lengths are spread over [hist / 2, hist]
        b = 2 * cells * esize(c["dtype"]) + (cells / 8 if c["mask"] else 0) + c["rows"] * (3 * c["hist"] + 8 * c["bias"] + 28)
        return {"bytes": b, "flops": 8.0 * cells}
    cells = c["n"] * c["k"]
    groups = c["n"] * -(-c["k"] // c["group"])
    # the matrix in, codes and scales out and in again, the values out
    return {"bytes": cells * (2 + 0.5 + 0.5 + 4) + 2 * groups * (3 if c["zeros"] else 2), "flops": 6.0 * cells}


# ------------------------------------------------------------------ the inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _ints(gen, low, high, *shape):
    return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int32)


def _matrix(gen, n, k, group, zeros):
    """Codes as rounded normal values have them, scales as a trained layer's: [n][k] codes, [n][groups] scales and zero points."""
    groups = -(-k // group)
    zero = _ints(gen, 6, 10, n, groups) if zeros else torch.full((n, groups), 8, device="cuda", dtype=torch.int32)
    codes = _randn(gen, n, k).mul_(2.5).round_().to(torch.int32).add_(8).clamp_(0, 15)
    scales = (torch.rand(n, groups, generator=gen, device="cuda") * 0.008 + 0.004).half()
    return codes, scales, zero


def _tiles(a, fill=0):
    """[n][q] -> [tile][q][8][2], the layout of scales and zero points."""
    n, q = a.shape
    a = torch.nn.functional.pad(a, (0, 0, 0, -n % 16), value=fill)
    return a.view(-1, 2, 8, q).permute(0, 3, 2, 1).contiguous()


def _pack(codes):
    """[n][k] codes -> int32 [tile][span][2][32][4]."""
    n, k = codes.shape
    a = torch.nn.functional.pad(codes, (0, -k % 128, 0, -n % 16), value=8)
    a = a.view(a.shape[0] // 16, 2, 8, a.shape[1] // 128, 4, 4, 8)  # tile, h, g, span, j, c, i
    word = torch.zeros(a.shape[:-1], dtype=torch.int32, device=a.device)
    for i, p in enumerate(PLACE):
        word |= a[..., i] << (4 * p)
    return word.permute(0, 3, 1, 2, 5, 4).reshape(a.shape[0], a.shape[3], 2, 32, 4).contiguous()


def _held(c, matrix):
    """What a program keeps of a 4-bit matrix."""
    codes, scales, zero = matrix
    return dict(codes=_pack(codes), scales=_tiles(scales), zeros=_tiles(zero.to(torch.uint8), 8) if c["zeros"] else None,
                n=c["n"], k=c["k"], group=c["group"])


def _matmul_inputs(c, seed):
    gen = _generator(seed)
    x = _randn(gen, c["m"], c["k"]).to(DTYPES[c["x"]])
    mats = [_matrix(gen, c["n"], c["k"], c["group"], c["zeros"]) for _ in range(2 if c["op"] == "gated" else 1)]
    bias = _randn(gen, c["n"]) if c.get("bias") else None
    residual = _randn(gen, c["m"], c["n"]).to(DTYPES[c["y"]]) if c.get("residual") else None
    return x, mats, bias, residual


def _logits_inputs(c, seed):
    gen = _generator(seed)
    r, v = c["rows"], c["vocab"]
    s = dict(logits=(_randn(gen, r, v) * 3).to(DTYPES[c["dtype"]]))
    # histories of [hist / 2, hist] ids, common words far more often than rare ones; -1 is padding, and counts for nothing
    lens = _ints(gen, max(1, c["hist"] // 2), c["hist"] + 1, r)
    s["hist_off"] = torch.nn.functional.pad(lens.cumsum(0, dtype=torch.int32), (1, 0)).to(torch.int32)
    total = r * c["hist"]  # room; the last offset says how much of it is used
    u = torch.rand(total, generator=gen, device="cuda")
    s["hist"] = (torch.exp(u * math.log(v)) - 1).to(torch.int32).clamp_(-1, v - 1)
    s["hist"][torch.rand(total, generator=gen, device="cuda") < 0.01] = -1
    s["gen_from"] = (lens * torch.rand(r, generator=gen, device="cuda")).to(torch.int32)
    s["repetition"] = 1 + 0.3 * torch.rand(r, generator=gen, device="cuda")
    s["presence"] = torch.rand(r, generator=gen, device="cuda") - 0.2
    s["frequency"] = 0.2 * torch.rand(r, generator=gen, device="cuda")
    s["bias_ids"] = s["bias"] = s["bias_off"] = s["mask"] = None
    if c["bias"]:
        s["bias_ids"] = _ints(gen, 0, v, r * c["bias"])  # an id may come twice: its last value counts
        s["bias"] = _randn(gen, r * c["bias"]) * 4
        s["bias_off"] = torch.arange(r + 1, device="cuda", dtype=torch.int32) * c["bias"]
    if c["mask"]:
        words = -(-v // 32)
        s["mask"] = _ints(gen, -(2**31), 2**31 - 1, r, words) & _ints(gen, -(2**31), 2**31 - 1, r, words)
        if r > 8:
            s["mask"][5] = 0  # a grammar that has ended
    return s


def _quantize_inputs(c, seed):
    gen = _generator(seed)
    w = _randn(gen, c["n"], c["k"]).mul_(0.02).to(DTYPES[c["dtype"]])
    w[c["n"] // 2, : min(c["k"], 200)] = 0  # a group of zeros
    return w


def prepare(case, seed):
    c = case
    if c["op"] in ("linear", "gated"):
        x, mats, bias, residual = _matmul_inputs(c, seed)
        state = dict(x=x, w=[_held(c, m) for m in mats], bias=bias, residual=residual)
        state["out"] = torch.empty(c["m"], c["n"], dtype=DTYPES[c["y"]], device="cuda")
    elif c["op"] == "logits":
        state = _logits_inputs(c, seed)
        state["out"] = torch.empty_like(state["logits"])
        state["pick"] = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
    else:
        state = dict(w=_quantize_inputs(c, seed))
    state["case"] = dict(c)
    return state


# ------------------------------------------------------------------ the plain forms
def _values(w):
    """A held 4-bit matrix as fp32 [n][k]: a code of 4 bits times a scale of 11 is exact."""
    t, s = w["codes"].shape[:2]
    shifts = torch.tensor([4 * p for p in PLACE], dtype=torch.int32, device=w["codes"].device)
    a = ((w["codes"].unsqueeze(-1) >> shifts) & 15).view(t, s, 2, 8, 4, 4, 8)  # tile, span, h, g, c, j, i
    codes = a.permute(0, 2, 3, 1, 5, 4, 6).reshape(16 * t, 128 * s)[: w["n"], : w["k"]].float()

    def rows(b):
        return b.permute(0, 3, 2, 1).reshape(16 * t, -1)[: w["n"]].float().repeat_interleave(w["group"], dim=1)[:, : w["k"]]

    return (codes - (rows(w["zeros"]) if w["zeros"] is not None else 8.0)) * rows(w["scales"])


def _plain_linear(s):
    y = s["x"].float() @ _values(s["w"][0]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out"].dtype)


def _plain_gated(s):
    x = s["x"].float()
    gate, up = x @ _values(s["w"][0]).t(), x @ _values(s["w"][1]).t()
    return (gate / (1 + torch.exp(-gate)) * up).to(s["out"].dtype)


def _cells(ids, off, rows, vocab):
    """For flat lists of ids, a row's from off[row] on: which entries count, their rows, and their places in [rows][vocab]."""
    at = torch.arange(ids.numel(), device=ids.device)
    row = torch.bucketize(at, off[1:].long(), right=True)
    fine = (row < rows) & (ids >= 0) & (ids < vocab)
    row = row.clamp(max=rows - 1)
    return fine, at, row, row * vocab + ids.long().clamp(0, vocab - 1)


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    fine, at, row, cell = _cells(s["hist"], s["hist_off"], rows, vocab)
    seen = torch.zeros(rows * vocab, device=x.device).index_add_(0, cell, fine.float()).view(rows, vocab) > 0
    new = fine & (at - s["hist_off"].long()[row] >= s["gen_from"].long()[row])
    count = torch.zeros(rows * vocab, device=x.device).index_add_(0, cell, new.float()).view(rows, vocab)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        fine, at, row, cell = _cells(s["bias_ids"], s["bias_off"], rows, vocab)
        last = torch.full((rows * vocab,), -1, device=x.device).scatter_reduce_(0, cell, torch.where(fine, at, -1), "amax")
        last = last.view(rows, vocab)
        x = x + torch.where(last >= 0, s["bias"][last.clamp(min=0)], 0.0)
    if s["mask"] is not None:
        bits = (s["mask"].unsqueeze(-1) >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.view(rows, -1)[:, :vocab] > 0, x, -math.inf)
    # the greedy choice: the lowest index of the largest value, -1 where no value is above the lowest finite one
    top = torch.where(x > torch.finfo(torch.float32).min, x, -math.inf).amax(1, keepdim=True)
    index = torch.arange(vocab, device=x.device, dtype=torch.int32)
    pick = torch.where((x == top) & (top > -math.inf), index, vocab).amin(1)
    return {"logits": x.to(s["out"].dtype), "pick": torch.where(pick < vocab, pick, -1).to(torch.int32)}


def _plain_quantize(s):
    c, w = s["case"], s["w"].float()
    n, k = w.shape
    a = torch.nn.functional.pad(w, (0, -k % c["group"])).view(n, -1, c["group"])
    if c["zeros"]:
        low, high = a.amin(2, keepdim=True).clamp(max=0), a.amax(2, keepdim=True).clamp(min=0)
        scale = ((high - low) / 15).half().float()
        some = scale > 0
        zero = torch.where(some, torch.round(-low / torch.where(some, scale, 1.0)).clamp(0, 15), 8.0)
    else:
        scale = (a.abs().amax(2, keepdim=True) / 7).half().float()
        some = scale > 0
        zero = torch.full_like(scale, 8.0)
    code = torch.where(some, torch.round(a / torch.where(some, scale, 1.0)) + zero, zero).clamp(0, 15)
    return ((code - zero) * scale).view(n, -1)[:, :k]


# ------------------------------------------------------------------ the framework's calls
_framework = []


def _kv():
    """The framework's package (its folder's name is no Python name)."""
    if not _framework:
        import importlib.util
        import os
        import sys

        name, folder = "rk3588_npu_b200", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rk3588-npu_b200")
        if name not in sys.modules:
            spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _framework.append(sys.modules[name])
    return _framework[0]


def _w4(state, i):
    """The framework's handle of matrix i: made at its first use and kept, as a program that holds the matrix keeps it."""
    handles = state.setdefault("handles", {})
    if i not in handles:
        w = state["w"][i]
        handles[i] = _kv().W4(w["codes"], w["scales"], w["zeros"], w["n"], w["k"], w["group"])
    return handles[i]


def _own_linear(s):
    _kv().w4_linear(_w4(s, 0), s["x"], s["out"], bias=s["bias"], residual=s["residual"])
    return s["out"]


def _own_gated(s):
    _kv().w4_gated(_w4(s, 0), _w4(s, 1), s["x"], s["out"])
    return s["out"]


def _own_logits(s):
    _kv().logits_adjust(s["logits"], s["out"], pick=s["pick"], hist=s["hist"], hist_off=s["hist_off"], gen_from=s["gen_from"],
                        repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
                        bias=s["bias"], bias_off=s["bias_off"], mask=s["mask"])
    return {"logits": s["out"], "pick": s["pick"]}


def _own_quantize(s):
    c = s["case"]
    return _kv().w4_quantize(s["w"], group=c["group"], zero_points=c["zeros"]).dequantize()


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "gated": _own_gated, "logits": _own_logits, "quantize": _own_quantize}[op](state)
    return {"linear": _plain_linear, "gated": _plain_gated, "logits": _plain_logits, "quantize": _plain_quantize}[op](state)


# ------------------------------------------------------------------ the definitions, in 64 bits
def _exact_weights(c, matrix):
    codes, scales, zero = matrix
    group_of = torch.arange(c["k"], device=codes.device) // c["group"]
    return (codes.double() - zero.double()[:, group_of]) * scales.double()[:, group_of]


def _exact_logits(c, s):
    x = s["logits"].double()
    off, ids = s["hist_off"].cpu().tolist(), s["hist"].long()
    bits = torch.arange(c["vocab"], device=x.device)
    for r in range(c["rows"]):
        mine = ids[off[r]:off[r + 1]]
        new = mine[int(s["gen_from"][r]):]
        mine, new = mine[mine >= 0], new[new >= 0]
        met = mine.unique()
        rep = s["repetition"][r].double()
        x[r, met] = torch.where(x[r, met] > 0, x[r, met] / rep, x[r, met] * rep)
        word, times = new.unique(return_counts=True)
        x[r, word] -= s["frequency"][r].double() * times + s["presence"][r].double()
        if s["bias"] is not None:
            a, b = r * c["bias"], (r + 1) * c["bias"]
            last = dict(zip(s["bias_ids"][a:b].tolist(), s["bias"][a:b].tolist()))
            x[r, list(last)] += torch.tensor(list(last.values()), dtype=torch.float64, device=x.device)
        if s["mask"] is not None:
            x[r, (s["mask"][r].long()[bits // 32] >> (bits % 32)) & 1 == 0] = -math.inf
    return {"logits": x, "pick": None}


def _exact_quantize(c, w):
    n, k = w.shape
    out = torch.empty(n, k, dtype=torch.float64, device=w.device)
    for a in range(0, k, c["group"]):
        part = w[:, a:a + c["group"]].double()
        if c["zeros"]:
            low, high = part.min(1).values.clamp(max=0), part.max(1).values.clamp(min=0)
            scale = ((high - low) / 15).to(torch.float16).double()
            zero = (-low / scale).round().clamp(0, 15)
            code = ((part / scale[:, None]).round() + zero[:, None]).clamp(0, 15) - zero[:, None]
        else:
            scale = (part.abs().max(1).values / 7).to(torch.float16).double()
            code = (part / scale[:, None]).round().clamp(-8, 7)
        out[:, a:a + c["group"]] = torch.where(scale[:, None] > 0, code * scale[:, None], 0.0)
    return out


def exact(case, seed):
    c = case
    if c["op"] == "logits":
        return _exact_logits(c, _logits_inputs(c, seed))
    if c["op"] == "quantize":
        return _exact_quantize(c, _quantize_inputs(c, seed))
    x, mats, bias, residual = _matmul_inputs(c, seed)
    y = [torch.einsum("mk,nk->mn", x.double(), _exact_weights(c, m)) for m in mats]
    if c["op"] == "gated":
        return y[0] * torch.sigmoid(y[0]) * y[1]
    y = y[0]
    if bias is not None:
        y = y + bias.double()
    if residual is not None:
        y = y + residual.double()
    return y
