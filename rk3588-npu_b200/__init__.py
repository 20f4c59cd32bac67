"""Python host binding of the B200 decode hot path (ctypes over include/kvattn.h).

The product is the C ABI in ``lib/libkvattn.so`` (CUDA kernels for sm_100a +
C++ host runtime).  This module only marshals arguments: device tensors are
torch tensors (used for device memory and streams), everything else is plain
Python.  There is no fallback: if the library is missing, ``load()`` raises.

Reference interfaces mirrored (Bobchasm/rk3588-npu):
  KVCache        worker/include/model/kv_cache.h:19-41  -> Pool + sequences
  op_rope + append loop + op_attention
                 worker/src/model/qwen2_model.cpp:180-206 -> Pool.plan / decode_layer / commit
  (no counterpart) placement of requests onto GPUs      -> Scheduler
"""
from __future__ import annotations

import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libkvattn.so")

KV_OK, KV_ERR_INVAL, KV_ERR_OOM, KV_ERR_BADSEQ, KV_ERR_CUDA, KV_ERR_RANGE, KV_ERR_STATE, \
    KV_ERR_TIMEOUT = range(8)
KV_F16, KV_BF16, KV_I8 = 0, 1, 2
KVP_HOST_ONLY = -1
KVP_MERGE_GRID, KVP_MERGE_CLUSTER = 0, 1
HEAD_DIM = 128
BLOCK_TOKENS = 16
KVX_HANDLE_BYTES = 64
KVN_UNIQUE_ID_BYTES = 128

_vp = C.c_void_p
_ip = C.POINTER(C.c_int)

# name -> argtypes (all return int status unless listed in _RESTYPE)
_SIGS = {
    "kv_last_error": [],
    "kv_status_str": [C.c_int],
    "kv_version": [],
    "kv_kernel_count": [C.POINTER(C.c_longlong)],
    "kvp_create": [C.c_int] * 10 + [C.c_float, C.POINTER(_vp)],
    "kvp_destroy": [_vp],
    "kvp_reset": [_vp, _vp],
    "kvp_free_blocks": [_vp, _ip],
    "kvp_num_blocks": [_vp, _ip],
    "kvp_storage": [_vp, C.POINTER(_vp), C.POINTER(_vp), C.POINTER(C.c_size_t)],
    "kvp_seq_alloc": [_vp, _ip],
    "kvp_seq_free": [_vp, C.c_int],
    "kvp_seq_reserve": [_vp, C.c_int, C.c_int],
    "kvp_seq_set_blocks": [_vp, C.c_int, _ip, C.c_int],
    "kvp_seq_len": [_vp, C.c_int, _ip],
    "kvp_seq_set_len": [_vp, C.c_int, C.c_int],
    "kvp_seq_blocks": [_vp, C.c_int, _ip, C.c_int, _ip],
    "kvp_import": [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp],
    "kvp_gather": [_vp, C.c_int, C.c_int, _vp, _vp, _vp],
    "kvp_import_i8": [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp, _vp, _vp],
    "kvp_gather_i8": [_vp, C.c_int, C.c_int, _vp, _vp, _vp, _vp, _vp],
    "kv_append_chunk": [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp],
    "attn_prefill": [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp],
    "attn_prefill_mma": [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp],
    "kv_append_chunk_batch": [_vp, C.c_int, C.c_int, _vp, _vp, _vp, _vp, _vp, _vp],
    "attn_prefill_batch": [_vp, C.c_int, C.c_int, _vp, _vp, _vp, _vp, _vp, _vp],
    "attn_decode_plan": [_vp, C.c_int, _ip, _vp],
    "attn_decode_plan_ex": [_vp, C.c_int, _ip, _ip, _ip, _vp],
    "attn_decode_append": [_vp, C.c_int, _vp, _vp, _vp, _vp, _vp],
    "attn_decode_append_partial": [_vp, C.c_int, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "attn_decode_commit": [_vp],
    "attn_combine_lse": [C.c_int, C.c_int, C.c_int, _vp, _vp, _vp, _vp, _vp],
    "attn_combine_lse_packed": [C.c_int, C.c_int, C.c_int, _vp, _vp, _vp],
    "kvp_device_status": [_vp, _vp, _ip],
    "kvp_plan_info": [_vp, _ip, _ip, _ip, _ip, _ip, _ip, _ip, C.c_int],
    "kvp_plan_cta_start": [_vp, _ip, C.c_int],
    "kvp_launch_info": [_vp, _ip, _ip],
    "kvp_timing_enable": [_vp, C.c_int],
    "kvp_set_overlap": [_vp, C.c_int],
    "kvp_set_merge_mode": [_vp, C.c_int],
    "kvp_plan_clusters": [_vp, _ip, _ip],
    "attn_contig_noalloc": [_vp, _vp, _vp, _vp] + [C.c_int] * 7 + [_vp],
    "kvp_timing_read": [_vp, C.POINTER(C.c_double), _ip],
    "kvx_create": [C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(_vp)],
    "kvx_handle": [_vp, _vp],
    "kvx_open": [_vp, C.c_int, _vp],
    "kvx_destroy": [_vp],
    "attn_decode_append_xgpu": [_vp, C.c_int, _vp, _vp, _vp, _vp, _vp, _vp],
    "kvn_unique_id": [_vp],
    "kvn_create": [C.c_int, C.c_int, C.c_int, _vp, C.c_int, C.POINTER(_vp)],
    "kvn_destroy": [_vp],
    "attn_decode_append_nccl": [_vp, C.c_int, _vp, _vp, _vp, _vp, _vp, _vp],
    "kvs_create": [C.c_int, C.c_int, C.POINTER(C.c_longlong), C.POINTER(_vp)],
    "kvs_destroy": [_vp],
    "kvs_place": [_vp, C.c_longlong, C.c_int, _ip],
    "kvs_resize": [_vp, C.c_longlong, C.c_int],
    "kvs_release": [_vp, C.c_longlong],
    "kvs_gpu_of": [_vp, C.c_longlong, _ip],
    "kvs_load": [_vp, C.c_int, C.POINTER(C.c_longlong), _ip],
}


class _W4Matrix(C.Structure):
    _fields_ = [("device", C.c_int), ("n", C.c_int), ("k", C.c_int), ("group", C.c_int), ("codes", _vp),
                ("scales", _vp), ("zeros", _vp)]


class _LogitsCall(C.Structure):
    _fields_ = [("device", C.c_int), ("rows", C.c_int), ("vocab", C.c_int), ("dtype", C.c_int), ("logits", _vp),
                ("ld_logits", C.c_longlong), ("out", _vp), ("ld_out", C.c_longlong), ("pick", _vp), ("hist", _vp),
                ("hist_off", _vp), ("gen_from", _vp), ("hist_n", C.c_longlong), ("repetition", _vp),
                ("presence", _vp), ("frequency", _vp), ("bias_ids", _vp), ("bias", _vp), ("bias_off", _vp),
                ("bias_n", C.c_longlong), ("mask", _vp), ("ld_mask", C.c_longlong)]


_SIGS.update({
    "w4_sizes": [C.c_int, C.c_int, C.c_int] + [C.POINTER(C.c_size_t)] * 3,
    "w4_quantize": [_vp, _vp, C.c_int, C.c_longlong, _vp],
    "w4_dequantize": [_vp, _vp, C.c_longlong, _vp],
    "w4_linear": [_vp, _vp, C.c_int, C.c_int, C.c_longlong, _vp, _vp, C.c_longlong, _vp, C.c_int, C.c_longlong, _vp, _vp],
    "w4_gated": [_vp, _vp, _vp, C.c_int, C.c_int, C.c_longlong, _vp, C.c_int, C.c_longlong, _vp, _vp],
    "w4_work_bytes": [C.c_int] * 6 + [C.POINTER(C.c_size_t)],
    "logits_adjust": [C.POINTER(_LogitsCall), _vp],
    "step_ops_status": [C.c_int, _ip],
    "step_ops_wait_limit": [C.c_longlong],
})
_RESTYPE = {"kv_last_error": C.c_char_p, "kv_status_str": C.c_char_p, "kv_version": C.c_char_p}

_lib = None


class KVError(RuntimeError):
    def __init__(self, status: int, fn: str, msg: str):
        self.status = status
        super().__init__(f"{fn}: {_lib.kv_status_str(status).decode()} ({msg})")


def load() -> C.CDLL:
    """Load libkvattn.so (build it with rk3588-npu_b200/build.py).  Raises
    FileNotFoundError when it is absent: there is no other implementation."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is missing; build it with `python rk3588-npu_b200/build.py`")
        L = C.CDLL(LIB_PATH)
        for name, args in _SIGS.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = _RESTYPE.get(name, C.c_int)
        _lib = L
    return _lib


def _check(rc: int, fn: str) -> None:
    if rc != KV_OK:
        raise KVError(rc, fn, _lib.kv_last_error().decode())


def call(fn: str, *args) -> None:
    """Call a status-returning C entry point, raising KVError on failure."""
    _check(getattr(load(), fn)(*args), fn)


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return t.data_ptr()


def _stream(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _ints(xs):
    xs = list(int(x) for x in xs)
    return (C.c_int * max(1, len(xs)))(*xs)


class Pool:
    """A paged KV pool on one GPU (or a host-only bookkeeping pool).

    Method names follow KVCache where one exists (kv_cache.h:19-41):
    ``reset``, ``cur_pos``/``set_cur_pos`` (per sequence), ``capacity``."""

    def __init__(self, device: int, num_layers: int, num_blocks: int, *, num_q_heads: int = 12,
                 num_kv_heads: int = 2, dtype: int = KV_F16, max_seqs: int = 256,
                 max_seq_len: int = 32768, rope_theta: float = 1e6):
        L = load()
        h = _vp()
        _check(L.kvp_create(device, num_layers, num_q_heads, num_kv_heads, HEAD_DIM, BLOCK_TOKENS,
                            num_blocks, dtype, max_seqs, max_seq_len, rope_theta, C.byref(h)),
               "kvp_create")
        self.h = h
        self.device = device
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.q_heads = num_q_heads
        self.kv_heads = num_kv_heads
        self.kv_dim = num_kv_heads * HEAD_DIM
        self.hidden = num_q_heads * HEAD_DIM
        self.dtype = dtype
        self.max_seqs = max_seqs
        self.max_seq_len = max_seq_len
        self._plan_n = 0

    def close(self) -> None:
        if self.h:
            _check(_lib.kvp_destroy(self.h), "kvp_destroy")
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- pool ----
    def reset(self, stream=None) -> None:
        call("kvp_reset", self.h, None if self.device < 0 else _stream(stream))

    def free_blocks(self) -> int:
        n = C.c_int()
        call("kvp_free_blocks", self.h, C.byref(n))
        return n.value

    def storage(self):
        k, v, lb = _vp(), _vp(), C.c_size_t()
        call("kvp_storage", self.h, C.byref(k), C.byref(v), C.byref(lb))
        return k.value, v.value, lb.value

    def launch_info(self):
        a, b = C.c_int(), C.c_int()
        call("kvp_launch_info", self.h, C.byref(a), C.byref(b))
        return a.value, b.value

    # ---- sequences ----
    def seq_alloc(self) -> int:
        s = C.c_int()
        call("kvp_seq_alloc", self.h, C.byref(s))
        return s.value

    def seq_free(self, seq: int) -> None:
        call("kvp_seq_free", self.h, seq)

    def reserve(self, seq: int, n_tokens: int) -> None:
        call("kvp_seq_reserve", self.h, seq, n_tokens)

    def set_blocks(self, seq: int, block_ids) -> None:
        ids = list(block_ids)
        call("kvp_seq_set_blocks", self.h, seq, _ints(ids), len(ids))

    def cur_pos(self, seq: int) -> int:
        n = C.c_int()
        call("kvp_seq_len", self.h, seq, C.byref(n))
        return n.value

    def set_cur_pos(self, seq: int, pos: int) -> None:
        call("kvp_seq_set_len", self.h, seq, pos)

    def blocks(self, seq: int) -> list[int]:
        n = C.c_int()
        call("kvp_seq_blocks", self.h, seq, None, 0, C.byref(n))
        buf = (C.c_int * max(1, n.value))()
        call("kvp_seq_blocks", self.h, seq, buf, n.value, C.byref(n))
        return list(buf[:n.value])

    def capacity(self, seq: int) -> int:
        return len(self.blocks(seq)) * BLOCK_TOKENS

    # ---- data movement (device tensors) ----
    def import_rows(self, layer, seq, pos0, k_rows, v_rows, stream=None) -> None:
        n = k_rows.shape[0]
        assert k_rows.shape == (n, self.kv_dim) and v_rows.shape == (n, self.kv_dim)
        call("kvp_import", self.h, layer, seq, pos0, n, _ptr(k_rows), _ptr(v_rows), _stream(stream))

    def gather(self, layer, seq, stream=None):
        import torch
        n = self.cur_pos(seq)
        dev = torch.device("cuda", self.device)
        rows = _on_stream(stream, dev, lambda: [torch.empty((n, self.kv_dim), dtype=torch.int16, device=dev) for _ in range(2)])
        k, v = rows
        call("kvp_gather", self.h, layer, seq, _ptr(k), _ptr(v), _stream(stream))
        _handed_over(stream, dev, *rows)
        return k, v

    def import_i8(self, layer, seq, pos0, k_codes, v_codes, k_scales, v_scales, stream=None) -> None:
        """INT8 pools: codes [n, kv_dim] int8, scales [n, kv_heads] fp32 (device tensors)."""
        n = k_codes.shape[0]
        call("kvp_import_i8", self.h, layer, seq, pos0, n, _ptr(k_codes), _ptr(v_codes), _ptr(k_scales),
             _ptr(v_scales), _stream(stream))

    def gather_i8(self, layer, seq, stream=None):
        """INT8 pools: (k_codes, v_codes, k_scales, v_scales) of positions [0, len)."""
        import torch
        n = self.cur_pos(seq)
        dev = torch.device("cuda", self.device)
        rows = _on_stream(stream, dev, lambda: [torch.empty((n, self.kv_dim), dtype=torch.int8, device=dev) for _ in range(2)] + [
            torch.empty((n, self.kv_dim // HEAD_DIM), dtype=torch.float32, device=dev) for _ in range(2)])
        kc, vc, ks, vs = rows
        call("kvp_gather_i8", self.h, layer, seq, _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), _stream(stream))
        _handed_over(stream, dev, *rows)
        return kc, vc, ks, vs

    def append_chunk(self, layer, seq, pos0, k, v, stream=None) -> None:
        n = k.shape[0]
        assert k.shape == (n, self.kv_dim) and v.shape == (n, self.kv_dim)
        call("kv_append_chunk", self.h, layer, seq, pos0, n, _ptr(k), _ptr(v), _stream(stream))

    def prefill(self, layer, seq, pos0, q, out, stream=None, kernel="tc") -> None:
        """Causal attention of q [n, hidden] (unrotated) at positions pos0.. over
        the pool (the chunk's K/V appended first); kernel "tc" (tcgen05) or
        "mma" (the mma.sync baseline)."""
        n = q.shape[0]
        fn = "attn_prefill" if kernel == "tc" else "attn_prefill_mma"
        call(fn, self.h, layer, seq, pos0, n, _ptr(q), _ptr(out), _stream(stream))

    def append_chunk_batch(self, layer, seqs, pos0s, k, v, ns=None, stream=None) -> None:
        """Chunks of several sequences in one call: chunk i is ns[i] rows of
        k / v [sum(ns), kv_dim] (in order) at positions pos0s[i].. of seqs[i]."""
        ns = list(ns) if ns is not None else [k.shape[0]]
        assert len(seqs) == len(pos0s) == len(ns) and sum(ns) == k.shape[0]
        call("kv_append_chunk_batch", self.h, layer, len(seqs), _ints(seqs), _ints(pos0s), _ints(ns), _ptr(k),
             _ptr(v), _stream(stream))

    def prefill_batch(self, layer, seqs, pos0s, ns, q, out, stream=None) -> None:
        """Causal attention of several chunks (rows concatenated in q / out, in
        order) in shared tcgen05 launches."""
        assert len(seqs) == len(pos0s) == len(ns) and sum(ns) == q.shape[0]
        call("attn_prefill_batch", self.h, layer, len(seqs), _ints(seqs), _ints(pos0s), _ints(ns), _ptr(q),
             _ptr(out), _stream(stream))

    # ---- decode ----
    def plan(self, seq_ids, rope_pos=None, append=None, stream=None) -> None:
        ids = list(seq_ids)
        st = None if self.device < 0 else _stream(stream)
        if rope_pos is None and append is None:
            call("attn_decode_plan", self.h, len(ids), _ints(ids), st)
        else:
            rp = _ints(rope_pos) if rope_pos is not None else None
            ap = _ints(append) if append is not None else None
            call("attn_decode_plan_ex", self.h, len(ids), _ints(ids), rp, ap, st)
        self._plan_n = len(ids)

    def plan_info(self):
        """The active plan: pieces (slot, kv head, b0, b1), CTA ranges, patches."""
        n, grid, npatch = C.c_int(), C.c_int(), C.c_int()
        call("kvp_plan_info", self.h, C.byref(n), C.byref(grid), C.byref(npatch), None, None, None,
             None, 0)
        cap = max(1, n.value)
        a, b, c, d = [(C.c_int * cap)() for _ in range(4)]
        call("kvp_plan_info", self.h, C.byref(n), C.byref(grid), C.byref(npatch), a, b, c, d, cap)
        cs = (C.c_int * (grid.value + 1))()
        call("kvp_plan_cta_start", self.h, cs, grid.value + 1)
        return {"nitems": n.value, "grid": grid.value, "npatch": npatch.value,
                "items": list(zip(a[:n.value], b[:n.value], c[:n.value], d[:n.value])),
                "cta_start": list(cs)}

    def decode_layer(self, layer, q, k_new, v_new, out, m=None, l=None, stream=None) -> None:
        n = self._plan_n
        assert q.shape[0] >= n and out.shape[0] >= n
        if m is None:
            call("attn_decode_append", self.h, layer, _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(out),
                 _stream(stream))
        else:
            call("attn_decode_append_partial", self.h, layer, _ptr(q), _ptr(k_new), _ptr(v_new),
                 _ptr(out), _ptr(m), _ptr(l), _stream(stream))

    def commit(self) -> None:
        call("attn_decode_commit", self.h)

    def timing(self, enable: bool) -> None:
        call("kvp_timing_enable", self.h, int(enable))

    def set_overlap(self, enable: bool) -> None:
        """kvp_set_overlap: decode launches may copy their first tiles while
        the previous kernel in the stream finishes (that kernel must not
        write this pool, other than as one of this pool's decode launches)."""
        call("kvp_set_overlap", self.h, int(enable))

    def set_merge_mode(self, mode: int) -> None:
        """kvp_set_merge_mode: KVP_MERGE_GRID (a merge launch behind the
        decode launch, the default) or KVP_MERGE_CLUSTER (splits merged inside
        8-CTA clusters when the packing balances)."""
        call("kvp_set_merge_mode", self.h, int(mode))

    def plan_clusters(self):
        """(launches of the active plan merging inside clusters, launches)."""
        a, b = C.c_int(), C.c_int()
        call("kvp_plan_clusters", self.h, C.byref(a), C.byref(b))
        return a.value, b.value

    def timing_read(self):
        """(summed decode-launch milliseconds, launches) since timing(True)."""
        ms, n = C.c_double(), C.c_int()
        call("kvp_timing_read", self.h, C.byref(ms), C.byref(n))
        return ms.value, n.value

    def device_status(self, stream=None) -> int:
        s = C.c_int()
        call("kvp_device_status", self.h, _stream(stream), C.byref(s))
        return s.value


def kernel_count() -> int:
    """Kernels the library has launched in this process so far."""
    n = C.c_longlong()
    call("kv_kernel_count", C.byref(n))
    return n.value


def combine_lse(m, l, o, out, stream=None) -> None:
    """out[rows, dim] = LSE merge of G partial states m, l [G, rows], o [G, rows, dim]."""
    G, rows, dim = o.shape
    call("attn_combine_lse", G, rows, dim, _ptr(m), _ptr(l), _ptr(o), _ptr(out), _stream(stream))


def combine_lse_packed(packed, rows, out, stream=None) -> None:
    """The same merge over packed [G, rows*(2+dim)] rows of [m | l | o]."""
    G = packed.shape[0]
    dim = packed.shape[1] // rows - 2
    call("attn_combine_lse_packed", G, rows, dim, _ptr(packed), _ptr(out), _stream(stream))


# ---------------------------------------------------------------- step_ops.h
STEP_F16, STEP_BF16, STEP_F32 = 0, 1, 2
_step_types = {}  # torch dtype -> STEP_*


def _step_dtype(t, what: str) -> int:
    if not _step_types:
        import torch
        _step_types.update({torch.float16: STEP_F16, torch.bfloat16: STEP_BF16, torch.float32: STEP_F32})
    d = _step_types.get(t.dtype)
    if d is None:
        raise ValueError(f"{what}: unsupported element type {t.dtype}")
    return d


def _rows(t, device: int, what: str, rows=None, cols=None) -> int:
    """A 2-D device tensor with contiguous rows: the elements from row to row."""
    shape = t.shape
    if len(shape) != 2 or t.get_device() != device:
        raise ValueError(f"{what}: a 2-D tensor on cuda:{device} is expected")
    m, n = shape
    if (rows is not None and m != rows) or (cols is not None and n != cols):
        raise ValueError(f"{what}: shape {tuple(shape)}, expected ({rows}, {cols})")
    if t.is_contiguous():
        return n
    ld, inner = t.stride()
    if inner != 1 and n > 1:
        raise ValueError(f"{what}: the elements of a row must be adjacent")
    return ld if m > 1 else n


def _words(t, device: int, what: str, dtype, n=None):
    """The address of a contiguous 1-D device tensor of 4-byte values (None: NULL)."""
    if t is None:
        return None
    shape = t.shape
    if t.dtype is not dtype or t.get_device() != device or len(shape) != 1 or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous 1-D {dtype} tensor on cuda:{device} is expected")
    if n is not None and shape[0] != n:
        raise ValueError(f"{what}: {shape[0]} values, expected {n}")
    return t.data_ptr()


_raw_stream = None  # device index -> address of torch's current stream


def _stream_on(stream, device: int):
    global _raw_stream
    if stream is None:
        if _raw_stream is None:
            import torch
            # the plain address where torch has it, without a Stream object around it
            _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
                (lambda d: torch.cuda.current_stream(d).cuda_stream)
        return _raw_stream(device)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _on_stream(stream, device, make):
    """make()'s tensors, allocated for the stream that a call runs on: a block of
    the current stream's may still be in use by that stream's pending work,
    which `stream` does not wait for."""
    if stream is None or _stream_on(stream, device.index) == _stream_on(None, device.index):
        return make()
    import torch
    s = torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream
    with torch.cuda.stream(s):
        return make()


def _handed_over(stream, device, *tensors):
    """Results made for `stream`, which the caller may use on the current stream and free there."""
    if stream is not None:
        import torch
        current = torch.cuda.current_stream(device)
        for t in tensors:
            if t is not None:
                t.record_stream(current)


def _scratch(w, x, dtype: int, m: int, ldx: int, gated: int, stream):
    """Scratch of w4_work_bytes() for an x that is fp32 or not in 16-byte aligned
    rows, held by the caching allocator for the call's stream; None where no
    rows go through it."""
    if dtype != STEP_F32 and ldx % 8 == 0 and x.data_ptr() % 16 == 0:
        return None
    key = (m, dtype == STEP_F32, gated)
    size = w._work.get(key)
    if size is None:  # the sizes of a matrix do not change
        n = C.c_size_t()
        call("w4_work_bytes", w.n, w.k, w.group, dtype, m, gated, C.byref(n))
        size = w._work[key] = n.value
    if not size:
        return None
    import torch
    return _on_stream(stream, x.device, lambda: torch.empty(size, dtype=torch.uint8, device=x.device))


class W4:
    """A matrix [n, k] in 4 bits (w4_matrix of include/step_ops.h, which gives
    the layout): codes int32 [T, S, 2, 32, 4], scales fp16 [T, Q, 8, 2] and
    zero points uint8 of that shape or None, with T = ceil(n / 16), S = ceil(k /
    128), Q = ceil(k / group).  Made by w4_quantize, or from such tensors."""

    def __init__(self, codes, scales, zeros, n: int, k: int, group: int):
        import torch
        load()
        sizes = [C.c_size_t() for _ in range(3)]
        call("w4_sizes", n, k, group, *[C.byref(x) for x in sizes])
        dev = codes.get_device()
        if dev < 0:
            raise ValueError("codes: a device tensor is expected")
        for t, size, dtype, what in ((codes, sizes[0], torch.int32, "codes"), (scales, sizes[1], torch.float16, "scales"),
                                     (zeros, sizes[2], torch.uint8, "zeros")):
            if t is None and what == "zeros":
                continue
            if t.dtype != dtype or t.get_device() != dev or not t.is_contiguous() or t.nbytes != size.value:
                raise ValueError(f"{what}: {size.value} contiguous bytes of {dtype} on cuda:{dev} are expected")
        self._hold(codes, scales, zeros, n, k, group, dev)

    def _hold(self, codes, scales, zeros, n, k, group, dev) -> None:
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.n, self.k, self.group, self.device = n, k, group, dev
        self._c = _W4Matrix(dev, n, k, group, codes.data_ptr(), scales.data_ptr(),
                            zeros.data_ptr() if zeros is not None else None)
        self._at = C.addressof(self._c)
        self._work = {}  # (rows, fp32, gated) -> w4_work_bytes

    def dequantize(self, out=None, stream=None):
        """The matrix's values, fp32 [n, k]."""
        import torch
        if out is None:
            dev = self.codes.device
            out = _on_stream(stream, dev, lambda: torch.empty(self.n, self.k, dtype=torch.float32, device=dev))
            _handed_over(stream, dev, out)
        elif out.dtype != torch.float32:
            raise ValueError("out: fp32 is expected")
        ld = _rows(out, self.device, "out", self.n, self.k)
        call("w4_dequantize", self._at, out.data_ptr(), ld, _stream_on(stream, self.device))
        return out


def w4_quantize(w, group: int = 128, zero_points: bool = False, stream=None) -> W4:
    """w [n, k] fp16 or bf16 -> W4 (w4_quantize of include/step_ops.h)."""
    import torch
    n, k = w.shape
    if not (n > 0 and k > 0 and group in (32, 64, 128)):
        raise ValueError(f"a 4-bit matrix of {n} x {k} in groups of {group}: groups of 32, 64 or 128 are supported")
    T, S, Q = (n + 15) // 16, (k + 127) // 128, (k + group - 1) // group
    dev, dtype = w.device, _step_dtype(w, "w")
    if dev.type != "cuda":
        raise ValueError("w: a device tensor is expected")
    load()
    m = W4.__new__(W4)
    arrays = _on_stream(stream, dev, lambda: (
        torch.empty((T, S, 2, 32, 4), dtype=torch.int32, device=dev), torch.empty((T, Q, 8, 2), dtype=torch.float16, device=dev),
        torch.empty((T, Q, 8, 2), dtype=torch.uint8, device=dev) if zero_points else None))
    m._hold(*arrays, n, k, group, dev.index)
    ld = _rows(w, m.device, "w")
    call("w4_quantize", m._at, w.data_ptr(), dtype, ld, _stream_on(stream, m.device))
    _handed_over(stream, dev, *arrays)
    return m


def w4_linear(w: W4, x, out, bias=None, residual=None, stream=None) -> None:
    """out [m, n] = x [m, k] W^T (+ bias [n] fp32) (+ residual [m, n], of out's
    type; may be out).  x and out fp16, bf16 or fp32, rows any distance apart."""
    dev = w.device
    ldx = _rows(x, dev, "x", None, w.k)
    m = x.shape[0]
    ldo = _rows(out, dev, "out", m, w.n)
    b = r = None
    ldr = 0
    xd = _step_dtype(x, "x")
    if bias is not None:
        import torch
        b = _words(bias, dev, "bias", torch.float32, w.n)
    if residual is not None:
        ldr = _rows(residual, dev, "residual", m, w.n)
        if residual.dtype != out.dtype:
            raise ValueError("residual: out's element type is expected")
        r = residual.data_ptr()
    work = _scratch(w, x, xd, m, ldx, 0, stream)
    rc = _lib.w4_linear(w._at, x.data_ptr(), xd, m, ldx, b, r, ldr, out.data_ptr(), _step_dtype(out, "out"), ldo,
                        work.data_ptr() if work is not None else None, _stream_on(stream, dev))
    if rc:
        _check(rc, "w4_linear")


def w4_gated(gate: W4, up: W4, x, out, stream=None) -> None:
    """out [m, n] = silu(x Wg^T) * (x Wu^T), types as w4_linear."""
    dev = gate.device
    ldx = _rows(x, dev, "x", None, gate.k)
    m = x.shape[0]
    ldo = _rows(out, dev, "out", m, gate.n)
    xd = _step_dtype(x, "x")
    work = _scratch(gate, x, xd, m, ldx, 1, stream)
    rc = _lib.w4_gated(gate._at, up._at, x.data_ptr(), xd, m, ldx, out.data_ptr(), _step_dtype(out, "out"), ldo,
                       work.data_ptr() if work is not None else None, _stream_on(stream, dev))
    if rc:
        _check(rc, "w4_gated")


def step_ops_status(device: int = 0) -> int:
    """KV_OK, or KV_ERR_TIMEOUT if a bounded wait ran out since the last call (synchronises the device)."""
    s = C.c_int()
    call("step_ops_status", device, C.byref(s))
    return s.value


def step_ops_wait_limit(clocks: int = -1) -> None:
    """The limit of those waits in SM clocks for launches from now on (0: what is not ready has run out; < 0: about a second)."""
    call("step_ops_wait_limit", clocks)


def logits_adjust(logits, out, pick=None, hist=None, hist_off=None, gen_from=None, repetition=None, presence=None,
                  frequency=None, bias_ids=None, bias=None, bias_off=None, mask=None, stream=None) -> None:
    """Penalties, biases and a mask on logits [rows, vocab] (fp32, fp16 or
    bf16) into out (may be logits), and the greedy choice of each row into
    pick [rows] int32 (-1: nothing is left): logits_adjust of
    include/step_ops.h.  hist / bias_ids are int32 lists cut by hist_off /
    bias_off [rows + 1]; gen_from int32 and the penalties fp32 have one value
    per row; mask is int32 [rows, >= ceil(vocab / 32)], a set bit allows."""
    import torch
    i32, f32 = torch.int32, torch.float32
    load()
    dev = logits.get_device()
    ld_in = _rows(logits, dev, "logits")
    rows, vocab = logits.shape
    ld_out = _rows(out, dev, "out", rows, vocab)
    if out.dtype != logits.dtype:
        raise ValueError("out: the logits' element type is expected")
    mask_ptr, ld_mask = None, 0
    if mask is not None:
        if mask.dtype != i32:
            raise ValueError("mask: int32 words are expected")
        ld_mask = _rows(mask, dev, "mask", rows)
        if mask.shape[1] < (vocab + 31) // 32:
            raise ValueError(f"mask: {mask.shape[1]} words per row for {vocab} tokens")
        mask_ptr = mask.data_ptr()
    if (hist is None) != (hist_off is None) or not ((bias is None) == (bias_ids is None) == (bias_off is None)):
        raise ValueError("hist and hist_off, and bias_ids, bias and bias_off, come together")
    if gen_from is not None and hist is None:
        raise ValueError("gen_from needs a history")
    bias_n = bias_ids.shape[0] if bias_ids is not None else 0
    c = _LogitsCall(dev, rows, vocab, _step_dtype(logits, "logits"), logits.data_ptr(), ld_in, out.data_ptr(), ld_out,
                    _words(pick, dev, "pick", i32, rows), _words(hist, dev, "hist", i32),
                    _words(hist_off, dev, "hist_off", i32, rows + 1), _words(gen_from, dev, "gen_from", i32, rows),
                    hist.shape[0] if hist is not None else 0, _words(repetition, dev, "repetition", f32, rows),
                    _words(presence, dev, "presence", f32, rows), _words(frequency, dev, "frequency", f32, rows),
                    _words(bias_ids, dev, "bias_ids", i32), _words(bias, dev, "bias", f32, bias_n),
                    _words(bias_off, dev, "bias_off", i32, rows + 1), bias_n, mask_ptr, ld_mask)
    rc = _lib.logits_adjust(C.byref(c), _stream_on(stream, dev))
    if rc:
        _check(rc, "logits_adjust")


class Scheduler:
    """Placement of requests onto GPUs by resident KV blocks (kvs_* C ABI).

    Deterministic: ranks that make the same calls in the same order agree
    on every placement without communicating."""

    def __init__(self, blocks_per_gpu, block_tokens: int = BLOCK_TOKENS):
        L = load()
        caps = (C.c_longlong * len(blocks_per_gpu))(*[int(b) for b in blocks_per_gpu])
        h = _vp()
        _check(L.kvs_create(len(blocks_per_gpu), block_tokens, caps, C.byref(h)), "kvs_create")
        self.h = h
        self.n_gpus = len(blocks_per_gpu)

    def close(self) -> None:
        if self.h:
            _check(_lib.kvs_destroy(self.h), "kvs_destroy")
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def place(self, request: int, tokens: int) -> int:
        g = C.c_int()
        call("kvs_place", self.h, request, tokens, C.byref(g))
        return g.value

    def resize(self, request: int, tokens: int) -> None:
        call("kvs_resize", self.h, request, tokens)

    def release(self, request: int) -> None:
        call("kvs_release", self.h, request)

    def gpu_of(self, request: int) -> int:
        g = C.c_int()
        call("kvs_gpu_of", self.h, request, C.byref(g))
        return g.value

    def load(self, gpu: int) -> tuple[int, int]:
        b, n = C.c_longlong(), C.c_int()
        call("kvs_load", self.h, gpu, C.byref(b), C.byref(n))
        return b.value, n.value
