"""Operators on torch CUDA tensors: a 4-bit key/value cache with its attention, and log probabilities of given tokens (``b200_kv4_*``,
``b200_log_probs`` in include/b200llama.h).

Every call runs on the current stream of its tensors' device, returns without waiting and can be captured into a CUDA graph.  Tensors are
checked here: a wrong type, shape, device or layout raises ``ValueError`` before anything is launched; what the library refuses raises
``native.B200Error``.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import native

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # B200_GGML_F32, _F16, _BF16
MAX_TOP = 32


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _rows(t: torch.Tensor, name: str, n: int, heads: int, head_size: int, device) -> int:
    """Checks rows [n, heads, head_size] whose heads lie one behind the other; entries between rows."""
    _need(t.dim() == 3 and t.shape[1] == heads and t.shape[2] == head_size and t.shape[0] == n, f"{name}: [{n}, {heads}, {head_size}] is wanted, got {tuple(t.shape)}")
    _need(t.device == device, f"{name} is on {t.device}, the cache on {device}")
    s = t.stride()
    _need(n == 0 or ((s[2] == 1 or head_size == 1) and (s[1] == head_size or heads == 1)), f"{name}: the heads of a row have to lie one behind the other")
    return s[0] if n > 1 else max(s[0], heads * head_size)


def _indices(t: torch.Tensor | None, name: str, n: int, device) -> int | None:
    if t is None:
        return None
    _need(t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == n, f"{name}: {n} entries of int32 are wanted, got {tuple(t.shape)} of {t.dtype}")
    _need(t.device == device, f"{name} is on {t.device}, not on {device}")
    _need(n <= 1 or t.stride(0) == 1, f"{name} has to be contiguous")
    return t.data_ptr()


def _vector(t: torch.Tensor | None, name: str, shape: tuple, device) -> int | None:
    if t is None:
        return None
    _need(t.dtype == torch.float32 and t.device == device and t.dim() == len(shape) and t.is_contiguous(), f"{name}: a contiguous float32 tensor of {len(shape)} dimensions on {device} is wanted")
    _need(t.shape[0] >= shape[0] and t.shape[1:] == shape[1:], f"{name}: {shape} is wanted, got {tuple(t.shape)}")
    return t.data_ptr()


class KV4Cache:
    """Keys and values of ``slots`` sequences of ``context`` positions in 4 bits (groups of 32 entries of a head share an FP16 scale).

    ``positions`` (and ``slots``) of a call are int32 tensors on the cache's device with an entry per row; ``slots=None`` is slot 0.  A row whose slot or position lies
    outside the cache is padding: nothing is read, stored or written for it.  Calls that store and read the same positions belong on one stream, or are ordered by events."""

    def __init__(self, slots: int, context: int, kv_heads: int, head_size: int, device: int | torch.device | str | None = None):
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
        _need(device.type == "cuda", f"a cache lives on a GPU, not on {device}")
        index = torch.cuda.current_device() if device.index is None else device.index
        self.device, self.slots, self.context, self.kv_heads, self.head_size = torch.device("cuda", index), slots, context, kv_heads, head_size
        self._p, out, err = None, C.c_void_p(), C.create_string_buffer(256)
        self._lib = native.lib()
        rc = self._lib.b200_kv4_create(slots, context, kv_heads, head_size, index, C.byref(out), err, 256)
        if rc != native.B200_OK:
            native._raise(rc, err.value.decode())
        self._p = out

    def _call(self, f, args):
        if self._p is None:
            raise native.B200Error(-6, "the cache has been freed")
        rc = f(self._p, C.byref(args), torch.cuda.current_stream(self.device).cuda_stream)
        if rc != native.B200_OK:
            native._raise(rc, self._lib.b200_kv4_last_error(self._p).decode())

    def append(self, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, q: torch.Tensor | None = None, slots: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
               k_norm: torch.Tensor | None = None, eps: float = 1e-6, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, layout: str = "half",
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Stores rows ``k``, ``v`` [n, kv_heads, head_size] (FP32, FP16 or BF16; parts of a wider row are fine).  ``q`` [n, heads, head_size] of the same type comes back in FP32.
        On the way the heads of q and k are RMS-normed (``q_norm`` / ``k_norm`` [head_size]) and rotated (``cos`` / ``sin`` [context, head_size / 2], pairs by ``layout``:
        "half" or "interleaved").  Two rows of a call must not name the same place; ``q_out`` is left as it was where a row is padding or has a negative position."""
        n, hs, dev = k.shape[0], self.head_size, self.device
        a = native.KV4Append()
        _need(k.dtype in _TYPES and v.dtype == k.dtype, f"k and v are FP32, FP16 or BF16, both the same: got {k.dtype} and {v.dtype}")
        _need(layout in native.ROPE_LAYOUTS, f"layout {layout!r}")
        a.n, a.type, a.rope_layout, a.eps = n, _TYPES[k.dtype], native.ROPE_LAYOUTS[layout], eps
        a.k_stride, a.v_stride = _rows(k, "k", n, self.kv_heads, hs, dev), _rows(v, "v", n, self.kv_heads, hs, dev)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        a.positions, a.slots = _indices(positions, "positions", n, dev), _indices(slots, "slots", n, dev)
        _need(a.positions is not None or n == 0, "positions are wanted")
        if q is not None:
            _need(q.dtype == k.dtype and q.dim() == 3, f"q: rows of {k.dtype} as k are wanted")
            a.heads = q.shape[1]
            a.q_stride, a.q = _rows(q, "q", n, a.heads, hs, dev), q.data_ptr()
            if q_out is None:
                q_out = torch.empty((n, a.heads, hs), dtype=torch.float32, device=dev)
            _need(q_out.dtype == torch.float32, "q_out is FP32")
            a.q_out_stride, a.q_out = _rows(q_out, "q_out", n, a.heads, hs, dev), q_out.data_ptr()
        else:
            _need(q_out is None and q_norm is None, "q_out and q_norm belong to q")
        a.q_norm, a.k_norm = _vector(q_norm, "q_norm", (hs,), dev), _vector(k_norm, "k_norm", (hs,), dev)
        _need((cos is None) == (sin is None), "a rotation needs cos and sin")
        if cos is not None:
            a.cos, a.sin = _vector(cos, "cos", (self.context, hs // 2), dev), _vector(sin, "sin", (self.context, hs // 2), dev)
        if n:
            self._call(self._lib.b200_kv4_append, a)
        return q_out

    def attention(self, q: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor | None = None, scale: float | None = None, window: int = 0, max_len: int = 0, chunk: int = 1,
                  dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of FP32 rows ``q`` [n, heads, head_size]: the row at position p sees the positions up to p of its slot, the last ``window`` of them (0: all); ``scale``
        is head_size ** -0.5 unless given.  Results are FP32, FP16 or BF16.  ``max_len`` (largest position + 1, 0: unknown) and ``chunk`` (neighbouring rows that are successive
        tokens of one sequence) only choose how the work is split.  A row that sees nothing is zeros."""
        n, hs, dev = q.shape[0], self.head_size, self.device
        _need(q.dim() == 3 and q.dtype == torch.float32, f"q: FP32 rows [n, heads, head_size] are wanted, got {tuple(q.shape)} of {q.dtype}")
        _need(q.shape[1] > 0 and q.shape[1] % self.kv_heads == 0, f"{q.shape[1]} query heads over {self.kv_heads} key/value heads")
        if out is None:
            out = torch.empty((n, q.shape[1], hs), dtype=dtype, device=dev)
        _need(out.dtype in _TYPES, f"results of {out.dtype}")
        a = native.KV4Attention()
        a.n, a.heads, a.window, a.max_len, a.chunk, a.out_type = n, q.shape[1], window, max_len, chunk, _TYPES[out.dtype]
        a.q_stride, a.out_stride = _rows(q, "q", n, a.heads, hs, dev), _rows(out, "out", n, a.heads, hs, dev)
        a.q, a.out = q.data_ptr(), out.data_ptr()
        a.positions, a.slots = _indices(positions, "positions", n, dev), _indices(slots, "slots", n, dev)
        _need(a.positions is not None or n == 0, "positions are wanted")
        a.scale = 1.0 / math.sqrt(hs) if scale is None else scale
        if n:
            self._call(self._lib.b200_kv4_attention, a)
        return out

    def read(self, positions: torch.Tensor, slots: torch.Tensor | None = None, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """The values held at some rows: (k, v), each [n, kv_heads, head_size] (not defined where a row is padding or has a negative position)."""
        _need(positions is not None and dtype in _TYPES, "positions, and a type of FP32, FP16 or BF16, are wanted")
        n = positions.shape[0]
        k, v = torch.empty((2, n, self.kv_heads, self.head_size), dtype=dtype, device=self.device).unbind(0)
        a = native.KV4Read()
        a.n, a.type, a.k, a.v = n, _TYPES[dtype], k.data_ptr(), v.data_ptr()
        a.positions, a.slots = _indices(positions, "positions", n, self.device), _indices(slots, "slots", n, self.device)
        if n:
            self._call(self._lib.b200_kv4_read, a)
        return k, v

    def reset(self):
        """Every position reads as zeros again (ordered on the current stream)."""
        if self._p is None:
            raise native.B200Error(-6, "the cache has been freed")
        rc = self._lib.b200_kv4_reset(self._p, torch.cuda.current_stream(self.device).cuda_stream)
        if rc != native.B200_OK:
            native._raise(rc, self._lib.b200_kv4_last_error(self._p).decode())

    @property
    def device_bytes(self) -> int:
        return self._lib.b200_kv4_device_bytes(self._p)

    def free(self):
        """Gives the memory back; waits for the device's work."""
        if self._p is not None:
            self._lib.b200_kv4_free(self._p)
            self._p = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def log_probs(logits: torch.Tensor, targets: torch.Tensor | None, top: int = 0):
    """Of rows ``logits`` [rows, vocab] (FP32, FP16 or BF16; rows may be parts of padded ones): the log probability of ``targets`` [rows] (int32; 0 where a target lies outside
    the vocabulary: no target), the entropy in nats, and the ``top`` (at most 32) most likely tokens with their log probabilities, equal ones by index:
    (logprobs [rows], entropy [rows], top_ids [rows, top] int32, top_logprobs [rows, top])."""
    _need(logits.dim() == 2 and logits.dtype in _TYPES and logits.is_cuda, f"logits: FP32, FP16 or BF16 rows [rows, vocab] on a GPU are wanted, got {tuple(logits.shape)} of {logits.dtype}")
    rows, vocab = logits.shape
    _need(vocab > 0 and 0 <= top <= min(MAX_TOP, vocab), f"{top} alternatives of {vocab} logits (at most {MAX_TOP})")
    _need(rows == 0 or vocab == 1 or logits.stride(1) == 1, "the logits of a row have to lie one behind the other")
    a = native.LogProbs()
    a.targets = _indices(targets, "targets", rows, logits.device)
    numbers = torch.empty((2, rows), dtype=torch.float32, device=logits.device)
    ids = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
    values = torch.empty((rows, top), dtype=torch.float32, device=logits.device)
    chosen, entropy = numbers.unbind(0)
    if rows:
        a.logits, a.row_stride, a.rows, a.vocab, a.type, a.top, a.device = logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, _TYPES[logits.dtype], top, logits.device.index
        a.logprobs, a.entropy, a.top_ids, a.top_logprobs = chosen.data_ptr(), entropy.data_ptr(), ids.data_ptr(), values.data_ptr()
        err = C.create_string_buffer(256)
        rc = native.lib().b200_log_probs(C.byref(a), torch.cuda.current_stream(logits.device).cuda_stream, err, 256)
        if rc != native.B200_OK:
            native._raise(rc, err.value.decode())
    return chosen, entropy, ids, values
