"""Operators on torch CUDA tensors: a 4-bit key/value cache and a 16-bit one in pages with their attention, log probabilities of given tokens and the verification of
drafted ones (``b200_kv4_*``, ``b200_paged_*``, ``b200_log_probs``, ``b200_verify_drafts`` in include/b200llama.h, on tensors through csrc/torch_ops.cpp).

Every call runs on the current stream of its tensors' device, returns without waiting and can be captured into a CUDA graph.  Tensors are
checked first: a wrong type, shape, device or layout raises ``ValueError`` (or ``TypeError``: no tensor at all) before anything is launched;
what the library refuses raises ``native.B200Error``.  There are no derivatives: a tensor that requires a gradient is refused unless gradients are off
(``torch.no_grad()``, ``torch.inference_mode()``), one that carries a forward-mode tangent is refused until it is detached.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch

from . import native

OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "_b200ops.so")


def _load():
    native.lib()  # the library that the binding links against, with its own message where it is missing
    if not os.path.exists(OPS_PATH):
        raise RuntimeError(f"{OPS_PATH} is missing: run `python -c 'import __graft_entry__ as g; g.build()'`")
    spec = importlib.util.spec_from_loader("_b200ops", importlib.machinery.ExtensionFileLoader("_b200ops", OPS_PATH))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.on_error(native._raise)
    return m


_ops = _load()
MAX_TOP = 32


class KV4Cache(_ops.Cache):
    """Keys and values of ``slots`` sequences of ``context`` positions in 4 bits (groups of 32 entries of a head share an FP16 scale; heads of 32, 64, 96, 128 or 256).

    ``positions`` (and ``slots``) of a call are int32 tensors on the cache's device with an entry per row; ``slots=None`` is slot 0.  A row whose slot or position lies
    outside the cache is padding: nothing is read, stored or written for it.  Calls that store and read the same positions belong on one stream, or are ordered by events.

    append(k, v, positions, q=None, slots=None, q_norm=None, k_norm=None, eps=1e-6, cos=None, sin=None, layout="half", q_out=None)
        Stores rows ``k``, ``v`` [n, kv_heads, head_size] (FP32, FP16 or BF16; parts of a wider row are fine).  ``q`` [n, heads, head_size] of the same type comes back in
        FP32.  On the way the heads of q and k are RMS-normed (``q_norm`` / ``k_norm`` [head_size]) and rotated (``cos`` / ``sin`` [context, head_size / 2], pairs by
        ``layout``: "half" or "interleaved").  Two rows of a call must not name the same place; ``q_out`` is left as it was where a row is padding or has a negative position.

    attention(q, positions, slots=None, scale=None, window=0, max_len=0, chunk=1, dtype=torch.float32, out=None)
        Causal attention of FP32 rows ``q`` [n, heads, head_size]: the row at position p sees the positions up to p of its slot, the last ``window`` of them (0: all);
        ``scale`` is head_size ** -0.5 unless given.  Results are FP32, FP16 or BF16.  ``max_len`` (largest position + 1, 0: unknown) only chooses how the work is split.  ``chunk``
        (neighbouring rows that are successive tokens of one sequence) does too, and with 16-bit results it chooses the precision: chunks of 64 rows (tokens x query heads of a key/value
        head) and more with heads of 64, 96 or 128 are multiplied as FP16 operands.  FP16 results are then off by 6e-4 of their norm where scores have a standard deviation of 2 and by
        1.8e-3 at 33 (with ``chunk=1`` 2e-4, their own rounding), BF16 results by 1.8e-3 and 2.4e-3 (1.7e-3); FP32 results are never rounded so.  A row that sees nothing is zeros.  (Should a wait inside
        a chunk's kernel ever run out, its rows are not written and the cache refuses further attention: B200Error with the state's code.)

    read(positions, slots=None, dtype=torch.float32)
        The values held at some rows: (k, v), each [n, kv_heads, head_size] (not defined where a row is padding or has a negative position).

    reset() makes every position read as zeros (ordered on the current stream); free() gives the memory back and waits for the device's work.  A cache's memory is not torch's: making one
    allocates from the driver and waits for the device."""

    def __init__(self, slots: int, context: int, kv_heads: int, head_size: int, device: int | torch.device | str | None = None):
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"a cache lives on a GPU, not on {device}")
        super().__init__(slots, context, kv_heads, head_size, torch.cuda.current_device() if device.index is None else device.index)

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self.device_index)


def log_probs(logits: torch.Tensor, targets: torch.Tensor | None, top: int = 0):
    """Of rows ``logits`` [rows, vocab] (FP32, FP16 or BF16; rows may be parts of padded ones): the log probability of ``targets`` [rows] (int32; 0 where a target lies outside
    the vocabulary: no target), the entropy in nats, and the ``top`` (at most 32) most likely tokens with their log probabilities, equal ones by index:
    (logprobs [rows], entropy [rows], top_ids [rows, top] int32, top_logprobs [rows, top])."""
    return _ops.log_probs(logits, targets, top)


class PagedKVCache(_ops.Paged):
    """Keys and values of any number of sequences in ``pages`` pages of ``page_size`` positions (a power of two), FP16 or BF16; heads of 32, 64, 96, 128 or 256.  Which page holds what is the
    caller's: ``tables`` of a call is int32 [sequences, width], and position p of sequence s lies in page ``tables[s, p // page_size]``.  Sequences may share pages.  ``keys`` and ``values``
    [pages, kv_heads, page_size, head_size] are the memory itself, torch's; zeros at first.

    ``positions`` (and ``sequences``) of a call are int32 tensors on the cache's device with an entry per row; ``sequences=None`` is the first table's.  A row whose sequence has no table or whose
    position lies behind its table is padding: nothing is stored or written for it, and what lies in its rows does not matter.  A table entry outside the pool is no page: nothing is stored there, nobody sees its positions.  At
    most 2^29 positions a table.  Calls that store and read the same positions belong on one stream, or are ordered by events.

    append(k, v, positions, tables, sequences=None, q=None, q_norm=None, k_norm=None, eps=1e-6, cos=None, sin=None, layout="half", q_out=None)
        Stores rows ``k``, ``v`` [n, kv_heads, head_size] (FP32, FP16 or BF16; parts of a wider row are fine), rounded once.  ``q`` [n, heads, head_size] of the same type comes back in the
        cache's type.  On the way the heads of q and k are RMS-normed (``q_norm`` / ``k_norm`` [head_size]) and their first 2 r entries rotated (``cos`` / ``sin`` [positions, r]; r is
        head_size / 2 for whole heads; scaled or stretched positions are a matter of these tables; pairs by ``layout``: "half": i and i + r, or "interleaved": 2 i and 2 i + 1).  A position
        behind these tables is padding.  Two rows of a call must not name the same place; ``q_out``, which may not overlap ``q``, ``k``, ``v`` or the cache (refused), is left as it was where a row is padding or has a negative position.

    attention(q, positions, tables, sequences=None, scale=None, window=0, max_len=0, chunk=1, dtype=None, out=None)
        Causal attention of rows ``q`` [n, heads, head_size] of the cache's type: the row at position p sees the positions up to p of its sequence, the last ``window`` of them (0: all);
        ``scale`` is head_size ** -0.5 unless given.  Results are of the cache's type unless ``dtype`` says FP32, FP16 or BF16.  ``chunk`` (neighbouring rows that are successive tokens of one
        sequence: drafted tokens, a prompt's chunk) and ``max_len`` (largest position + 1, 0: unknown) only choose how the work is split, but tell them: rows of a prompt without ``chunk`` read all pages once each, where a chunk's
        read them once for 32 rows or 128, tens of times as fast; and a call of more than 256 single rows (or of 256 groups) gives each its own CTAs, however long it is.  ``out`` may be ``q`` itself, but not overlap it or the cache
        otherwise (refused).  ``dtype`` chooses the precision too: 16-bit results come
        from probabilities of the cache's type, half a step off each, FP32 results from several such numbers (24 bits BF16, 22 FP16).  A row that sees nothing is zeros; a value that is
        infinite or NaN reaches the rows that see it, and only those."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_size: int, dtype: torch.dtype = torch.bfloat16, device: int | torch.device | str | None = None):
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"a cache lives on a GPU, not on {device}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a paged cache is FP16 or BF16, not {dtype}")
        if min(pages, page_size, kv_heads, head_size) <= 0:
            raise ValueError("pages, page_size, kv_heads and head_size must be positive")
        keys, values = (torch.zeros(pages, kv_heads, page_size, head_size, dtype=dtype, device=device) for _ in range(2))
        super().__init__(keys, values)

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self.device_index)


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor | None, draft_logits: torch.Tensor | None = None, temperature: float = 1.0):
    """How many drafted tokens of each sequence stand, and the token behind them, so that all of them are distributed as the target's own samples (temperature 0: are its most likely ones).

    ``logits`` [sequences, drafts + 1, vocab] (FP32, FP16 or BF16; rows may be parts of padded ones): the target's, the first behind what was there, the others behind a draft each.
    ``drafts`` [sequences, drafts] int32: the first negative one (or one outside the vocabulary) ends a sequence's.  ``draft_logits`` [sequences, drafts, vocab] of the same type: what the drafts were sampled
    from, at the same ``temperature`` (0, or 1e-4 to 1e4); None: they were not sampled (looked up).  ``uniforms`` [sequences, drafts + 1] FP32 in [0, 1): one for each draft, the last for the
    token (None with temperature 0).  Draft i stands when uniforms[i] q_i(draft) < p_i(draft) and those in front of it do; the token is drawn from p of its row where no draft was left, else from
    max(p - q, 0) (None: p without the draft), as the first index whose running sum passes uniforms[drafts] times the whole.  At most 64 drafts.

    Returns (tokens [sequences, drafts + 1] int32: the drafts that stand, the token, then -1; accepted [sequences] int32).  A row that has no distribution (a NaN, an infinite logit, none
    above -inf) ends its sequence where it is reached: its draft does not stand, the token is -1."""
    return _ops.verify_drafts(logits, drafts, uniforms, draft_logits, temperature)
