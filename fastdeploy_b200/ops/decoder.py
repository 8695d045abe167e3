"""Attention of generating text models (csrc/kernels/decoder_attention_sm100.cu).

* :class:`CausalAttention` - attention over whole prompts: packed sequences of any length, causal or not, grouped heads;
* :class:`SharedPrefixAttention` - one new token per batch item over a prefix that all items share (its keys are read
  once for the whole batch) and the item's own keys in a cache.

Both are planned over fixed buffers like the operators of :mod:`.transformer`; the lengths are device tensors that every
launch reads, so that one plan (and one CUDA graph) serves every batch composition that fits the buffers. A plan owns its
workspace, which is ready on every stream when the constructor returns (one made during a graph capture is that graph's):
launches of one plan have to be ordered (one stream, or streams that wait for one another); two plans are independent.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .. import _native
from .base import DT_BF16, DT_F16, DeviceOp, StatusWord, settle

KEY_TILE = 128          # keys per tile of the tensor-core kernel


class _DecoderAttnDesc(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("status", ctypes.c_void_p), ("seq_start", ctypes.c_void_p), ("seq_len", ctypes.c_void_p),
                ("pk", ctypes.c_void_p), ("pv", ctypes.c_void_p), ("prefix_len", ctypes.c_void_p),
                ("part_o", ctypes.c_void_p), ("part_ml", ctypes.c_void_p), ("own_o", ctypes.c_void_p),
                ("own_ml", ctypes.c_void_p), ("counter", ctypes.c_void_p)] + \
               [(n, ctypes.c_longlong) for n in ("q_ld", "k_ld", "v_ld", "o_ld", "pk_ld", "pv_ld", "k_item", "v_item")] + \
               [(n, ctypes.c_int) for n in ("dtype", "prefix_form", "n_seq", "rows", "max_len", "prefix_rows", "own_rows",
                                            "H", "Hk", "D", "causal", "splits", "own_splits")] + [("scale", ctypes.c_float)]


def _lib():
    lib = _native.kernels()
    if not getattr(lib, "_decoder_ready", False):
        lib.fdb_decoder_attention_create.restype = ctypes.c_void_p
        lib.fdb_decoder_attention_create.argtypes = [ctypes.POINTER(_DecoderAttnDesc)]
        if lib.fdb_decoder_attention_desc_size() != ctypes.sizeof(_DecoderAttnDesc):
            raise RuntimeError("libfdb200_kernels.so is out of date: DecoderAttnDesc layout differs; rebuild with "
                               "`python -m fastdeploy_b200._native.build`")
        lib._decoder_ready = True
    return lib


_DTYPES = {torch.float16: DT_F16, torch.bfloat16: DT_BF16}


def _check_heads(heads: int, kv_heads: int, width: int, scale: Optional[float]):
    """(head dim, score scale) after checking what the kernels take."""
    if heads < 1 or kv_heads < 1 or heads % kv_heads or heads // kv_heads > 128:
        raise ValueError(f"{heads} query heads do not divide into groups of at most 128 over {kv_heads} key heads")
    if width % heads:
        raise ValueError(f"{width} columns of q do not divide into {heads} heads")
    d = width // heads
    if d % 8 or not 8 <= d <= 128:
        raise ValueError(f"head dim {d}: a multiple of 8 up to 128 is needed")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (0.0 < scale < math.inf):
        raise ValueError(f"the score scale must be positive and finite, got {scale}")
    return d, scale


def _check_rows(name: str, t: torch.Tensor, like: torch.Tensor, dims: int, width: int) -> None:
    if t.dim() != dims or t.shape[-1] != width:
        raise ValueError(f"{name}: expected {dims} dimensions with {width} columns, got {tuple(t.shape)}")
    if t.dtype not in _DTYPES or t.dtype != like.dtype:
        raise TypeError(f"{name}: all operands must be fp16 or all bf16, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, q on {like.device}")
    if t.numel() == 0:
        raise ValueError(f"{name} is empty")
    if t.stride(-1) != 1 or t.data_ptr() % 16:
        raise ValueError(f"{name}: columns must be contiguous and the first row 16-byte aligned")
    for dim in range(dims - 1):
        if t.shape[dim] > 1 and (t.stride(dim) % 8 or t.stride(dim) < (width if dim == dims - 2 else 0)):
            raise ValueError(f"{name}: stride {t.stride(dim)} of dimension {dim} must be a multiple of 8 that holds a row")


def _check_ints(name: str, t: torch.Tensor, like: torch.Tensor, count: int) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() != count or t.device != like.device:
        raise ValueError(f"{name}: {count} contiguous int32 values on {like.device} are needed")


def _check_cuda(q: torch.Tensor) -> None:
    if q.device.type != "cuda":
        raise ValueError(f"q is on {q.device}: the kernels run on a GPU")


def _pitch(t: torch.Tensor, dim: int, least: int) -> int:
    """Stride of a dimension; of one that has a single row, any pitch the kernels accept."""
    return t.stride(dim) if t.shape[dim] > 1 else (least + 7) // 8 * 8


def _own_splits(own: int, ctas: int, d: int, sms: int) -> int:
    """Pieces that an item's own keys are cut into, from the rows of its cache (the lengths are only known on the device).

    Uncut, a CTA reads all own keys of an item and key head (of up to 16 query heads). Where such CTAs leave SMs without
    work, caches of 512 rows or more are cut, into pieces of at least 256 rows, until every SM has one CTA, or two of heads
    of up to 64 columns, whose rings hold half the bytes. That is half of what fits on an SM (98 and 49 KB of shared memory
    a CTA): the ring of one CTA keeps enough bytes on their way, and each further piece is a part that goes through memory
    and is joined. 128 columns, one CTA an SM against four: 1 item, 8 key heads, 32768 keys 48 and 54 us; 1 item, 1 key
    head of 16 query heads, 120000 keys 81 and 200 us; 4 items, 8 key heads, 16384 keys 72 and 77 us. 64 columns, two
    against four: 1 item, 12 key heads, 32768 keys 41 and 44 us (one: 43)."""
    per_sm = 1 if d > 64 else 2
    return max(1, min(own // 256, per_sm * sms // ctas))


def _make(desc: _DecoderAttnDesc, keep, name: str, device: torch.device) -> DeviceOp:
    op = DeviceOp(lambda: _lib().fdb_decoder_attention_create(ctypes.byref(desc)), keep, name, device)
    op.create = ("fdb_decoder_attention_create", None, desc)
    settle(device)
    return op


class CausalAttention:
    """Attention over whole prompts that lie back to back in ``q`` ``[T, heads * D]``, ``k`` and ``v``
    ``[T, kv_heads * D]`` (fp16 or bf16; row pitches may differ, e.g. slices of one projection's output).

    Sequence ``i`` is rows ``seq_start[i] .. seq_start[i] + seq_len[i]`` (int32 device tensors, read at every launch; a
    length of zero is allowed, at most ``max_len``, sequences must not overlap). Token ``t`` of a sequence attends to
    its tokens ``0 .. t`` (``causal``) or to all of them; query head ``h`` uses key head ``h // (heads // kv_heads)``.
    Rows of ``out`` outside the sequences are left as they were, and rows of ``k`` / ``v`` outside them may hold
    anything. A sequence that does not fit is not computed and reported through ``status``."""

    def __init__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, *, heads: int,
                 kv_heads: Optional[int] = None, seq_start: torch.Tensor, seq_len: torch.Tensor,
                 max_len: Optional[int] = None, scale: Optional[float] = None, causal: bool = True,
                 status: Optional[StatusWord] = None):
        kv_heads = heads if kv_heads is None else kv_heads
        d, scale = _check_heads(heads, kv_heads, q.shape[-1], scale)
        for name, t, width in (("q", q, heads * d), ("k", k, kv_heads * d), ("v", v, kv_heads * d), ("out", out, heads * d)):
            _check_rows(name, t, q, 2, width)
            if t.shape[0] != q.shape[0]:
                raise ValueError(f"{name} has {t.shape[0]} rows, q {q.shape[0]}")
        rows = q.shape[0]
        n = int(seq_len.numel())
        if n < 1:
            raise ValueError("seq_len holds no sequence")
        _check_ints("seq_start", seq_start, q, n)
        _check_ints("seq_len", seq_len, q, n)
        max_len = rows if max_len is None else int(max_len)
        if max_len < 1:
            raise ValueError(f"max_len must be positive, got {max_len}")
        _check_cuda(q)
        self.status = status or StatusWord(q.device)
        dd = _DecoderAttnDesc()
        dd.q, dd.k, dd.v, dd.out, dd.status = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), self.status.ptr
        dd.seq_start, dd.seq_len = seq_start.data_ptr(), seq_len.data_ptr()
        dd.q_ld, dd.o_ld = _pitch(q, 0, heads * d), _pitch(out, 0, heads * d)
        dd.k_ld, dd.v_ld = _pitch(k, 0, kv_heads * d), _pitch(v, 0, kv_heads * d)
        dd.dtype, dd.n_seq, dd.rows, dd.max_len = _DTYPES[q.dtype], n, rows, min(max_len, rows)
        dd.H, dd.Hk, dd.D, dd.causal, dd.scale = heads, kv_heads, d, int(bool(causal)), scale
        self.ops = [_make(dd, [q, k, v, out, seq_start, seq_len, self.status], "causal_attention", q.device)]

    def launch(self, stream: Optional[int] = None) -> None:
        for op in self.ops:
            op.launch(stream)


class SharedPrefixAttention:
    """One decoding step of a batch whose items share their first keys. ``q`` and ``out`` are ``[B, heads * D]`` (one new
    token per item); ``prefix_k`` / ``prefix_v`` ``[P, kv_heads * D]`` hold the shared keys, of which the first
    ``prefix_len`` (int32 device tensor of one value; ``None``: all) count; ``k`` / ``v`` ``[B, L, kv_heads * D]`` are
    the items' own caches, of which item ``b`` uses the first ``seq_len[b]`` rows (the new token's own key included).

    ``out[b] = softmax(scale * q[b] . [prefix_k; k[b]]) [prefix_v; v[b]]``. Either part may be absent (``None``) or, by its
    length, empty; an item without any key gets zeros. Lengths are read at every launch; one that does not fit its buffer
    is cut to it and reported through ``status``. Rows behind a length may hold anything."""

    def __init__(self, q: torch.Tensor, prefix_k: Optional[torch.Tensor], prefix_v: Optional[torch.Tensor],
                 k: Optional[torch.Tensor], v: Optional[torch.Tensor], out: torch.Tensor, *, heads: int,
                 kv_heads: Optional[int] = None, seq_len: Optional[torch.Tensor] = None,
                 prefix_len: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                 status: Optional[StatusWord] = None):
        kv_heads = heads if kv_heads is None else kv_heads
        d, scale = _check_heads(heads, kv_heads, q.shape[-1], scale)
        _check_rows("q", q, q, 2, heads * d)
        _check_rows("out", out, q, 2, heads * d)
        b = q.shape[0]
        if out.shape[0] != b:
            raise ValueError(f"out has {out.shape[0]} rows, q {b}")
        if (prefix_k is None) != (prefix_v is None) or (k is None) != (v is None):
            raise ValueError("keys and values come together")
        if prefix_k is None and k is None:
            raise ValueError("neither a prefix nor own keys are given")
        rows = own = 0
        if prefix_k is not None:
            _check_rows("prefix_k", prefix_k, q, 2, kv_heads * d)
            _check_rows("prefix_v", prefix_v, q, 2, kv_heads * d)
            rows = prefix_k.shape[0]
            if prefix_v.shape[0] != rows:
                raise ValueError(f"prefix_k has {rows} rows, prefix_v {prefix_v.shape[0]}")
            if prefix_len is not None:
                _check_ints("prefix_len", prefix_len, q, 1)
        elif prefix_len is not None:
            raise ValueError("prefix_len without a prefix")
        if k is not None:
            _check_rows("k", k, q, 3, kv_heads * d)
            _check_rows("v", v, q, 3, kv_heads * d)
            if k.shape[0] != b or v.shape[0] != b or k.shape[1] != v.shape[1]:
                raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match {b} items")
            if seq_len is None:
                raise ValueError("own keys need seq_len")
            _check_ints("seq_len", seq_len, q, b)
            own = k.shape[1]
        elif seq_len is not None:
            raise ValueError("seq_len without own keys")
        _check_cuda(q)
        dev = q.device
        self.status = status or StatusWord(dev)
        sms = torch.cuda.get_device_properties(dev).multi_processor_count
        group = heads // kv_heads
        # The prefix is cut until every SM has a piece of it, but no piece is shorter than four key tiles: each piece
        # costs a launch of its own softmax and a part that the join reads (64 items, 4096 shared keys, 8 key heads of
        # 128: 18 pieces 57 us, 8 pieces 42).
        splits = 1
        if rows:
            pairs = -(-b // (2 * (128 // group)))
            splits = max(1, min(-(-rows // (4 * KEY_TILE)), sms // (pairs * kv_heads)))
        per_head = 8 if group <= 8 else 16
        columns = kv_heads * -(-group // per_head)
        own_splits = _own_splits(own, b * columns, d, sms)

        def space(*shape, dtype=torch.float32):
            return torch.zeros(*shape, dtype=dtype, device=dev)
        self.part_o = space(splits, b, heads, d) if rows else None
        self.part_ml = space(splits, b, heads, 2) if rows else None
        self.own_o = space(own_splits, b, heads, d) if own_splits > 1 else None
        self.own_ml = space(own_splits, b, heads, 2) if own_splits > 1 else None
        self.counter = space(b * columns, dtype=torch.int32) if own_splits > 1 else None
        dd = _DecoderAttnDesc()
        dd.q, dd.out, dd.status = q.data_ptr(), out.data_ptr(), self.status.ptr
        for field, t in (("pk", prefix_k), ("pv", prefix_v), ("k", k), ("v", v), ("seq_len", seq_len),
                         ("prefix_len", prefix_len), ("part_o", self.part_o), ("part_ml", self.part_ml),
                         ("own_o", self.own_o), ("own_ml", self.own_ml), ("counter", self.counter)):
            setattr(dd, field, t.data_ptr() if t is not None else None)
        dd.q_ld, dd.o_ld = _pitch(q, 0, heads * d), _pitch(out, 0, heads * d)
        if rows:
            dd.pk_ld, dd.pv_ld = _pitch(prefix_k, 0, kv_heads * d), _pitch(prefix_v, 0, kv_heads * d)
        if own:
            dd.k_ld, dd.v_ld = _pitch(k, 1, kv_heads * d), _pitch(v, 1, kv_heads * d)
            dd.k_item, dd.v_item = _pitch(k, 0, 0), _pitch(v, 0, 0)
        dd.dtype, dd.prefix_form, dd.rows, dd.prefix_rows, dd.own_rows = _DTYPES[q.dtype], 1, b, rows, own
        dd.H, dd.Hk, dd.D, dd.splits, dd.own_splits, dd.scale = heads, kv_heads, d, splits, own_splits, scale
        self.ops = [_make(dd, [q, prefix_k, prefix_v, k, v, out, seq_len, prefix_len, self.part_o, self.part_ml,
                               self.own_o, self.own_ml, self.counter, self.status], "shared_prefix_attention", dev)]

    def launch(self, stream: Optional[int] = None) -> None:
        for op in self.ops:
            op.launch(stream)
