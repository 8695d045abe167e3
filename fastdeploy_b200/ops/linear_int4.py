"""Products with 4-bit weights and group scales (csrc/kernels/linear_int4.cu).

``y = x @ W^T + bias`` with ``W[n, k] = (q[n, k] - z[n, k // group]) * s[n, k // group]``, ``q`` and ``z`` in 0..15. The
weight comes in the layout of the ONNX operator ``com.microsoft::MatMulNBits`` (bits = 4) and is laid out once for the
kernel by :func:`pack_linear_weight_int4`; :class:`Int4Linear` is a planned product over fixed buffers. Sums are in fp32 and
the weights are never rounded; the kernel is made for few rows of ``x`` (up to 64 per pass over the weight, more rows
take several passes).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _native
from .base import DT_BF16, DT_F16, DT_F32, DeviceOp, StatusWord, current_stream_ptr, settle

GROUPS = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: DT_F16, torch.bfloat16: DT_BF16}
_SCALE_DTYPES = {torch.float16: DT_F16, torch.bfloat16: DT_BF16, torch.float32: DT_F32}


class _Int4Desc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "y", "bias", "w", "x_pad", "status")] + \
               [("x_ld", ctypes.c_longlong), ("y_ld", ctypes.c_longlong)] + \
               [(n, ctypes.c_int) for n in ("dtype", "scale_dtype", "has_zeros", "m", "n", "k", "group", "tile_rows", "splits")]


def _lib():
    lib = _native.kernels()
    if not getattr(lib, "_int4_ready", False):
        lib.fdb_int4_linear_create.restype = ctypes.c_void_p
        lib.fdb_int4_linear_create.argtypes = [ctypes.POINTER(_Int4Desc)]
        lib.fdb_int4_pack.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_int] * 4 + [ctypes.c_void_p]
        lib.fdb_int4_packed_bytes.argtypes = [ctypes.c_int] * 5
        lib.fdb_int4_packed_bytes.restype = ctypes.c_longlong
        if lib.fdb_int4_desc_size() != ctypes.sizeof(_Int4Desc):
            raise RuntimeError("libfdb200_kernels.so is out of date: Int4Desc layout differs; rebuild with "
                               "`python -m fastdeploy_b200._native.build`")
        lib._int4_ready = True
    return lib


@dataclass
class Int4Weight:
    """A 4-bit weight ``[n, k]`` as the kernel reads it."""
    data: torch.Tensor              # blocks of 128 rows x 128 columns: weights, scales, zero points
    scale_dtype: torch.dtype
    has_zeros: bool
    n: int
    k: int
    group: int


def quantize_groups_int4(w: torch.Tensor, group: int = 128, symmetric: bool = True
                         ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Round-to-nearest 4-bit quantisation of ``w`` ``[n, k]`` per group of ``group`` elements along ``k``: the bytes
    ``[n, groups, group // 2]``, fp32 scales ``[n, groups]`` and, unless ``symmetric``, zero points
    ``[n, (groups + 1) // 2]`` (two to a byte) that :func:`pack_linear_weight_int4` takes."""
    if group not in GROUPS:
        raise ValueError(f"group size {group}: one of {GROUPS} is needed")
    if w.dim() != 2 or w.numel() == 0:
        raise ValueError(f"a weight [n, k] is needed, got {tuple(w.shape)}")
    n, k = w.shape
    groups = -(-k // group)
    wf = torch.zeros(n, groups * group, dtype=torch.float32, device=w.device)
    wf[:, :k] = w.float()
    wf = wf.view(n, groups, group)
    if symmetric:
        scale = wf.abs().amax(-1) / 7.0
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        zero = torch.full_like(scale, 8.0)
    else:
        low, high = wf.amin(-1).clamp(max=0.0), wf.amax(-1).clamp(min=0.0)
        scale = (high - low) / 15.0
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))
        zero = (-low / scale).round().clamp(0, 15)
    q = (torch.round(wf / scale[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8)
    packed = q[..., 0::2] | (q[..., 1::2] << 4)
    if symmetric:
        return packed.contiguous(), scale, None
    z = torch.zeros(n, (groups + 1) // 2 * 2, dtype=torch.uint8, device=w.device)
    z[:, :groups] = zero.to(torch.uint8)
    return packed.contiguous(), scale, (z[:, 0::2] | (z[:, 1::2] << 4)).contiguous()


def _per_row(t: torch.Tensor, n: int, count: int) -> bool:
    """Whether ``t`` holds ``count`` values for each of ``n`` rows: ``[n, count]`` (1s may follow) or flat."""
    return t.numel() == n * count and (t.dim() == 1 or tuple(t.shape[:2]) == (n, count))


def pack_linear_weight_int4(qweight: torch.Tensor, scales: torch.Tensor, zero_points: Optional[torch.Tensor] = None, *,
                            k: Optional[int] = None) -> Int4Weight:
    """Lays out ``qweight`` uint8 ``[n, groups, group // 2]`` (even element in the low half of a byte), ``scales``
    ``[n, groups]`` (fp16, bf16 or fp32, kept as they are) and ``zero_points`` uint8 ``[n, (groups + 1) // 2]`` (two to a
    byte; ``None``: 8 everywhere) for the kernel; scales and zero points may also come flat. ``k`` is the weight's real
    column count when the last group is partly padding."""
    if qweight.dim() != 3 or qweight.dtype != torch.uint8 or qweight.numel() == 0:
        raise ValueError(f"qweight: uint8 [n, groups, group // 2] is needed, got {qweight.dtype} {tuple(qweight.shape)}")
    n, groups, half = qweight.shape
    group = half * 2
    if group not in GROUPS:
        raise ValueError(f"group size {group}: one of {GROUPS} is needed")
    k = groups * group if k is None else int(k)
    if not (groups - 1) * group < k <= groups * group:
        raise ValueError(f"k = {k} does not fill {groups} groups of {group}")
    if scales.dtype not in _SCALE_DTYPES:
        raise TypeError(f"scales must be fp16, bf16 or fp32, got {scales.dtype}")
    if not _per_row(scales, n, groups):
        raise ValueError(f"scales: {n} x {groups} values are needed, got {tuple(scales.shape)}")
    if zero_points is not None:
        if zero_points.dtype != torch.uint8:
            raise TypeError(f"zero points must be packed uint8, got {zero_points.dtype}")
        if not _per_row(zero_points, n, (groups + 1) // 2):
            raise ValueError(f"zero_points: {n} x {(groups + 1) // 2} bytes are needed, got {tuple(zero_points.shape)}")
    for name, t in (("scales", scales), ("zero_points", zero_points)):
        if t is not None and t.device != qweight.device:
            raise ValueError(f"{name} is on {t.device}, qweight on {qweight.device}")
    if qweight.device.type != "cuda":
        raise ValueError(f"qweight is on {qweight.device}: the kernels run on a GPU")
    q, s = qweight.contiguous(), scales.contiguous()
    z = zero_points.contiguous() if zero_points is not None else None
    dev = q.device
    code = _SCALE_DTYPES[s.dtype]
    data = torch.empty(_lib().fdb_int4_packed_bytes(code, int(z is not None), n, k, group), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = _lib().fdb_int4_pack(q.data_ptr(), s.data_ptr(), z.data_ptr() if z is not None else None, data.data_ptr(), code,
                                  n, k, group, current_stream_ptr(dev))
    if rc != 0:
        raise RuntimeError(f"int4 pack: {_native.last_error()}")
    return Int4Weight(data, s.dtype, z is not None, n, k, group)


# Up to this many rows of x take the vector kernel, whose CTAs of 16 weight rows each read x again; more the tensor-core kernel,
# whose blocks cost the same up to 32 rows. Microseconds of both, fp16, at 16 and at 17 rows: 28672 x 8192 64 and 68, then 96
# and 68; 14336 x 8192 39 and 37, then 53 and 37; 9472 x 4096 16 and 20, then 25 and 20; 4096 x 4096 12 and 16, then 14 and 16.
# Weights of a few MB would keep the vector kernel a little longer (768 x 768 at 32 rows: 6 and 12).
VECTOR_ROWS = 16


def _tile_form(m: int, weight: Int4Weight, sms: int) -> Tuple[int, int]:
    """(rows of x per tile, splits of K) of the tensor-core kernel, (0, 1) for the vector kernel."""
    if m <= VECTOR_ROWS:
        return 0, 1
    rows = 32 if m <= 32 else 64
    ctas, k_tiles = -(-weight.n // 128) * -(-m // rows), -(-weight.k // 128)
    return rows, max(1, min(8, sms // ctas, k_tiles // 4))


class Int4Linear(DeviceOp):
    """Planned ``y[M, n] = x[M, k] @ W^T + bias`` over fixed buffers: ``x`` and ``y`` fp16 or bf16 with any row pitch,
    ``bias`` fp32 ``[n]``."""
    _any_stream = True

    def __init__(self, x: torch.Tensor, weight: Int4Weight, y: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                 status: Optional[StatusWord] = None, name: str = "int4_linear"):
        if x.dim() != 2 or y.dim() != 2 or x.shape[0] != y.shape[0] or x.shape[0] < 1:
            raise ValueError(f"x [M, {weight.k}] and y [M, {weight.n}] are needed, got {tuple(x.shape)} and {tuple(y.shape)}")
        if x.shape[1] != weight.k or y.shape[1] != weight.n:
            raise ValueError(f"x has {x.shape[1]} columns and y {y.shape[1]}, the weight is {weight.n} x {weight.k}")
        if x.dtype not in _DTYPES or y.dtype != x.dtype:
            raise TypeError(f"x and y must both be fp16 or both bf16, got {x.dtype} and {y.dtype}")
        if weight.scale_dtype not in (x.dtype, torch.float32):
            raise TypeError(f"the weight's scales are {weight.scale_dtype}: pack it with scales of {x.dtype} or fp32")
        m = x.shape[0]
        for what, t in (("x", x), ("y", y)):
            if t.stride(1) != 1 and t.shape[1] > 1:
                raise ValueError(f"{what}: columns must be contiguous")
            if m > 1 and t.stride(0) < t.shape[1]:
                raise ValueError(f"{what}: rows overlap (pitch {t.stride(0)})")
        if bias is not None and (bias.dtype != torch.float32 or bias.numel() != weight.n or not bias.is_contiguous()):
            raise ValueError(f"bias: {weight.n} contiguous fp32 values are needed")
        for what, t in (("x", x), ("y", y), ("bias", bias)):
            if t is not None and t.device != weight.data.device:
                raise ValueError(f"{what} is on {t.device}, the weight on {weight.data.device}")
        d = _Int4Desc()
        d.x_ld, d.y_ld = (x.stride(0), y.stride(0)) if m > 1 else (-(-weight.k // 8) * 8, weight.n)
        aligned = x.data_ptr() % 16 == 0 and d.x_ld % 8 == 0 and weight.k % 8 == 0
        # rows that 16-byte loads cannot take are copied to aligned ones first (every launch writes all of them)
        self.x_pad = None if aligned else torch.empty(m, -(-weight.k // 8) * 8, dtype=x.dtype, device=x.device)
        d.x, d.y, d.w = x.data_ptr(), y.data_ptr(), weight.data.data_ptr()
        self.status = status or StatusWord(x.device)
        tile_rows, splits = _tile_form(m, weight, torch.cuda.get_device_properties(x.device).multi_processor_count)
        d.tile_rows, d.splits, d.status = tile_rows, splits, self.status.ptr
        for field, t in (("bias", bias), ("x_pad", self.x_pad)):
            setattr(d, field, t.data_ptr() if t is not None else None)
        d.dtype, d.scale_dtype, d.has_zeros = _DTYPES[x.dtype], _SCALE_DTYPES[weight.scale_dtype], int(weight.has_zeros)
        d.m, d.n, d.k, d.group = m, weight.n, weight.k, weight.group
        super().__init__(lambda: _lib().fdb_int4_linear_create(ctypes.byref(d)),
                         [x, y, bias, weight.data, self.x_pad, self.status], name, x.device)
        self.create = ("fdb_int4_linear_create", None, d)
        if self._any_stream:
            settle(x.device)


class _SameStream(Int4Linear):
    """A product that is launched on the stream it was made on, which orders its workspace: nothing to wait for."""
    _any_stream = False


def linear_int4(x: torch.Tensor, weight: Int4Weight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Eager ``x @ W^T + bias`` for ``x`` ``[M, k]``."""
    y = torch.empty(x.shape[0], weight.n, dtype=x.dtype, device=x.device)
    _SameStream(x, weight, y, bias=bias.float().contiguous() if bias is not None else None).launch()
    return y
