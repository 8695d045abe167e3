"""Interpreter operators of generating text models: the standard ONNX ``Attention`` (opset 23: grouped heads, causal mask,
past keys) and ONNX Runtime's ``MatMulNBits`` (4-bit weights with group scales)."""
from __future__ import annotations

import math

import torch

from .interp import _OPS, op

_encoder_attention = _OPS["Attention"]


def is_standard_attention(node) -> bool:
    """The standard operator; the fused encoder node (domain ``fdb``) carries ``num_heads``."""
    return node.attr("num_heads") is None


@op("Attention")
def _attention(node, q, k, v, mask=None, past_k=None, past_v=None):
    if not is_standard_attention(node):
        return _encoder_attention(node, q, k, v) if mask is None else _encoder_attention(node, q, k, v, mask)
    flat = q.dim() == 3
    if flat:
        heads, kv_heads = node.attr("q_num_heads"), node.attr("kv_num_heads")
        if not heads or not kv_heads:
            raise ValueError("Attention: three-dimensional inputs need q_num_heads and kv_num_heads")

        def split(t, n):
            return t.reshape(t.shape[0], t.shape[1], n, t.shape[2] // n).transpose(1, 2)
        q, k, v = split(q, heads), split(k, kv_heads), split(v, kv_heads)
    if past_k is not None:
        k, v = torch.cat([past_k, k], 2), torch.cat([past_v, v], 2)
    heads, kv_heads = q.shape[1], k.shape[1]
    if heads % kv_heads:
        raise ValueError(f"Attention: {heads} query heads over {kv_heads} key heads")
    kk, vv = k.repeat_interleave(heads // kv_heads, 1), v.repeat_interleave(heads // kv_heads, 1)
    w = torch.matmul(q, kk.transpose(-1, -2)) * node.attr("scale", 1.0 / math.sqrt(q.shape[-1]))
    cap = float(node.attr("softcap", 0.0))
    if cap > 0:
        w = cap * torch.tanh(w / cap)
    seen = None
    if node.attr("is_causal", 0):
        rows, cols = w.shape[-2:]
        past = 0 if past_k is None else past_k.shape[2]
        seen = torch.arange(cols, device=w.device)[None, :] <= torch.arange(rows, device=w.device)[:, None] + past
    if mask is not None and mask.dtype == torch.bool:
        seen = mask if seen is None else seen & mask
    elif mask is not None:
        w = w + mask
    if seen is not None:
        w = w.masked_fill(~seen, -math.inf)
    o = torch.matmul(torch.softmax(w, -1), vv)
    if flat:
        o = o.transpose(1, 2).reshape(o.shape[0], o.shape[2], -1)
    if len(node.outputs) > 3 and node.outputs[3]:
        raise NotImplementedError("Attention: the score output is not implemented")
    return (o, k, v) if len(node.outputs) > 1 else o


@op("MatMulNBits")
def _matmul_nbits(node, a, b, scales, zero_points=None, g_idx=None, bias=None):
    n, k, bits, group = (int(node.attr(x, d)) for x, d in (("N", 0), ("K", 0), ("bits", 4), ("block_size", 0)))
    if bits != 4:
        raise NotImplementedError(f"MatMulNBits with {bits} bits (4 are supported)")
    groups = -(-k // group)
    b = b.reshape(n, groups * (group // 2))
    q = torch.stack([b & 15, b >> 4], -1).reshape(n, groups * group)[:, :k].to(a.dtype)
    if zero_points is None:
        zero = torch.full((n, groups), 8.0, dtype=a.dtype, device=a.device)
    elif zero_points.dtype == torch.uint8:
        z = zero_points.reshape(n, (groups + 1) // 2)
        zero = torch.stack([z & 15, z >> 4], -1).reshape(n, -1)[:, :groups].to(a.dtype)
    else:
        zero = zero_points.reshape(n, groups).to(a.dtype)
    of = (torch.arange(k, device=a.device) // group) if g_idx is None else g_idx.reshape(-1)[:k].long()
    s = scales.reshape(n, groups).to(a.dtype)
    y = torch.matmul(a, ((q - zero[:, of]) * s[:, of]).t())
    return y if bias is None else y + bias
