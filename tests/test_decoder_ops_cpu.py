"""Generating text models on the host: the standard Attention and MatMulNBits operators of the interpreter against written
out formulas, their way through the ONNX writer and reader, and the refusals of the GPU operators (no GPU needed)."""
import math

import numpy as np
import pytest
import torch

from fastdeploy_b200.ir.graph import Graph, Node
from fastdeploy_b200.ir.interp import _OPS, Interpreter


def naive_attention(q, k, v, scale, causal, past=0):
    """float64, q [B, H, S, D], k / v [B, Hk, L, D], one row at a time."""
    b, h, s, _ = q.shape
    out = np.zeros(q.shape[:3] + v.shape[3:])
    for i in range(b):
        for j in range(h):
            kv = j // (h // k.shape[1])
            for t in range(s):
                n = t + past + 1 if causal else k.shape[2]
                w = np.exp(scale * (k[i, kv, :n] @ q[i, j, t]) - np.max(scale * (k[i, kv, :n] @ q[i, j, t])))
                out[i, j, t] = w @ v[i, kv, :n] / w.sum()
    return out


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("causal", [0, 1])
def test_standard_attention(flat, causal):
    rng = np.random.default_rng(0)
    b, h, hk, s, d = 2, 6, 2, 5, 8
    q, k, v = (rng.standard_normal((b, n, s, d)).astype(np.float32) for n in (h, hk, hk))
    want = naive_attention(q.astype(np.float64), k, v, 0.3, causal)
    attrs = dict(is_causal=causal, scale=0.3)
    ins = [torch.from_numpy(x) for x in (q, k, v)]
    if flat:
        ins = [x.transpose(1, 2).reshape(b, s, -1) for x in ins]
        attrs.update(q_num_heads=h, kv_num_heads=hk)
        want = want.transpose(0, 2, 1, 3).reshape(b, s, -1)
    got = _OPS["Attention"](Node("Attention", ["q", "k", "v"], ["y"], attrs), *ins).numpy()
    # sums of at most 8 products and 5 weights in fp32 of values around 1: 2^-20 is ample
    assert np.abs(got - want).max() < 2 ** -18


def test_standard_attention_past_mask_and_cap():
    rng = np.random.default_rng(1)
    q, k, v, pk, pv = (rng.standard_normal((1, 2, n, 4)).astype(np.float32) for n in (3, 3, 3, 4, 4))
    node = Node("Attention", ["q", "k", "v", "", "pk", "pv"], ["y", "nk", "nv"], dict(is_causal=1))
    y, nk, nv = _OPS["Attention"](node, *(torch.from_numpy(x) if x is not None else None for x in (q, k, v, None, pk, pv)))
    kk, vv = np.concatenate([pk, k], 2), np.concatenate([pv, v], 2)
    assert np.array_equal(nk.numpy(), kk) and np.array_equal(nv.numpy(), vv)
    assert np.abs(y.numpy() - naive_attention(q.astype(np.float64), kk, vv, 0.5, True, past=4)).max() < 2 ** -18
    seen = np.tril(np.ones((3, 3), bool))
    plain = Node("Attention", ["q", "k", "v", "m"], ["y"], {})
    got = _OPS["Attention"](plain, *(torch.from_numpy(x) for x in (q, k, v, seen))).numpy()
    assert np.abs(got - naive_attention(q.astype(np.float64), k, v, 0.5, True)).max() < 2 ** -18
    capped = _OPS["Attention"](Node("Attention", ["q", "k", "v"], ["y"], dict(softcap=2.0)),
                               *(torch.from_numpy(x) for x in (q, k, v)))
    w = torch.softmax(2 * torch.tanh(torch.from_numpy(q @ k.transpose(0, 1, 3, 2)) * 0.5 / 2), -1)
    assert torch.allclose(capped, w @ torch.from_numpy(v), atol=1e-5)


def nbits_weight(rng, n, k, group, zero):
    groups = -(-k // group)
    q = rng.integers(0, 16, (n, groups * group))
    z = rng.integers(0, 16, (n, groups)) if zero else np.full((n, groups), 8)
    s = (0.05 + 0.1 * rng.random((n, groups))).astype(np.float32)
    dense = ((q - np.repeat(z, group, 1)) * np.repeat(s.astype(np.float64), group, 1))[:, :k]
    packed = (q[:, 0::2] | (q[:, 1::2] << 4)).astype(np.uint8).reshape(n, groups, group // 2)
    zp = np.pad(z, ((0, 0), (0, groups % 2)))
    return dense, packed, s, (zp[:, 0::2] | (zp[:, 1::2] << 4)).astype(np.uint8) if zero else None


@pytest.mark.parametrize("zero", [False, True])
def test_matmul_nbits_through_the_onnx_file(zero):
    from fastdeploy_b200.importer.onnx_format import load_onnx, save_onnx
    rng = np.random.default_rng(2)
    n, k, group = 7, 50, 16
    dense, packed, s, z = nbits_weight(rng, n, k, group, zero)
    bias = rng.standard_normal(n).astype(np.float32)
    g = Graph("m", 21)
    g.add_input("x", "float32", [None, k])
    for name, value in (("w", packed), ("s", s.reshape(-1)), ("b", bias)) + ((("z", z.reshape(-1)),) if zero else ()):
        g.add_initializer(name, value)
    g.add_node("MatMulNBits", ["x", "w", "s", "z" if zero else "", "", "b"], ["y"], domain="com.microsoft", N=n, K=k, bits=4,
               block_size=group)
    g.add_output("y", "float32", [None, n])
    x = rng.standard_normal((3, k)).astype(np.float32)
    want = x.astype(np.float64) @ dense.T + bias
    for graph in (g, load_onnx(save_onnx(g))):
        got = np.asarray(Interpreter(graph).run({"x": x})["y"])
        # 50 products of up to 15 * 0.15 * 3 in fp32
        assert np.abs(got - want).max() < 50 * 8 * 2 ** -23 * 8


def test_refusals_of_the_attention_operators():
    from fastdeploy_b200.ops.decoder import CausalAttention, SharedPrefixAttention
    q, k, out = torch.zeros(16, 128, dtype=torch.float16), torch.zeros(16, 64, dtype=torch.float16), torch.zeros(16, 128, dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32)

    def causal(q=q, k=k, v=k, out=out, heads=2, kv_heads=1, start=ints, length=ints, **kw):
        return CausalAttention(q, k, v, out, heads=heads, kv_heads=kv_heads, seq_start=start, seq_len=length, **kw)
    for bad in (dict(heads=3), dict(heads=2, kv_heads=3), dict(k=k[:, :60]), dict(k=k.t()), dict(k=k[:8]), dict(out=out[:4]),
                dict(start=ints.long()), dict(length=ints[:0]), dict(start=ints[:1]), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(max_len=0),
                dict(k=torch.zeros(16, 65, dtype=torch.float16)[:, :64]),      # rows that are not 16 bytes apart
                dict(k=torch.zeros(16 * 64 + 8, dtype=torch.float16)[4:-4].view(16, 64)),
                dict(q=torch.zeros(16, 20, dtype=torch.float16), heads=2),     # head dim 10
                dict(q=torch.zeros(16, 272, dtype=torch.float16), heads=2),    # head dim 136
                dict()):                                                       # all right, but not on a GPU
        with pytest.raises(ValueError):
            causal(**bad)
    for bad in (dict(k=k.float()), dict(q=q.float(), k=k.float(), v=k.float(), out=out.float()), dict(out=out.bfloat16())):
        with pytest.raises(TypeError):
            causal(**bad)
    qb, ob, cache = torch.zeros(2, 128, dtype=torch.float16), torch.zeros(2, 128, dtype=torch.float16), torch.zeros(2, 10, 64, dtype=torch.float16)

    def prefix(q=qb, pk=k, pv=k, k=cache, v=cache, out=ob, seq_len=ints, **kw):
        return SharedPrefixAttention(q, pk, pv, k, v, out, heads=2, kv_heads=1, seq_len=seq_len, **kw)
    for bad in (dict(pk=None), dict(k=None), dict(pk=None, pv=None, k=None, v=None, seq_len=None), dict(seq_len=None),
                dict(seq_len=ints[:1]), dict(k=cache[:1]), dict(v=cache[:, :9]), dict(pv=k[:5]), dict(k=cache[0]),
                dict(k=None, v=None), dict(prefix_len=ints), dict(pk=None, pv=None, prefix_len=ints[:1]), dict(out=ob[:1]),
                dict(pk=k[:0], pv=k[:0]), dict(scale=0.0), dict()):
        with pytest.raises(ValueError):
            prefix(**bad)


def test_refusals_of_the_int4_operators():
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, Int4Weight, pack_linear_weight_int4, quantize_groups_int4
    q, s = torch.zeros(4, 3, 16, dtype=torch.uint8), torch.ones(4, 3)
    for args, kw in (((q[0], s), {}), ((q.int(), s), {}), ((q[:, :, :5], s), {}), ((q, s[:2]), {}), ((q, s), dict(k=97)),
                     ((q, s), dict(k=64)), ((q, s, torch.zeros(4, 1, dtype=torch.uint8)), {}), ((q, s), {})):
        with pytest.raises(ValueError):
            pack_linear_weight_int4(*args, **kw)
    for args in ((q, s.double()), (q, s, torch.zeros(4, 2))):
        with pytest.raises(TypeError):
            pack_linear_weight_int4(*args)
    for args in ((torch.zeros(4), 16), (torch.zeros(4, 4), 20), (torch.zeros(0, 4), 16)):
        with pytest.raises(ValueError):
            quantize_groups_int4(*args)
    w = Int4Weight(torch.zeros(1, dtype=torch.uint8), torch.float16, False, 4, 96, 32)
    x, y = torch.zeros(2, 96, dtype=torch.float16), torch.zeros(2, 4, dtype=torch.float16)
    for a, b, bias in ((x[0], y, None), (x[:, :95], y, None), (x, y[:, :3], None), (x[:1], y, None),
                       (torch.zeros(96, 2, dtype=torch.float16).t(), y, None), (x, y, torch.zeros(3)),
                       (x, y, torch.zeros(4, dtype=torch.float16)), (x[:1].expand(2, 96), y, None)):
        with pytest.raises(ValueError):
            Int4Linear(a, w, b, bias=bias)
    for a, b in ((x.float(), y.float()), (x, y.bfloat16()), (x.bfloat16(), y.bfloat16())):
        with pytest.raises(TypeError):
            Int4Linear(a, w, b)


def test_quantised_groups_reproduce_representable_weights():
    from fastdeploy_b200.ops.linear_int4 import quantize_groups_int4
    w = torch.arange(-7, 8).float().repeat(2, 3)[:, :40] * 0.5          # every group of 16 holds -3.5 and 3.5 or is covered
    q, s, z = quantize_groups_int4(w, 16)
    back = (torch.stack([q & 15, q >> 4], -1).reshape(2, -1)[:, :40].float() - 8) * s.repeat_interleave(16, 1)[:, :40]
    assert z is None and ((back - w).abs() <= s.repeat_interleave(16, 1)[:, :40] * 0.5 + 1e-6).all()
