"""Prompt attention (causal, grouped heads, packed sequences) and shared-prefix decode attention against 64 bits.

Tolerance, element by element, from the arithmetic of the kernels. With u half a step of the 16-bit type
(``finfo.eps / 2``), weights p_j, l = sum p_j, A = sum p_j |v_j| / l and n keys:

* each weight is rounded to 16 bits before it multiplies V: at most u A (in fp16, weights under 2^-14 have an absolute
  step: n 2^-25 max|v| / l more, and l >= 1 / 2^8 of its true scale is covered by the factor below);
* a score is a sum of d products in fp32, off by at most (d + 8) 2^-23 S with S = scale max |q| . |k|, scaled to log2
  units in fp32 and put through a 2-ulp exponential: a relative error of each weight of at most
  e = 2 (d + 8) 2^-23 S + 2^-20, which moves the quotient by at most 2 e A;
* the sums over n keys are in fp32: n 2^-23 A for the numerator and as much for l;
* the result is rounded once: u |o|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def reference(q, k, v, scale, visible):
    """(o, tolerance) in 64 bits for q [n, d], k / v [m, d] and a boolean visible [n, m]; rows that see nothing are 0."""
    dt, (n, d), m = q.dtype, q.shape, k.shape[0]
    u = torch.finfo(dt).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    k = torch.where(visible.any(0)[:, None], k, 0)
    v = torch.where(visible.any(0)[:, None], v, 0)
    s = (q @ k.T * scale).masked_fill(~visible, -math.inf)
    top = s.amax(1, keepdim=True)
    p = torch.exp(s - torch.where(top.isinf(), 0, top))
    l = p.sum(1, keepdim=True)
    some = l > 0
    l = torch.where(some, l, 1)
    o = torch.where(some, p @ v / l, 0)
    a = p @ v.abs() / l
    big_s = (scale * (q.abs() @ k.abs().T)).amax()
    e = 2 * (d + 8) * 2 ** -23 * big_s + 2 ** -20
    tol = a * (u + 2 * e + 2 * m * 2 ** -23) + u * o.abs() + 2 ** -40
    if dt == torch.float16:
        tol = tol + m * 2 ** -25 * v.abs().amax() / l + 2 ** -25
    return o, tol


def make_packed(lens, gaps, heads, kv_heads, d, dt, seed, junk=float("nan")):
    """One projection buffer with sequences of ``lens`` tokens, ``gaps[i]`` junk rows before each and some behind."""
    gen = torch.Generator().manual_seed(seed)
    starts, at = [], 0
    for n, g in zip(lens, gaps):
        at += g
        starts.append(at)
        at += n
    rows = at + 5
    qkv = torch.full((rows, (heads + 2 * kv_heads) * d), junk, dtype=dt)
    for st, n in zip(starts, lens):
        qkv[st:st + n] = torch.randn(n, qkv.shape[1], generator=gen).to(dt)
    qkv = qkv.cuda()
    q, k, v = qkv.split([heads * d, kv_heads * d, kv_heads * d], 1)
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, lens)]
    return q, k, v, ints[0], ints[1]


def check_packed(q, k, v, out, starts, lens, heads, kv_heads, d, scale, causal, mark):
    outside = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    for st, n in zip(starts, lens):
        outside[st:st + n] = False
        vis = torch.ones(n, n, dtype=torch.bool, device="cuda")
        vis = vis.tril() if causal else vis
        for h in range(heads):
            if n == 0:
                continue
            j = h // (heads // kv_heads)
            o, tol = reference(q[st:st + n, h * d:(h + 1) * d], k[st:st + n, j * d:(j + 1) * d],
                               v[st:st + n, j * d:(j + 1) * d], scale, vis)
            diff = (out[st:st + n, h * d:(h + 1) * d].double() - o).abs()
            assert (diff <= tol).all(), (st, n, h, diff.max().item(), (diff / tol).max().item())
    assert (out[outside] == mark).all()


PROMPTS = [
    # lens, gaps, heads, kv_heads, d
    ([1], [0], 1, 1, 64),
    ([128], [0], 1, 1, 128),
    ([129, 1, 0, 255], [0, 0, 3, 1], 2, 2, 64),
    ([300, 17], [2, 1], 4, 2, 128),
    ([1025], [0], 3, 1, 80),
    ([513, 64, 2], [1, 0, 7], 7, 1, 32),
    ([200, 333], [0, 0], 12, 4, 96),
    ([77, 130], [0, 1], 2, 2, 72),
    ([40], [3], 1, 1, 8),
    ([700], [0], 16, 1, 64),
    ([65, 33], [1, 1], 128, 1, 16),
    ([2000, 1, 1, 1999], [0, 0, 0, 0], 4, 1, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_causal_attention(case, causal, dtype):
    from fastdeploy_b200.ops.decoder import CausalAttention
    lens, gaps, heads, kv_heads, d = case
    q, k, v, start, length = make_packed(lens, gaps, heads, kv_heads, d, dtype, 1)
    out = torch.full((q.shape[0], heads * d), 7.0, dtype=dtype, device="cuda")
    att = CausalAttention(q, k, v, out, heads=heads, kv_heads=kv_heads, seq_start=start, seq_len=length, causal=causal,
                          max_len=max(lens))
    att.launch()
    att.status.check()
    check_packed(q, k, v, out, start.tolist(), lens, heads, kv_heads, d, 1 / math.sqrt(d), causal, 7.0)


PREFIXES = [
    # batch, prefix, capacity, lens, heads, kv_heads, d
    (1, 1, 0, None, 1, 1, 64),
    (1, 0, 5, [5], 2, 1, 64),
    (3, 0, 40, [0, 1, 40], 4, 4, 128),
    (3, 129, 40, [0, 17, 39], 8, 2, 128),
    (2, 1000, 2000, [1999, 3], 12, 12, 64),
    (130, 257, 20, [(7 * i) % 21 for i in range(130)], 6, 2, 80),
    (5, 4100, 33, [33, 32, 31, 16, 15], 20, 2, 128),
    (4, 300, 64, [64, 1, 0, 50], 32, 1, 32),
    (2, 70, 30, [30, 29], 14, 2, 72),
    (1, 9000, 5000, [4999], 4, 2, 96),
    (9, 128, 16, [16] * 9, 128, 1, 8),
]


def make_prefix(case, dtype, seed, junk=float("nan")):
    b, p, cap, lens, heads, kv_heads, d = case
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen).to(dtype).cuda()
    q = randn(b, heads * d)
    pk, pv = (randn(p, kv_heads * d), randn(p, kv_heads * d)) if p else (None, None)
    k = v = length = None
    if cap:
        k, v = randn(b, cap, kv_heads * d), randn(b, cap, kv_heads * d)
        for i, n in enumerate(lens):
            k[i, n:] = junk
            v[i, n:] = junk
        length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return q, pk, pv, k, v, length


def check_prefix(q, pk, pv, k, v, lens, out, heads, kv_heads, d, scale):
    for i in range(q.shape[0]):
        n = lens[i] if k is not None else 0
        parts_k = ([pk] if pk is not None else []) + ([k[i, :n]] if n else [])
        if not parts_k:
            assert (out[i] == 0).all()
            continue
        kk = torch.cat(parts_k)
        vv = torch.cat(([pv] if pv is not None else []) + ([v[i, :n]] if n else []))
        group = heads // kv_heads
        for j in range(kv_heads):
            o, tol = reference(q[i].view(heads, d)[j * group:(j + 1) * group], kk[:, j * d:(j + 1) * d],
                               vv[:, j * d:(j + 1) * d], scale,
                               torch.ones(group, kk.shape[0], dtype=torch.bool, device="cuda"))
            diff = (out[i].view(heads, d)[j * group:(j + 1) * group].double() - o).abs()
            assert (diff <= tol).all(), (i, j, diff.max().item(), (diff / tol).max().item())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PREFIXES, ids=lambda c: "-".join(str(x) for x in c[:3] + c[4:]))
def test_shared_prefix_attention(case, dtype):
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    b, p, cap, lens, heads, kv_heads, d = case
    q, pk, pv, k, v, length = make_prefix(case, dtype, 2)
    out = torch.full((b, heads * d), 7.0, dtype=dtype, device="cuda")
    att = SharedPrefixAttention(q, pk, pv, k, v, out, heads=heads, kv_heads=kv_heads, seq_len=length)
    for _ in range(2):                      # the second launch finds the workspace as the first one left it
        out.fill_(7.0)
        att.launch()
        att.status.check()
        check_prefix(q, pk, pv, k, v, lens, out, heads, kv_heads, d, 1 / math.sqrt(d))
