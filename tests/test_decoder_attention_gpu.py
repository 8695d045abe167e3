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


def test_lengths_are_read_at_launch_and_bad_ones_are_reported():
    """One plan, several compositions, on a side stream and as a replayed graph; a sequence that does not fit its buffer is
    left out and reported, the others are computed."""
    from fastdeploy_b200.ops.decoder import CausalAttention
    heads, kv_heads, d, rows = 4, 2, 64, 400
    torch.manual_seed(3)
    q, k, v = (torch.randn(rows, n * d, device="cuda").half() for n in (heads, kv_heads, kv_heads))
    out = torch.empty(rows, heads * d, device="cuda", dtype=torch.float16)
    start, lens = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
    att = CausalAttention(q, k, v, out, heads=heads, kv_heads=kv_heads, seq_start=start, seq_len=lens, max_len=300)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.launch()
    for how, (st, ln) in enumerate([([0, 100, 399], [100, 299, 1]), ([5, 0, 0], [300, 0, 5]), ([10, 20, 300], [1, 200, 100])]):
        start.copy_(torch.tensor(st)), lens.copy_(torch.tensor(ln)), out.fill_(7.0)
        torch.cuda.synchronize()
        if how == 0:
            with torch.cuda.stream(side):
                att.launch()
        elif how == 1:
            att.launch(side.cuda_stream)
        else:
            graph.replay()
        torch.cuda.synchronize()
        att.status.check()
        check_packed(q, k, v, out, st, ln, heads, kv_heads, d, d ** -0.5, True, 7.0)
    for st, ln, good in (([0, 390, 50], [20, 11, 10], [0, 2]), ([0, -1, 50], [20, 4, 10], [0, 2]), ([0, 60, 50], [20, -5, 10], [0, 2]),
                         ([0, 60, 370], [20, 301, 30], [0, 2])):
        start.copy_(torch.tensor(st)), lens.copy_(torch.tensor(ln)), out.fill_(7.0)
        att.launch()
        with pytest.raises(RuntimeError, match="bad shape"):
            att.status.check()
        check_packed(q, k, v, out, [st[i] for i in good], [ln[i] for i in good], heads, kv_heads, d, d ** -0.5, True, 7.0)


def test_prefix_lengths_are_read_at_launch_and_cut_to_the_buffers():
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    case = (4, 700, 50, [50, 0, 1, 20], 8, 2, 64)
    q, pk, pv, k, v, length = make_prefix(case, torch.bfloat16, 4)
    plen = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty(4, 512, device="cuda", dtype=torch.bfloat16)
    att = SharedPrefixAttention(q, pk, pv, k, v, out, heads=8, kv_heads=2, seq_len=length, prefix_len=plen)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.launch()
    for n in (700, 0, 1, 129, 512):
        plen.fill_(n)
        out.fill_(7.0)
        graph.replay()
        att.status.check()
        check_prefix(q, pk[:n] if n else None, pv[:n], k, v, case[3], out, 8, 2, 64, 0.125)
    plen.fill_(701)
    att.launch()
    with pytest.raises(RuntimeError, match="bad shape"):
        att.status.check()
    check_prefix(q, pk, pv, k, v, case[3], out, 8, 2, 64, 0.125)
    plen.fill_(700)
    k2, v2 = torch.nan_to_num(k), torch.nan_to_num(v)
    k.copy_(k2), v.copy_(v2)
    length.copy_(torch.tensor([51, -1, 1, 20]))
    att.launch()
    with pytest.raises(RuntimeError, match="bad shape"):
        att.status.check()
    check_prefix(q, pk, pv, k, v, [50, 0, 1, 20], out, 8, 2, 64, 0.125)


def test_strided_caches_and_broadcast_items():
    """Caches as [B, L] slices of a wider buffer, K and V interleaved, and one item's cache read by every item."""
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    torch.manual_seed(5)
    b, cap, hk, d, heads = 3, 37, 2, 96, 6
    kv = torch.randn(b, 64, 2, hk * d, device="cuda").half()
    k, v = kv[:, 10:10 + cap, 0], kv[:, 10:10 + cap, 1]
    pkv = torch.randn(300, 2 * hk * d + 8, device="cuda").half()
    pk, pv = pkv[:, :hk * d], pkv[:, hk * d:2 * hk * d]
    qo = torch.randn(b, 2, heads * d, device="cuda").half()
    lens = [37, 5, 16]
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    att = SharedPrefixAttention(qo[:, 0], pk, pv, k, v, qo[:, 1], heads=heads, kv_heads=hk, seq_len=length, scale=0.2)
    att.launch()
    att.status.check()
    check_prefix(qo[:, 0], pk, pv, k, v, lens, qo[:, 1], heads, hk, d, 0.2)
    one_k, one_v = k[:1].expand(b, -1, -1), v[:1].expand(b, -1, -1)
    att = SharedPrefixAttention(qo[:, 0], pk, pv, one_k, one_v, qo[:, 1], heads=heads, kv_heads=hk, seq_len=length, scale=0.2)
    att.launch()
    check_prefix(qo[:, 0], pk, pv, one_k, one_v, lens, qo[:, 1], heads, hk, d, 0.2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_rescale_and_equal_scores(dtype):
    """Maxima that grow by far more than the rescaling threshold from tile to tile, and rows of equal scores."""
    from fastdeploy_b200.ops.decoder import CausalAttention, SharedPrefixAttention
    torch.manual_seed(6)
    n, d = 700, 64
    q = torch.randn(n, d, device="cuda").to(dtype)
    ramp = torch.linspace(0, 4, n, device="cuda")[:, None]
    k = (q.float().mean(0, keepdim=True) * 30 * ramp + torch.randn(n, d, device="cuda") * ramp).to(dtype)
    v = torch.randn(n, d, device="cuda").to(dtype)
    ints = [torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, n)]
    for keys in (k, k.flip(0).contiguous(), torch.zeros_like(k)):
        for causal in (True, False):
            out = torch.empty_like(q)
            CausalAttention(q, keys, v, out, heads=1, seq_start=ints[0], seq_len=ints[1], causal=causal).launch()
            check_packed(q, keys, v, out, [0], [n], 1, 1, d, d ** -0.5, causal, 7.0)
        out = torch.empty(1, d, dtype=dtype, device="cuda")
        own = torch.tensor([n - 300], dtype=torch.int32, device="cuda")
        SharedPrefixAttention(q[:1], keys[:300], v[:300], keys[None, 300:], v[None, 300:], out, heads=1, seq_len=own).launch()
        check_prefix(q[:1], keys[:300], v[:300], keys[None, 300:], v[None, 300:], [n - 300], out, 1, 1, d, d ** -0.5)


def test_prompt_then_decoding_steps_together():
    """As a program uses them: a shared prompt goes through 4-bit projections and prompt attention, its keys become the
    prefix; then three items decode five steps each, a captured step replayed, keys appended to their caches. Every
    attention output is held against 64 bits over the very buffers it read."""
    from fastdeploy_b200.ops.decoder import CausalAttention, SharedPrefixAttention
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4, quantize_groups_int4
    torch.manual_seed(7)
    b, n, heads, hk, d, c, dt = 3, 150, 8, 2, 64, 512, torch.bfloat16
    width = (heads + 2 * hk) * d
    w = pack_linear_weight_int4(*quantize_groups_int4(torch.randn(width, c, device="cuda") * c ** -0.5, 32, symmetric=False))
    x, qkv = torch.randn(n, c, device="cuda").to(dt), torch.empty(n, width, dtype=dt, device="cuda")
    out = torch.empty(n, heads * d, dtype=dt, device="cuda")
    q, pk, pv = qkv.split([heads * d, hk * d, hk * d], 1)
    ints = [torch.tensor([z], dtype=torch.int32, device="cuda") for z in (0, n)]
    proj = Int4Linear(x, w, qkv)
    prompt = CausalAttention(q, pk, pv, out, heads=heads, kv_heads=hk, seq_start=ints[0], seq_len=ints[1])
    proj.launch(), prompt.launch()
    proj.status.check(), prompt.status.check()
    check_packed(q, pk, pv, out, [0], [n], heads, hk, d, d ** -0.5, True, 7.0)

    xs, step = torch.randn(b, c, device="cuda").to(dt), torch.empty(b, width, dtype=dt, device="cuda")
    cache_k, cache_v = (torch.full((b, 6, hk * d), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    lens, o = torch.zeros(b, dtype=torch.int32, device="cuda"), torch.empty(b, heads * d, dtype=dt, device="cuda")
    sq, sk, sv = step.split([heads * d, hk * d, hk * d], 1)
    sproj = Int4Linear(xs, w, step)
    att = SharedPrefixAttention(sq, pk, pv, cache_k, cache_v, o, heads=heads, kv_heads=hk, seq_len=lens)
    at = torch.arange(b, device="cuda")

    def one_step():
        sproj.launch()
        cache_k[at, lens.long()] = sk
        cache_v[at, lens.long()] = sv
        lens.add_(1)
        att.launch()
    one_step()
    graph = torch.cuda.CUDAGraph()
    check_prefix(sq, pk, pv, cache_k, cache_v, [1] * b, o, heads, hk, d, d ** -0.5)
    with torch.cuda.graph(graph):
        one_step()
    for t in range(2, 6):
        xs.copy_(torch.randn(b, c, device="cuda"))
        graph.replay()
        att.status.check(), sproj.status.check()
        assert lens.tolist() == [t] * b
        check_prefix(sq, pk, pv, cache_k, cache_v, [t] * b, o, heads, hk, d, d ** -0.5)


def test_plans_of_one_kernel_with_different_shared_memory():
    """A later plan that needs less shared memory leaves an earlier one launchable."""
    from fastdeploy_b200.ops.decoder import CausalAttention, SharedPrefixAttention
    plans = []
    for d in (128, 64):
        q, k, v, start, length = make_packed([40], [0], 2, 2, d, torch.float16, 8)
        out = torch.full((q.shape[0], 2 * d), 7.0, dtype=torch.float16, device="cuda")
        plans.append((CausalAttention(q, k, v, out, heads=2, seq_start=start, seq_len=length), q, k, v, out, start, d))
    for att, q, k, v, out, start, d in plans:
        att.launch()
        check_packed(q, k, v, out, start.tolist(), [40], 2, 2, d, d ** -0.5, True, 7.0)
    plans = []
    for cap in (120000, 300):                      # many splits of the own keys, then one
        case = (1, 0, cap, [cap], 16, 1, 128)
        q, pk, pv, k, v, length = make_prefix(case, torch.float16, 9)
        out = torch.empty(1, 16 * 128, dtype=torch.float16, device="cuda")
        plans.append((SharedPrefixAttention(q, pk, pv, k, v, out, heads=16, kv_heads=1, seq_len=length), q, k, v, cap, out))
    for att, q, k, v, cap, out in plans:
        att.launch()
        att.status.check()
        check_prefix(q, None, None, k, v, [cap], out, 16, 1, 128, 128 ** -0.5)
