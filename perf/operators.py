"""Cases that time and check the operators a generating text model runs on: attention over whole prompts
(``ops.decoder.CausalAttention``), attention of one new token per item over a prefix that the whole batch shares and
the item's own keys (``ops.decoder.SharedPrefixAttention``) and products with 4-bit weights
(``ops.linear_int4.Int4Linear``).

``run`` computes an operator either with elementary torch operations in 32 bits (``own`` false) or through this
package (``own`` true), on what ``prepare`` made; ``exact`` computes the same in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a handful of chat turns of a few tokens each: the latency of one small launch
        {"name": "prompt_short", "op": "prompt", "dtype": "fp16", "heads": 12, "kv_heads": 12, "d": 64, "seqs": 4,
         "shortest": 1, "longest": 64, "tail": 0, "causal": True},
        # the text benchmark's batch (64 texts of 16 to 512 tokens, 12 heads of 64) scored by a causal model
        {"name": "prompt_batch", "op": "prompt", "dtype": "bf16", "heads": 12, "kv_heads": 12, "d": 64, "seqs": 64,
         "shortest": 16, "longest": 512, "tail": 5, "causal": True},
        # prompts of very different lengths in one packed step, four query heads to a key head
        {"name": "prompt_ragged", "op": "prompt", "dtype": "fp16", "heads": 32, "kv_heads": 8, "d": 128, "seqs": 9,
         "shortest": 1, "longest": 4097, "tail": 3, "causal": True},
        # one long document
        {"name": "prompt_long", "op": "prompt", "dtype": "bf16", "heads": 16, "kv_heads": 4, "d": 128, "seqs": 1,
         "shortest": 16384, "longest": 16384, "tail": 0, "causal": True},
        # two samples of a short prompt, a multi-head model: the latency of one decoding step
        {"name": "prefix_short", "op": "prefix", "dtype": "fp16", "heads": 12, "kv_heads": 12, "d": 64, "batch": 2,
         "prefix": 257, "shortest": 1, "longest": 33},
        # an odd batch behind one instruction text, six query heads to a key head
        {"name": "prefix_odd", "op": "prefix", "dtype": "fp16", "heads": 24, "kv_heads": 4, "d": 80, "batch": 17,
         "prefix": 1999, "shortest": 0, "longest": 300},
        # a usual serving batch behind a system prompt
        {"name": "prefix_batch", "op": "prefix", "dtype": "bf16", "heads": 32, "kv_heads": 8, "d": 128, "batch": 64,
         "prefix": 4096, "shortest": 1, "longest": 512},
        # many questions on one long document
        {"name": "prefix_long", "op": "prefix", "dtype": "bf16", "heads": 32, "kv_heads": 8, "d": 128, "batch": 128,
         "prefix": 32768, "shortest": 64, "longest": 1024},
        # one token through a projection of the text benchmark's hidden size: latency
        {"name": "int4_small", "op": "int4", "dtype": "fp16", "rows": 1, "n": 768, "k": 768, "group": 32,
         "zero": False, "bias": True},
        # sizes that are no multiple of anything, with zero points
        {"name": "int4_odd", "op": "int4", "dtype": "bf16", "rows": 5, "n": 5003, "k": 4000, "group": 64, "zero": True,
         "bias": False},
        # one token through the widest projection of a large model: the weights' bytes count alone
        {"name": "int4_large", "op": "int4", "dtype": "fp16", "rows": 1, "n": 28672, "k": 8192, "group": 128,
         "zero": False, "bias": False},
        # a serving batch through the same kind of projection
        {"name": "int4_batch", "op": "int4", "dtype": "bf16", "rows": 64, "n": 14336, "k": 8192, "group": 128,
         "zero": True, "bias": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt", "prefix", "int4"])
    case = {"op": op, "dtype": rng.choice(["fp16", "bf16"])}
    if op == "int4":
        rows = _log_int(rng, 1, 64)
        n = _log_int(rng, 256, 16384)
        k = _log_int(rng, 256, 8192)
        case.update(rows=rows, n=n, k=k, group=rng.choice([16, 32, 64, 128, 256]), zero=rng.random() < 0.5,
                    bias=rng.random() < 0.5)
        return case
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    case.update(heads=heads, kv_heads=kv_heads, d=rng.choice([32, 64, 64, 80, 96, 128, 128, 128]))
    if op == "prompt":
        longest = _log_int(rng, 1, 6000)
        # padded scores of the plain form stay below 3e9 values
        most = max(1, min(64, int(3e9 / (heads * longest * longest))))
        case.update(seqs=_log_int(rng, 1, most), shortest=max(1, longest // rng.choice([1, 2, 8, 100])),
                    longest=longest, tail=rng.choice([0, 1, 17]), causal=rng.random() < 0.8)
    else:
        longest = _log_int(rng, 1, 1024)
        case.update(batch=_log_int(rng, 1, 128), prefix=_log_int(rng, 1, 16384), shortest=rng.randint(0, longest),
                    longest=longest)
    return case


# ----------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed, count):
    """Lengths spread evenly over the case's shortest to longest, in an order that the seed gives."""
    some = torch.linspace(case["longest"], case["shortest"], count, dtype=torch.float64).round().to(torch.int32)
    return some[torch.randperm(count, generator=torch.Generator().manual_seed(seed))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).to(dt)
    if case["op"] == "prompt":
        h, hk, d = case["heads"], case["kv_heads"], case["d"]
        lens = _lengths(case, seed, case["seqs"])
        starts = torch.cumsum(lens, 0, dtype=torch.int32) - lens
        rows = int(lens.sum()) + case["tail"]
        qkv = randn(rows, (h + 2 * hk) * d)          # the projection's one buffer: queries, keys, values side by side
        s = {"q": qkv[:, :h * d], "k": qkv[:, h * d:(h + hk) * d], "v": qkv[:, (h + hk) * d:],
             "out": torch.zeros(rows, h * d, device="cuda", dtype=dt), "start": starts.cuda(), "len": lens.cuda(),
             "longest": case["longest"]}
        if own:
            from fastdeploy_b200.ops.decoder import CausalAttention
            s["plan"] = CausalAttention(s["q"], s["k"], s["v"], s["out"], heads=h, kv_heads=hk, seq_start=s["start"],
                                        seq_len=s["len"], max_len=case["longest"], causal=case["causal"])
    elif case["op"] == "prefix":
        h, hk, d, b, p = case["heads"], case["kv_heads"], case["d"], case["batch"], case["prefix"]
        lens = _lengths(case, seed, b)
        s = {"q": randn(b, h * d), "prefix_k": randn(p, hk * d), "prefix_v": randn(p, hk * d),
             "k": randn(b, case["longest"], hk * d), "v": randn(b, case["longest"], hk * d),
             "out": torch.zeros(b, h * d, device="cuda", dtype=dt), "len": lens.cuda()}
        if own:
            from fastdeploy_b200.ops.decoder import SharedPrefixAttention
            s["plan"] = SharedPrefixAttention(s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], s["out"], heads=h,
                                              kv_heads=hk, seq_len=s["len"])
    else:
        m, n, k, g = case["rows"], case["n"], case["k"], case["group"]
        groups = (k + g - 1) // g
        s = {"x": randn(m, k),
             "w": torch.randint(0, 256, (n, groups, g // 2), device="cuda", generator=gen, dtype=torch.uint8),
             "scale": (0.005 + 0.01 * torch.rand(n, groups, device="cuda", generator=gen)).to(dt),
             "zero": torch.randint(0, 256, (n, (groups + 1) // 2), device="cuda", generator=gen, dtype=torch.uint8)
             if case["zero"] else None,
             "bias": torch.randn(n, device="cuda", generator=gen) if case["bias"] else None,
             "out": torch.zeros(m, n, device="cuda", dtype=dt)}
        if own:
            from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
            packed = pack_linear_weight_int4(s["w"], s["scale"], s["zero"], k=k)
            s["plan"] = Int4Linear(s["x"], packed, s["out"], bias=s["bias"])
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------------- the plain forms
def _prompt_plain(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["d"]
    n, m = s["len"].numel(), s["longest"]
    at = torch.arange(m, device="cuda")
    real = at[None, :] < s["len"][:, None]                                            # [sequences, longest]
    rows = torch.where(real, s["start"][:, None] + at[None, :], 0).long()
    q = s["q"].float()[rows].view(n, m, hk, h // hk, d).permute(0, 2, 3, 1, 4)        # sequence, kv head, group, token
    k = s["k"].float()[rows].view(n, m, hk, 1, d).permute(0, 2, 3, 4, 1)
    v = s["v"].float()[rows].view(n, m, hk, 1, d).permute(0, 2, 3, 1, 4)
    w = torch.matmul(q, k).mul_(1.0 / math.sqrt(d))
    seen = real[:, None, :] & (at[None, None, :] <= at[None, :, None]) if c["causal"] else real[:, None, :]
    w.masked_fill_(~seen[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, m, h * d)
    out = torch.zeros_like(s["out"])
    out[rows[real]] = o[real].to(out.dtype)
    return out


def _prefix_plain(s):
    c = s["case"]
    h, hk, d, b = c["heads"], c["kv_heads"], c["d"], c["batch"]
    q = s["q"].float().view(b, hk, h // hk, d)
    pk, pv = s["prefix_k"].float().view(-1, hk, d), s["prefix_v"].float().view(-1, hk, d)
    k, v = s["k"].float().view(b, -1, hk, d), s["v"].float().view(b, -1, hk, d)
    w0 = torch.einsum("bhgd,phd->bhgp", q, pk)
    w1 = torch.einsum("bhgd,blhd->bhgl", q, k)
    real = torch.arange(k.shape[1], device="cuda")[None, :] < s["len"][:, None]
    w1 = w1.masked_fill(~real[:, None, None, :], -math.inf)
    w = torch.cat([w0, w1], -1) / math.sqrt(d)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    p = pk.shape[0]
    o = torch.einsum("bhgp,phd->bhgd", w[..., :p], pv) + torch.einsum("bhgl,blhd->bhgd", w[..., p:], v)
    return o.reshape(b, h * d).to(s["q"].dtype)


def _int4_plain(s):
    c = s["case"]
    low, high = s["w"] & 15, s["w"] >> 4                                              # the even and the odd elements
    q = torch.stack([low, high], -1).view(c["n"], -1, c["group"]).float()
    zero = 8.0
    if s["zero"] is not None:
        z = torch.stack([s["zero"] & 15, s["zero"] >> 4], -1).view(c["n"], -1)[:, :q.shape[1]]
        zero = z.float()[:, :, None]
    w = ((q - zero) * s["scale"].float()[:, :, None]).view(c["n"], -1)[:, :c["k"]]
    y = torch.matmul(s["x"].float(), w.t())
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def run(state):
    if own:
        state["plan"].launch()
        return state["out"]
    op = state["case"]["op"]
    if op == "prompt":
        return _prompt_plain(state)
    if op == "prefix":
        return _prefix_plain(state)
    return _int4_plain(state)


# ------------------------------------------------------------------------------------------- what a pass cannot avoid
def work(case):
    if case["op"] == "prompt":
        h, hk, d = case["heads"], case["kv_heads"], case["d"]
        lens = [float(x) for x in _lengths(case, 1, case["seqs"])]
        pairs = sum(n * (n + 1) / 2 if case["causal"] else n * n for n in lens)
        return {"bytes": 2.0 * sum(lens) * d * (2 * h + 2 * hk), "flops": 4.0 * h * d * pairs}
    if case["op"] == "prefix":
        h, hk, d, b, p = case["heads"], case["kv_heads"], case["d"], case["batch"], case["prefix"]
        own_keys = float(sum(int(x) for x in _lengths(case, 1, b)))
        return {"bytes": 2.0 * (2 * b * h * d + 2 * hk * d * (p + own_keys)), "flops": 4.0 * h * d * (b * p + own_keys)}
    m, n, k, g = case["rows"], case["n"], case["k"], case["group"]
    groups = (k + g - 1) // g
    weights = n * k / 2 + 2 * n * groups + (n * ((groups + 1) // 2) if case["zero"] else 0)
    return {"bytes": weights + 2.0 * m * (k + n) + (4.0 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "prompt":
        h, hk, d = case["heads"], case["kv_heads"], case["d"]
        out = torch.zeros(s["out"].shape, dtype=f64, device="cuda")
        for st, n in zip(s["start"].tolist(), s["len"].tolist()):
            for head in range(h):
                j = head // (h // hk)
                q = s["q"][st:st + n, head * d:(head + 1) * d].to(f64)
                k = s["k"][st:st + n, j * d:(j + 1) * d].to(f64)
                v = s["v"][st:st + n, j * d:(j + 1) * d].to(f64)
                a = (q @ k.T) / d ** 0.5
                if case["causal"]:
                    a += torch.full((n, n), -math.inf, dtype=f64, device="cuda").triu_(1)
                out[st:st + n, head * d:(head + 1) * d] = torch.softmax(a, 1) @ v
        return out
    if case["op"] == "prefix":
        h, hk, d, b = case["heads"], case["kv_heads"], case["d"], case["batch"]
        out = torch.zeros(b, h * d, dtype=f64, device="cuda")
        for i, n in enumerate(s["len"].tolist()):
            keys = torch.cat([s["prefix_k"], s["k"][i, :n]]).to(f64).unflatten(1, (hk, d)).permute(1, 2, 0)
            vals = torch.cat([s["prefix_v"], s["v"][i, :n]]).to(f64).unflatten(1, (hk, d)).permute(1, 0, 2)
            q = s["q"][i].to(f64).view(hk, h // hk, d)
            out[i] = (torch.softmax(q @ keys / d ** 0.5, -1) @ vals).reshape(-1)
        return out
    n, k, g = case["n"], case["k"], case["group"]
    element = torch.arange(k, device="cuda")
    byte = s["w"].view(n, -1)[:, element // 2].to(torch.int32)
    w = torch.where(element % 2 == 0, byte % 16, byte // 16).to(f64)
    if s["zero"] is None:
        w -= 8
    else:
        group = element // g
        zero = s["zero"][:, group // 2].to(torch.int32)
        w -= torch.where(group % 2 == 0, zero % 16, zero // 16)
    w *= s["scale"].to(f64)[:, element // g]
    y = s["x"].to(f64) @ w.T
    return y if s["bias"] is None else y + s["bias"].to(f64)
