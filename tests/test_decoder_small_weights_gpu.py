"""Weights far below the largest one count in fp16 too.

One key has weight 1 and a value of zero, n - 1 keys have weight w = 2^-b and values of one, so o = (n - 1) w / (1 + (n - 1) w).
Every such weight is held in fp16 after a multiplication by 2^7 (the largest one may lag by 2^8 more), where the step below 2^-14
is 2^-24: off by at most e = 2^-25 / 2^7 / w of itself, or half a step 2^-11. The other errors are those of
test_decoder_attention_gpu: a score's rounding and the exponential (2^-18 here: products of powers of two), sums of n terms in
fp32, and the result's rounding.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("n,b", [(4096, 14.3), (16384, 18.6), (32768, 21.4), (32768, 23.5), (32768, 25.5)])
@pytest.mark.parametrize("form", ["prompt", "prefix", "own"])
def test_small_weights(form, n, b, first):
    from fastdeploy_b200.ops.decoder import CausalAttention, SharedPrefixAttention
    d, dt = 64, torch.float16
    q = torch.zeros(1, d, dtype=dt, device="cuda")
    q[0, 0] = 1.0
    k = torch.zeros(n, d, dtype=dt, device="cuda")
    v = torch.ones(n, d, dtype=dt, device="cuda")
    top = 0 if first else n - 1
    k[top, 0], v[top] = 4.0, 0.0                                    # score 4 / 4 * b ln 2 above the others'
    scale = b * 0.6931471805599453 / 4
    out = torch.zeros(1, d, dtype=dt, device="cuda")
    if form == "prompt":
        qs = q.expand(n, d).contiguous()
        full = torch.zeros(n, d, dtype=dt, device="cuda")
        ints = [torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, n)]
        CausalAttention(qs, k, v, full, heads=1, seq_start=ints[0], seq_len=ints[1], scale=scale, causal=False).launch()
        out = full
    elif form == "prefix":
        SharedPrefixAttention(q, k, v, None, None, out, heads=1, scale=scale).launch()
    else:
        length = torch.tensor([n], dtype=torch.int32, device="cuda")
        SharedPrefixAttention(q, None, None, k[None], v[None], out, heads=1, seq_len=length, scale=scale).launch()
    w = 2.0 ** -b
    o = (n - 1) * w / (1 + (n - 1) * w)
    tol = o * (max(2.0 ** -11, 2.0 ** -32 / w) + 2.0 ** -18 + 2 * n * 2.0 ** -23) + 2.0 ** -11 * o + 2.0 ** -25
    diff = (out.double() - o).abs().max().item()
    assert diff <= tol, (diff / o, tol / o)
