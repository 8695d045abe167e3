"""NaN scores of keys that count reach the outputs that see them, and no others."""
import pytest
import torch

from test_decoder_attention_gpu import make_packed, make_prefix

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix,cap,lens,bad", [
    # one or all of few own keys, next to a prefix
    (300, 20, [1, 5], [0]), (300, 20, [20, 20], list(range(20))), (300, 20, [20, 20], [7]),
    # a warp's share and a split's share of many own keys, with and without a prefix
    (0, 2048, [2048, 1500], list(range(64, 80))), (129, 4096, [4096, 100], list(range(0, 512))),
    (1, 4096, [4096, 4096], list(range(4000, 4096)))])
def test_nan_own_keys(prefix, cap, lens, bad, dtype):
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    q, pk, pv, k, v, length = make_prefix((2, prefix, cap, lens, 4, 2, 64), dtype, 3)
    k[0, bad, 64:] = float("nan")                                   # item 0, the second key head
    out = torch.empty(2, 256, dtype=dtype, device="cuda")
    SharedPrefixAttention(q, pk, pv, k, v, out, heads=4, kv_heads=2, seq_len=length).launch()
    nan = out.isnan().view(2, 4, 64)
    assert nan[0, 2:].all() and not nan[0, :2].any() and not nan[1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [slice(5, 6), slice(0, 512), slice(512, 1024), slice(1920, 2000), slice(0, 2000)])
def test_nan_prefix_keys(bad, dtype):
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    q, pk, pv, k, v, length = make_prefix((3, 2000, 40, [0, 1, 40], 4, 2, 64), dtype, 4)
    pk[bad, :64] = float("nan")
    out = torch.empty(3, 256, dtype=dtype, device="cuda")
    SharedPrefixAttention(q, pk, pv, k, v, out, heads=4, kv_heads=2, seq_len=length).launch()
    nan = out.isnan().view(3, 4, 64)
    assert nan[:, :2].all() and not nan[:, 2:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [0, 100, 128, 399])
def test_nan_prompt_keys(first, dtype):
    from fastdeploy_b200.ops.decoder import CausalAttention
    q, k, v, start, length = make_packed([400, 50], [1, 2], 4, 2, 64, dtype, 5)
    k[1 + first, 64:] = float("nan")
    out = torch.zeros(q.shape[0], 256, dtype=dtype, device="cuda")
    CausalAttention(q, k, v, out, heads=4, kv_heads=2, seq_start=start, seq_len=length).launch()
    nan = out.isnan().view(-1, 4, 64)
    want = torch.zeros_like(nan)
    want[1 + first:401, 2:] = True
    assert torch.equal(nan, want)
