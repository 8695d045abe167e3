"""Prompt attention over more sequences than one look of the unit search takes (32), empty and bad ones among them.
Tolerances as derived in test_decoder_attention_gpu."""
import math

import pytest
import torch

from test_decoder_attention_gpu import check_packed, make_packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("count", [31, 32, 33, 64, 70])
def test_many_sequences(count, causal):
    from fastdeploy_b200.ops.decoder import CausalAttention
    lens = [(37 * i + 11) % 90 if i % 7 else 0 for i in range(count)]
    lens[-1] = 300
    q, k, v, start, length = make_packed(lens, [i % 3 for i in range(count)], 4, 2, 64, torch.bfloat16, 11)
    out = torch.full((q.shape[0], 256), 7.0, dtype=torch.bfloat16, device="cuda")
    att = CausalAttention(q, k, v, out, heads=4, kv_heads=2, seq_start=start, seq_len=length, causal=causal, max_len=300)
    att.launch()
    att.status.check()
    check_packed(q, k, v, out, start.tolist(), lens, 4, 2, 64, 1 / math.sqrt(64), causal, 7.0)


@pytest.mark.parametrize("bad_start,bad_len", [(0, 301), (-4, 5), (3, -2), (590, 20)])
def test_a_bad_sequence_is_reported_whatever_empty_ones_follow(bad_start, bad_len):
    """Empty sequences may start anywhere, also outside the buffer; one in the same place of the next 32 hides nothing."""
    from fastdeploy_b200.ops.decoder import CausalAttention
    count = 70
    starts, lens = [-1] * count, [0] * count
    starts[2], lens[2] = bad_start, bad_len
    good = {40: (10, 200), 69: (300, 33)}
    for i, (st, n) in good.items():
        starts[i], lens[i] = st, n
    q, k, v, _, _ = make_packed([600], [0], 2, 1, 64, torch.float16, 12)
    out = torch.full((q.shape[0], 128), 7.0, dtype=torch.float16, device="cuda")
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, lens)]
    att = CausalAttention(q, k, v, out, heads=2, kv_heads=1, seq_start=ints[0], seq_len=ints[1], max_len=300)
    att.launch()
    with pytest.raises(RuntimeError, match="bad shape"):
        att.status.check()
    check_packed(q, k, v, out, [s for s, _ in good.values()], [n for _, n in good.values()], 2, 1, 64, 0.125, True, 7.0)
    ints[1][2] = 0
    out.fill_(7.0)
    att.launch()
    att.status.check()
    check_packed(q, k, v, out, [s for s, _ in good.values()], [n for _, n in good.values()], 2, 1, 64, 0.125, True, 7.0)
