"""A plan of the generating models' operators made while its stream is still busy may be launched on any stream at once: its
workspace is ready when the constructor returns. Tolerances as derived in the operators' own tests."""
import pytest
import torch

from test_decoder_attention_gpu import check_packed, check_prefix, make_packed, make_prefix
from test_linear_int4_gpu import check, dense, make

pytestmark = pytest.mark.gpu


def poison_and_stall():
    """Small blocks that the allocator hands out again hold ones, and the current stream has half a second of work."""
    blocks = [torch.ones(n, dtype=torch.int32, device="cuda") for n in (1, 2, 16, 128, 128) for _ in range(40)]
    torch.cuda.synchronize()
    del blocks
    torch.cuda._sleep(10 ** 9)


def on_another_stream(op):
    side = torch.cuda.Stream()
    op.launch(side.cuda_stream)
    side.synchronize()


def test_split_own_keys():
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    case = (2, 70, 3000, [3000, 1234], 8, 2, 128)
    q, pk, pv, k, v, length = make_prefix(case, torch.bfloat16, 21)
    out = torch.zeros(2, 1024, dtype=torch.bfloat16, device="cuda")
    poison_and_stall()
    att = SharedPrefixAttention(q, pk, pv, k, v, out, heads=8, kv_heads=2, seq_len=length)
    assert att.own_o is not None
    on_another_stream(att)
    torch.cuda.synchronize()
    att.status.check()
    check_prefix(q, pk, pv, k, v, case[3], out, 8, 2, 128, 128 ** -0.5)


def test_prompt_status():
    """The report of a bad sequence is not wiped out by the plan's own set-up."""
    from fastdeploy_b200.ops.decoder import CausalAttention
    q, k, v, _, _ = make_packed([100], [0], 2, 2, 64, torch.float16, 22)
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 200], [100, 5])]
    out = torch.full((q.shape[0], 128), 7.0, dtype=torch.float16, device="cuda")
    poison_and_stall()
    att = CausalAttention(q, k, v, out, heads=2, seq_start=ints[0], seq_len=ints[1])
    on_another_stream(att)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bad shape"):
        att.status.check()
    check_packed(q, k, v, out, [0], [100], 2, 2, 64, 0.125, True, 7.0)


@pytest.mark.parametrize("m", [3, 40])
def test_unaligned_rows_of_a_product(m):
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
    x, q, s, z = make(m, 90, 130, 32, True, torch.bfloat16, torch.bfloat16)
    w = pack_linear_weight_int4(q, s, z, k=130)
    y = torch.zeros(m, 90, dtype=torch.bfloat16, device="cuda")
    poison_and_stall()
    op = Int4Linear(x, w, y)
    on_another_stream(op)
    torch.cuda.synchronize()
    on_another_stream(op)
    torch.cuda.synchronize()
    op.status.check()
    check(y, x, dense(q, s, z, 130), None)


def test_a_plan_made_during_a_capture():
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    case = (1, 0, 2000, [1999], 4, 2, 64)
    q, pk, pv, k, v, length = make_prefix(case, torch.float16, 23)
    out = torch.zeros(1, 256, dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att = SharedPrefixAttention(q, pk, pv, k, v, out, heads=4, kv_heads=2, seq_len=length)
        att.launch()
    for _ in range(2):
        out.zero_()
        graph.replay()
        att.status.check()
        check_prefix(q, pk, pv, k, v, case[3], out, 4, 2, 64, 0.125)
