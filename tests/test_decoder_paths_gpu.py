"""Uses of the generating models' operators that their own tests leave out: rows further than 2^31 elements apart, outputs over the
queries, two captured plans at once, and a decoder layer through Runtime and the plan runner. Tolerances as derived in the
operators' own tests; the last one compares bits."""
import numpy as np
import pytest
import torch

from test_decoder_attention_gpu import check_packed, check_prefix, make_packed, make_prefix
from test_linear_int4_gpu import check, dense, make
from test_plan_file_gpu import _roundtrip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def far():
    """A buffer of more than 2^31 elements; rows(count, width, pitch, column) views it."""
    buf = torch.empty(40 * ((1 << 26) + 8), dtype=torch.float16, device="cuda")

    def rows(shape, strides, at):
        assert at + sum((n - 1) * s for n, s in zip(shape, strides)) < buf.numel()
        t = torch.as_strided(buf, shape, strides, at)
        t.copy_(torch.randn(shape, generator=torch.Generator().manual_seed(at)))
        return t
    yield rows
    del buf


def test_far_prompt_rows(far):
    from fastdeploy_b200.ops.decoder import CausalAttention
    pitch, n = (1 << 28) + 8, 9
    q, k, v, out = (far((n, w), (pitch, 1), at) for w, at in ((256, 0), (128, 256), (128, 384), (256, 512)))
    ints = [torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, n)]
    att = CausalAttention(q, k, v, out, heads=4, kv_heads=2, seq_start=ints[0], seq_len=ints[1])
    att.launch()
    att.status.check()
    check_packed(q, k, v, out, [0], [n], 4, 2, 64, 0.125, True, 7.0)


def test_far_caches(far):
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    item, pitch = (1 << 31) + 8, (1 << 28) + 8
    k, v = (far((2, 20, 128), (item, 128, 1), at) for at in (0, 4096))
    pk, pv = (far((9, 128), (pitch, 1), at) for at in (8192, 8320))
    q, out = (far((2, 256), (item, 1), at) for at in (9000, 9256))
    lens = [20, 13]
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    att = SharedPrefixAttention(q, pk, pv, k, v, out, heads=4, kv_heads=2, seq_len=length)
    att.launch()
    att.status.check()
    check_prefix(q, pk, pv, k, v, lens, out, 4, 2, 64, 0.125)
    # one item whose own rows are far apart
    fk, fv = (far((1, 9, 128), (8, pitch, 1), at) for at in (20000, 20128))
    one = torch.full((1,), 9, dtype=torch.int32, device="cuda")
    att = SharedPrefixAttention(q[:1], None, None, fk, fv, out[:1], heads=4, kv_heads=2, seq_len=one)
    att.launch()
    check_prefix(q[:1], None, None, fk, fv, [9], out[:1], 4, 2, 64, 0.125)


@pytest.mark.parametrize("m,pitch,k", [(9, (1 << 28) + 8, 128), (9, (1 << 28) + 3, 130), (40, (1 << 26) + 8, 128), (40, (1 << 26) + 5, 130)])
def test_far_rows_of_a_product(far, m, pitch, k):
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
    _, q, s, z = make(m, 70, k, 32, True, torch.float16, torch.float16)
    x, y = (far((m, w), (pitch, 1), at) for w, at in ((k, 0), (70, 200)))
    op = Int4Linear(x, pack_linear_weight_int4(q, s, z, k=k), y)
    op.launch()
    op.status.check()
    check(y, x, dense(q, s, z, k), None)


def test_outputs_over_the_queries():
    """A query tile, or an item's heads, are read before the same CTA or a later launch writes there."""
    from fastdeploy_b200.ops.decoder import CausalAttention, SharedPrefixAttention
    lens = [700, 33, 260]
    q, k, v, start, length = make_packed(lens, [0, 2, 0], 6, 2, 64, torch.bfloat16, 31, junk=7.0)
    was = q.clone()
    CausalAttention(q, k, v, q, heads=6, kv_heads=2, seq_start=start, seq_len=length, max_len=700).launch()
    check_packed(was, k, v, q, start.tolist(), lens, 6, 2, 64, 0.125, True, 7.0)
    for case in ((70, 300, 40, [i % 41 for i in range(70)], 12, 2, 64), (2, 300, 3000, [3000, 700], 40, 2, 128)):
        q, pk, pv, k, v, length = make_prefix(case, torch.float16, 32)
        was = q.clone()
        heads, hk, d = case[4:]
        SharedPrefixAttention(q, pk, pv, k, v, q, heads=heads, kv_heads=hk, seq_len=length).launch()
        check_prefix(was, pk, pv, k, v, case[3], q, heads, hk, d, d ** -0.5)


def test_two_captured_plans_at_once():
    from fastdeploy_b200.ops.decoder import SharedPrefixAttention
    case = (3, 500, 3000, [3000, 0, 1500], 8, 2, 128)
    runs = []
    for seed in (41, 42):
        q, pk, pv, k, v, length = make_prefix(case, torch.bfloat16, seed)
        out = torch.zeros(3, 1024, dtype=torch.bfloat16, device="cuda")
        att = SharedPrefixAttention(q, pk, pv, k, v, out, heads=8, kv_heads=2, seq_len=length)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                att.launch()
        runs.append((graph, torch.cuda.Stream(), att, q, pk, pv, k, v, out))
    for _ in range(5):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for graph, stream, att, q, pk, pv, k, v, out in runs:
        att.status.check()
        check_prefix(q, pk, pv, k, v, case[3], out, 8, 2, 128, 128 ** -0.5)


@pytest.mark.parametrize("s,c", [(6, 96), (150, 100)])           # 100 columns: rows that the product copies to aligned ones
def test_decoder_layer_through_runtime_and_without_python(tmp_path, s, c):
    import fastdeploy_b200 as fd
    from fastdeploy_b200.importer.onnx_format import load_onnx, save_onnx
    from fastdeploy_b200.ir.graph import Graph
    from fastdeploy_b200.runtime.native_backend import build_plan
    rng = np.random.default_rng(5)
    b, heads, hk, d, group = 2, 4, 2, 24, 32
    g = Graph("layer", 23)
    g.add_input("x", "float32", [b, s, c])

    def nbits(x, y, n, k):
        q = rng.integers(0, 256, (n, -(-k // group), group // 2)).astype(np.uint8)
        g.add_initializer(y + "w", q)
        g.add_initializer(y + "s", (0.02 + 0.02 * rng.random((n, q.shape[1]))).astype(np.float16))
        g.add_node("MatMulNBits", [x, y + "w", y + "s"], [y], domain="com.microsoft", N=n, K=k, bits=4, block_size=group)
    for name, n in (("q", heads), ("k", hk), ("v", hk)):
        nbits("x", name, n * d, c)
    g.add_node("Attention", ["q", "k", "v"], ["a"], q_num_heads=heads, kv_num_heads=hk, is_causal=1)
    nbits("a", "y", c, heads * d)
    g.add_output("y", "float32", [b, s, c])
    path = str(tmp_path / "layer.onnx")
    open(path, "wb").write(save_onnx(g))
    x = (rng.standard_normal((b, s, c)) * 0.5).astype(np.float32)
    plan = build_plan(load_onnx(save_onnx(g)), {"x": [b, s, c]}, "cuda:0")
    feed = torch.from_numpy(x).cuda()
    _roundtrip(plan, {"x": feed}, tmp_path, "layer")
    want = plan.outputs["y"].logical().float().cpu().numpy()
    opt = fd.RuntimeOption()
    opt.set_model_path(path, model_format=fd.ModelFormat.ONNX)
    opt.use_gpu(0)
    rt = fd.Runtime(opt)
    for _ in range(2):
        got = np.asarray(rt.infer({"x": x})[0], np.float32)
        assert np.array_equal(got, want)
