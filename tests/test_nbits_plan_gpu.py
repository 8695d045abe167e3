"""``MatMulNBits`` nodes as native plans against 64 bits: nodes that share a weight, and a bias that the graph computes.

Tolerance: x (in 16 bits already) meets exact weights, sums over K are in fp32, and the result is rounded to 16 bits once: with
A = sum |x| |w| at most K 2^-23 A + 2^-11 |y|; the fp16 steps of the interpreter (scales and weights rounded, 2^-11 each, the
product's result and the sum with the bias once more each) add 2^-11 (3 A + |y|).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40])
def test_nodes_with_one_weight_and_a_computed_bias(rows):
    from fastdeploy_b200.ir.graph import Graph
    from fastdeploy_b200.runtime.native_backend import build_plan
    rng = np.random.default_rng(0)
    n, k = 24, 128
    w = rng.integers(0, 256, (n, k // 2)).astype(np.uint8)
    q = np.stack([w & 15, w >> 4], -1).reshape(n, k).astype(np.float64)
    g = Graph("m", 21)
    g.add_input("x", "float32", [rows, k])
    g.add_initializer("w", w)
    want = {}
    x = (rng.integers(-64, 65, (rows, k)) / 32).astype(np.float32)          # exact in 16 bits
    for i, (group, zero, bias) in enumerate(((32, None, None), (32, None, None), (32, 3, None), (64, None, None), (32, 3, "b"))):
        groups = k // group
        s = (rng.integers(1, 65, (n, groups)) / 1024).astype(np.float32)
        g.add_initializer(f"s{i}", s)
        z = np.full((n, groups), 8 if zero is None else zero)
        if zero is not None:
            g.add_initializer(f"z{i}", np.full((n, (groups + 1) // 2), zero * 17, np.uint8))
        ins = ["x", "w", f"s{i}", f"z{i}" if zero is not None else "", "", bias or ""]
        g.add_node("MatMulNBits", ins, [f"y{i}"], domain="com.microsoft", N=n, K=k, bits=4, block_size=group)
        g.add_output(f"y{i}", "float32", [rows, n])
        dense = (q - np.repeat(z, group, 1)) * np.repeat(s.astype(np.float64), group, 1)
        want[f"y{i}"] = (x.astype(np.float64) @ dense.T, np.abs(x).astype(np.float64) @ np.abs(dense).T)
    base = rng.integers(-8, 9, n).astype(np.float32)
    g.add_input("base", "float32", [n])
    g.nodes.insert(0, g.nodes.pop())                                          # its bias is made first
    two = g.add_initializer("two", np.array([2.0], np.float32))
    g.add_node("Mul", ["base", two], ["b"])
    g.nodes.insert(0, g.nodes.pop())
    want["y4"] = (want["y4"][0] + 2 * base, want["y4"][1])
    plan = build_plan(g, {"x": [rows, k], "base": [n]}, "cuda:0")
    assert sum(s.name.startswith("int4") for s in plan.steps) == 4
    plan.inputs["x"].t.copy_(torch.from_numpy(x))
    plan.inputs["base"].t.copy_(torch.from_numpy(base))
    plan.run()
    torch.cuda.synchronize()
    plan.status.check()
    for name, (y, a) in want.items():
        got = plan.outputs[name].logical().double().cpu().numpy()
        tol = k * 2.0 ** -23 * a + 2.0 ** -11 * (np.abs(y) + (3 * a + np.abs(y) if name == "y4" else 0)) + 2.0 ** -24
        assert (np.abs(got - y) <= tol).all(), (name, np.abs(got - y).max())


def test_expanded_values_feed_the_operators():
    """Rows that an Expand makes share memory; results are those of the graph with the values written out, bit for bit."""
    from fastdeploy_b200.ir.graph import Graph
    from fastdeploy_b200.runtime.native_backend import build_plan
    rng = np.random.default_rng(1)
    b, n, k, group, d = 5, 32, 64, 32, 16
    w = rng.integers(0, 256, (n, k // 2)).astype(np.uint8)
    s = (rng.integers(1, 65, (n, k // group)) / 1024).astype(np.float32)
    x, y = rng.standard_normal((1, 1, k)).astype(np.float32), rng.standard_normal((b, 1, n)).astype(np.float32)
    outs = []
    for expand in (True, False):
        g = Graph("m", 23)
        g.add_input("x", "float32", [1 if expand else b, 1, k])
        g.add_input("q", "float32", [b, 1, n])
        g.add_initializer("w", w), g.add_initializer("s", s)
        name = "x"
        if expand:
            g.add_node("Cast", ["x"], ["x16"], to=10)
            g.add_node("Expand", ["x16", g.add_initializer("shape", np.array([b, 1, k], np.int64))], ["wide"])
            name = "wide"
        g.add_node("MatMulNBits", [name, "w", "s"], ["p"], domain="com.microsoft", N=n, K=k, bits=4, block_size=group)
        kv = name
        g.add_node("Slice", [name] + [g.add_initializer(f"c{i}", np.array([v], np.int64)) for i, v in enumerate((0, n, 2))], ["kv"])
        kv = "kv"
        g.add_node("Attention", ["q", kv, kv], ["a"], q_num_heads=n // d, kv_num_heads=n // d)
        for o in "pa":
            g.add_output(o, "float32", [b, 1, n])
        plan = build_plan(g, {"x": [1 if expand else b, 1, k], "q": [b, 1, n]}, "cuda:0")
        names = [st.name for st in plan.steps]
        assert any(m.startswith("int4") for m in names) and "causal_attention" in names
        plan.inputs["x"].t.copy_(torch.from_numpy(x if expand else np.repeat(x, b, 0)))
        plan.inputs["q"].t.copy_(torch.from_numpy(y))
        plan.run()
        torch.cuda.synchronize()
        plan.status.check()
        outs.append({o: plan.outputs[o].logical().float().cpu() for o in "pa"})
    assert all(torch.equal(outs[0][o], outs[1][o]) for o in "pa")
    assert outs[0]["p"].abs().max() > 0 and outs[0]["a"].abs().max() > 0
