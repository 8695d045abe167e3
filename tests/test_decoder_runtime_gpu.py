"""A decoder layer from an ONNX graph (4-bit projections, causal attention with grouped heads) as a native plan against the
fp32 interpreter."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("four_d", [False, True])
@pytest.mark.parametrize("causal", [1, 0])
def test_decoder_layer_plan(causal, four_d):
    from fastdeploy_b200.importer.onnx_format import load_onnx, save_onnx
    from fastdeploy_b200.ir.graph import Graph
    from fastdeploy_b200.ir.interp import Interpreter
    from fastdeploy_b200.runtime.native_backend import build_plan
    rng = np.random.default_rng(0)
    b, s, c, heads, hk, d, group = 2, 200, 96, 6, 2, 24, 32
    g = Graph("layer", 23)
    g.add_input("x", "float32", [b, s, c])
    dense = {}

    def nbits(x, y, n, k):
        q = rng.integers(0, 256, (n, -(-k // group), group // 2)).astype(np.uint8)
        scale = (0.02 + 0.02 * rng.random((n, q.shape[1]))).astype(np.float16)
        zero = rng.integers(0, 256, (n, (q.shape[1] + 1) // 2)).astype(np.uint8)
        for name, value in (("w", q), ("s", scale), ("z", zero)):
            g.add_initializer(y + name, value)
        g.add_node("MatMulNBits", [x, y + "w", y + "s", y + "z"], [y], domain="com.microsoft", N=n, K=k, bits=4, block_size=group)
        e = np.stack([q & 15, q >> 4], -1).reshape(n, -1)[:, :k].astype(np.float64)
        zz = np.stack([zero & 15, zero >> 4], -1).reshape(n, -1)[:, :q.shape[1]]
        dense[y] = (e - np.repeat(zz, group, 1)[:, :k]) * np.repeat(scale.astype(np.float64), group, 1)[:, :k]
    nbits("x", "q", heads * d, c)
    nbits("x", "k", hk * d, c)
    nbits("x", "v", hk * d, c)
    names = ["q", "k", "v"]
    attrs = dict(is_causal=causal, scale=0.05)
    if four_d:
        for i, (nm, n) in enumerate(zip(names, (heads, hk, hk))):
            shape = g.add_initializer(nm + "_shape", np.array([b, s, n, d], np.int64))
            g.add_node("Reshape", [nm, shape], [nm + "4"])
            g.add_node("Transpose", [nm + "4"], [nm + "t"], perm=[0, 2, 1, 3])
            names[i] = nm + "t"
        g.add_node("Attention", names, ["at"], **attrs)
        g.add_node("Transpose", ["at"], ["at4"], perm=[0, 2, 1, 3])
        shape = g.add_initializer("o_shape", np.array([b, s, heads * d], np.int64))
        g.add_node("Reshape", ["at4", shape], ["a"])
    else:
        g.add_node("Attention", names, ["a"], q_num_heads=heads, kv_num_heads=hk, **attrs)
    nbits("a", "y", c, heads * d)
    g.add_output("y", "float32", [b, s, c])
    g = load_onnx(save_onnx(g))
    x = (rng.standard_normal((b, s, c)) * 0.5).astype(np.float32)
    want = np.asarray(Interpreter(g).run({"x": x})["y"], np.float64)
    plan = build_plan(g, {"x": [b, s, c]}, "cuda:0")
    assert not [st.name for st in plan.steps if st.name.startswith("torch:")]
    plan.inputs["x"].t.copy_(torch.from_numpy(x).cuda())
    plan.run()
    torch.cuda.synchronize()
    plan.status.check()
    got = plan.outputs["y"].logical().float().cpu().numpy()
    # Half a step u = 2^-11 at x, at q / k / v, at the weights, at the attention's result and at y. With the layer's
    # largest magnitudes: dq of a projection, ds of a score, da of the attention (a weight moves by twice its score's error).
    u = 2.0 ** -11
    big = {n: np.abs(x.reshape(-1, c) @ dense[n].T).max() for n in ("q", "k", "v")}
    dp = {n: u * (np.abs(x.reshape(-1, c)) @ np.abs(dense[n].T)).max() + u * big[n] for n in big}
    ds = 0.05 * d * (big["q"] * dp["k"] + big["k"] * dp["q"] + dp["q"] * dp["k"])
    da = (2 * ds + u) * big["v"] + dp["v"] + u * big["v"]
    tol = np.abs(dense["y"]).sum(1).max() * da + u * np.abs(want).max() + 1e-4
    assert np.abs(got - want).max() <= tol, (np.abs(got - want).max(), tol)
    # the bound above adds every magnitude up; errors of independent roundings stay far below it
    assert np.linalg.norm(got - want) <= 0.02 * np.linalg.norm(want)
