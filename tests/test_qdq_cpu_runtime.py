"""A quantised export on the CPU keeps its quantise / dequantise pairs: values round and saturate as the model says. All numbers
are small multiples of powers of two, so that every sum is exact in fp32 and results have to be equal."""
import numpy as np
import pytest


@pytest.mark.parametrize("spread", [1.0, 6.0])       # inside the range, and far outside of it
def test_cpu_runtime_rounds_and_saturates_like_the_exported_graph(tmp_path, spread):
    import fastdeploy_b200 as fd
    from fastdeploy_b200.importer.onnx_format import save_onnx
    from fastdeploy_b200.ir.graph import Graph
    rng = np.random.default_rng(0)
    g = Graph("m", 17)
    g.add_input("x", "float32", [8, 16])
    step = np.float32(1 / 32)
    w = [(rng.integers(-8, 9, (16, 16)) / 16).astype(np.float32) for _ in range(2)]
    bias = (rng.integers(-16, 17, 16) / 16).astype(np.float32)
    for name, value in (("s", step), ("z", np.int8(0)), ("w0", w[0]), ("w1", w[1]), ("b", bias)):
        g.add_initializer(name, np.asarray(value))
    cur = "x"
    for i in range(2):
        g.add_node("QuantizeLinear", [cur, "s", "z"], [f"q{i}"])
        g.add_node("DequantizeLinear", [f"q{i}", "s", "z"], [f"d{i}"])
        g.add_node("MatMul", [f"d{i}", f"w{i}"], [f"m{i}"])
        cur = f"m{i}"
        if i == 0:
            g.add_node("Add", ["m0", "b"], ["a"])
            g.add_node("Relu", ["a"], ["r"])
            cur = "r"
    g.add_output("m1", "float32", [8, 16])
    x = (rng.uniform(-spread, spread, (8, 16)) * 64).round().astype(np.float32) / 64

    def fake(v):
        return np.clip(np.rint(v.astype(np.float64) * 32), -128, 127) / 32
    want = fake(np.maximum(fake(x) @ w[0] + bias, 0)) @ w[1]
    path = str(tmp_path / "m.onnx")
    open(path, "wb").write(save_onnx(g))
    opt = fd.RuntimeOption()
    opt.set_model_path(path, model_format=fd.ModelFormat.ONNX)
    got = np.asarray(fd.Runtime(opt).infer({"x": x})[0])
    assert np.array_equal(got, want.astype(np.float32))
