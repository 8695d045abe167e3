"""How ``MatMulNBits`` nodes become planned 4-bit products: which weights are laid out for which node, and which nodes are
left to the interpreter. The kernel objects are stand-ins that record what they were given (no GPU needed)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from fastdeploy_b200.ir.graph import Graph
from fastdeploy_b200.runtime import native_backend


class Recorder:
    """The part of a plan builder that the lowering uses."""

    def __init__(self, graph, shapes, dtype=torch.float16):
        self.g, self.dtype, self.device = graph, dtype, torch.device("cpu")
        self.info = SimpleNamespace(shapes=shapes)
        self.packed, self.vals, self.launched = {}, {}, []
        self.plan = SimpleNamespace(add_native=lambda op, node: None, status=None)

    def rows_view(self, name, rows, cols):
        return torch.zeros(rows, cols, dtype=self.dtype)

    def const_f32(self, name):
        return torch.from_numpy(self.g.initializers[name])


@pytest.fixture
def recorded(monkeypatch):
    """Runs the lowering over a graph's nodes: (result, weight given to the product) per node."""
    from fastdeploy_b200.ops import linear_int4
    products = []

    class Product:
        def __init__(self, x, weight, y, **kw):
            products.append(weight)

        def launch(self):
            pass
    monkeypatch.setattr(linear_int4, "pack_linear_weight_int4",
                        lambda q, s, z=None, *, k=None: (q.clone(), s.clone(), None if z is None else z.clone(), k))
    monkeypatch.setattr(linear_int4, "Int4Linear", Product)

    def run(graph, shapes):
        rec = Recorder(graph, shapes)
        results = [native_backend._lower_MatMulNBits(rec, node) for node in graph.nodes]
        return results, products, rec
    return run


N, K = 4, 64


def shared_weight_graph(*nodes):
    """Nodes (scales, zeros, block size) that share one ``B`` initializer of N x K."""
    g = Graph("m", 21)
    g.add_input("x", "float32", [3, K])
    g.add_initializer("w", np.arange(N * K // 2, dtype=np.uint8).reshape(N, -1))
    for i, (s, z, group) in enumerate(nodes):
        groups = K // group
        g.add_initializer(f"s{i}", np.full((N, groups), s, np.float32))
        if z is not None:
            g.add_initializer(f"z{i}", np.full((N, (groups + 1) // 2), z, np.uint8))
        g.add_node("MatMulNBits", ["x", "w", f"s{i}", f"z{i}" if z is not None else ""], [f"y{i}"], domain="com.microsoft",
                   N=N, K=K, bits=4, block_size=group)
    return g


def test_nodes_that_share_the_weight_keep_their_own_scales_zero_points_and_groups(recorded):
    forms = [(1.0, None, 32), (2.0, None, 32), (1.0, 0x77, 32), (1.0, 0x99, 32), (1.0, None, 16)]
    results, products, _ = recorded(shared_weight_graph(*forms), {"x": [3, K]})
    assert results == [None] * len(forms)
    for (s, z, group), (q, scales, zeros, k) in zip(forms, products):
        assert q.shape == (N, K // group, group // 2) and k == K
        assert (scales == s).all()
        assert zeros is None if z is None else (zeros == z).all()


def test_a_weight_that_two_equal_nodes_share_is_laid_out_once(recorded):
    g = shared_weight_graph((1.0, 0x77, 32))
    g.add_node("MatMulNBits", list(g.nodes[0].inputs), ["again"], domain="com.microsoft", N=N, K=K, bits=4, block_size=32)
    results, products, _ = recorded(g, {"x": [3, K]})
    assert results == [None, None] and products[0] is products[1]


def test_a_computed_bias_is_left_to_the_interpreter(recorded):
    g = shared_weight_graph((1.0, None, 32))
    g.add_initializer("b0", np.ones(N, np.float32))
    nodes = [["x", "w", "s0", "", "", b] for b in ("b0", "b")]
    g.nodes.clear()
    g.add_input("b", "float32", [N])
    for i, ins in enumerate(nodes):
        g.add_node("MatMulNBits", ins, [f"y{i}"], domain="com.microsoft", N=N, K=K, bits=4, block_size=32)
    results, products, _ = recorded(g, {"x": [3, K]})
    assert results == [None, False] and len(products) == 1


@pytest.mark.parametrize("shape", [[K], [0, K], [2, 0, K]])
def test_vectors_and_empty_inputs_are_left_to_the_interpreter(recorded, shape):
    results, products, _ = recorded(shared_weight_graph((1.0, None, 32)), {"x": shape})
    assert results == [False] and not products


def test_broadcast_rows_are_copied_apart(monkeypatch, recorded):
    """An Expand is a view whose rows share memory; the product wants them one behind the other."""
    from fastdeploy_b200.ops import linear_int4
    seen = []
    row = torch.arange(K).to(torch.float16)
    product = linear_int4.Int4Linear
    monkeypatch.setattr(linear_int4, "Int4Linear", lambda x, *a, **kw: seen.append(x.clone()) or seen.append(x.stride(0)) or product(x, *a, **kw))
    monkeypatch.setattr(Recorder, "rows_view", lambda self, name, rows, cols: row.expand(rows, cols))
    monkeypatch.setattr(Recorder, "copy", lambda self, src, dst, *a: dst.copy_(src), raising=False)
    results, _, _ = recorded(shared_weight_graph((1.0, None, 32)), {"x": [5, K]})
    assert results == [None] and torch.equal(seen[0], row.expand(5, K)) and seen[1] >= K


@pytest.mark.parametrize("shape", [[0, 5, 16], [2, 0, 16]])
@pytest.mark.parametrize("scale", [0.25, None])
def test_empty_attention_and_odd_scales_are_left_to_the_interpreter(shape, scale):
    for value in ([scale] if scale else [float("nan"), float("inf"), 0.0, -1.0]):
        g = Graph("m", 23)
        g.add_node("Attention", ["q", "k", "v"], ["y"], q_num_heads=2, kv_num_heads=2, scale=value)
        rec = Recorder(g, dict.fromkeys("qkv", shape if scale else [2, 5, 16]))
        assert native_backend._lower_standard_attention(rec, g.nodes[0]) is False
