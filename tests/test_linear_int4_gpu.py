"""Products with 4-bit weights against 64 bits.

Tolerance, element by element: q - z is exact, products of two 16-bit floats are exact in fp32, and the sums over K are in
fp32, so with A = sum |x| |q - z| s the sum is off by at most (K + 8) 2^-23 A (2^-23: the tensor core's adder may truncate);
the result is rounded once, by half a step of its type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def dense(qweight, scales, zero_points, k):
    n, groups, half = qweight.shape
    q = torch.stack([qweight & 15, qweight >> 4], -1).reshape(n, groups, half * 2).double()
    if zero_points is None:
        z = torch.full((n, groups), 8.0, dtype=torch.float64, device=q.device)
    else:
        z = torch.stack([zero_points & 15, zero_points >> 4], -1).reshape(n, -1)[:, :groups].double()
    return ((q - z[..., None]) * scales.double().reshape(n, groups)[..., None]).reshape(n, -1)[:, :k]


def check(y, x, w, bias):
    u = torch.finfo(y.dtype).eps / 2
    want = x.double() @ w.T + (0 if bias is None else bias.double())
    a = x.double().abs() @ w.abs().T + (0 if bias is None else bias.double().abs())
    tol = a * (x.shape[1] + 8) * 2 ** -23 + u * want.abs() + 2 ** -25
    diff = (y.double() - want).abs()
    assert (diff <= tol).all(), (diff.max().item(), (diff / tol).max().item())


def make(m, n, k, group, zero, dtype, scale_dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    q = torch.randint(0, 256, (n, groups, group // 2), generator=gen, dtype=torch.uint8).cuda()
    s = (0.01 + 0.02 * torch.rand(n, groups, generator=gen)).to(scale_dtype).cuda()
    z = torch.randint(0, 256, (n, (groups + 1) // 2), generator=gen, dtype=torch.uint8).cuda() if zero else None
    x = torch.randn(m, k, generator=gen).to(dtype).cuda()
    return x, q, s, z


CASES = [
    # m, n, k, group, zero points, bias
    (1, 1, 1, 16, False, False),
    (1, 16, 128, 128, False, True),
    (1, 768, 768, 32, False, True),
    (2, 17, 130, 16, True, False),
    (3, 100, 1000, 64, True, True),
    (8, 333, 257, 32, True, False),
    (9, 64, 512, 256, True, True),
    (16, 200, 776, 16, False, False),
    (17, 4099, 384, 128, True, False),
    (33, 48, 2048, 32, True, True),
    (64, 500, 1024, 256, False, True),
    (65, 129, 640, 64, True, False),
    (200, 80, 96, 16, True, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_int4_linear(case, dtype):
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
    m, n, k, group, zero, use_bias = case
    for scale_dtype in (dtype, torch.float32):
        x, q, s, z = make(m, n, k, group, zero, dtype, scale_dtype)
        bias = torch.randn(n, device="cuda") if use_bias else None
        packed = pack_linear_weight_int4(q, s, z, k=k)
        y = torch.full((m, n + 3), 7.0, dtype=dtype, device="cuda")
        op = Int4Linear(x, packed, y[:, :n], bias=bias)
        op.launch()
        check(y[:, :n], x, dense(q, s, z, k), bias)
        assert (y[:, n:] == 7.0).all()


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("pitch", [512, 515, 520])
def test_int4_linear_strided_rows(offset, pitch):
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
    m, n, k = 5, 90, 500
    _, q, s, z = make(m, n, k, 32, True, torch.bfloat16, torch.bfloat16)
    buf = torch.full((m * pitch + 64,), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (m, k), (pitch, 1), offset)
    x.copy_(torch.randn(m, k))
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    Int4Linear(x, pack_linear_weight_int4(q, s, z, k=k), y).launch()
    check(y, x, dense(q, s, z, k), None)


def test_quantised_weight_is_within_half_a_step():
    from fastdeploy_b200.ops.linear_int4 import linear_int4, pack_linear_weight_int4, quantize_groups_int4
    torch.manual_seed(3)
    w = torch.randn(70, 300, device="cuda")
    x = torch.randn(4, 300, device="cuda").half()
    for symmetric in (True, False):
        q, s, z = quantize_groups_int4(w, 64, symmetric)
        back = dense(q, s, z, 300)
        step = s.repeat_interleave(64, 1)[:, :300]
        # half a step, and with zero points half a step more where rounding the zero point cuts the range's end
        assert ((back - w).abs() <= step * (0.5 if symmetric else 1.0) + 1e-6).all()
        check(linear_int4(x, pack_linear_weight_int4(q, s, z, k=300)), x, back, None)


def test_plans_of_one_kernel_with_different_shared_memory():
    """A later plan that needs less shared memory leaves an earlier one launchable."""
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
    plans = []
    for zero, scale_dtype in ((False, torch.bfloat16), (True, torch.float32), (False, torch.bfloat16)):
        x, q, s, z = make(40, 130, 512, 16, zero, torch.bfloat16, scale_dtype)
        y = torch.empty(40, 130, dtype=torch.bfloat16, device="cuda")
        plans.append((Int4Linear(x, pack_linear_weight_int4(q, s, z), y), x, y, dense(q, s, z, 512)))
    for op, x, y, w in plans:
        op.launch()
        op.status.check()
        check(y, x, w, None)
