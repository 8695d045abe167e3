"""4-bit products of more rows than a grid dimension of 65535 holds, with rows that 16-byte loads can and cannot take.
Tolerance as derived in test_linear_int4_gpu."""
import pytest
import torch

from test_linear_int4_gpu import check, dense, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [65535, 65537, 200001])
@pytest.mark.parametrize("k,pitch", [(33, 33), (32, 41), (32, 32)])
def test_more_rows_than_a_grid_dimension(m, k, pitch):
    from fastdeploy_b200.ops.linear_int4 import Int4Linear, pack_linear_weight_int4
    x, q, s, z = make(m, 24, k, 16, True, torch.float16, torch.float16)
    rows = torch.zeros(m, pitch, dtype=torch.float16, device="cuda")
    rows[:, :k] = x
    x = rows[:, :k]
    y = torch.zeros(m, 24, dtype=torch.float16, device="cuda")
    op = Int4Linear(x, pack_linear_weight_int4(q, s, z, k=k), y)
    op.launch()
    op.status.check()
    check(y, x, dense(q, s, z, k), None)
