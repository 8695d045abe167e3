"""Shapes that the packing of 4-bit weights takes and refuses (checked before the device: no GPU needed)."""
import pytest
import torch

from fastdeploy_b200.ops.linear_int4 import pack_linear_weight_int4

N, GROUPS = 6, 4
Q = torch.zeros(N, GROUPS, 16, dtype=torch.uint8)


@pytest.mark.parametrize("scales,zeros", [((GROUPS, N), None), ((N * GROUPS // 2, 2), None), ((1, N * GROUPS), None),
                                          ((N, GROUPS), (GROUPS // 2, N)), ((N, GROUPS), (3, N * GROUPS // 6))])
def test_transposed_scales_or_zero_points_are_refused(scales, zeros):
    with pytest.raises(ValueError, match="are needed"):
        pack_linear_weight_int4(Q, torch.ones(scales), None if zeros is None else torch.zeros(zeros, dtype=torch.uint8))


@pytest.mark.parametrize("scales", [(N, GROUPS), (N * GROUPS,), (N, GROUPS, 1)])
@pytest.mark.parametrize("zeros", [None, (N, GROUPS // 2), (N * GROUPS // 2,)])
def test_flat_and_two_dimensional_forms_pass_the_shape_checks(scales, zeros):
    with pytest.raises(ValueError, match="run on a GPU"):
        pack_linear_weight_int4(Q, torch.ones(scales), None if zeros is None else torch.zeros(zeros, dtype=torch.uint8))
