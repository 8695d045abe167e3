"""Which kernel form a 4-bit product takes, by its rows and the weight's size (a rule on sizes: no GPU needed)."""
import pytest
import torch

from fastdeploy_b200.ops.linear_int4 import Int4Weight, _tile_form

SMS = 148


def weight(n, k):
    return Int4Weight(torch.zeros(1, dtype=torch.uint8), torch.float16, False, n, k, 128)


@pytest.mark.parametrize("n,k", [(1, 1), (128, 8192), (4096, 4096), (28672, 8192)])
def test_every_form_is_taken_and_no_other(n, k):
    rows = [_tile_form(m, weight(n, k), SMS)[0] for m in range(1, 300)]
    assert rows == [0] * 16 + [32] * 16 + [64] * (299 - 32)


@pytest.mark.parametrize("m", [17, 32, 33, 64, 65, 1000])
@pytest.mark.parametrize("n,k", [(1, 1), (100, 130), (128, 100000), (4096, 4096), (28672, 8192)])
def test_pieces_of_k_fit_a_cluster_and_the_machine(m, n, k):
    rows, splits = _tile_form(m, weight(n, k), SMS)
    ctas = -(-n // 128) * -(-m // rows)
    assert 1 <= splits <= 8 and splits <= -(-k // 128)
    assert splits == 1 or splits * ctas <= SMS
