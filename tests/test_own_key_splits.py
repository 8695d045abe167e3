"""How many pieces the own keys of a decoding step are cut into (a rule on sizes: no GPU needed)."""
import pytest

from fastdeploy_b200.ops.decoder import _own_splits

SMS = 148


@pytest.mark.parametrize("d,fit", [(8, 4), (64, 4), (72, 2), (128, 2)])      # CTAs whose rings an SM's shared memory holds
@pytest.mark.parametrize("ctas", [1, 3, 8, 100, 148, 149, 5000])
@pytest.mark.parametrize("own", [0, 1, 511, 512, 4096, 120000, 1 << 22])
def test_pieces_are_whole_and_run_at_once(own, ctas, d, fit):
    n = _own_splits(own, ctas, d, SMS)
    assert n >= 1
    if n > 1:
        assert own // n >= 256                  # a piece is worth its part
        assert n * ctas <= fit * SMS            # no second wave of pieces
    assert (own < 512) <= (n == 1)
