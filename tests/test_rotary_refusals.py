"""A rotation that no call could use is refused when it is made."""
import pytest

from magpie_tts_rt_b200 import rotary


@pytest.mark.parametrize("eps", [1e39, float("inf"), -1.0, float("nan")])
def test_eps_that_single_precision_does_not_hold(eps):
    with pytest.raises(ValueError):
        rotary.Rotation(64, eps=eps, device="cpu")


@pytest.mark.parametrize("eps", [0.0, 1e-60, 1e-6, 3.4e38])
def test_eps_of_single_precision(eps):
    assert rotary.Rotation(64, eps=eps, device="cpu").eps == eps
