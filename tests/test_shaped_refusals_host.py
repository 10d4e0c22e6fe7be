"""Refusals of the shaped token attention that guard against a call that runs as another, on
the CPU.  No kernel runs."""
import pytest
import torch


@pytest.mark.parametrize("cap", [1e-46, 5e-324, 7e-46])
def test_a_cap_that_float32_takes_for_none(cap):
    """Caps below half of Float32's least number (1.4e-45) would arrive as 0, which is no cap."""
    from circulant_attention import tokens as T
    q = torch.zeros(2, 9, 32)
    with pytest.raises(AssertionError, match="is 0 in Float32"):
        T._shape(q, 2, 4, cap, None, None)


def test_no_cap_and_least_caps():
    """0 and None are no cap; what Float32 holds goes to the C entry, which has bounds of its own."""
    from circulant_attention import tokens as T
    q = torch.zeros(2, 9, 32)
    slopes = torch.zeros(4)
    for cap in (0, 0.0, None, False):
        assert T._shape(q, 2, 4, cap, slopes, None).args()[0] == 0.0
    assert T._shape(q, 2, 4, 2e-45, None, None).args()[0] == 2e-45
