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


def test_workspaces_behind_a_prefix():
    """One token of one sequence, a small window: alone it has one part, behind a prefix of what
    the table holds several; batches that fill the chip, and chunks, have no more for it."""
    from circulant_attention import _lib
    plain, shaped = _lib.lib.circatt_paged_workspace_bytes, _lib.lib.circatt_shaped_paged_workspace_bytes
    one = (3, 1, 1, 8, 8, 128, 32, 0, 16, 1024)
    assert plain(*one) == shaped(*one, 0) == 0
    assert shaped(*one, 1) >= 2 * 8 * 32 * (128 + 2) * 4      # two parts of eight blocks at least
    short = (3, 1, 1, 8, 8, 128, 32, 0, 16, 2)                # a table of 32 tokens: nothing to share
    assert shaped(*short, 1) == plain(*short) == 0
    for full in ((3, 64, 64, 8, 8, 128, 32, 0, 16, 1024), (3, 1024, 2, 32, 8, 128, 256, 0, 16, 512)):
        assert shaped(*full, 1) == plain(*full)
    assert shaped(3, 0, 1, 8, 8, 128, 32, 0, 16, 8, 1) == 0 and shaped(3, 1, 1, 8, 3, 128, 32, 0, 16, 8, 1) == -1
