"""w4.quantize of matrices in 64 bits takes the nearest values of the numbers as they are, not of their roundings to 32 (no GPU needed)."""
import pytest
import torch

import w4_reference as R


def test_numbers_next_to_a_tie():
    from uwc_amd import w4
    tiny = 2.0 ** -40  # fp32 rounds it away
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    w = torch.zeros((1, 32), dtype=torch.float64)
    w[0, :7], w[0, 7:14], w[0, 14:21], w[0, 31] = ties * (1 - tiny), ties * (1 + tiny), -ties * (1 + tiny), 6
    v = w4.values(*w4.quantize(w), torch.float64)[0]
    up = [0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    assert v[:7].tolist() == [0.0] + up[:-1] and v[7:14].tolist() == up and v[14:21].tolist() == [-u for u in up]


def test_a_largest_number_below_a_power_of_two():
    from uwc_amd import w4
    w = torch.zeros((1, 32), dtype=torch.float64)
    w[0, 0], w[0, 1] = 8 * (1 - 2.0 ** -50), 0.5
    codes, scales = w4.quantize(w)
    assert scales.item() == 127 and w4.values(codes, scales)[0, :2].tolist() == [6.0, 0.5]


def test_numbers_below_32_bits_and_past_them():
    from uwc_amd import w4
    w = torch.zeros((2, 32), dtype=torch.float64)
    w[0, 0], w[1, 0], w[1, 1] = 1e-300, 6 * 2.0 ** -127, -2.0 ** -127
    codes, scales = w4.quantize(w)
    assert scales.flatten().tolist() == [0, 0] and torch.equal(R.values(codes, scales)[1], w[1]) and not R.values(codes, scales)[0].any()
    for big in (1e39, 1e300, float("inf"), float("nan")):
        w[0, 0] = big
        with pytest.raises(AssertionError, match="w4.quantize"):
            w4.quantize(w)
