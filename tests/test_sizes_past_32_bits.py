"""Sizes that the C-ABI's 32-bit arguments do not hold are refused, not cut (no GPU needed)."""
import pytest
import torch

MORE = 2 ** 32 + 1  # one, if it were cut


def u8(*s):
    return torch.empty(s, dtype=torch.uint8, device="meta")


@pytest.mark.parametrize("fn", ["linear", "gated"])
def test_rows_and_outputs_of_4_bit_linears(fn):
    from uwc_amd import w4
    f = getattr(w4, fn)
    x = torch.zeros((1, 32), dtype=torch.bfloat16)
    codes, scales = torch.zeros((2, 16), dtype=torch.uint8), torch.zeros((2, 1), dtype=torch.uint8)
    for rows in (MORE, 2 ** 31):
        with pytest.raises(AssertionError, match=f"w4.{fn}: .*2\\^31"):
            f(x.expand(rows, 32), codes, scales)
    with pytest.raises(AssertionError, match=f"w4.{fn}: .*2\\^31"):
        f(x.to("meta"), u8(2 ** 32 + 2, 16), u8(2 ** 32 + 2, 1))
    with pytest.raises(AssertionError, match=f"w4.{fn}: .*2\\^31"):
        f(x.to("meta")[:, :1].expand(1, 2 ** 32 + 32), u8(2, 2 ** 31 + 16), u8(2, 2 ** 27 + 1))
