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


def test_tables_and_rows_of_the_cache():
    from uwc_amd import kv, pages
    cache = kv.new_cache(4, 2, 64, 16, "cpu")
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    cos = torch.zeros((4, 64))
    q = torch.zeros((2, 512), dtype=torch.bfloat16)
    wide = torch.empty((2, MORE), dtype=torch.int32, device="meta")
    meta = tuple(x.to("meta") for x in cache)
    m = lambda x: x.to("meta")  # noqa: E731
    for f in (lambda: pages.fork([meta], wide, m(i(2)), m(i(4)), m(i(2))), lambda: pages.compact([meta], wide, m(i(4))),
              lambda: kv.append(meta, m(q), wide, m(i(2)), m(cos), m(cos)), lambda: kv.attend(meta, m(q).view(2, 8, 64), wide, m(i(2))),
              lambda: kv.read(meta, wide, m(i(2)), m(i(3)), 1)):
        with pytest.raises(AssertionError, match=r"table .*2\^31"):
            f()
    many = m(q)[:1].expand(MORE, 512)
    for f in (lambda: kv.append(meta, many, m(i(2, 3)), m(i(2)), m(cos), m(cos), cu=m(i(3))),
              lambda: kv.attend(meta, many.view(MORE, 8, 64), m(i(2, 3)), m(i(2)), cu=m(i(3)))):
        with pytest.raises(AssertionError, match=r"rows.*2\^31"):
            f()
