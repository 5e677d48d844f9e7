"""Example bank, without a GPU: arguments at the ends of what the kernels take."""
import pytest
import torch

from test_bank_host import _calls, _struct


@pytest.mark.parametrize("scale", [2.36e38, 2.9e38, 3.4e38])
def test_scales_whose_power_of_two_form_is_not_finite_are_refused(scale):
    """The kernels multiply logits by scale * log2 e, which is past float32's range from 2.3587e38 on."""
    calls, lib = _calls(_struct(), scale=scale)
    for name in ("attend", "pages"):
        assert calls[name]() == -1 and b"scale" in lib.gpsr_last_error()


@pytest.mark.parametrize("rows", [2 ** 31, 2 ** 32 + 5])
def test_more_rows_than_a_call_can_count_are_refused(rows):
    """The library counts rows in 32 bits: 2^32 + 5 of them would have been 5.  One row repeated, so that they need no memory."""
    from super_resolution_amd import _lib, ops
    q = torch.zeros(64).expand(1, rows, 1, 64)
    with pytest.raises(_lib.GpsrError, match="rows"):
        ops._strided(q, 1, None, 64, q.get_device(), "bank_attend: q")
    assert ops._strided(q[:, :7], 1, None, 64, q.get_device(), "bank_attend: q")[1] == 2
    table = torch.empty(1, rows, dtype=torch.int32, device="meta")
    with pytest.raises(_lib.GpsrError, match="pages"):
        ops._bank_index(table, (torch.zeros(1, dtype=torch.int32),), -1, "bank_attend")


def test_a_bank_without_heads_is_refused():
    """Before the query heads are divided by its number of heads."""
    from super_resolution_amd import _lib, ops
    u8, f32 = (lambda *s: torch.zeros(s, dtype=torch.uint8)), (lambda *s: torch.zeros(s))
    for heads in (0, 1):
        bank = ops.Bank(u8(2, heads, 16, 32), u8(2, heads, 16, 2), u8(2, heads, 16, 32), u8(2, heads, 16, 2), f32(2, heads, 16), f32(2, heads, 64))
        if heads:
            assert ops._bank(bank, -1)[1:] == (1, 64)
        else:
            with pytest.raises(_lib.GpsrError, match="heads"):
                ops._bank(bank, -1)
