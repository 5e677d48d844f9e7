"""Example bank, without a GPU: arguments at the ends of what the kernels take."""
import pytest

from test_bank_host import _calls, _struct


@pytest.mark.parametrize("scale", [2.36e38, 2.9e38, 3.4e38])
def test_scales_whose_power_of_two_form_is_not_finite_are_refused(scale):
    """The kernels multiply logits by scale * log2 e, which is past float32's range from 2.3587e38 on."""
    calls, lib = _calls(_struct(), scale=scale)
    for name in ("attend", "pages"):
        assert calls[name]() == -1 and b"scale" in lib.gpsr_last_error()
