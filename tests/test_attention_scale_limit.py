"""The largest scale of attention: checked before the device is touched."""
import pytest

from test_block_operators_refusals import attention_parts, call_attention, refused


@pytest.mark.parametrize("backward", [False, True])
def test_scales_whose_exponents_leave_f32_are_refused(backward):
    _, good = attention_parts(backward)
    for scale in (2.4e38, 3.4e38):                          # times log2(e): beyond the largest f32
        refused(lambda: call_attention({**good, "scale": scale}), "positive")
    for scale in (2.0 ** 127, 1.0, 1e-30):
        refused(lambda: call_attention({**good, "scale": scale}), "null context")
