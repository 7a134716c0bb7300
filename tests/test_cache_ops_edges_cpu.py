"""Refusals of the operators around a long paged cache that need no GPU."""
import pytest

P = 4096   # an address that no call below gets to use


def _refused(name, args, text):
    from ssd_b200 import lib
    so = lib.load()
    assert len(args) == len(lib.SIGNATURES[name][1])
    assert getattr(so, name)(*args) < 0
    got = so.ssdk_last_error().decode()
    assert text in got, got


@pytest.mark.parametrize("scale", [2.4e38, -3e38])
def test_scales_past_32_bits_in_base_2(scale):
    """Scores are scaled by scale log2(e): where that is infinite a score of 0 would be NaN."""
    for q_len in (1, 40):
        _refused("ssdk_span_attn", [P * i for i in range(1, 8)] + [2, q_len, 4, 2, 64, 32, 2, 4, 16, 3, scale, None], "scale")
