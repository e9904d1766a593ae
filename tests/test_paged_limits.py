"""Ends of the paged operators' argument ranges (refused before a GPU is reached)."""

from test_native_build import built  # noqa: F401  (fixture)
from test_paged import _attend, lib  # noqa: F401  (fixture)


def test_scale_times_log2_e_has_to_be_a_number(lib):  # noqa: F811
    """The kernels take scale * log2(e): the largest fp32 over that is the last
    one accepted (and goes on to the next check, a workspace that is missing)."""
    most = 3.4028234663852886e38 / 1.4426950408889634
    for scale, want in ((most * 0.999999, 6), (most * 1.000001, 2), (3.4e38, 2), (1e-38, 6), (1e-45, 6)):
        assert _attend(lib, scale=scale, ws=None) == want, scale
