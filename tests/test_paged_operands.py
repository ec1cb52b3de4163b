"""What the operators over a paged cache refuse of operands that a kernel could not read, before anything touches a device: scales whose steps of log2 are not finite, arrays of 32-bit
values that are not aligned to them."""
import pytest

from test_paged_refusals import A, append_of, attn_of, cache_of, p, refused, reorder_of, select_of  # noqa: F401


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scales_beyond_the_range_of_their_logarithm(p, scale):
    refused(attn_of(p, scale=scale), "not finite")
