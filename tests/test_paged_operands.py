"""What the operators over a paged cache refuse of operands that a kernel could not read, before anything touches a device: scales whose steps of log2 are not finite, arrays of 32-bit
values that are not aligned to them."""
import pytest

from test_paged_refusals import A, append_of, attn_of, cache_of, p, refused, reorder_of, select_of  # noqa: F401


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scales_beyond_the_range_of_their_logarithm(p, scale):
    refused(attn_of(p, scale=scale), "not finite")


@pytest.mark.parametrize("name", ["pos", "seq", "rope"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_append_operands_of_32_bits(p, name, off):
    refused(append_of(p, **{name: A + off}), "aligned to 4 bytes")


@pytest.mark.parametrize("name", ["lens", "shared", "group_first", "sinks"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_attention_operands_of_32_bits(p, name, off):
    refused(attn_of(p, **{name: A + off}), "aligned to 4 bytes")


@pytest.mark.parametrize("off", [1, 2, 3])
def test_tables(p, off):
    refused(append_of(p, cache_of(p, tables=A + off)), "aligned to 4 bytes")
    refused(attn_of(p, cache_of(p, tables=A + off)), "aligned to 4 bytes")


@pytest.mark.parametrize("name", ["scores", "out_scores", "out_tokens", "out_parents"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_choice_operands_of_32_bits(p, name, off):
    apart = dict(scores=2 * A, out_scores=3 * A, out_tokens=4 * A, out_parents=5 * A, workspace=(8 * A, 1 << 19))
    apart[name] += off
    refused(select_of(p, **apart), "aligned to 4 bytes")


@pytest.mark.parametrize("name,at", [("parents", A), ("tables_in", 2 * A), ("tables_out", 3 * A), ("lens_in", 4 * A), ("lens_out", 5 * A), ("row_of", 6 * A)])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_reorder_operands_of_32_bits(p, name, at, off):
    refused(reorder_of(p, **{name: at + off}), "aligned to 4 bytes")
