"""Batches whose pages cannot be counted in 32 bits are refused on the host (fake,
never dereferenced pointers; no GPU needed)."""
import pytest

from test_span_refusals import SHARED, UNSUPPORTED, WINDOW, refused


def test_window_decode_counts_the_pages_that_a_row_may_see(native):
    refused(native.tvp_paged_window_decode_attention, WINDOW, [
        ({"batch": 1 << 5, "stride": 1 << 26, "window": 1 << 30, "sinks": 0}, UNSUPPORTED),
        ({"batch": 33, "stride": 1 << 26, "window": 1 << 30, "sinks": 1 << 30}, UNSUPPORTED),
        ({"batch": 2 ** 31 - 1, "stride": 2, "window": 64}, UNSUPPORTED),
        ({"batch": 1 << 29, "stride": 1 << 20, "window": 33, "sinks": 1}, UNSUPPORTED)])


@pytest.mark.parametrize("groups", [0, 1])
def test_shared_prefix_counts_the_tables_pages(native, groups):
    refused(native.tvp_paged_shared_prefix_decode_attention, SHARED, [
        ({"batch": 1 << 5, "stride": 1 << 26, "groups": groups}, UNSUPPORTED),
        ({"batch": 2 ** 31 - 1, "stride": 2, "groups": groups}, UNSUPPORTED)])
