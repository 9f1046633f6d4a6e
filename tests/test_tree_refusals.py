"""Calls of the tree operators that are refused on the host for what a kernel would do with them."""
import pytest

from test_tree_abi import FAKE, attn


@pytest.mark.parametrize("B,pages,page_size,rc", [
    (1024, 1 << 22, 16, 1), (1024, (1 << 22) - 400, 16, 1), (1024, (1 << 22) - 4800, 16, 3), (32, 127, 1 << 24, 3),
    (33, 127, 1 << 24, 1), (1024, 1 << 21, 16, 3)])
def test_a_batch_of_more_tiles_than_a_run_can_count(fl, B, pages, page_size, rc):
    """A run is up to 1.0001 times all tiles and starts long, in 32 bits: with nearly 2^31 of them (and one
    workgroup a kv head) it would come out negative, and the merge would read slots that nobody wrote.
    Status 3: only the work is too small."""
    assert attn(fl, B=B, max_pages=pages, stride=pages, page_size=page_size, n_pages=8) == rc
    if rc == 1:
        assert b"max_pages" in fl._lib.lib().fl_last_error()
