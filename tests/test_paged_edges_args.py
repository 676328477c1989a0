"""Refusals at the ends of the paged operators' ranges, on the host before the
context is touched (no GPU)."""
import pytest

import cw
from test_paged_args import CTX, P, batch, pages, refused


@pytest.mark.parametrize("max_path", [(1 << 30) + 1, (1 << 31) - 1, -1])
def test_kv_accept_paths_longer_than_positions(max_path):
    """Steps of 64 nodes end before 2^31."""
    refused(cw.lib().cw_kv_accept(CTX, pages(), batch(), P, max_path, P, None), f"max_path={max_path}")
