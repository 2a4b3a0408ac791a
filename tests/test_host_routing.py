"""The routing order's scratch, whose size callers may have written down."""

import pytest

import pearl_b200 as pg


@pytest.mark.parametrize("slots,blocks", [(0, 0), (1, 1), (8192, 1), (8193, 2), (131072, 16)])
def test_scratchpad_bytes(slots, blocks):
    assert pg.moe.get_build_routing_data_scratchpad_bytes(slots) == blocks * 256 * 4
