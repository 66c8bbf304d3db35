"""More of what the serving entry points refuse or pass over before anything reaches a device (no GPU needed)."""

import pytest

from test_serving_ops_cpu import COPY, INVALID, call, with_args


@pytest.mark.parametrize("pairs", [(1 << 20) + 1, (1 << 31) - 1])
def test_copy_blocks_refuses_more_pairs_than_a_launch_can_check(rt, pairs):
    """Each pair is checked against all others: without a limit a call could keep the GPU busy for minutes."""
    rc, text = call(rt, "ttb_paged_copy_blocks", with_args(COPY, np=pairs, heads=1, bs=1, d=8))
    assert rc == INVALID and "2^20" in text, (rc, text)
