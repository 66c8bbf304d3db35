"""More of what the serving entry points refuse or pass over before anything reaches a device (no GPU needed)."""

import ctypes

import pytest

from test_serving_ops_cpu import COMMIT, COPY, DECODE, INVALID, N, SAMPLE, TREE, WINDOW, call, with_args


@pytest.mark.parametrize("pairs", [(1 << 20) + 1, (1 << 31) - 1])
def test_copy_blocks_refuses_more_pairs_than_a_launch_can_check(rt, pairs):
    """Each pair is checked against all others: without a limit a call could keep the GPU busy for minutes."""
    rc, text = call(rt, "ttb_paged_copy_blocks", with_args(COPY, np=pairs, heads=1, bs=1, d=8))
    assert rc == INVALID and "2^20" in text, (rc, text)


@pytest.mark.parametrize("nulls", [("q", "out"), ("q", "k", "v", "out")])
def test_a_prompt_without_queries_needs_no_addresses(rt, nulls):
    rc, text = call(rt, "ttb_sdpa_window", with_args(WINDOW, sq=0, **{n: N for n in nulls}))
    assert rc == 0, text


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_a_prompt_with_queries_and_keys_needs_addresses(rt, name):
    rc, text = call(rt, "ttb_sdpa_window", with_args(WINDOW, **{name: N}))
    assert rc == INVALID and "null" in text


@pytest.mark.parametrize("name,base,field,off", [
    *[("ttb_sdpa_window", WINDOW, f, 1) for f in ("q", "k", "v", "out")], ("ttb_sdpa_window", WINDOW, "lens", 2),
    ("ttb_sdpa_window_decode", DECODE, "table", 2), ("ttb_sdpa_window_decode", DECODE, "pos", 2),
    *[("ttb_sdpa_tree", TREE, f, 2) for f in ("table", "lens", "parents", "drafts")],
    *[("ttb_paged_commit_draft", COMMIT, f, 2) for f in ("table", "lens", "path", "plens")],
    *[("ttb_sample_logits", SAMPLE, f, 2) for f in ("x", "u", "t", "k", "p", "m", "out", "prob")]])
def test_addresses_that_split_an_element_are_refused(rt, name, base, field, off):
    """A load through such an address faults the GPU."""
    rc, text = call(rt, name, with_args(base, **{field: ctypes.c_void_p((1 << 20) + off)}))
    assert rc == INVALID and "aligned" in text, (rc, text)
