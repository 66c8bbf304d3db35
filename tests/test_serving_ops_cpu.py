"""What the serving entry points refuse, before anything reaches a device (no GPU needed: every refused call returns
from its argument checks)."""

import ctypes

import pytest

P = ctypes.c_void_p(1 << 20)      # a non-null, aligned address that nothing reads
ODD = ctypes.c_void_p((1 << 20) + 2)
N = ctypes.c_void_p(None)
INVALID, UNSUPPORTED = 2, 3
BF16, F32, I8 = 2, 0, 17


def call(rt, name, values):
    conv = []
    for v in values:
        conv.append(ctypes.c_float(v) if isinstance(v, float) else ctypes.c_int64(v) if isinstance(v, int) else v)
    return getattr(rt.lib, name)(*conv), rt.lib.ttb_last_error().decode()


def with_args(base, **kw):
    args = dict(base)
    assert set(kw) <= set(args)
    args.update(kw)
    return list(args.values())


WINDOW = dict(q=P, k=P, v=P, lens=N, out=P, dtype=BF16, batch=1, hq=4, hkv=2, sq=8, skv=8, d=64, qs=N, ks=N, vs=N, os=N, offset=0, window=4,
              sinks=0, scale=0.5, stream=N)
DECODE = dict(q=P, k=P, v=P, table=P, pos=P, out=P, dtype=BF16, batch=2, h=4, hkv=2, blocks=9, bs=16, pages=4, d=64, window=4, sinks=0, scale=0.5,
              ws=P, wsb=1 << 30, stream=N)
TREE = dict(q=P, kd=P, vd=P, k=P, v=P, table=P, lens=P, parents=P, drafts=N, out=P, dtype=BF16, batch=2, nodes=8, h=4, hkv=2, blocks=9, bs=16, pages=4,
            d=64, pu=2, window=0, sinks=0, scale=0.5, ws=P, wsb=1 << 30, stream=N)
SAMPLE = dict(x=P, u=P, t=N, k=N, p=N, m=N, out=P, prob=N, dtype=F32, rows=2, vocab=100, stride=100, ws=P, wsb=1 << 30, stream=N)
HOST2 = (ctypes.c_void_p * 2)(1 << 20, 1 << 21)
HOLE2 = (ctypes.c_void_p * 2)(1 << 20, None)
COPY = dict(caches=HOST2, n=2, pairs=P, np=3, dtype=BF16, blocks=9, heads=2, bs=16, d=64, stream=N)
COMMIT = dict(caches=HOST2, drafts=HOST2, n=2, table=P, lens=P, path=P, plens=P, dtype=BF16, users=2, nodes=4, heads=2, blocks=9, bs=16, pages=4, d=64,
              stream=N)


@pytest.mark.parametrize("name,base,bad,code", [
    ("ttb_sdpa_window", WINDOW, dict(q=N), INVALID), ("ttb_sdpa_window", WINDOW, dict(out=N), INVALID),
    ("ttb_sdpa_window", WINDOW, dict(hq=5), INVALID), ("ttb_sdpa_window", WINDOW, dict(batch=0), INVALID),
    ("ttb_sdpa_window", WINDOW, dict(window=0), INVALID), ("ttb_sdpa_window", WINDOW, dict(sinks=-1), INVALID),
    ("ttb_sdpa_window", WINDOW, dict(offset=-1), INVALID), ("ttb_sdpa_window", WINDOW, dict(offset=1 << 40), INVALID),
    ("ttb_sdpa_window", WINDOW, dict(sq=1 << 40), INVALID), ("ttb_sdpa_window", WINDOW, dict(scale=float("nan")), INVALID),
    ("ttb_sdpa_window", WINDOW, dict(dtype=I8), UNSUPPORTED), ("ttb_sdpa_window", WINDOW, dict(d=264), UNSUPPORTED),
    ("ttb_sdpa_window_decode", DECODE, dict(pos=N), INVALID), ("ttb_sdpa_window_decode", DECODE, dict(h=5), INVALID),
    ("ttb_sdpa_window_decode", DECODE, dict(window=0), INVALID), ("ttb_sdpa_window_decode", DECODE, dict(window=-3), INVALID),
    ("ttb_sdpa_window_decode", DECODE, dict(pages=0), INVALID), ("ttb_sdpa_window_decode", DECODE, dict(q=ODD), INVALID),
    ("ttb_sdpa_window_decode", DECODE, dict(table=N), INVALID), ("ttb_sdpa_window_decode", DECODE, dict(bs=1 << 28), INVALID),
    ("ttb_sdpa_window_decode", DECODE, dict(dtype=F32), UNSUPPORTED), ("ttb_sdpa_window_decode", DECODE, dict(d=96), UNSUPPORTED),
    ("ttb_sdpa_window_decode", DECODE, dict(scale=float("inf")), INVALID),
    ("ttb_sdpa_window_decode", DECODE, dict(pages=4000, blocks=9000, window=60000, wsb=64), INVALID),
    ("ttb_sdpa_window_decode", DECODE, dict(pages=4000, blocks=9000, window=60000, ws=N), INVALID),
    ("ttb_sdpa_tree", TREE, dict(parents=N), INVALID), ("ttb_sdpa_tree", TREE, dict(nodes=0), INVALID),
    ("ttb_sdpa_tree", TREE, dict(nodes=65), INVALID), ("ttb_sdpa_tree", TREE, dict(pu=3), INVALID),
    ("ttb_sdpa_tree", TREE, dict(window=-1), INVALID), ("ttb_sdpa_tree", TREE, dict(sinks=-1), INVALID),
    ("ttb_sdpa_tree", TREE, dict(kd=ODD), INVALID), ("ttb_sdpa_tree", TREE, dict(d=48), UNSUPPORTED),
    ("ttb_sdpa_tree", TREE, dict(pages=4000, blocks=9000, wsb=64), INVALID),
    ("ttb_sample_logits", SAMPLE, dict(x=N), INVALID), ("ttb_sample_logits", SAMPLE, dict(u=N), INVALID),
    ("ttb_sample_logits", SAMPLE, dict(vocab=0), INVALID), ("ttb_sample_logits", SAMPLE, dict(vocab=(1 << 22) + 1, stride=1 << 23), INVALID),
    ("ttb_sample_logits", SAMPLE, dict(stride=99), INVALID), ("ttb_sample_logits", SAMPLE, dict(rows=-1), INVALID),
    ("ttb_sample_logits", SAMPLE, dict(dtype=I8), UNSUPPORTED),
    ("ttb_paged_copy_blocks", COPY, dict(caches=HOLE2), INVALID), ("ttb_paged_copy_blocks", COPY, dict(pairs=N), INVALID),
    ("ttb_paged_copy_blocks", COPY, dict(pairs=ODD), INVALID), ("ttb_paged_copy_blocks", COPY, dict(np=-1), INVALID),
    ("ttb_paged_copy_blocks", COPY, dict(blocks=0), INVALID), ("ttb_paged_copy_blocks", COPY, dict(dtype=99), INVALID),
    ("ttb_paged_copy_blocks", COPY, dict(heads=1 << 20, bs=1 << 20, d=1 << 20), INVALID),
    ("ttb_paged_commit_draft", COMMIT, dict(drafts=HOLE2), INVALID), ("ttb_paged_commit_draft", COMMIT, dict(table=N), INVALID),
    ("ttb_paged_commit_draft", COMMIT, dict(users=65536), INVALID), ("ttb_paged_commit_draft", COMMIT, dict(pages=0), INVALID),
    ("ttb_paged_commit_draft", COMMIT, dict(nodes=-1), INVALID), ("ttb_paged_commit_draft", COMMIT, dict(heads=1 << 20, d=1 << 20), INVALID),
])
def test_refusals(rt, name, base, bad, code):
    rc, text = call(rt, name, with_args(base, **bad))
    assert rc == code and text, (rc, text)


@pytest.mark.parametrize("name,base,empty", [
    ("ttb_sdpa_window", WINDOW, dict(sq=0)), ("ttb_sample_logits", SAMPLE, dict(rows=0, x=N)), ("ttb_paged_copy_blocks", COPY, dict(np=0, pairs=N)),
    ("ttb_paged_copy_blocks", COPY, dict(n=0)), ("ttb_paged_commit_draft", COMMIT, dict(users=0)), ("ttb_paged_commit_draft", COMMIT, dict(nodes=0)),
])
def test_nothing_to_do_is_not_an_error(rt, name, base, empty):
    rc, text = call(rt, name, with_args(base, **empty))
    assert rc == 0, text


def test_workspace_sizes_of_impossible_problems_are_zero(rt):
    for n in ("ttb_sdpa_window_decode_workspace_bytes", "ttb_sdpa_tree_workspace_bytes"):
        getattr(rt.lib, n).restype = ctypes.c_size_t
    I, L = ctypes.c_int, ctypes.c_int64
    assert rt.lib.ttb_sdpa_window_decode_workspace_bytes(I(0), I(8), I(2), I(128), L(100), L(10), L(0)) == 0
    assert rt.lib.ttb_sdpa_window_decode_workspace_bytes(I(1), I(8), I(3), I(128), L(100), L(10), L(0)) == 0
    assert rt.lib.ttb_sdpa_tree_workspace_bytes(I(1), I(0), I(8), I(2), I(128), L(100)) == 0
    # one user with a long cache: the keys are split, two floats and head_dim partial sums per row and part
    size = rt.lib.ttb_sdpa_window_decode_workspace_bytes(I(1), I(8), I(1), I(128), L(1 << 20), L(1 << 19), L(0))
    assert size > 0 and size % (8 * 130 * 4) == 0
