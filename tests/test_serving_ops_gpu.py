"""Window attention with sinks, attention of draft trees, block copies, committing drafts and sampling, against plain
64-bit forms (tests/serving.py)."""

import ctypes
import math

import pytest
import torch

from serving import Kernels, TAG, attend, check, sample_row, tree_lines, window_seen

pytestmark = pytest.mark.gpu


@pytest.fixture
def kn(rt, device):
    h = Kernels(rt)
    yield h
    h.close()


def rand(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


# ---- prompts -------------------------------------------------------------------------------------------------------
PROMPTS = [  # dtype, batch, heads, kv heads, queries, keys, dim, offset, window, sinks, lens, permuted
    (torch.bfloat16, 1, 4, 2, 1, 1, 128, 0, 1, 0, None, False),
    (torch.bfloat16, 1, 4, 1, 200, 200, 128, 0, 64, 4, None, False),
    (torch.bfloat16, 2, 8, 2, 333, 333, 128, 0, 100, 7, [333, 90], False),
    (torch.float16, 2, 6, 2, 129, 640, 64, 511, 300, 65, [640, 600], False),
    (torch.float16, 1, 3, 3, 70, 70, 64, 0, 1, 0, None, False),
    (torch.bfloat16, 1, 2, 1, 150, 150, 256, 0, 77, 200, None, False),
    (torch.bfloat16, 1, 12, 2, 65, 165, 32, 100, 33, 1, None, False),
    (torch.bfloat16, 2, 8, 2, 257, 300, 128, 43, 128, 128, [0, 300], True),
    (torch.float16, 1, 8, 1, 300, 300, 128, 0, 10 ** 12, 10 ** 12, None, True),
    (torch.bfloat16, 1, 4, 2, 513, 513, 64, 0, 256, 3, None, False),
    (torch.bfloat16, 1, 8, 8, 400, 400, 128, 0, 130, 130, None, False),
    (torch.bfloat16, 1, 2, 1, 40, 20, 128, 0, 8, 2, None, False),          # fewer keys than queries: late rows keep the sinks
    (torch.bfloat16, 1, 2, 2, 33, 50, 80, 17, 20, 3, None, False),         # head_dim the tensor-core kernels do not take
    (torch.float16, 1, 2, 1, 9, 9, 7, 0, 4, 1, None, False),
    (torch.float32, 2, 4, 2, 50, 83, 64, 33, 20, 5, [83, 40], False),
    (torch.float32, 1, 2, 1, 70, 70, 256, 0, 70, 0, None, True),
]


@pytest.mark.parametrize("dtype,B,H,Hkv,S,N,D,offset,window,sinks,lens,permuted", PROMPTS)
def test_window_prompt(kn, dtype, B, H, Hkv, S, N, D, offset, window, sinks, lens, permuted):
    gen = torch.Generator().manual_seed(S * 7 + D)
    q, k, v = rand(gen, B, H, S, D, dtype=dtype), rand(gen, B, Hkv, N, D, dtype=dtype), rand(gen, B, Hkv, N, D, dtype=dtype)
    pos = torch.arange(S) + offset
    seen = []
    for b in range(B):
        s = window_seen(pos, N, window, sinks)
        if lens:
            s[:, lens[b]:] = False
        seen.append(s)
        dead = ~s.any(dim=0)                    # keys no row sees: NaN must stay outside
        k[b][:, dead] = float("nan")
        v[b][:, dead] = float("inf")
    got = kn.window(q, k, v, offset, window, sinks, torch.tensor(lens, dtype=torch.int32) if lens else None, permuted=permuted)
    for b in range(B):
        want, tol = attend(q[b], k[b], v[b], seen[b], 1 / math.sqrt(D), dtype)
        check(got[b], want, tol, f"user {b}")
        assert (got[b][:, ~seen[b].any(dim=1)] == 0).all()


def test_window_prompt_equals_causal_attention_when_the_window_covers_it(kn, rt):
    gen = torch.Generator().manual_seed(3)
    q, k, v = rand(gen, 1, 8, 512, 128), rand(gen, 1, 2, 512, 128), rand(gen, 1, 2, 512, 128)
    got = kn.window(q, k, v, 0, 512, 0)
    want, tol = attend(q[0], k[0], v[0], torch.ones(512, 512, dtype=torch.bool).tril(), 1 / math.sqrt(128), torch.bfloat16)
    check(got[0], want, tol)


@pytest.mark.parametrize("scale", [0.5, -0.25, 0.0])
def test_window_prompt_scales(kn, scale):
    gen = torch.Generator().manual_seed(11)
    q, k, v = rand(gen, 1, 4, 140, 64), rand(gen, 1, 2, 140, 64), rand(gen, 1, 2, 140, 64)
    got = kn.window(q, k, v, 0, 50, 3, scale=scale)
    want, tol = attend(q[0], k[0], v[0], window_seen(torch.arange(140), 140, 50, 3), scale, torch.bfloat16)
    check(got[0], want, tol)


@pytest.mark.parametrize("shift", [-300.0, 300.0])
def test_window_prompt_with_scores_far_from_zero(kn, shift):
    """Every score lies near `shift`: the reference maximum has to follow it from the first key that a row sees."""
    gen = torch.Generator().manual_seed(12)
    S, D = 300, 128
    q, k, v = rand(gen, 1, 2, S, D), rand(gen, 1, 1, S, D), rand(gen, 1, 1, S, D)
    q[..., 0], k[..., 0] = 16.0, shift / 16.0 * math.sqrt(D) / 1.0
    got = kn.window(q, k, v, 0, 40, 2)
    want, tol = attend(q[0], k[0], v[0], window_seen(torch.arange(S), S, 40, 2), 1 / math.sqrt(D), torch.bfloat16)
    check(got[0], want, tol)


# ---- one token per user -----------------------------------------------------------------------------------------------
def paged(gen, dense_k, dense_v, block, lens, dtype):
    """Lays [B, Hkv, N, D] out in blocks in random order; positions at and behind lens[b], and spare blocks, hold NaN."""
    B, Hkv, N, D = dense_k.shape
    pages = (N + block - 1) // block
    order = torch.randperm(B * pages + 2, generator=gen)[:B * pages].view(B, pages).to(torch.int32)
    k = torch.full((B * pages + 2, Hkv, block, D), float("nan"), dtype=dtype)
    v = torch.full((B * pages + 2, Hkv, block, D), float("inf"), dtype=dtype)
    table = order.clone()
    for b in range(B):
        for j in range(lens[b]):
            k[order[b, j // block], :, j % block] = dense_k[b, :, j]
            v[order[b, j // block], :, j % block] = dense_v[b, :, j]
        table[b, (lens[b] + block - 1) // block:] = -1
    return k, v, table


DECODES = [  # dtype, heads, kv heads, dim, positions, block, window, sinks, cur_pos
    (torch.bfloat16, 8, 2, 128, 300, 32, 64, 4, [299, 0, -1, 63, 64, 70]),
    (torch.float16, 8, 8, 64, 1500, 16, 1000, 4, [1499, 1003]),
    (torch.bfloat16, 6, 2, 128, 200, 7, 33, 0, [199, 31, 32, 33]),
    (torch.bfloat16, 64, 2, 128, 700, 64, 10 ** 12, 0, [699, 128]),
    (torch.bfloat16, 40, 2, 64, 130, 1, 90, 50, [129, 95]),
    (torch.float16, 3, 1, 256, 400, 100, 128, 300, [399, 250]),
    (torch.bfloat16, 16, 1, 32, 520, 24, 1, 0, [519, 0]),
    (torch.bfloat16, 8, 1, 256, 5000, 64, 4096, 16, [4999, 4200, 12]),
]


@pytest.mark.parametrize("dtype,H,Hkv,D,N,block,window,sinks,pos", DECODES)
def test_window_decode(kn, dtype, H, Hkv, D, N, block, window, sinks, pos):
    gen = torch.Generator().manual_seed(N + D)
    B = len(pos)
    q = rand(gen, 1, B, H, D, dtype=dtype)
    dk, dv = rand(gen, B, Hkv, N, D, dtype=dtype), rand(gen, B, Hkv, N, D, dtype=dtype)
    k, v, table = paged(gen, dk, dv, block, [p + 1 for p in pos], dtype)
    cur = torch.tensor(pos, dtype=torch.int32)
    got = kn.decode(q, k, v, table, cur, window, sinks)
    again = kn.decode(q, k, v, table, cur, window, sinks)
    assert torch.equal(got, again)
    dense = kn.decode(q, dk, dv, None, cur, window, sinks)
    assert torch.equal(got, dense)                       # same slots in the same order, whatever the pages
    for b in range(B):
        want, tol = attend(q[0, b][:, None], dk[b], dv[b], window_seen(cur[b:b + 1].long(), N, window, sinks), 1 / math.sqrt(D), dtype)
        check(got[0, b][:, None], want, tol, f"user {b}")
    assert kn.bad() == 0


def test_window_decode_past_the_end_of_the_table(kn):
    """A position behind the cache sees the part of its window that is there."""
    gen = torch.Generator().manual_seed(5)
    q, k, v = rand(gen, 1, 2, 4, 64), rand(gen, 2, 2, 100, 64), rand(gen, 2, 2, 100, 64)
    got = kn.decode(q, k, v, None, torch.tensor([110, 2 ** 31 - 1], dtype=torch.int32), 50, 3)
    for b, p in enumerate((110, 2 ** 31 - 1)):
        want, tol = attend(q[0, b][:, None], k[b], v[b], window_seen(torch.tensor([p]), 100, 50, 3), 1 / math.sqrt(64), torch.bfloat16)
        check(got[0, b][:, None], want, tol)


# ---- trees ------------------------------------------------------------------------------------------------------------
def some_parents(gen, T, kind):
    if kind == "chain":
        return [t - 1 for t in range(T)]
    if kind == "star":
        return [-1] * T
    return [int(torch.randint(-1, t, (1,), generator=gen)) if t else -1 for t in range(T)]


TREES = [  # dtype, heads, kv heads, dim, block, cached tokens, nodes, kind, window, sinks, draft_lens, shared parents
    (torch.bfloat16, 8, 2, 128, 32, [100, 0, 1], 1, "star", 0, 0, None, False),
    (torch.bfloat16, 8, 2, 128, 16, [100, 64, 31], 8, "random", 0, 0, None, False),
    (torch.float16, 4, 4, 64, 24, [333, 5], 13, "random", 50, 4, [13, 6], False),
    (torch.bfloat16, 16, 2, 128, 64, [700, 129], 64, "random", 0, 0, [64, 63], True),
    (torch.bfloat16, 6, 2, 256, 7, [90, 200], 17, "chain", 12, 3, None, True),
    (torch.float16, 3, 1, 32, 100, [1000], 64, "chain", 30, 1010, None, False),
    (torch.bfloat16, 8, 1, 128, 64, [3000, 2000], 31, "random", 0, 0, [31, 0], False),
    (torch.bfloat16, 32, 4, 128, 64, [513], 33, "star", 100, 0, None, False),
    (torch.float16, 8, 1, 64, 8, [2049, 64], 40, "random", 2000, 5, None, False),
]


@pytest.mark.parametrize("dtype,H,Hkv,D,block,lens,T,kind,window,sinks,drafts,shared", TREES)
def test_tree(kn, dtype, H, Hkv, D, block, lens, T, kind, window, sinks, drafts, shared, room=0):
    gen = torch.Generator().manual_seed(T * 31 + D)
    B, N = len(lens), max(max(lens), 1, room)
    q, kd, vd = rand(gen, B, T, H, D, dtype=dtype), rand(gen, B, T, Hkv, D, dtype=dtype), rand(gen, B, T, Hkv, D, dtype=dtype)
    dk, dv = rand(gen, B, Hkv, N, D, dtype=dtype), rand(gen, B, Hkv, N, D, dtype=dtype)
    k, v, table = paged(gen, dk, dv, block, lens, dtype)
    parents = torch.tensor([some_parents(gen, T, kind) for _ in range(1 if shared else B)], dtype=torch.int32)
    live = drafts or [T] * B
    for b in range(B):
        kd[b, live[b]:] = float("nan")
        vd[b, live[b]:] = float("nan")
    before = rand(gen, B, T, H, D, dtype=dtype)
    args = (q, kd, vd, k, v, table, torch.tensor(lens, dtype=torch.int32), parents, window, sinks,
            torch.tensor(drafts, dtype=torch.int32) if drafts else None)
    got = kn.tree(*args, out=before)
    assert torch.equal(got, kn.tree(*args, out=before))
    for b in range(B):
        n, t = lens[b], live[b]
        assert torch.equal(got[b, t:], before[b, t:])    # padding nodes are left as they were
        related = tree_lines(parents[0 if shared else b].tolist())[:t, :t]
        where = n + related.sum(dim=1) - 1
        cached = window_seen(where, N, window, sinks)
        cached[:, n:] = False
        fresh = related
        if window:
            fresh = related & ((where[None, :] > where[:, None] - window) | (where[None, :] < sinks))
        keys = torch.cat([dk[b], kd[b, :t].transpose(0, 1)], dim=1)
        vals = torch.cat([dv[b], vd[b, :t].transpose(0, 1)], dim=1)
        want, tol = attend(q[b, :t].transpose(0, 1), keys, vals, torch.cat([cached, fresh], dim=1), 1 / math.sqrt(D), dtype)
        check(got[b, :t].transpose(0, 1), want, tol, f"user {b}")
    assert kn.bad() == 0


@pytest.mark.parametrize("room", [2304, 4352])
@pytest.mark.parametrize("dtype,H,Hkv,D,block,lens,T,kind,window,sinks,drafts,shared", [
    (torch.bfloat16, 8, 2, 128, 32, [100, 0, 1, 2300], 1, "star", 0, 0, None, False),
    (torch.float16, 4, 4, 64, 24, [333, 5, 2200], 13, "random", 50, 4, [13, 6, 0], False),
    (torch.bfloat16, 16, 2, 128, 64, [700, 129, 2304], 64, "random", 0, 0, [64, 63, 1], True),
    (torch.bfloat16, 3, 1, 128, 7, [90, 2200], 17, "chain", 12, 3, None, True),
    (torch.float16, 5, 1, 64, 100, [1000], 64, "chain", 30, 1010, None, False),
    (torch.bfloat16, 32, 4, 128, 64, [2303, 513], 33, "star", 100, 0, None, False),
    (torch.bfloat16, 8, 8, 64, 128, [2048, 127, 128], 5, "random", 1500, 33, None, False),
    (torch.float16, 8, 1, 128, 40, [2280], 40, "random", 10 ** 12, 2, [33], False)])
def test_tree_in_a_large_cache(kn, dtype, H, Hkv, D, block, lens, T, kind, window, sinks, drafts, shared, room):
    test_tree(kn, dtype, H, Hkv, D, block, lens, T, kind, window, sinks, drafts, shared, room=room)


def test_tree_of_many_users_in_a_middling_cache(kn):
    lens = torch.randint(0, 2100, (40,), generator=torch.Generator().manual_seed(61)).tolist()
    test_tree(kn, torch.bfloat16, 8, 2, 64, 32, lens, 9, "random", 0, 0, None, False, room=2304)


def test_tree_reports_a_parent_that_is_not_an_earlier_node(kn):
    gen = torch.Generator().manual_seed(2)
    q, kd, vd = rand(gen, 1, 4, 4, 64), rand(gen, 1, 4, 2, 64), rand(gen, 1, 4, 2, 64)
    k, v = rand(gen, 1, 2, 50, 64), rand(gen, 1, 2, 50, 64)
    lens = torch.tensor([50], dtype=torch.int32)
    good = kn.tree(q, kd, vd, k, v, None, lens, torch.tensor([[-1, 0, -1, 1]], dtype=torch.int32))
    assert kn.bad() == 0
    for parent in (2, 3, 64, -5, 2 ** 31 - 1):
        got = kn.tree(q, kd, vd, k, v, None, lens, torch.tensor([[-1, 0, parent, 1]], dtype=torch.int32))
        assert kn.bad() == 1 and kn.bad() == 0
        assert torch.equal(got, good)


def test_tree_chain_equals_decode_steps(kn):
    """A chain of drafts gives each node what a decode step would give once the drafts before it are cached."""
    gen = torch.Generator().manual_seed(8)
    B, T, H, Hkv, D, n = 2, 5, 8, 2, 128, 70
    q, kd, vd = rand(gen, B, T, H, D), rand(gen, B, T, Hkv, D), rand(gen, B, T, Hkv, D)
    k, v = rand(gen, B, Hkv, n + T, D), rand(gen, B, Hkv, n + T, D)
    k[:, :, n:], v[:, :, n:] = kd.transpose(1, 2), vd.transpose(1, 2)
    lens = torch.full((B,), n, dtype=torch.int32)
    chain = torch.arange(-1, T - 1, dtype=torch.int32)[None]
    got = kn.tree(q, kd, vd, k, v, None, lens, chain, window=20, sinks=2)
    for t in range(T):
        step = kn.decode(q[:, t][None], k, v, None, lens + t, 20, 2)
        for b in range(B):
            want, tol = attend(q[b, t][:, None], k[b], v[b], window_seen(torch.tensor([n + t]), n + T, 20, 2), 1 / math.sqrt(D), torch.bfloat16)
            check(step[0, b][:, None], want, tol)
            check(got[b, t][:, None], want, tol)


# ---- pages -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,caches,shape", [(torch.bfloat16, 3, (20, 2, 16, 64)), (torch.float32, 1, (9, 1, 3, 5)), (torch.int8, 2, (12, 3, 5, 7)),
                                                (torch.float16, 300, (6, 1, 4, 6)), (torch.uint8, 2, (8, 2, 64, 130))])
def test_copy_blocks(kn, dtype, caches, shape):
    gen = torch.Generator().manual_seed(caches)
    ts = [torch.randint(-100, 100, shape, generator=gen).to(dtype) for _ in range(caches)]
    pairs = torch.tensor([[0, 3], [-1, -1], [0, 5], [2, 1], [4, 4]], dtype=torch.int32)
    got = kn.copy_blocks(ts, pairs)
    for g, t in zip(got, ts):
        want = t.clone()
        for s, d in ((0, 3), (0, 5), (2, 1)):
            want[d] = t[s]
        assert torch.equal(g, want)
    assert kn.bad() == 0


@pytest.mark.parametrize("pairs,done", [
    ([[0, 1], [2, 1]], [(0, 1)]),                        # one destination twice: the first stays
    ([[0, 1], [1, 2]], [(1, 2)]),                        # a destination that is a source
    ([[0, 8], [3, 4]], [(3, 4)]), ([[8, 0], [3, 4]], [(3, 4)]), ([[-1, 0], [3, 4]], [(3, 4)]), ([[0, -2], [3, 4]], [(3, 4)]),
    ([[0, 1], [1, 0]], []),                              # a swap needs a third block
])
def test_copy_blocks_leaves_out_what_has_no_defined_result(kn, pairs, done):
    gen = torch.Generator().manual_seed(1)
    t = rand(gen, 8, 2, 8, 64)
    got = kn.copy_blocks([t], torch.tensor(pairs, dtype=torch.int32))[0]
    want = t.clone()
    for s, d in done:
        want[d] = t[s]
    assert torch.equal(got, want)
    assert kn.bad() == 1


def test_copy_blocks_many_pairs(kn):
    gen = torch.Generator().manual_seed(4)
    t = rand(gen, 1300, 1, 2, 40)
    order = torch.randperm(1300, generator=gen).to(torch.int32)
    pairs = torch.stack([order[:650], order[650:]], dim=1).contiguous()
    got = kn.copy_blocks([t, t + 1], pairs)
    want = t.clone()
    want[pairs[:, 1].long()] = t[pairs[:, 0].long()]
    assert torch.equal(got[0], want) and kn.bad() == 0


@pytest.mark.parametrize("dtype,caches,heads,block,dim,nodes", [(torch.bfloat16, 4, 2, 16, 64, 9), (torch.float32, 2, 3, 5, 7, 4), (torch.int8, 1, 2, 3, 10, 64),
                                                               (torch.float16, 2, 8, 32, 128, 31), (torch.float16, 257, 1, 4, 8, 3)])
def test_commit_draft(kn, dtype, caches, heads, block, dim, nodes):
    gen = torch.Generator().manual_seed(nodes)
    users, pages = 4, 90 // block + nodes // block + 2
    lens = torch.tensor([0, 1, 90, 37], dtype=torch.int32)
    counts = torch.tensor([nodes, 0, min(2, nodes), -3], dtype=torch.int32)
    table = torch.randperm(users * pages + 3, generator=gen)[:users * pages].view(users, pages).to(torch.int32).contiguous()
    ts = [torch.randint(-100, 100, (users * pages + 3, heads, block, dim), generator=gen).to(dtype) for _ in range(caches)]
    ds = [torch.randint(-100, 100, (users, nodes, heads, dim), generator=gen).to(dtype) for _ in range(caches)]
    path = torch.stack([torch.randperm(nodes, generator=gen) for _ in range(users)]).to(torch.int32)
    got = kn.commit(ts, ds, table, lens, path, counts)
    for g, t, d in zip(got, ts, ds):
        want = t.clone()
        for b in range(users):
            for i in range(max(0, int(counts[b]))):
                at = int(lens[b]) + i
                want[table[b, at // block], :, at % block] = d[b, path[b, i]]
        assert torch.equal(g, want)
    assert kn.bad() == 0


def test_commit_draft_leaves_out_rows_without_a_place(kn):
    gen = torch.Generator().manual_seed(6)
    t, d = rand(gen, 6, 2, 4, 64), rand(gen, 2, 5, 2, 64)
    table = torch.tensor([[3, -1], [0, 6]], dtype=torch.int32)
    path = torch.tensor([[0, 7, 1, -1, 2], [4, 3, 2, 1, 0]], dtype=torch.int32)
    got = kn.commit([t], [d], table, torch.tensor([1, 2], dtype=torch.int32), path, torch.tensor([5, 5], dtype=torch.int32))[0]
    want = t.clone()
    want[3, :, 1], want[3, :, 3] = d[0, 0], d[0, 1]       # node 7 has no row; positions 4 and 5 have no block
    want[0, :, 2], want[0, :, 3] = d[1, 4], d[1, 3]       # block 6 does not exist
    assert torch.equal(got, want)
    assert kn.bad() == 1
    got = kn.commit([t], [d], table, torch.tensor([-4, 2 ** 31 - 1], dtype=torch.int32), path, torch.tensor([5, 5], dtype=torch.int32))[0]
    assert torch.equal(got, t) and kn.bad() == 1


def test_commit_draft_of_many_users(kn):
    """More users and pieces than fill the GPU: every CTA serves all caches in turn."""
    gen = torch.Generator().manual_seed(51)
    users, nodes, heads, block, dim, caches = 1200, 33, 8, 8, 64, 3
    pages = 6
    blocks = users * pages
    table = torch.randperm(blocks, generator=gen).view(users, pages).to(torch.int32)
    lens = torch.randint(0, pages * block - nodes + 1, (users,), generator=gen).to(torch.int32)
    count = torch.randint(0, nodes + 1, (users,), generator=gen).to(torch.int32)
    path = torch.stack([torch.randperm(nodes, generator=gen) for _ in range(users)]).to(torch.int32)
    before = [torch.randint(-128, 128, (blocks, heads, block, dim), generator=gen, dtype=torch.int8) for _ in range(caches)]
    drafts = [torch.randint(-128, 128, (users, nodes, heads, dim), generator=gen, dtype=torch.int8) for _ in range(caches)]
    got = kn.commit(before, drafts, table, lens, path, count)
    who = torch.arange(users)[:, None].expand(users, nodes)
    step = torch.arange(nodes)[None].expand(users, nodes)
    live = step < count[:, None]
    at = lens[:, None].long() + step
    who, node, at = who[live], path[live].long(), at[live]
    for b, d, g in zip(before, drafts, got):
        want = b.clone()
        want[table[who, at // block].long(), :, at % block] = d[who, node]
        assert torch.equal(g, want)
    assert kn.bad() == 0


def test_more_caches_than_a_launch_takes(kn):
    gen = torch.Generator().manual_seed(52)
    caches = [torch.randint(-128, 128, (4, 1, 2, 16), generator=gen, dtype=torch.int8) for _ in range(259)]
    drafts = [torch.randint(-128, 128, (1, 2, 1, 16), generator=gen, dtype=torch.int8) for _ in range(259)]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    for c, g in zip(caches, kn.copy_blocks(caches, i32([1, 3], [1, 0]))):
        assert torch.equal(g, c[[1, 1, 2, 1]])
    for c, d, g in zip(caches, drafts, kn.commit(caches, drafts, i32([2, 0]), i32(1), i32([1, 0]), i32(2))):
        want = c.clone()
        want[2, 0, 1], want[0, 0, 0] = d[0, 1, 0], d[0, 0, 0]
        assert torch.equal(g, want)
    assert kn.bad() == 0


# ---- sampling -----------------------------------------------------------------------------------------------------------
def check_samples(kn, logits, u, heat=None, k=None, p=None, low=None):
    rows = logits.shape[0]
    f = lambda x: None if x is None else torch.tensor(x, dtype=torch.float32)
    uu = torch.tensor(u, dtype=torch.float32)
    args = (logits, uu, f(heat), None if k is None else torch.tensor(k, dtype=torch.int32), f(p), f(low))
    token, prob = kn.sample(*args)
    token2, prob2 = kn.sample(*args)
    assert torch.equal(token, token2) and torch.equal(prob, prob2)
    for r in range(rows):
        one = lambda x, d: d if x is None else float(torch.tensor(x[r], dtype=torch.float32))
        want, share = sample_row(logits[r], float(uu[r]), one(heat, 1.0), k[r] if k else 0, one(p, 1.0), one(low, 0.0))
        assert int(token[r]) == want, f"row {r}: token {int(token[r])} != {want}"
        # a weight is off by some 2^-22 of itself, the total by no more, the share is rounded to f32
        assert abs(float(prob[r]) - share) <= 2.0 ** -20 * share + 1e-9, f"row {r}: {float(prob[r])} != {share}"
    return token


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 5003, 50001])
def test_sample_settings(kn, dtype, vocab):
    gen = torch.Generator().manual_seed(vocab)
    heat = [1.0, 0.7, 1.5, 0.0, 1.0, 1.0, 1.0, 0.9, 1.2, -1.0, 0.05, 30.0, 1.0, 1.0, 1.0, 2.0]
    k = [0, 0, 5, 3, 1, 40, 0, 20, 700, 0, 0, 4000, 10 ** 9, -4, 0, 300]
    p = [1.0, 0.9, 1.0, 0.5, 0.9, 0.95, 0.3, 0.8, 0.99, 0.5, 0.9, 0.999, 0.0, 2.0, 1e-6, 0.97]
    low = [0.0, 0.0, 0.0, 0.1, 0.5, 0.0, 0.1, 0.02, 1e-4, 0.3, 0.0, 0.9, 1.0, 1.5, 0.0, 1e-3]
    rows = len(heat)
    logits = (torch.randn(rows, vocab, generator=gen) * 3).to(dtype)
    u = torch.rand(rows, generator=gen).tolist()
    check_samples(kn, logits, u, heat, k, p, low)
    check_samples(kn, logits, u)
    check_samples(kn, logits, u, p=[0.9] * rows)
    check_samples(kn, logits, u, k=[7] * rows)


def test_sample_cuts_deep_in_large_rows(kn):
    """Borders far below the largest logits, where the row has to be searched again."""
    gen = torch.Generator().manual_seed(21)
    vocab = 128000
    k = [40000, 0, 127999, 60000, 3000, 0, 100000, 0, 2500, 9000, 0, 20000]
    p = [1.0, 0.99, 1.0, 0.97, 0.999, 0.5, 0.9, 0.9999, 1.0, 0.3, 0.8, 1.0]
    heat = [1.0, 1.5, 1.0, 3.0, 0.7, 8.0, 1.0, 1.0, 0.2, 100.0, 1.0, 0.6]
    low = [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 1e-5, 1e-4]
    logits = torch.randn(len(k), vocab, generator=gen) * 2.5
    for dtype in (torch.float32, torch.bfloat16):
        check_samples(kn, logits.to(dtype), torch.rand(len(k), generator=gen).tolist(), heat, k, p, low)


def test_sample_rows_that_mislead_a_sample(kn):
    """Few distinct values, masks of the type's lowest value, almost everything masked, one logit far above the rest."""
    gen = torch.Generator().manual_seed(22)
    vocab = 50001
    x = torch.randn(10, vocab, generator=gen) * 2.5
    x[0] = 1.25
    x[1] = torch.randint(0, 3, (vocab,), generator=gen).float()
    x[2, torch.randperm(vocab, generator=gen)[:49000]] = torch.finfo(torch.float32).min
    x[3, torch.randperm(vocab, generator=gen)[:49900]] = float("-inf")
    x[4, 12345] = 900.0
    x[5, 777] = 3e38
    x[6, :] = -1e30
    x[6, 40000:] = 2.0
    x[7, torch.randperm(vocab, generator=gen)[:vocab - 1]] = float("-inf")
    x[8, 30000:] = x[8, 0]
    x[9, 33333] = float("inf")
    for heat, k, p, low in ((1.0, 0, 1.0, 0.0), (1.0, 30000, 1.0, 0.0), (0.5, 0, 0.95, 0.0), (2.0, 20000, 0.9, 0.01), (0.01, 50, 0.5, 0.0),
                            (1.0, 0, 1.0, 0.3), (50.0, 45000, 0.99, 0.0), (float("inf"), 49000, 0.75, 0.0), (1e-30, 9, 0.9, 0.5)):
        check_samples(kn, x, torch.rand(10, generator=gen).tolist(), [heat] * 10, [k] * 10, [p] * 10, [low] * 10)


def test_sample_ties_go_to_the_lower_index(kn):
    logits = torch.zeros(6, 1000)
    logits[1, 500:] = 1.0
    logits[2, ::2] = 2.0
    logits[3, 999] = logits[3, 998] = 5.0
    logits[4] = -0.0
    logits[4, ::3] = 0.0
    check_samples(kn, logits, [0.999] * 6, heat=[0.0] * 6)
    check_samples(kn, logits, [0.999] * 6, k=[10, 3, 499, 1, 700, 999])
    check_samples(kn, logits, [0.999, 0.0, 0.5, 0.7, 0.25, 0.3], p=[0.5, 0.25, 0.1, 0.2, 0.75, 0.125], k=[700, 600, 800, 900, 0, 3])


def test_sample_rows_with_nothing_or_little_to_take(kn):
    inf, nan = float("inf"), float("nan")
    logits = torch.randn(8, 300, generator=torch.Generator().manual_seed(0))
    logits[0] = -inf
    logits[1] = nan
    logits[2] = -inf
    logits[2, 17] = -3e38
    logits[3, ::2] = nan
    logits[4, 5] = logits[4, 250] = inf
    logits[5] = -inf
    logits[5, 200:] = 3e38
    logits[6, :299] = -inf
    for heat in (1.0, 0.0, 1e-30, inf):
        check_samples(kn, logits, [0.1, 0.2, 0.9999999, 0.6, 0.7, 0.5, 0.3, 0.99], [heat] * 8, [0, 0, 5, 0, 1, 50, 0, 100], [1.0, 0.9] * 4)


def test_sample_draws_follow_the_uniform_numbers(kn):
    """u sweeps the shares of four tokens, in index order; u = 0 never takes a token without weight."""
    logits = torch.tensor([[float("-inf"), 0.0, 0.0, -1e30, 0.0, 0.0]]).repeat(9, 1)
    u = [0.0, 0.2499, 0.25, 0.4999, 0.5, 0.7499, 0.75, 0.9999999, 1.0]
    token, prob = kn.sample(logits, torch.tensor(u))
    assert token.tolist() == [1, 1, 2, 2, 4, 4, 5, 5, 5]
    assert prob.tolist() == [0.25] * 9


def test_sample_reads_rows_through_their_stride(kn):
    gen = torch.Generator().manual_seed(9)
    wide = torch.randn(5, 1037, generator=gen)
    u = torch.rand(5, generator=gen)
    got, _ = kn.sample(wide, u, stride=1001)
    want, _ = kn.sample(wide[:, :1001].contiguous(), u)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_deep_cuts_under_a_few_heavy_tokens(kn, dtype):
    """A few tokens, which a sample of the row hardly sees, hold most of the weight; top-k is deep, min-p lies on either
    side of its border."""
    gen = torch.Generator().manual_seed(31)
    vocab, rows = 100003, 14
    logits = torch.randn(rows, vocab, generator=gen) * 2.5
    for r in range(rows):
        logits[r, torch.randperm(vocab, generator=gen)[:24]] += torch.rand(24, generator=gen) * 12
        logits[r, torch.randperm(vocab, generator=gen)[:1000]] = float("-inf")
    k = [40000, 40000, 1501, 30000, 2000, 60000, 40000, 99999, 1600, 40000, 5000, 40000, 1400, 80000]
    p = [1.0, 0.5, 0.9, 0.99, 1.0, 0.95, 1.0, 0.99, 0.999, 1.0, 0.7, 0.9, 0.99, 0.5]
    heat = [1.0, 1.0, 0.8, 0.5, 0.5, 1.0, 0.6, 0.8, 0.5, 0.3, 1.0, 0.5, 0.7, 0.8]
    low = [0.0, 0.0, 0.0, 0.0, 1e-6, 0.02, 1e-3, 0.0, 1e-4, 1e-12, 1e-7, 0.1, 0.0, 1e-9]
    check_samples(kn, logits.to(dtype), torch.rand(rows, generator=gen).tolist(), heat, k, p, low)


def test_sample_the_longest_rows(kn):
    gen = torch.Generator().manual_seed(32)
    logits = (torch.randn(4, 2 ** 22, generator=gen) * 2).to(torch.bfloat16)
    logits[3, 2 ** 22 - 1] = 60.0
    check_samples(kn, logits, [0.3, 0.8, 0.5, 0.5], heat=[0.5, 0.7, 0.0, 1.0], k=[50, 0, 0, 0], p=[1.0, 0.4, 1.0, 1.0])


def test_sample_many_short_rows(kn):
    logits = torch.randn(70001, 5, generator=torch.Generator().manual_seed(53))
    token, prob = kn.sample(logits, torch.zeros(70001), torch.zeros(70001))
    assert torch.equal(token.long(), logits.argmax(dim=1)) and bool((prob == 1).all())


# ---- sizes and streams -----------------------------------------------------------------------------------------------------
def test_caches_of_more_than_2_to_the_31_elements(kn):
    """The last blocks of large caches give what the same blocks give in small ones; everything else holds NaN."""
    gen = torch.Generator().manual_seed(41)
    blocks, pages, Hkv, H, block, D, T = 33000, 68, 8, 16, 64, 128, 5
    one = Hkv * block * D * 2
    k, v = rand(gen, pages, Hkv, block, D), rand(gen, pages, Hkv, block, D)
    big = []
    for t in (k, v):
        ptr = ctypes.c_void_p()
        kn._check(kn.lib.ttb_malloc(ctypes.byref(ptr), ctypes.c_size_t(blocks * one), kn.stream))
        kn._bufs.append(ptr)
        kn._check(kn.lib.ttb_memset(ptr, 0xff, ctypes.c_size_t(blocks * one), kn.stream))
        kn._check(kn.lib.ttb_memcpy_h2d(ctypes.c_void_p(ptr.value + (blocks - pages) * one), ctypes.c_void_p(t.data_ptr()), ctypes.c_size_t(pages * one),
                                        kn.stream))
        kn.sync()
        big.append(ptr)
    table = torch.randperm(pages, generator=gen)[None].to(torch.int32)
    far = kn.up(table + (blocks - pages))
    size = max(kn.lib.ttb_sdpa_window_decode_workspace_bytes(*kn.args(1, H, Hkv, D, pages * block, 10 ** 6, 0)),
               kn.lib.ttb_sdpa_tree_workspace_bytes(*kn.args(1, T, H, Hkv, D, pages * block)), 16)
    work, scale = kn.empty((size,), torch.uint8), 1 / math.sqrt(D)

    n = 4310
    q, pos = rand(gen, 1, 1, H, D), torch.tensor([n - 1], dtype=torch.int32)
    out = kn.empty(q.shape, q.dtype)
    kn.call("ttb_sdpa_window_decode", kn.up(q), *big, far, kn.up(pos), out, TAG[q.dtype], 1, H, Hkv, blocks, block, pages, D, 10 ** 6, 0, scale,
            work, ctypes.c_size_t(size), kn.stream)
    assert torch.equal(kn.download(out, q.shape, q.dtype), kn.decode(q, k, v, table, pos, 10 ** 6, 0))

    q, kd, vd = rand(gen, 1, T, H, D), rand(gen, 1, T, Hkv, D), rand(gen, 1, T, Hkv, D)
    lens, parents = torch.tensor([n], dtype=torch.int32), torch.tensor([[-1, 0, 0, 2, 1]], dtype=torch.int32)
    out = kn.empty(q.shape, q.dtype)
    kn.call("ttb_sdpa_tree", kn.up(q), kn.up(kd), kn.up(vd), *big, far, kn.up(lens), kn.up(parents), None, out, TAG[q.dtype], 1, T, H, Hkv, blocks, block,
            pages, D, 1, 0, 0, scale, work, ctypes.c_size_t(size), kn.stream)
    assert torch.equal(kn.download(out, q.shape, q.dtype), kn.tree(q, kd, vd, k, v, table, lens, parents))

    arr, darr = (ctypes.c_void_p * 2)(*[b.value for b in big]), (ctypes.c_void_p * 2)(kn.up(kd).value, kn.up(vd).value)
    path, count = torch.tensor([[0, 2, 3, 0, 0]], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    kn.call("ttb_paged_commit_draft", arr, darr, 2, far, kn.up(lens), kn.up(path), kn.up(count), TAG[q.dtype], 1, T, Hkv, blocks, block, pages, D, kn.stream)
    last = int(table[0, n // block])
    kn.call("ttb_paged_copy_blocks", arr, 2, kn.up(torch.tensor([[blocks - pages + last, 0]], dtype=torch.int32)), 1, TAG[q.dtype], blocks, Hkv, block, D,
            kn.stream)
    for ptr, t, d in zip(big, (k, v), (kd, vd)):
        want = t[last].clone()
        for i, node in enumerate((0, 2, 3)):
            want[:, n % block + i] = d[0, node]
        assert torch.equal(kn.download(ptr, want.shape, want.dtype), want)   # block 0, a copy of the one written
    assert kn.bad() == 0


def test_calls_on_two_streams_at_once(kn):
    """Each stream with buffers and workspaces of its own: what they give alone."""
    gen = torch.Generator().manual_seed(42)
    H, Hkv, D, n, vocab = 8, 2, 128, 5000, 60000
    other = ctypes.c_void_p()
    kn._check(kn.lib.ttb_stream_create(ctypes.byref(other)))
    jobs = []
    for stream in (kn.stream, other):
        logits, u, top_k = torch.randn(40, vocab, generator=gen) * 3, torch.rand(40, generator=gen), torch.randint(1, 20000, (40,), generator=gen).int()
        q, kd, vd = rand(gen, 2, 6, H, D), rand(gen, 2, 6, Hkv, D), rand(gen, 2, 6, Hkv, D)
        k, v, lens = rand(gen, 2, Hkv, n, D), rand(gen, 2, Hkv, n, D), torch.tensor([n, 1234], dtype=torch.int32)
        parents = torch.tensor([[-1, 0, 1, 0, 3, 3]], dtype=torch.int32)
        want = kn.sample(logits, u, None, top_k)[0], kn.tree(q, kd, vd, k, v, None, lens, parents)
        size = kn.lib.ttb_sdpa_tree_workspace_bytes(*kn.args(2, 6, H, Hkv, D, n))
        work, token, out = kn.empty((max(size, 16),), torch.uint8), kn.empty((40,), torch.int32), kn.empty(q.shape, q.dtype)
        sample = (kn.up(logits), kn.up(u), None, kn.up(top_k), None, None, token, None, TAG[logits.dtype], 40, vocab, vocab, None, ctypes.c_size_t(0), stream)
        tree = (kn.up(q), kn.up(kd), kn.up(vd), kn.up(k), kn.up(v), None, kn.up(lens), kn.up(parents), None, out, TAG[q.dtype], 2, 6, H, Hkv, 2, n, 1, D, 1, 0, 0,
                1 / math.sqrt(D), work, ctypes.c_size_t(size), stream)
        jobs.append((sample, tree, token, out, want))
    for _ in range(5):
        for sample, tree, *_ in jobs:
            kn.call("ttb_sdpa_tree", *tree)
            kn.call("ttb_sample_logits", *sample)
    kn._check(kn.lib.ttb_stream_sync(other))
    kn.sync()
    for _, _, token, out, (want, want_out) in jobs:
        assert torch.equal(kn.download(token, (40,), torch.int32), want)
        assert torch.equal(kn.download(out, want_out.shape, want_out.dtype), want_out)
    kn._check(kn.lib.ttb_stream_destroy(other))


# ---- together ------------------------------------------------------------------------------------------------------------
def test_a_speculative_step(kn):
    """Draft tree -> attention -> logits -> greedy tokens -> accepted path -> cache -> next token's attention, and a fork."""
    gen = torch.Generator().manual_seed(77)
    B, T, H, Hkv, D, block, vocab = 2, 6, 4, 2, 64, 8, 97
    lens = torch.tensor([29, 12], dtype=torch.int32)
    pages = 6
    dk, dv = rand(gen, B, Hkv, 48, D), rand(gen, B, Hkv, 48, D)
    k, v, table = paged(gen, dk, dv, block, [48, 48], torch.bfloat16)
    q, kd, vd = rand(gen, B, T, H, D), rand(gen, B, T, Hkv, D), rand(gen, B, T, Hkv, D)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 4], [-1, -1, 1, 2, 3, 0]], dtype=torch.int32)
    head = rand(gen, vocab, H * D, scale=0.05)
    out = kn.tree(q, kd, vd, k, v, table, lens, parents)
    logits = (out.reshape(B * T, H * D).float() @ head.float().T).to(torch.bfloat16)
    token, _ = kn.sample(logits, torch.zeros(B * T), torch.zeros(B * T))
    assert torch.equal(token.long(), logits.float().argmax(dim=1))
    # say the verifier accepts the path 0, 2, 4 of the first user and 1, 2 of the second
    path = torch.tensor([[0, 2, 4, 9, 9, 9], [1, 2, 9, 9, 9, 9]], dtype=torch.int32)
    count = torch.tensor([3, 2], dtype=torch.int32)
    k2, v2 = kn.commit([k, v], [kd, vd], table, lens, path, count)
    full_k, full_v = dk.clone(), dv.clone()
    for b in range(B):
        for i in range(int(count[b])):
            full_k[b, :, lens[b] + i], full_v[b, :, lens[b] + i] = kd[b, path[b, i]], vd[b, path[b, i]]
    pos = lens + count - 1
    q1 = rand(gen, 1, B, H, D)
    got = kn.decode(q1, k2, v2, table, pos, 16, 2)
    for b in range(B):
        want, tol = attend(q1[0, b][:, None], full_k[b], full_v[b], window_seen(pos[b:b + 1].long(), 48, 16, 2), 1 / math.sqrt(D), torch.bfloat16)
        check(got[0, b][:, None], want, tol)
    # the first user forks: its last block is copied to a spare one, the table of the copy points there
    used = set(table.flatten().tolist())
    spare = next(i for i in range(k.shape[0]) if i not in used)
    last = int(pos[0]) // block
    k3, v3 = kn.copy_blocks([k2, v2], torch.tensor([[int(table[0, last]), spare]], dtype=torch.int32))
    forked = table.clone()
    forked[1] = table[0]
    forked[1, last] = spare
    two = kn.decode(q1[:, :1].repeat(1, 2, 1, 1), k3, v3, forked, pos[:1].repeat(2), 16, 2)
    assert torch.equal(two[0, 0], two[0, 1]) and torch.equal(two[0, 0], got[0, 0])
    assert kn.bad() == 0


@pytest.mark.parametrize("n", [900, 9000])
def test_serving_step_as_a_replayed_trace(kn, n):
    """The calls record into a trace and replay on new contents of the same buffers, on a stream of their own."""
    gen = torch.Generator().manual_seed(13)
    B, T, H, Hkv, D = 1, 4, 8, 1, 128
    mk = lambda: [rand(gen, B, T, H, D), rand(gen, B, T, Hkv, D), rand(gen, B, T, Hkv, D)]
    k, v = rand(gen, B, Hkv, n, D), rand(gen, B, Hkv, n, D)
    parents, lens = torch.tensor([[-1, 0, 1, 0]], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    first, second = mk(), mk()
    want = [kn.tree(*x, k, v, None, lens, parents) for x in (first, second)]
    bufs = [kn.upload(t) for t in first]
    pk, pv, pl, pp = kn.upload(k), kn.upload(v), kn.upload(lens), kn.upload(parents)
    size = kn.lib.ttb_sdpa_tree_workspace_bytes(*kn.args(B, T, H, Hkv, D, n))
    assert (size > 0) == (n > 4096)                       # one user: the keys are split, over a cluster or over more CTAs
    work, out = kn.empty((max(size, 16),), torch.uint8), kn.empty((B, T, H, D), torch.bfloat16)
    logits = kn.upload(torch.randn(3, 500, generator=gen))
    u, token = kn.upload(torch.tensor([0.1, 0.5, 0.9])), kn.empty((3,), torch.int32)
    size2 = kn.lib.ttb_sample_logits_workspace_bytes(*kn.args(3, 500))
    work2 = kn.empty((max(size2, 16),), torch.uint8)
    drawn, _ = kn.sample(kn.download(logits, (3, 500), torch.float32), torch.tensor([0.1, 0.5, 0.9]))
    stream, trace = ctypes.c_void_p(), ctypes.c_void_p()
    kn._check(kn.lib.ttb_stream_create(ctypes.byref(stream)))
    kn._check(kn.lib.ttb_trace_begin(stream))
    kn.call("ttb_sdpa_tree", *bufs, pk, pv, None, pl, pp, None, out, TAG[torch.bfloat16], B, T, H, Hkv, B, n, 1, D, 1, 0, 0,
            1 / math.sqrt(D), work, ctypes.c_size_t(size), stream)
    kn.call("ttb_sample_logits", logits, u, None, None, None, None, token, None, 0, 3, 500, 500, work2, ctypes.c_size_t(size2), stream)
    kn._check(kn.lib.ttb_trace_end(stream, ctypes.byref(trace)))
    for x, w in ((first, want[0]), (second, want[1])):
        for p, t in zip(bufs, x):
            t = t.contiguous()
            kn._check(kn.lib.ttb_memcpy_h2d(p, ctypes.c_void_p(t.data_ptr()), ctypes.c_size_t(t.numel() * 2), stream))
        kn._check(kn.lib.ttb_trace_launch(trace, stream))
        kn._check(kn.lib.ttb_stream_sync(stream))
        assert torch.equal(kn.download(out, (B, T, H, D), torch.bfloat16), w)
        assert torch.equal(kn.download(token, (3,), torch.int32), drawn)
    kn._check(kn.lib.ttb_trace_destroy(trace))
    kn._check(kn.lib.ttb_stream_destroy(stream))
