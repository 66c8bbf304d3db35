"""Serving operators at their edges: NaN among the operands, scales that the tensor-core kernels hand on, bad parents in a
long cache, and calls whose first use is inside a recording."""

import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

from serving import TAG, Kernels, attend, check, tree_lines, window_seen

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture
def kn(rt, device):
    h = Kernels(rt)
    yield h
    h.close()


def rand(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen).to(dtype)


def check_poison(got, clean, poisoned):
    """Rows (`poisoned`, of got's shape without the last dimension) are NaN throughout, the others are what they are
    without the NaN."""
    assert torch.isnan(got[poisoned]).all(), f"{int((~torch.isnan(got[poisoned])).sum())} elements of poisoned rows are not NaN"
    assert torch.equal(got[~poisoned], clean[~poisoned])


# ---- NaN: a softmax over a NaN score is NaN, in that row only -----------------------------------------------------------
@pytest.mark.parametrize("dtype,H,Hkv,S,D,window,sinks,scale", [
    (torch.bfloat16, 4, 2, 300, 128, 100, 4, None), (torch.float16, 6, 2, 290, 64, 70, 0, None), (torch.bfloat16, 2, 1, 150, 256, 77, 3, None),
    (torch.bfloat16, 4, 2, 100, 32, 33, 0, None), (torch.bfloat16, 4, 2, 200, 128, 64, 2, -0.25), (torch.bfloat16, 2, 1, 90, 80, 20, 1, None),
    (torch.float32, 2, 2, 90, 64, 20, 1, None)])
def test_nan_in_a_prompt_reaches_the_rows_that_see_it(kn, dtype, H, Hkv, S, D, window, sinks, scale):
    gen = torch.Generator().manual_seed(S + D)
    q, k, v = rand(gen, 1, H, S, D, dtype=dtype), rand(gen, 1, Hkv, S, D, dtype=dtype), rand(gen, 1, Hkv, S, D, dtype=dtype)
    clean = kn.window(q, k, v, 0, window, sinks, scale=scale)
    seen = window_seen(torch.arange(S), S, window, sinks)
    G = H // Hkv
    q2 = q.clone()
    q2[0, 1, S // 2, D - 1] = NAN
    poisoned = torch.zeros(1, H, S, dtype=torch.bool)
    poisoned[0, 1, S // 2] = True
    check_poison(kn.window(q2, k, v, 0, window, sinks, scale=scale), clean, poisoned)
    for keys in ([S // 3], list(range(S // 4, S // 2))):             # one key, and all that some rows see
        k2 = k.clone()
        k2[0, Hkv - 1, keys, 0] = NAN
        poisoned = torch.zeros(1, H, S, dtype=torch.bool)
        poisoned[0, (Hkv - 1) * G:] = seen[:, keys].any(dim=1)
        check_poison(kn.window(q, k2, v, 0, window, sinks, scale=scale), clean, poisoned)


@pytest.mark.parametrize("N", [90, 700, 5000])                      # one part, a cluster's parts, parts joined by a second kernel
@pytest.mark.parametrize("dtype,H,Hkv,D", [(torch.bfloat16, 8, 2, 128), (torch.float16, 3, 1, 256)])
def test_nan_in_a_decode_step(kn, dtype, H, Hkv, D, N):
    gen = torch.Generator().manual_seed(N)
    q, k, v = rand(gen, 1, 2, H, D, dtype=dtype), rand(gen, 2, Hkv, N, D, dtype=dtype), rand(gen, 2, Hkv, N, D, dtype=dtype)
    pos = torch.tensor([N - 1, N // 2], dtype=torch.int32)
    run = lambda q, k: kn.decode(q, k, v, None, pos, 10 ** 6, 0)
    clean = run(q, k)
    q2 = q.clone()
    q2[0, 1, 2] = NAN
    poisoned = torch.zeros(1, 2, H, dtype=torch.bool)
    poisoned[0, 1, 2] = True
    check_poison(run(q2, k), clean, poisoned)
    for keys in (slice(N // 3, N // 3 + 1), slice(0, N // 2 - 8)):
        k2 = k.clone()
        k2[1, Hkv - 1, keys] = NAN
        poisoned = torch.zeros(1, 2, H, dtype=torch.bool)
        poisoned[0, 1, (Hkv - 1) * (H // Hkv):] = True
        check_poison(run(q, k2), clean, poisoned)


@pytest.mark.parametrize("B,H,Hkv,D,N", [
    (2, 4, 2, 128, 90), (2, 6, 2, 256, 700), (1, 4, 1, 32, 5000),   # mma.sync: one part, a cluster, a second kernel
    (1, 4, 1, 64, 4400), (5, 16, 8, 128, 4400), (18, 8, 8, 64, 4400)])  # tcgen05: many parts, three, one
def test_nan_in_a_tree(kn, B, H, Hkv, D, N):
    gen = torch.Generator().manual_seed(N + B)
    T = 5
    q, kd, vd = rand(gen, B, T, H, D), rand(gen, B, T, Hkv, D), rand(gen, B, T, Hkv, D)
    k, v = rand(gen, B, Hkv, N, D), rand(gen, B, Hkv, N, D)
    lens, parents = torch.full((B,), N - 3, dtype=torch.int32), torch.tensor([[-1, 0, 0, 1, 2]], dtype=torch.int32)
    run = lambda q, kd, k: kn.tree(q, kd, vd, k, v, None, lens, parents)
    clean = run(q, kd, k)
    G, b = H // Hkv, B - 1
    none = lambda: torch.zeros(B, T, H, dtype=torch.bool)
    q2, poisoned = q.clone(), none()
    q2[b, 3, 1], poisoned[b, 3, 1] = NAN, True
    check_poison(run(q2, kd, k), clean, poisoned)
    kd2, poisoned = kd.clone(), none()
    kd2[b, 2, Hkv - 1, 3] = NAN                                      # node 2 and its child 4
    poisoned[b, [2, 4], (Hkv - 1) * G:] = True
    check_poison(run(q, kd2, k), clean, poisoned)
    for keys in (slice(N // 2, N // 2 + 1), slice(0, N // 2), slice(0, N)):
        k2, poisoned = k.clone(), none()
        k2[b, Hkv - 1, keys] = NAN
        poisoned[b, :, (Hkv - 1) * G:] = True
        check_poison(run(q, kd, k2), clean, poisoned)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 64)])
def test_a_prompt_without_keys_is_zero(kn, dtype, D):
    q = rand(torch.Generator().manual_seed(1), 2, 4, 40, D, dtype=dtype)
    out = kn.upload(torch.ones_like(q))
    kn.call("ttb_sdpa_window", kn.up(q), None, None, None, out, TAG[dtype], 2, 4, 2, 40, 0, D, None, None, None, None, 0, 8, 1, 0.1, kn.stream)
    assert (kn.download(out, q.shape, dtype) == 0).all()


# ---- long prompts, far positions ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,H,Hkv,S,N,D,offset,window,sinks,lens", [
    (torch.bfloat16, 4, 1, 1100, 4700, 128, 3600, 2900, 70, None),          # some 47 key tiles: the ring turns many times
    (torch.float16, 2, 2, 900, 5000, 64, 4100, 10 ** 9, 0, None),
    (torch.bfloat16, 3, 1, 700, 4000, 128, 3300, 3100, 1, [3777]),
    (torch.float16, 4, 2, 300, 3000, 256, 2700, 2000, 5, None),
    (torch.bfloat16, 4, 2, 140, 90, 128, 2 ** 29, 300, 3, None),            # the last positions there are: only the sinks are near
    (torch.float16, 4, 2, 140, 90, 64, 2 ** 29, 2 ** 31, 0, [77]),          # ... or everything is
    (torch.bfloat16, 2, 1, 70, 90, 32, 2 ** 29, 64, 80, None),
    (torch.float32, 2, 1, 70, 90, 64, 2 ** 29, 2 ** 40, 80, None)])
def test_long_and_far_prompts(kn, dtype, H, Hkv, S, N, D, offset, window, sinks, lens):
    gen = torch.Generator().manual_seed(N + S)
    q, k, v = rand(gen, 1, H, S, D, dtype=dtype), rand(gen, 1, Hkv, N, D, dtype=dtype), rand(gen, 1, Hkv, N, D, dtype=dtype)
    seen = window_seen(torch.arange(S) + offset, N, window, sinks)
    if lens:
        seen[:, lens[0]:] = False
    dead = ~seen.any(dim=0)
    k[0][:, dead], v[0][:, dead] = NAN, float("inf")
    got = kn.window(q, k, v, offset, window, sinks, torch.tensor(lens, dtype=torch.int32) if lens else None)
    want, tol = attend(q[0], k[0], v[0], seen, 1 / math.sqrt(D), dtype)
    check(got[0], want, tol)


# ---- scales and parents in long caches -----------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [0.0, -0.5])
@pytest.mark.parametrize("B,H,Hkv,D,room", [(1, 4, 1, 64, 4352), (5, 16, 8, 128, 4352), (18, 8, 8, 64, 4352), (2, 8, 2, 128, 300)])
def test_tree_scales_that_are_not_positive(kn, scale, B, H, Hkv, D, room):
    """The rows are planned for the tensor-core kernel (many parts, three, one) and computed by the other one."""
    gen = torch.Generator().manual_seed(B)
    T = 4
    q, kd, vd = rand(gen, B, T, H, D), rand(gen, B, T, Hkv, D), rand(gen, B, T, Hkv, D)
    k, v = rand(gen, B, Hkv, room, D), rand(gen, B, Hkv, room, D)
    lens = torch.randint(0, room + 1, (B,), generator=gen).to(torch.int32)
    lens[0] = room
    parents = torch.tensor([[-1, 0, 0, 2]], dtype=torch.int32)
    got = kn.tree(q, kd, vd, k, v, None, lens, parents, scale=scale)
    related = tree_lines(parents[0].tolist())
    for b in sorted({0, B // 2, B - 1}):
        cached = (torch.arange(room) < lens[b]).expand(T, room)
        keys, vals = torch.cat([k[b], kd[b].transpose(0, 1)], dim=1), torch.cat([v[b], vd[b].transpose(0, 1)], dim=1)
        want, tol = attend(q[b].transpose(0, 1), keys, vals, torch.cat([cached, related], dim=1), scale, torch.bfloat16)
        check(got[b].transpose(0, 1), want, tol, f"user {b}")


@pytest.mark.parametrize("scale", [0.0, -0.5])
@pytest.mark.parametrize("N", [90, 700, 5000])
def test_decode_scales_that_are_not_positive(kn, scale, N):
    gen = torch.Generator().manual_seed(N)
    q, k, v = rand(gen, 1, 1, 4, 64), rand(gen, 1, 2, N, 64), rand(gen, 1, 2, N, 64)
    got = kn.decode(q, k, v, None, torch.tensor([N - 1], dtype=torch.int32), 10 ** 6, 0, scale=scale)
    want, tol = attend(q[0, 0][:, None], k[0], v[0], torch.ones(1, N, dtype=torch.bool), scale, torch.bfloat16)
    check(got[0, 0][:, None], want, tol)


def test_tree_in_a_long_cache_reports_a_parent_that_is_not_an_earlier_node(kn):
    gen = torch.Generator().manual_seed(2)
    N = 4400
    q, kd, vd = rand(gen, 1, 4, 4, 64), rand(gen, 1, 4, 2, 64), rand(gen, 1, 4, 2, 64)
    k, v = rand(gen, 1, 2, N, 64), rand(gen, 1, 2, N, 64)
    lens = torch.tensor([N - 7], dtype=torch.int32)
    i32 = lambda *x: torch.tensor([x], dtype=torch.int32)
    good = kn.tree(q, kd, vd, k, v, None, lens, i32(-1, 0, -1, 1))
    assert kn.bad() == 0
    for parent in (2, 3, 64, -5, 2 ** 31 - 1):
        got = kn.tree(q, kd, vd, k, v, None, lens, i32(-1, 0, parent, 1))
        assert kn.bad() == 1 and kn.bad() == 0
        assert torch.equal(got, good)
    # a node that does not exist may name any parent
    got = kn.tree(q, kd, vd, k, v, None, lens, i32(-1, 0, 0, 77), draft_lens=torch.tensor([3], dtype=torch.int32))
    assert kn.bad() == 0 and (got[0, 3] == 0).all()


# ---- block copies -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("caches,blocks,moves", [(9, 2100, 1000), (5, 30, 12), (9, 50, 20), (260, 900, 420)])
def test_copy_blocks_of_many_caches_and_pairs(kn, caches, blocks, moves):
    """Each piece of a pair serves several caches in turn; among the pairs are paddings, blocks outside and destinations twice."""
    gen = torch.Generator().manual_seed(blocks)
    ts = [torch.randint(-128, 128, (blocks, 1, 2, 24), generator=gen, dtype=torch.int8) for _ in range(caches)]
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    pairs = torch.stack([order[:moves], order[blocks - moves:]], dim=1).contiguous()
    assert kn.bad() == 0
    done = torch.ones(moves, dtype=torch.bool)
    pairs[3] = -1
    done[3] = False
    for g, t in zip(kn.copy_blocks(ts, pairs), ts):
        want = t.clone()
        want[pairs[done, 1].long()] = t[pairs[done, 0].long()]
        assert torch.equal(g, want)
    assert kn.bad() == 0
    pairs[moves - 1, 1] = pairs[0, 1]       # a destination twice: the first stays
    pairs[moves - 2, 0] = blocks            # outside
    pairs[moves - 3, 1] = pairs[1, 0]       # onto a source
    done[moves - 3:] = False
    for g, t in zip(kn.copy_blocks(ts, pairs), ts):
        want = t.clone()
        want[pairs[done, 1].long()] = t[pairs[done, 0].long()]
        assert torch.equal(g, want)
    assert kn.bad() == 1


# ---- sampling next to a border ---------------------------------------------------------------------------------------------
def flat_rows(gen, rows, vocab, dtype, kind):
    """Rows whose weight is spread over many tokens: noise under a few likely tokens, or one token over equal others."""
    if kind == "noise":
        x = torch.randn(rows, vocab, generator=gen) * 2.5
        x.scatter_add_(1, torch.randint(0, vocab, (rows, 24), generator=gen), torch.rand(rows, 24, generator=gen) * 12)
    else:
        x = torch.full((rows, vocab), 0.7133)
        x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=gen)] = 8 + 6 * torch.rand(rows, generator=gen)
    return x.to(dtype)


def near_border(shares, above):
    """(i, u): a multiple u of 2^-24 in (0.5, 1), exact in f32, that lies 2^-31 .. 2^-29 above (below) shares[i]."""
    steps = torch.ceil(shares * 2 ** 24) if above else torch.floor(shares * 2 ** 24)
    far = (steps * 2.0 ** -24 - shares).abs()
    ok = (far > 2.0 ** -31) & (far < 2.0 ** -29) & (shares > 0.5) & (shares < 0.999)
    own = torch.diff(shares) > 2.0 ** -27                            # between neighbours that the distance does not reach
    ok[1:-1] &= own[:-1] & own[1:]
    ok[0] = ok[-1] = False
    i = int(ok.nonzero()[0])
    return i, float(steps[i] * 2.0 ** -24)


@pytest.mark.parametrize("kind", ["noise", "equal"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_draws_next_to_a_border(kn, dtype, kind):
    """u lies within 2^-29 of the border between two tokens.  The running sums' shares are off by less than 2^-36 (2^-38 for
    each weight, above and below the fraction bar; f64 sums add 2^-36 of that), so the token is the definition's."""
    gen = torch.Generator().manual_seed(71)
    logits = flat_rows(gen, 24, 128000, dtype, kind)
    us, want = [], []
    for r in range(logits.shape[0]):
        x = logits[r].double()
        run = torch.cumsum(torch.exp(x - x.max()), 0)
        i, u = near_border((run / run[-1])[1000:-1000], r % 2 == 0)
        us.append(u)
        want.append(1000 + i + (1 if r % 2 == 0 else 0))          # above the end of i's share: the next token
    token, prob = kn.sample(logits, torch.tensor(us))
    assert token.tolist() == want
    x = logits.double()
    w = torch.exp(x - x.amax(dim=1, keepdim=True))
    share = w[torch.arange(len(want)), want] / w.sum(dim=1)
    assert ((prob.double() - share).abs() <= 2.0 ** -23 * share).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 60000])
def test_sample_keeps_the_prefix_next_to_a_border(kn, dtype, k):
    """top-p lies within 2^-29 of a prefix's share: one entry more or less would show in the share of the token drawn, which
    is off by at most half a step of f32 and 2^-36."""
    gen = torch.Generator().manual_seed(72)
    logits = flat_rows(gen, 16, 128000, dtype, "noise")
    ps, want, shares = [], [], []
    u = torch.tensor(0.3)
    for r in range(logits.shape[0]):
        x = logits[r].double()
        order = torch.sort(x, descending=True, stable=True).indices
        kept = order[:k] if k else order
        mass = torch.exp(x[kept] - x[order[0]])
        run = torch.cumsum(mass, 0)
        i, p = near_border((run / run[-1])[:40000], r % 2 == 0)
        ps.append(p)
        kept = kept[:i + (2 if r % 2 == 0 else 1)]                # above the prefix's share: it takes one more
        kept = torch.sort(kept).values
        mass = torch.exp(x[kept] - x[order[0]])
        run = torch.cumsum(mass, 0)
        at = int((run <= float(u) * run[-1]).sum())
        want.append(int(kept[at]))
        shares.append(float(mass[at] / run[-1]))
    rows = logits.shape[0]
    token, prob = kn.sample(logits, u.repeat(rows), None, torch.full((rows,), k, dtype=torch.int32), torch.tensor(ps))
    assert token.tolist() == want
    shares = torch.tensor(shares, dtype=torch.float64)
    assert ((prob.double() - shares).abs() <= 2.0 ** -23 * shares).all()


@pytest.mark.parametrize("vocab", [9000, 60000])
def test_sample_rows_whose_tops_a_sample_misses(kn, vocab):
    """A few logits far above all others, by 20 to 1500 nats, the next ones 5 and 9 nats below: what top-p and top-k keep is
    among them, whatever the reference that the first pass took its weights against."""
    gen = torch.Generator().manual_seed(74)
    rise = [20, 60, 150, 204, 206, 215, 250, 270, 280, 300, 400, 500, 600, 620, 640, 700, 1000, 1500]
    rows = 4 * len(rise)
    logits = torch.randn(rows, vocab, generator=gen)
    for r in range(rows):
        at = torch.randperm(vocab, generator=gen)[:4]
        logits[r, at] = rise[r // 4] + torch.tensor([0.0, -5.0, -9.0, -9.0])
    p = [0.9, 0.999, 0.9999, 1.0] * len(rise)
    k = [0, 0, 3, 0] * len(rise)
    token, prob = kn.sample(logits, torch.rand(rows, generator=gen), None, torch.tensor(k, dtype=torch.int32), torch.tensor(p))
    for r in range(rows):
        x = logits[r].double()
        kept = torch.sort(x, descending=True, stable=True).indices[:k[r] or vocab]
        w = torch.exp(x[kept] - x[kept[0]])
        limit = float(torch.tensor(p[r], dtype=torch.float32))
        kept = kept[(torch.cumsum(w, 0) - w) < limit * w.sum()] if p[r] < 1 else kept
        w = torch.exp(x[kept] - x[kept[0]])
        share = float(w[kept == int(token[r])].sum() / w.sum())
        assert share > 0 and abs(float(prob[r]) - share) <= 2.0 ** -23 * share, (r, float(prob[r]), share)


def test_sample_min_p_at_its_border(kn):
    """min-p is the weight of one token, rounded down or up to f32: the token stays or goes.  Under a very high temperature
    every finite logit weighs 1, which min-p 1 keeps."""
    gen = torch.Generator().manual_seed(73)
    x = torch.randn(12, 3000, generator=gen)
    low, want = [], []
    for r in range(12):
        w = torch.exp(x[r].double() - x[r].double().max())
        at = int(torch.sort(w, descending=True).indices[100 + r])
        m = torch.tensor(float(w[at]), dtype=torch.float64).to(torch.float32)
        inf = torch.tensor(float("inf") if r % 2 else 0.0)
        m = torch.nextafter(m, inf) if (m.double() < w[at]) == bool(r % 2) else m
        low.append(float(m))
        want.append(int((w >= m.double()).sum()))
        assert want[-1] == 100 + r + (0 if r % 2 else 1)
    # a draw of u -> 1 takes the last token that stayed, in the vocabulary's order
    token, _ = kn.sample(x, torch.full((12,), 1.0 - 2.0 ** -24), None, None, None, torch.tensor(low))
    for r in range(12):
        w = torch.exp(x[r].double() - x[r].double().max())
        assert int(token[r]) == int((w >= low[r]).nonzero()[-1])
    for heat in (float("inf"), 1e30):
        u = torch.rand(12, generator=gen)
        token, prob = kn.sample(x, u, torch.full((12,), heat), None, None, torch.ones(12))
        assert token.tolist() == [min(int(float(v) * 3000), 2999) for v in u] and torch.allclose(prob, torch.tensor(1 / 3000))


# ---- the first call of a process inside a recording --------------------------------------------------------------------
FIRST = r"""
import ctypes, math, sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from __graft_entry__ import load_package
load_package()
from ttmlir_b200 import runtime_api as rt
from serving import Kernels, TAG
kn = Kernels(rt)
gen = torch.Generator().manual_seed(1)
r = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16)
i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
B, T, H, Hkv, D, n = 1, 4, 4, 2, 64, 5000
q, kd, vd, k, v = r(B, T, H, D), r(B, T, Hkv, D), r(B, T, Hkv, D), r(B, Hkv, n, D), r(B, Hkv, n, D)
q1, qp, kp, vp = r(1, 1, H, D), r(1, H, 130, D), r(1, Hkv, 130, D), r(1, Hkv, 130, D)
logits, u = torch.randn(2, 9000, generator=gen), torch.tensor([0.3, 0.7])
caches, pairs = [r(4, Hkv, 8, D)], i32([0, 2], [1, 3])
up = kn.upload
P = dict((name, up(t)) for name, t in dict(q=q, kd=kd, vd=vd, k=k, v=v, q1=q1, qp=qp, kp=kp, vp=vp, logits=logits, u=u, cache=caches[0], pairs=pairs,
         lens=i32(4900), pos=i32(4800), parents=i32([-1, 0, 1, 0]), path=i32([0, 2, 3, 0]), count=i32(3), table=i32([1]), short=i32(2)).items())
outs = dict(tree=kn.empty(q.shape, q.dtype), decode=kn.empty(q1.shape, q.dtype), prompt=kn.empty(qp.shape, q.dtype), token=kn.empty((2,), torch.int32))
sizes = [kn.lib.ttb_sdpa_tree_workspace_bytes(*kn.args(B, T, H, Hkv, D, n)), kn.lib.ttb_sdpa_window_decode_workspace_bytes(*kn.args(1, H, Hkv, D, n, 10 ** 6, 0))]
works = [kn.empty((max(s, 16),), torch.uint8) for s in sizes]
arr, darr = (ctypes.c_void_p * 1)(P["cache"].value), (ctypes.c_void_p * 1)(P["kd"].value)
stream, trace = ctypes.c_void_p(), ctypes.c_void_p()
kn._check(kn.lib.ttb_stream_create(ctypes.byref(stream)))
kn._check(kn.lib.ttb_trace_begin(stream))
bf, sc = TAG[torch.bfloat16], 1 / math.sqrt(D)
kn.call("ttb_paged_copy_blocks", arr, 1, P["pairs"], 2, bf, 4, Hkv, 8, D, stream)
kn.call("ttb_paged_commit_draft", arr, darr, 1, P["table"], P["short"], P["path"], P["count"], bf, 1, T, Hkv, 4, 8, 1, D, stream)
kn.call("ttb_sdpa_tree", P["q"], P["kd"], P["vd"], P["k"], P["v"], None, P["lens"], P["parents"], None, outs["tree"], bf, B, T, H, Hkv, 1, n, 1, D, 1, 0, 0, sc,
        works[0], ctypes.c_size_t(sizes[0]), stream)
kn.call("ttb_sdpa_window_decode", P["q1"], P["k"], P["v"], None, P["pos"], outs["decode"], bf, 1, H, Hkv, 1, n, 1, D, 10 ** 6, 0, sc, works[1],
        ctypes.c_size_t(sizes[1]), stream)
kn.call("ttb_sdpa_window", P["qp"], P["kp"], P["vp"], None, outs["prompt"], bf, 1, H, Hkv, 130, 130, D, None, None, None, None, 0, 40, 1, sc, stream)
kn.call("ttb_sample_logits", P["logits"], P["u"], None, None, None, None, outs["token"], None, 0, 2, 9000, 9000, None, ctypes.c_size_t(0), stream)
kn._check(kn.lib.ttb_trace_end(stream, ctypes.byref(trace)))
kn._check(kn.lib.ttb_trace_launch(trace, stream))
kn._check(kn.lib.ttb_stream_sync(stream))
got = [kn.download(outs["tree"], q.shape, q.dtype), kn.download(outs["decode"], q1.shape, q.dtype), kn.download(outs["prompt"], qp.shape, q.dtype),
       kn.download(outs["token"], (2,), torch.int32), kn.download(P["cache"], caches[0].shape, q.dtype)]
want = [kn.tree(q, kd, vd, k, v, None, i32(4900), i32([-1, 0, 1, 0])), kn.decode(q1, k, v, None, i32(4800), 10 ** 6, 0), kn.window(qp, kp, vp, 0, 40, 1),
        kn.sample(logits, u)[0], kn.commit(kn.copy_blocks(caches, pairs), [kd], i32([1]), i32(2), i32([0, 2, 3, 0]), i32(3))[0]]
assert all(torch.equal(g, w) for g, w in zip(got, want)), [torch.equal(g, w) for g, w in zip(got, want)]
assert kn.bad() == 0
print("same")
"""


def test_first_calls_of_a_process_record_into_a_trace(device):
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST.format(root=os.path.dirname(here), tests=here)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("same"), res.stdout + res.stderr
