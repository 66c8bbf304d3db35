"""Serving operators at their edges: NaN among the operands."""

import pytest
import torch

from serving import Kernels, window_seen

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
