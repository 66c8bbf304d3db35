"""sliding_window_size on the attention ops of a program, through tt::runtime::submit against the oracle."""

import math

import pytest
import torch

from helpers import assert_matches, run_body

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,B,H,Hkv,S,D,window", [
    (torch.bfloat16, 1, 8, 2, 300, 128, 64), (torch.float16, 2, 4, 4, 130, 64, 1), (torch.bfloat16, 1, 4, 2, 96, 32, 200), (torch.float32, 1, 2, 1, 70, 64, 33)])
def test_sdpa_with_a_sliding_window(rt, device, dtype, B, H, Hkv, S, D, window):
    torch.manual_seed(S)
    q, k, v = (torch.randn(B, h, S, D).to(dtype) for h in (H, Hkv, Hkv))
    got, want = run_body(rt, device, lambda b, x, y, z: b.scaled_dot_product_attention(x, y, z, True, None, None, window), [q, k, v])
    assert_matches(got[0], want[0], f"window {window}")


@pytest.mark.parametrize("window", [1, 100, 5000])
def test_decode_with_a_sliding_window(rt, device, window):
    torch.manual_seed(window)
    B, H, Hkv, S, D = 3, 8, 2, 700, 128
    q = torch.randn(1, B, H, D).to(torch.bfloat16)
    k, v = torch.randn(B, Hkv, S, D).to(torch.bfloat16), torch.randn(B, Hkv, S, D).to(torch.bfloat16)
    pos = torch.tensor([699, 0, 150], dtype=torch.int32)
    got, want = run_body(rt, device, lambda b, x, y, z, p: b.scaled_dot_product_attention_decode(x, y, z, p, None, True, 1 / math.sqrt(D), window),
                         [q, k, v, pos])
    assert_matches(got[0], want[0], f"window {window}", (0.999, 1e-2, 2.0 ** -6))


@pytest.mark.parametrize("block,window", [(32, 100), (16, 1), (64, 4000)])
def test_paged_decode_with_a_sliding_window(rt, device, block, window):
    torch.manual_seed(block)
    B, H, Hkv, D, pages = 4, 8, 4, 64, 9
    q = torch.randn(B, 1, H, D).to(torch.bfloat16)
    blocks = B * pages + 5
    k, v = torch.randn(blocks, Hkv, block, D).to(torch.bfloat16), torch.randn(blocks, Hkv, block, D).to(torch.bfloat16)
    table = torch.randperm(blocks)[:B * pages].view(B, pages).to(torch.int32)
    pos = torch.tensor([pages * block - 1, 0, block, 2 * block - 1], dtype=torch.int32)
    got, want = run_body(rt, device, lambda b, x, y, z, t, p: b.paged_scaled_dot_product_attention_decode(x, y, z, t, p, None, True, None, window),
                         [q, k, v, table, pos])
    assert_matches(got[0], want[0], f"window {window}", (0.999, 1e-2, 2.0 ** -6))


def test_a_window_with_a_mask_is_refused(rt, device):
    q, k = torch.randn(1, 2, 40, 64).to(torch.bfloat16), torch.randn(1, 2, 40, 64).to(torch.bfloat16)
    mask = torch.zeros(1, 1, 40, 40).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="sliding window"):
        run_body(rt, device, lambda b, x, y, m: b.scaled_dot_product_attention(x, y, y, False, m, None, 8), [q, k, mask])
    with pytest.raises(RuntimeError, match="sliding window"):
        run_body(rt, device, lambda b, x, y: b.scaled_dot_product_attention(x, y, y, False, None, None, 8), [q, k])
