"""CPU: the 64-bit restatements of the dense block and of 4-bit weights against independent ones."""
import pytest
import torch

import oracle


def _block(M, D, H, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *size: torch.randn(*size, generator=g, dtype=torch.float64)
    return r(M, D), r(D, 2 * H) / D ** 0.5, r(H, D) / H ** 0.5, r(M, D)


@pytest.mark.parametrize("M,D,H", [(1, 3, 2), (5, 8, 6), (7, 4, 9)])
def test_swiglu_block_is_one_expert(M, D, H):
    x, W1, W2, _ = _block(M, D, H)
    ref = oracle.experts_forward(x, W1[None], W2[None], torch.ones(1, M, dtype=torch.int32), torch.ones(1, M, dtype=torch.float64), dtype=torch.float64)
    a, b, h, y = oracle.swiglu_block(x, W1, W2)
    assert torch.allclose(y, ref.double(), rtol=1e-12, atol=1e-12)
    assert torch.equal(torch.cat([a, b], 1), x @ W1) and torch.allclose(h, a * torch.nn.functional.silu(b), rtol=1e-12)


@pytest.mark.parametrize("M,D,H", [(1, 3, 2), (5, 8, 6)])
def test_swiglu_block_gradients_by_autograd_and_differences(M, D, H):
    x, W1, W2, Gy = _block(M, D, H)
    got = oracle.swiglu_block_gradients(x, W1, W2, Gy)
    leaves = [t.clone().requires_grad_() for t in (x, W1, W2)]
    want = torch.autograd.grad(oracle.swiglu_block(*leaves)[3], leaves, Gy)
    value = lambda *t: (oracle.swiglu_block(*t)[3] * Gy).sum().item()
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)
        step = torch.zeros_like(a)
        step.view(-1)[a.numel() // 2] = 1e-5
        up, down = [t + step if j == i else t for j, t in enumerate((x, W1, W2))], [t - step if j == i else t for j, t in enumerate((x, W1, W2))]
        assert abs((value(*up) - value(*down)) / 2e-5 - a.reshape(-1)[a.numel() // 2].item()) < 1e-7


def test_int4_weights_by_hand_and_by_loops():
    codes = torch.tensor([[0x51], [0xF0]], dtype=torch.uint8)  # 1, 5, 0, 15
    assert oracle.int4_weights(codes, torch.tensor([[0.5]]), None, 32).flatten().tolist() == [-3.5, -1.5, -4.0, 3.5]
    assert oracle.int4_weights(codes, torch.tensor([[0.5], [2.0]]), torch.tensor([[1], [0]], dtype=torch.uint8), 2).flatten().tolist() == [0, 2, 0, 30]
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 256, (2, 48, 3), generator=g, dtype=torch.uint8)
    scale, zero = torch.rand(2, 3, 3, generator=g), torch.randint(0, 16, (2, 3, 3), generator=g, dtype=torch.uint8)
    got = oracle.int4_weights(codes, scale, zero, 32)
    for n in range(2):
        for k in range(96):
            for c in range(3):
                q = codes[n, k // 2, c].item() >> 4 if k % 2 else codes[n, k // 2, c].item() & 15
                assert got[n, k, c].item() == (q - zero[n, k // 32, c].item()) * scale[n, k // 32, c].double().item()
