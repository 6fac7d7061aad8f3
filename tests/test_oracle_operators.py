"""CPU: the 64-bit restatements of the operators beside the reference's path."""
import torch

import oracle
from helpers import make_routing


def test_balance_loss_is_one_where_all_is_even():
    M, N = 12, 4
    mask = torch.zeros(N, M, dtype=torch.int32)
    mask[torch.arange(M) % N, torch.arange(M)] = 1
    loss, counts, grad = oracle.balance_loss(torch.zeros(M, N), mask)
    assert loss == 1 and torch.equal(counts, torch.full((1, N), M // N)) and grad.abs().max() < 1e-18


def test_balance_loss_by_hand():
    # two experts, both tokens at the first; p = (3/4, 1/4) and (1/2, 1/2): 2 * (1 * 5/8)
    logits = torch.tensor([[3.0, 1.0], [1.0, 1.0]], dtype=torch.float64).log()
    mask = torch.tensor([[1, 1], [0, 0]], dtype=torch.int32)
    loss, _, grad = oracle.balance_loss(logits, mask)
    torch.testing.assert_close(loss, torch.tensor(1.25, dtype=torch.float64))
    torch.testing.assert_close(grad[0], torch.tensor([3 / 16, -3 / 16], dtype=torch.float64))


def test_balance_loss_gradient_is_that_of_autograd():
    B, S, N, K, Ks = 3, 7, 10, 4, 1
    mask, _ = make_routing(B * S, N, K, Ks, seed=3)
    logits = torch.randn(B * S, N, generator=torch.Generator().manual_seed(1)).double().requires_grad_()
    valid = torch.rand(B * S, generator=torch.Generator().manual_seed(2)) < 0.6
    valid[S:2 * S] = False  # a sequence without a token
    p = torch.softmax(logits[:, :N - Ks], -1)
    terms = []
    for b in (0, 2):
        on = torch.arange(b * S, (b + 1) * S)[valid[b * S:(b + 1) * S]]
        c = mask[:N - Ks, on].sum(1).double()
        terms.append((N - Ks) * (c / c.sum() * p[on].mean(0)).sum())
    ref = sum(terms) / 2
    ref.backward()
    loss, counts, grad = oracle.balance_loss(logits.detach(), mask, Ks, valid, B)
    torch.testing.assert_close(loss, ref.detach())
    torch.testing.assert_close(grad, logits.grad)
    assert counts[1].sum() == 0 and counts[0, -1] == valid[:S].sum()


def test_balance_loss_without_pairs_is_zero():
    loss, counts, grad = oracle.balance_loss(torch.randn(4, 3), torch.zeros(3, 4, dtype=torch.int32))
    assert loss == 0 and counts.sum() == 0 and grad.abs().sum() == 0
