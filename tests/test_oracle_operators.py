"""CPU: the 64-bit restatements of the operators beside the reference's path."""
import torch

import oracle
from helpers import make_layer_inputs, make_routing


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


def test_e4m3_is_that_of_torch():
    v = torch.cat([torch.linspace(-448, 448, 100001), torch.linspace(-0.03, 0.03, 20001), torch.exp2(torch.arange(-12.0, 9.0)),
                   torch.tensor([0.0, 448.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 432.0])])
    v = v.to(torch.float32)
    assert torch.equal(oracle.e4m3(v.double()).float(), v.to(torch.float8_e4m3fn).float())


def test_rows_in_8_bits():
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(0))
    x[1, :128] = 0
    x[2, 130] = 448
    x[3, :128] *= 2.0 ** -120
    q, e = oracle.rows_in_8_bits(x)
    assert q.abs().max() <= 448 and (q[2, 128:256] == oracle.e4m3(x[2, 128:256].double())).all()
    assert (q[1, :128] == 0).all() and (q[3, :128] == 0).all() and (e[[1, 3], 0] == -108).all()  # 2^-108 * 448 > 2^-100
    top = x.abs()[0, 256:].max()
    assert 224 < top / 2.0 ** e[0, 2] <= 448
    assert ((oracle.rounded_rows(x) - x).abs() <= x.abs() * 2.0 ** -4 + 2.0 ** -10 * torch.exp2(e.double()).repeat_interleave(128, 1)[:, :300]).all()


def test_experts_fp8_without_rounding_is_the_layer():
    """Whole numbers of four bits, and an h that is one of them: nothing is rounded."""
    M, D, H, N, K = 20, 64, 32, 4, 2
    _, W1, W2, mask, s, _ = make_layer_inputs(M, D, H, N, K)
    x = torch.randint(-8, 9, (M, D), generator=torch.Generator().manual_seed(1)).float()
    y = oracle.experts_fp8(x, W1.double() * 0, W2.double(), mask, s)
    assert (y == 0).all()
    W1[:, :, H:] = 0  # h = a * 0 * sigmoid(0)
    W1[:, 0, H:] = 64
    x[:, 0] = 8       # b = 512: sigmoid 1
    W1[:, :, :H] = torch.randint(-1, 2, (N, D, H), generator=torch.Generator().manual_seed(2)).float() * 0
    W1[:, 1, :H] = 2.0 ** -6
    x[:, 1:] = 4
    torch.testing.assert_close(oracle.experts_fp8(x, W1.double(), W2.double(), mask, s),
                               oracle.experts_forward(x, W1, W2, mask, s, dtype=torch.float64))
