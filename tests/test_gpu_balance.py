"""GPU: the balance loss and its gradient against 64 bits, alone, behind the router and in the `MoE`."""
import pytest
import torch

import momoe_amd
import oracle
from helpers import make_routing

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24  # half a step of fp32, relative


def _inputs(B, S, N, K, Ks, dtype, seed=0, skew=0.5):
    mask, _ = make_routing(B * S, N, K, Ks, seed=seed, skew=skew)
    logits = 2 * torch.randn(B, S, N, generator=torch.Generator().manual_seed(seed + 1))
    return logits.to(dtype), mask


def _check(logits, mask, Ks, valid, per_sequence, loss, counts, grad, weight):
    """Every p is off by its exponent's argument (at most 32, of which each rounding takes 2^-24), exp, sum and quotient, some
    64 + 8 half steps in all; a column sum adds chains of at most 64 + 256 terms, the last sums some 20 more: 512 half steps
    bound the loss, whose terms are all positive.  The gradient is p_j (c_j - sum c_i p_i) of such p, then
    rounded once."""
    B, S, N = logits.shape
    groups = B if per_sequence else 1
    flat = None if valid is None else valid.reshape(-1)
    ref, n, g = oracle.balance_loss(logits.reshape(-1, N), mask, Ks, flat, groups, weight)
    assert counts.dtype == torch.int64 and torch.equal(counts.cpu().reshape(groups, N), n)
    assert loss.dtype == torch.float32 and abs(loss.item() - ref.item()) <= 512 * E * abs(ref.item())
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    # the size of the two terms of the difference, each good to 128 half steps
    Nr = N - Ks
    p = torch.softmax(logits.reshape(-1, N)[:, :Nr].double().nan_to_num(0, 0, 0), -1)
    share = (n[:, :Nr].double() / n[:, :Nr].sum(1, keepdim=True).clamp_min(1)).repeat_interleave(B * S // groups, 0)
    on = torch.ones(groups, B * S // groups) if flat is None else flat.reshape(groups, -1).double()
    live = (n[:, :Nr].sum(1) > 0).sum().clamp_min(1)
    size = abs(weight) * Nr / on.sum(1).clamp_min(1).repeat_interleave(B * S // groups)[:, None] / live * p * (
        share + (share * p).sum(-1, keepdim=True))
    info = torch.finfo(logits.dtype)
    bound = torch.zeros(B * S, N, dtype=torch.float64)
    bound[:, :Nr] = 128 * E * size
    bound += g.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2  # (half a step, among subnormals too)
    off = (grad.cpu().reshape(-1, N).double() - g).abs()
    assert torch.isfinite(off).all() and (off <= bound).all(), ((off - bound).max(), (off / bound.clamp_min(1e-30)).max())


def _run(logits, mask, Ks, valid, per_sequence, weight=1.0):
    leaf = logits.to(DEV).detach().requires_grad_()
    loss, counts = momoe_amd.balance_loss(leaf, mask.to(DEV), Ks, None if valid is None else valid.to(DEV), per_sequence)
    assert loss.shape == () and counts.shape == ((logits.shape[0], logits.shape[-1]) if per_sequence else (logits.shape[-1],))
    assert not counts.requires_grad
    (loss * weight).backward()
    return loss.detach(), counts, leaf.grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("B,S,N,K,Ks", [
    (1, 1, 1, 1, 0), (1, 1, 8, 2, 0), (1, 3, 2, 1, 0), (2, 1, 33, 4, 1), (1, 128, 8, 2, 0), (3, 85, 60, 6, 2), (1, 257, 64, 8, 0),
    (4, 300, 100, 8, 0), (2, 1000, 128, 8, 4), (65, 17, 130, 4, 0), (70, 5, 32, 3, 0), (1, 700, 257, 5, 1), (5, 64, 512, 8, 0),
    (1, 5000, 31, 2, 0),
])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_balance_loss(B, S, N, K, Ks, dtype, per_sequence):
    logits, mask = _inputs(B, S, N, K, Ks, dtype)
    weight = 4096.0 if dtype == torch.float16 else 0.01
    _check(logits, mask, Ks, None, per_sequence, *_run(logits, mask, Ks, None, per_sequence, weight), weight)


@pytest.mark.parametrize("N", [60, 64])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_tokens_that_do_not_count_may_hold_anything(N, per_sequence):
    """Padding of NaN, infinities and of a mask that takes every expert; a sequence of padding only."""
    B, S, K = 4, 300, 4
    logits, mask = _inputs(B, S, N, K, 0, torch.float32)
    valid = torch.arange(S)[None] < torch.tensor([[S], [0], [1], [S // 2]])
    clean = _run(logits, mask, 0, valid, per_sequence)
    _check(logits, mask, 0, valid, per_sequence, *clean, 1.0)
    dirty, dmask = logits.clone(), mask.clone()
    dirty[~valid] = torch.tensor([float("nan"), float("inf"), float("-inf")]).repeat(N)[:N]
    dmask[:, ~valid.reshape(-1)] = 1
    for a, b in zip(clean, _run(dirty, dmask, 0, valid, per_sequence)):
        assert torch.equal(a, b)


def test_no_token_counts():
    logits, mask = _inputs(2, 40, 16, 2, 0, torch.bfloat16)
    for per_sequence in (False, True):
        for m, v in ((mask, torch.zeros(2, 40, dtype=torch.bool)), (torch.zeros_like(mask), None)):
            loss, counts, grad = _run(logits, m, 0, v, per_sequence)
            assert loss == 0 and counts.sum() == 0 and grad.abs().sum() == 0
    empty = torch.zeros(0, 5, 16, device=DEV, requires_grad=True)
    loss, counts = momoe_amd.balance_loss(empty, torch.zeros(16, 0, dtype=torch.int32, device=DEV))
    loss.backward()
    assert loss == 0 and counts.sum() == 0 and empty.grad.shape == (0, 5, 16)


def test_masked_logits():
    """-inf, and the lowest value, in places: no probability, no gradient; a token of -inf only makes the loss NaN and no other
    token's gradient."""
    logits, mask = _inputs(1, 200, 24, 2, 0, torch.float32)
    logits[0, :, 5] = float("-inf")
    logits[0, ::3, 7] = torch.finfo(torch.float32).min
    out = _run(logits, mask, 0, None, False)
    _check(logits, mask, 0, None, False, *out, 1.0)
    assert out[2][0, :, 5].abs().sum() == 0
    logits[0, 11] = float("-inf")
    loss, _, grad = _run(logits, mask, 0, None, False)
    keep = torch.arange(200) != 11
    assert loss.isnan() and grad[0, 11].isnan().all() and torch.equal(grad[0, keep], out[2][0, keep])


def test_strides_and_other_types_of_the_arguments():
    B, S, N, K = 2, 150, 48, 4
    logits, mask = _inputs(B, S, N, K, 0, torch.bfloat16)
    ref = _run(logits, mask, 0, None, True)
    wide = torch.zeros(B, S, 80, dtype=torch.bfloat16)
    wide[:, :, 5:5 + N] = logits  # rows with a pitch, off a 16-byte boundary: the column-by-column loads
    base = wide.to(DEV).requires_grad_()
    for m in (mask.to(DEV), mask.T.contiguous().to(DEV).T, mask.to(DEV).repeat(1, 2)[:, :B * S], mask.repeat_interleave(2, 0).to(DEV)[::2],
              mask.to(DEV).bool(), mask.to(DEV).repeat_interleave(3, 1)[:, ::3]):
        base.grad = None
        loss, counts = momoe_amd.balance_loss(base[:, :, 5:5 + N], m, 0, None, True)
        loss.backward()
        assert torch.equal(counts, ref[1])
        torch.testing.assert_close(loss, ref[0], rtol=16 * E, atol=0)
        torch.testing.assert_close(base.grad[:, :, 5:5 + N], ref[2], rtol=2.0 ** -7, atol=1e-9)  # (a step of bf16)
        assert base.grad[:, :, :5].abs().sum() == 0 and base.grad[:, :, 5 + N:].abs().sum() == 0
    columns = logits.transpose(1, 2).contiguous().to(DEV).transpose(1, 2).requires_grad_()
    loss, _ = momoe_amd.balance_loss(columns, mask.to(DEV), per_sequence=True)
    loss.backward()
    assert torch.equal(loss, ref[0]) and torch.equal(columns.grad, ref[2])
    # one row for all tokens: autograd sums what comes back
    row = logits[0, :1].float().to(DEV).requires_grad_()
    loss, _ = momoe_amd.balance_loss(row.expand(B * S, N), mask.to(DEV))
    loss.backward()
    full = logits[0, :1].float().expand(B * S, N)
    _, _, g = oracle.balance_loss(full, mask)
    torch.testing.assert_close(row.grad.cpu().double(), g.sum(0, keepdim=True), rtol=1e-4, atol=1e-7)


def test_gradient_against_differences():
    logits, mask = _inputs(2, 12, 10, 3, 1, torch.float32)
    _, _, grad = _run(logits, mask, 1, None, True)
    f = lambda t: oracle.balance_loss(t.reshape(-1, 10), mask, 1, None, 2)[0].item()
    h = 1e-5
    for b, s, n in ((0, 0, 0), (1, 5, 3), (0, 11, 8), (1, 2, 9)):
        up, down = logits.double().clone(), logits.double().clone()
        up[b, s, n] += h
        down[b, s, n] -= h
        # differences of 64-bit values at 1e-5: good to 1e-10 of the curvature and 1e-11 of the roundings
        assert abs((f(up) - f(down)) / (2 * h) - grad[b, s, n].item()) < 1e-8


@pytest.mark.parametrize("size", [(2, 30), (60,)])
def test_flags_that_changed_since_the_forward_are_refused(size):
    N = 16
    l = torch.randn(2, 30, N, device=DEV, requires_grad=True)
    mask = (torch.rand(N, 60, device=DEV) < 0.3).int()
    valid = torch.ones(size, dtype=torch.bool, device=DEV)
    loss, _ = momoe_amd.balance_loss(l, mask, valid=valid)
    valid.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("B,S", [(0, 5), (3, 0)])
def test_counts_of_no_tokens(B, S):
    loss, counts = momoe_amd.balance_loss(torch.zeros(B, S, 8, device=DEV), torch.zeros(8, 0, dtype=torch.int32, device=DEV),
                                          per_sequence=True)
    assert loss == 0 and counts.shape == (B, 8) and counts.sum() == 0


def test_logits_past_32_bit_offsets():
    """Tokens behind 2^31 logits: their counts, and their gradient against the formula."""
    M, N = 4_300_000, 512
    logits = torch.zeros(M, N, device=DEV, dtype=torch.bfloat16)
    mask = torch.zeros(N, M, dtype=torch.int32, device=DEV)
    logits[-3:] = torch.randn(3, N, device=DEV).bfloat16()
    mask[7, -3:] = mask[500, -1] = mask[1, 0] = 1
    logits.requires_grad_()
    loss, counts = momoe_amd.balance_loss(logits, mask)
    want = torch.zeros(N, dtype=torch.int64)
    want[7], want[500], want[1] = 3, 1, 1
    assert torch.equal(counts.cpu(), want)
    (loss * 2.0 ** 30).backward()
    p = torch.softmax(logits.detach()[-3:].cpu().double(), -1)
    c = want.double()
    g = 2.0 ** 30 * N / (M * 5.0) * p * (c - p @ c[:, None])
    got = logits.grad[-3:].cpu().double()
    # the sum over c in fp32, and one rounding to bf16
    assert ((got - g).abs() <= g.abs() * (2.0 ** -8 + 2.0 ** -14) + 2.0 ** 30 * N / (M * 5.0) * p * 5 * 2.0 ** -18).all()
    # nearly all tokens are even: p = 1 / N, and with it the loss is 1, but for three tokens of M
    assert abs(loss.item() - 1) <= 3 * N / M + 2.0 ** -10


def test_traced_modules_with_a_balance_loss():
    """A graph of torch.jit.trace does on inputs of other sizes what the module does."""
    D, H, N, K, Ks = 64, 32, 8, 3, 1
    torch.manual_seed(4)
    moe = momoe_amd.MoE(D, H, N, K, Ks, bias_update_rate=0.0, balance="sequence")
    x = torch.randn(2, 20, D, device=DEV, dtype=torch.bfloat16)
    traced = torch.jit.trace(moe, x)
    for B, S in ((2, 20), (3, 31)):
        results = []
        for module in (moe, traced):
            moe.zero_grad(set_to_none=True)
            xr = torch.randn(B, S, D, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(DEV).manual_seed(B)).requires_grad_()
            y, loss = module(xr)
            torch.autograd.backward([y, loss], [torch.ones_like(y), torch.full_like(loss, 3.0)])
            results.append([y, loss, xr.grad, moe.router.Wg_DN.grad])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_refusals():
    logits, mask = _inputs(2, 10, 8, 2, 0, torch.float32)
    l, m = logits.to(DEV), mask.to(DEV)
    with pytest.raises(AssertionError, match="bfloat16, float32 or float16"):
        momoe_amd.balance_loss(l.double(), m)
    for bad in (dict(mask_NM=m[:7]), dict(mask_NM=m[:, :-1]), dict(num_shared_experts=8), dict(num_shared_experts=-1),
                dict(valid=torch.ones(2, 9, dtype=torch.bool)), dict(valid=torch.ones(2, 10)), dict(logits=l[0, 0]),
                dict(logits=l.reshape(20, 8), per_sequence=True),
                dict(logits=torch.zeros(4, 600, device=DEV), mask_NM=torch.zeros(600, 4, dtype=torch.int32, device=DEV))):
        with pytest.raises(RuntimeError):
            momoe_amd.balance_loss(**{**dict(logits=l, mask_NM=m), **bad})
    leaf = l.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(momoe_amd.balance_loss(leaf, m)[0], leaf, create_graph=True)
    with torch.no_grad():
        loss, _ = momoe_amd.balance_loss(leaf, m)
    assert not loss.requires_grad
    # logits changed between forward and backward
    loss, _ = momoe_amd.balance_loss(leaf * 1.0, m)
    mid = leaf * 1.0
    loss, _ = momoe_amd.balance_loss(mid, m)
    mid.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_same_bits_each_time_on_another_stream_and_in_a_graph():
    logits, mask = _inputs(8, 700, 64, 8, 0, torch.bfloat16)
    m = mask.to(DEV)
    ref = _run(logits, mask, 0, None, True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(ref, _run(logits, mask, 0, None, True)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaf = logits.to(DEV).requires_grad_()
    with torch.cuda.stream(side):
        for _ in range(2):
            leaf.grad = None
            loss, counts = momoe_amd.balance_loss(leaf, m, per_sequence=True)
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, (loss.detach(), counts, leaf.grad)))
    del loss
    leaf.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts = momoe_amd.balance_loss(leaf, m, per_sequence=True)
        loss.backward()
    for seed in (5, 6, 7):
        other, _ = _inputs(8, 700, 64, 8, 0, torch.bfloat16, seed)
        want = _run(other, mask, 0, None, True)
        with torch.no_grad():
            leaf.copy_(other.to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (loss.detach(), counts, leaf.grad)))


@pytest.mark.parametrize("M,D,N,K,Ks", [(3, 64, 8, 2, 0), (300, 256, 60, 6, 2), (2500, 128, 64, 4, 0)])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_router_with_balance_loss(M, D, N, K, Ks, per_sequence):
    """The router's results stay what they are, and the gradients are those of the two losses together."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, M, D, generator=g).to(DEV, torch.bfloat16)
    router = momoe_amd.TopKRouter(D, N, K, Ks, Wg_DN=(torch.randn(D, N, generator=g) / D ** 0.5).to(DEV))
    bias = torch.cat([torch.zeros(N - Ks), torch.full((Ks,), float("-inf"))]).to(DEV)
    Gs = torch.randn(N, M, generator=g).to(DEV)
    logits = (x[0] @ router.Wg_DN).detach().requires_grad_()
    loss, counts = momoe_amd.balance_loss(logits.view(1, M, N) if per_sequence else logits, router(x, bias)[1], Ks, None, per_sequence)
    (2.0 * M * loss).backward()
    plain = [x.clone().requires_grad_(), router.Wg_DN]
    _, mask0, s0 = router(plain[0], bias)
    # (few tokens take their logits from a product of the library's own, whose sums may round otherwise)
    same = torch.equal(mask0, router.with_balance_loss(x, bias)[1])
    grads0 = torch.autograd.grad((s0 * Gs).sum(), plain)
    xr = x.clone().requires_grad_()
    y, mask, s, got, n = router.with_balance_loss(xr, bias, None, per_sequence)
    assert torch.equal(got, loss) and torch.equal(n, counts) and y.data_ptr() == xr.data_ptr()
    only = torch.autograd.grad(2.0 * M * got, [xr, router.Wg_DN], retain_graph=True)
    both = torch.autograd.grad(2.0 * M * got + (s * Gs).sum(), [xr, router.Wg_DN])
    G, W, X = logits.grad.double().cpu(), router.Wg_DN.detach().double().cpu(), x[0].double().cpu()
    want = (G @ W.T)[None], X.T @ G
    for a, b, size in zip(only, want, ((G.abs() @ W.abs().T)[None], X.abs().T @ G.abs())):
        # fp32 sums of exact products (M or N of them), one rounding to bf16
        assert ((a.double().cpu() - b).abs() <= b.abs() * 2.0 ** -8 + 2 * max(M, N) * E * size + 1e-30).all()
    if same:
        for a, b, c in zip(both, only, grads0):
            ref = b.double() + c.double()
            assert (a.double() - ref).norm() <= 2e-2 * ref.norm()
    # the loss alone in an evaluation
    with torch.no_grad():
        assert torch.equal(router.with_balance_loss(x, bias, None, per_sequence)[3], loss)


def test_moe_trains_with_a_balance_loss():
    """Router, experts and loss in one step: the gradients of the layer without it, and the loss's."""
    D, H, N, K, B, S = 128, 64, 16, 2, 3, 50
    g = torch.Generator().manual_seed(9)
    w = dict(Wg_DN=(torch.randn(D, N, generator=g) / D ** 0.5).to(DEV), Wl1_ND2H=(0.05 * torch.randn(N, D, 2 * H, generator=g)).to(DEV),
             Wl2_NHD=(0.05 * torch.randn(N, H, D, generator=g)).to(DEV))
    x = torch.randn(B, S, D, generator=g).to(DEV, torch.bfloat16)
    valid = (torch.arange(S)[None] < torch.tensor([[50], [20], [0]])).to(DEV)
    for balance in ("batch", "sequence"):
        moe = momoe_amd.MoE(D, H, N, K, 0, bias_update_rate=0.0, balance=balance, **w)
        y, loss = moe(x, valid)
        logits = (x.view(-1, D) @ moe.router.Wg_DN).detach()
        _, mask, _ = moe.router(x, moe.biases_N)
        want, _ = momoe_amd.balance_loss(logits.view(B, S, N), mask, 0, valid, balance == "sequence")
        torch.testing.assert_close(loss, want, rtol=1e-3, atol=0)
        (y.float().pow(2).mean() + 0.1 * loss).backward()
        full = moe.router.Wg_DN.grad.float()
        moe.zero_grad()
        y, loss = moe(x, valid)
        y.float().pow(2).mean().backward()
        part = moe.router.Wg_DN.grad.float().clone()
        moe.zero_grad()
        y, loss = moe(x, valid)
        (0.1 * loss).backward()
        assert moe.momoe.Wl1_ND2H.grad is None or moe.momoe.Wl1_ND2H.grad.abs().sum() == 0
        ref = part + moe.router.Wg_DN.grad.float()
        assert (full - ref).norm() <= 2e-2 * ref.norm()
    plain = momoe_amd.MoE(D, H, N, K, 0, bias_update_rate=0.0, **w)
    assert isinstance(plain(x), torch.Tensor)
    with pytest.raises(ValueError, match="valid"):
        plain(x, valid)


@pytest.mark.parametrize("per_sequence", [False, True])
def test_counts_are_the_callers_own(per_sequence):
    """Summed over ranks or added up in place between the forward and the backward: the gradient stays what it is.  (A collective
    changes a tensor without autograd's knowledge, as `.data` does.)"""
    B, S, N, K, D = 3, 200, 24, 3, 64
    logits, mask = _inputs(B, S, N, K, 0, torch.float32)
    want = _run(logits, mask, 0, None, per_sequence)
    leaf = logits.to(DEV).requires_grad_()
    router = momoe_amd.TopKRouter(D, N, K, 0, Wg_DN=torch.randn(D, N, generator=torch.Generator().manual_seed(1)).to(DEV))
    x = torch.randn(B, S, D, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    bias = torch.zeros(N, device=DEV)
    loss, _ = router.with_balance_loss(x, bias, None, per_sequence)[3:]
    through_gate, = torch.autograd.grad(1e3 * loss, router.Wg_DN)
    for change in (lambda c: c.data.add_(1000), lambda c: c.add_(1000), lambda c: c.data.zero_()):
        leaf.grad = None
        loss, counts = momoe_amd.balance_loss(leaf, mask.to(DEV), 0, None, per_sequence)
        assert torch.equal(counts, want[1])
        change(counts)
        loss.backward()
        assert torch.equal(leaf.grad, want[2])
        loss, counts = router.with_balance_loss(x, bias, None, per_sequence)[3:]
        change(counts)
        got, = torch.autograd.grad(1e3 * loss, router.Wg_DN)
        assert torch.equal(got, through_gate)


def test_flags_of_other_shapes_are_refused():
    """As many flags as tokens, but in another order than theirs."""
    B, S, N, K, D = 3, 20, 8, 2, 32
    logits, mask = _inputs(B, S, N, K, 0, torch.float32)
    l, m = logits.to(DEV), mask.to(DEV)
    flags = torch.ones(B * S, dtype=torch.bool, device=DEV)
    flags[50:] = False
    want, _ = momoe_amd.balance_loss(l, m, valid=flags)
    moe = momoe_amd.MoE(D, 32, N, K, 0, bias_update_rate=0.0, balance="batch")
    x = torch.randn(B, S, D, device=DEV, dtype=torch.bfloat16)
    _, through_moe = moe(x, flags)
    for good in (flags.view(B, S), flags):
        assert torch.equal(momoe_amd.balance_loss(l, m, valid=good)[0], want)
        assert torch.equal(momoe_amd.balance_loss(l.view(B * S, N), m, valid=good)[0], want)
        assert torch.equal(moe(x, good)[1], through_moe)
    for bad in (flags.view(S, B), flags.view(B, S).T, flags.view(1, B * S), flags.view(B, S, 1), flags.view(2, B, S // 2)):
        for per_sequence in (False, True):
            with pytest.raises(RuntimeError, match="valid must be"):
                momoe_amd.balance_loss(l, m, valid=bad, per_sequence=per_sequence)
        with pytest.raises(RuntimeError, match="valid must be"):
            moe(x, bad)
    with pytest.raises(RuntimeError, match="valid must be"):
        momoe_amd.balance_loss(l.view(B * S, N), m, valid=flags.view(B, S, 1))


@pytest.mark.parametrize("M,D,N,K,Ks", [(1, 64, 8, 2, 0), (128, 256, 16, 2, 0), (300, 512, 64, 6, 2), (1000, 1024, 128, 8, 0), (3000, 128, 60, 4, 0)])
def test_the_loss_leaves_the_routing_as_it_is(M, D, N, K, Ks):
    """Mask, gate weights, their gradients and the layer's result, bit by bit those without the loss."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, M, D, generator=g).to(DEV, torch.bfloat16)
    router = momoe_amd.TopKRouter(D, N, K, Ks, Wg_DN=(torch.randn(D, N, generator=g) / D ** 0.5).to(DEV))
    bias = torch.cat([torch.zeros(N - Ks), torch.full((Ks,), float("-inf"))]).to(DEV)
    Gs = torch.randn(N, M, generator=g).to(DEV)
    with torch.no_grad():
        _, mask, s = router(x, bias)
        _, mask1, s1, _, counts = router.with_balance_loss(x, bias)
    assert torch.equal(mask, mask1) and torch.equal(s, s1) and torch.equal(counts, mask.sum(1))
    results = []
    for with_loss in (False, True):
        xr = x.clone().requires_grad_()
        _, mask1, s1 = (router.with_balance_loss if with_loss else router)(xr, bias)[:3]
        assert torch.equal(mask, mask1) and torch.equal(s, s1)
        results.append(torch.autograd.grad((s1 * Gs).sum(), [xr, router.Wg_DN]))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    plain = momoe_amd.MoE(D, 32, N, K, Ks, bias_update_rate=0.0)
    balanced = momoe_amd.MoE(D, 32, N, K, Ks, bias_update_rate=0.0, balance="batch")
    balanced.load_state_dict(plain.state_dict())
    with torch.no_grad():
        assert torch.equal(plain(x), balanced(x)[0])


def test_sums_over_many_tokens():
    """2^27 tokens of the same logits: column sums whose terms would all be rounded the same way."""
    M, N = 1 << 27, 2
    logits = torch.tensor([0.0, 0.84375], device=DEV, dtype=torch.bfloat16).repeat(M, 1)
    mask = torch.zeros(N, M, dtype=torch.int32, device=DEV)
    mask[0] = 1
    loss, counts = momoe_amd.balance_loss(logits, mask)
    assert torch.equal(counts.cpu(), torch.tensor([M, 0]))
    want = 2 * torch.softmax(torch.tensor([0.0, 0.84375], dtype=torch.float64), 0)[0].item()
    # the bound of _check: 512 half steps, of p and of chains of some hundred terms at each level of the sums
    assert abs(loss.item() - want) <= 512 * E * want


@pytest.mark.parametrize("B,S,N,K", [(65, 500, 64, 4), (70, 1000, 33, 2), (130, 910, 16, 2), (130, 911, 16, 2), (260, 2000, 8, 1)])
@pytest.mark.parametrize("padded", [False, True])
def test_many_long_sequences(B, S, N, K, padded):
    """More than 64 sequences, on both sides of the line from which each is cut into pieces."""
    logits, mask = _inputs(B, S, N, K, 0, torch.bfloat16)
    valid = torch.arange(S)[None] < torch.arange(0, B * 37, 37)[:, None] % (S + 1) if padded else None
    _check(logits, mask, 0, valid, True, *_run(logits, mask, 0, valid, True, 0.01), 0.01)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_gradient_of_an_even_load(dtype, per_sequence):
    """Counts that are all the same: none.  Counts of half a million that differ by a few: as exact as their differences, which is what
    the loss is there for."""
    B, S, N, Ks = 2, 1 << 18, 5, 1
    logits = torch.randn(B, S, N, generator=torch.Generator().manual_seed(3)).to(dtype)
    mask = torch.ones(N, B * S, dtype=torch.int32)
    _, _, grad = _run(logits, mask, Ks, None, per_sequence, 1e6)
    assert (grad == 0).all()
    mask[1, [0, S + 7]] = 0
    mask[2, [5, 9, S, S + 1]] = 0
    loss, counts, grad = _run(logits, mask, Ks, None, per_sequence, 1e6)
    _check(logits, mask, Ks, None, per_sequence, loss, counts, grad, 1e6)
    groups = B if per_sequence else 1
    _, n, g = oracle.balance_loss(logits.reshape(-1, N), mask, Ks, None, groups, 1e6)
    n, p = n[:, :N - Ks].double(), torch.softmax(logits.reshape(-1, N)[:, :N - Ks].double(), -1)
    # Written with the counts' distances from their whole mean, which changes nothing as the p add up to one, the two terms of the
    # difference are p_j |c_j - mean| and p_j sum_i p_i |c_i - mean|: with every p good to 64 + 8 half steps as in _check, 128 of
    # these bound it.
    apart = (n - n.mean(1, keepdim=True).floor()).abs().repeat_interleave(B * S // groups, 0)
    scale = 1e6 * (N - Ks) / (B * S // groups) / n.sum(1).repeat_interleave(B * S // groups)[:, None] / groups
    bound = 128 * E * scale * p * (apart + (apart * p).sum(-1, keepdim=True))
    bound += g[:, :N - Ks].abs() * torch.finfo(dtype).eps / 2
    off = (grad.cpu().reshape(-1, N).double() - g)[:, :N - Ks].abs()
    assert (off <= bound).all(), (off / bound).max()
