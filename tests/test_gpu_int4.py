"""GPU: blocks with 4-bit weights, the experts' and the dense one, against 64 bits."""
import copy

import pytest
import torch

import momoe_amd
import oracle
from helpers import make_routing

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24


def _x(M, D, dtype=torch.bfloat16, seed=0):
    x = torch.randn(M, D, generator=torch.Generator().manual_seed(seed))
    return (x * torch.exp2(torch.randint(-6, 7, (M, 1), generator=torch.Generator().manual_seed(seed + 1)).float())).to(dtype)


def _weights(lead, D, H, group, zeros=True, scale_type=torch.bfloat16, seed=0):
    """(Wl1, S1, Wl2, S2, Z1, Z2): any codes, zeros of 0 to 15, scales of any size."""
    g = torch.Generator().manual_seed(seed)

    def of(R, C):
        G = -(-R // group)
        codes = torch.randint(0, 256, (*lead, R // 2, C), generator=g, dtype=torch.uint8)
        scale = ((0.5 + torch.rand(*lead, G, C, generator=g)) / (8 * R ** 0.5)).to(scale_type)
        return codes, scale, torch.randint(0, 16, (*lead, G, C), generator=g, dtype=torch.uint8) if zeros else None
    (q1, s1, z1), (q2, s2, z2) = of(D, 2 * H), of(H, D)
    return q1, s1, q2, s2, z1, z2


def _values(w, group):
    return oracle.int4_weights(w[0], w[1], w[4], group), oracle.int4_weights(w[2], w[3], w[5], group)


def _on(w):
    return [None if t is None else t.to(DEV) for t in w]


def _sum_bound(x, scale, group):
    """How far a sum over the contraction may be off: what is added up in a group is at most 143 |x| and what is subtracted 143 times the
    sum of x, each of at most group + 2 roundings, then, scaled, 143 of up to four groups stand in the sum until they are taken away again:
    two roundings a group, of the values of up to four; then the sum over the groups (of which the values are at most 15 |x| scale)."""
    k = x.shape[1]
    s = scale.double().abs().repeat_interleave(group, -2)[:k]
    return (x.abs() @ s) * E * (2 * 143 * (group + 4 + 4) + 15 * (scale.shape[-2] + 8))


def _block(x, w, group, kept=False):
    """(y, how far it may be off before its last rounding) of rows x (64 bits) through one block w.  kept: what bf16 leaves of h is bf16, too."""
    H = 2 * w[2].shape[0]
    W1, W2 = _values(w, group)
    a, b, h, y = oracle.swiglu_block(x, W1, W2)
    d = _sum_bound(x, w[1], group)
    da, db = d[:, :H], d[:, H:]
    # |d (b sig) / d b| <= 1.1; exp and reciprocal of the sigmoid, the products: some 16 + |b| roundings; h to bf16
    dh = da * (b * torch.sigmoid(b)).abs() + (a.abs() + da) * db * 1.1 + h.abs() * (16 + b.abs()) * 2 * E
    dh = dh + (h.abs() + dh) * 2.0 ** (-16 if kept else -8)
    return y, dh @ W2.abs() + _sum_bound(h.abs() + dh, w[3], group)


def _check(y, want, off):
    y = y.detach().cpu().double().reshape(want.shape)
    off = off + (want.abs() + off) * 2.0 ** -8 + 1e-38
    assert torch.isfinite(y).all() and ((y - want).abs() <= off).all(), ((y - want).abs() / off).max()


# M, D, H, group, zeros: one row, tiles of up to 32 and of 64 and their ends, widths below, at and past a block of 128 and of 64 columns,
# contractions past what is held of the rows at a time, shared by wavefronts or not
DENSE = [
    (1, 32, 32, 32, True), (1, 32, 32, 128, False), (1, 2080, 64, 128, True), (2, 64, 2080, 64, True), (7, 96, 160, 64, True), (16, 128, 128, 128, False),
    (17, 288, 96, 32, True), (32, 160, 416, 128, True), (33, 288, 1056, 64, False), (64, 1056, 288, 32, True), (65, 128, 64, 128, True),
    (131, 96, 2208, 32, False), (200, 640, 352, 64, True), (300, 2080, 96, 128, True), (517, 64, 640, 128, False), (1000, 160, 160, 32, True),
    # tiles of 64 rows, contractions cut into slices and whole: their ends in rows and columns, half a block of 128 left over
    (300, 1056, 160, 32, True), (270, 416, 416, 128, False), (33, 2080, 1408, 64, True), (70, 1408, 2080, 32, False), (129, 2208, 1312, 128, True),
    (400, 352, 352, 64, True), (1000, 288, 160, 128, True), (2100, 160, 160, 32, False), (5000, 96, 96, 64, True), (12000, 64, 64, 128, True),
]


@pytest.mark.parametrize("scale_type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,D,H,group,zeros", DENSE)
def test_dense_block(M, D, H, group, zeros, scale_type):
    w = _weights((), D, H, group, zeros, scale_type)
    block = momoe_amd.FeedForwardInt4(D, H, *_on(w), group_size=group)
    x = _x(M, D)
    y = block(x.to(DEV))
    assert y.dtype == torch.bfloat16 and y.shape == (M, D)
    _check(y, *_block(x.double(), w, group, M <= 16))


@pytest.mark.parametrize("M,D,H,group,zeros", [(20, 1056, 96, 128, True), (700, 1056, 160, 32, True), (700, 1120, 160, 64, False), (700, 1184, 160, 128, True)])
def test_rows_of_one_sign(M, D, H, group, zeros):
    """The most that codes' offsets add up to, and is to be taken away again; the last groups of four not all there."""
    w = _weights((), D, H, group, zeros)
    x = (3 + 0.1 * _x(M, D).float().sign()).to(torch.bfloat16)
    x[1::2] = -x[1::2]
    block = momoe_amd.FeedForwardInt4(D, H, *_on(w), group_size=group)
    _check(block(x.to(DEV)), *_block(x.double(), w, group))


# M, D, H, N, K, Ks, skew, group: experts without a token and with nearly all
EXPERTS = [
    (1, 32, 32, 2, 1, 0, 0, 32), (1, 256, 128, 8, 8, 0, 0, 128), (7, 96, 160, 4, 2, 0, 0, 64), (50, 288, 416, 5, 2, 1, 0, 128),
    (33, 2208, 64, 3, 1, 0, 0, 64), (64, 64, 2208, 2, 2, 1, 0, 32), (200, 128, 128, 16, 2, 0, 1.5, 128), (300, 96, 64, 4, 2, 0, 0, 32),
    (517, 288, 160, 5, 2, 1, 0, 64), (700, 128, 416, 4, 3, 1, 2.0, 128), (90, 1056, 352, 40, 4, 0, 0, 128), (300, 128, 96, 40, 2, 0, 2.0, 64),
    # tiles of 64 rows, few of them in an expert and many
    (300, 288, 416, 5, 2, 1, 2.0, 64), (100, 1056, 352, 8, 2, 0, 0, 32), (330, 2080, 96, 3, 1, 0, 1.0, 128), (3000, 160, 96, 3, 1, 0, 0, 32),
]


@pytest.mark.parametrize("M,D,H,N,K,Ks,skew,group", EXPERTS)
def test_experts(M, D, H, N, K, Ks, skew, group):
    w = _weights((N,), D, H, group, zeros=M % 2 == 0)
    layer = momoe_amd.MoMoEInt4(D, H, N, K, *_on(w), group_size=group)
    mask, s = make_routing(M, N, K, Ks, seed=5, skew=skew)
    x = _x(M, D)
    y, sizes = layer(x.view(1, M, D).to(DEV), mask.to(DEV), s.to(DEV))
    assert y.shape == (1, M, D) and y.dtype == torch.bfloat16 and torch.equal(sizes.cpu(), mask.sum(1))
    want, off = torch.zeros(M, D, dtype=torch.float64), torch.zeros(M, D, dtype=torch.float64)
    for i in range(N):
        rows = mask[i].nonzero().flatten()
        if len(rows):
            out, d = _block(x[rows].double(), [None if t is None else t[i] for t in w], group, len(rows) <= 16 and M * K <= 16 * N)
            sr = s[i, rows].double()[:, None]
            want.index_add_(0, rows, sr * out)
            off.index_add_(0, rows, sr * d + (sr * out).abs() * (K + 2) * 2 * E)
    _check(y, want, off)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("D,H", [(32, 32), (160, 96), (288, 416)])
def test_weights_come_back(D, H, group):
    for zeros, scale_type in ((True, torch.bfloat16), (False, torch.float16)):
        w = _weights((3,), D, H, group, zeros, scale_type)
        back = momoe_amd.MoMoEInt4(D, H, 3, 1, *_on(w), group_size=group).weights()
        one = momoe_amd.FeedForwardInt4(D, H, *[None if t is None else t[1] for t in _on(w)], group_size=group).weights()
        for a, b, c in zip(back, w, one):
            b = torch.full_like(a.cpu(), 8) if b is None else b
            assert a.dtype == b.dtype and torch.equal(a.cpu(), b) and torch.equal(c.cpu(), b[1])


@pytest.mark.parametrize("M", [1, 40, 200, 8000])
def test_strides_types_and_places_of_x(M):
    D, H, group = 96, 64, 32
    w = _weights((), D, H, group)
    block = momoe_amd.FeedForwardInt4(D, H, *_on(w), group_size=group)
    x = _x(M, D).to(DEV)
    ref = block(x)
    wide = torch.zeros(2 * M, D + 24, device=DEV, dtype=torch.bfloat16)
    for at in (0, 3, 8):
        wide[::2, at:D + at] = x
        assert torch.equal(block(wide[::2, at:D + at]), ref)
    assert torch.equal(block(x.T.contiguous().T), ref) and torch.equal(block(x.float()), ref) and torch.equal(block(x.double()), ref)
    assert torch.equal(block(x.half()), block(x.half().to(torch.bfloat16)))
    assert block(x.view(M, 1, 1, D)).shape == (M, 1, 1, D) and torch.equal(block(x.view(M, 1, 1, D)).view(M, D), ref)
    assert torch.equal(block(x[0]), block(x[:1])[0]) and block(x[:0]).shape == (0, D)
    assert torch.equal(block(x.cpu()), ref.cpu())
    assert torch.equal(block(x[:1].expand(M, D)), block(x[:1].repeat(M, 1)))


@pytest.mark.parametrize("M", [30, 40, 600])
def test_tokens_of_nan_and_infinity_stay_with_themselves(M):
    D, H, N, K, group = 288, 160, 4, 2, 64
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, K, *_on(w), group_size=group)
    block = momoe_amd.FeedForwardInt4(D, H, *[t[0] for t in _on(w)], group_size=group)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    bad = x.clone()
    bad[0, 3, 100], bad[0, 17, 200], bad[0, M - 1, 0], bad[0, 20] = float("nan"), float("inf"), float("-inf"), 0
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[[3, 17, 20, M - 1]] = False
    for call in (lambda t: layer(t, mask, s)[0], block):
        y, ref = call(bad), call(x)
        assert y[0, [3, 17, M - 1]].isnan().all() and (y[0, 20] == 0).all() and torch.equal(y[0, keep], ref[0, keep])


@pytest.mark.parametrize("M", [40, 600, 8000])
def test_routing_that_is_not_k_of_n(M, monkeypatch):
    """Too few experts: what is missing is absent.  Too many: zeros.  CHECK_ROUTING raises for both."""
    D, H, N, K, group = 96, 64, 4, 2, 32
    layer = momoe_amd.MoMoEInt4(D, H, N, K, *_on(_weights((N,), D, H, group)), group_size=group)
    mask, s = make_routing(M, N, K, seed=2)
    x = _x(M, D).view(1, M, D).to(DEV)
    few = mask.clone()
    few[:, 5] = 0
    few[mask[:, 6].nonzero()[0], 6] = 0
    y, ref = layer(x, few.to(DEV), s.to(DEV))[0], layer(x, mask.to(DEV), s.to(DEV))[0]
    keep = torch.arange(M, device=DEV) > 6
    assert (y[0, 5] == 0).all() and torch.equal(y[0, keep], ref[0, keep]) and not torch.equal(y[0, 6], ref[0, 6])
    many = torch.ones_like(mask)
    assert (layer(x, many.to(DEV), s.to(DEV))[0] == 0).all()
    monkeypatch.setattr(momoe_amd.experts, "CHECK_ROUTING", True)
    for m in (few, many):
        with pytest.raises(RuntimeError, match="exactly K"):
            layer(x, m.to(DEV), s.to(DEV))


@pytest.mark.parametrize("M", [3, 150, 500])
def test_streams_and_replayed_graphs(M):
    """Two calls at once on streams of their own, and a graph of both replayed on other inputs between eager calls."""
    D, H, N, K, group = 288, 416, 8, 2, 64
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, K, *_on(w), group_size=group)
    block = momoe_amd.FeedForwardInt4(D, H, *[t[0] for t in _on(w)], group_size=group)
    ins = [(_x(M, D, seed=i).view(1, M, D).to(DEV), *[t.to(DEV) for t in make_routing(M, N, K, seed=i)]) for i in range(3)]
    both = lambda x, mask, s: (layer(x, mask, s)[0], block(x))
    ref = [both(*t) for t in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    out = []
    for t, st in zip(ins, streams):
        with torch.cuda.stream(st):
            out.append(both(*t))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for u, v in zip(out, ref) for a, b in zip(u, v))
    held = [t.clone() for t in ins[0]]
    with torch.cuda.stream(streams[0]):
        both(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(*held)
    for i in (1, 2, 0, 1):
        for h, t in zip(held, ins[i]):
            h.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, ref[i]))
        assert all(torch.equal(a, b) for a, b in zip(both(*ins[i]), ref[i]))


def test_quantized_layers():
    """from_momoe, to_int4: the values that `quantize` gives, and those of a `MoE` with its router; state moves as it is."""
    D, H, N, K, M = 96, 160, 4, 2, 30
    g = torch.Generator().manual_seed(3)
    moe = momoe_amd.MoE(D, H, N, K, 0, Wg_DN=torch.randn(D, N, generator=g).to(DEV), Wl1_ND2H=torch.randn(N, D, 2 * H, generator=g).to(DEV),
                        Wl2_NHD=torch.randn(N, H, D, generator=g).to(DEV))
    x = _x(M, D).view(1, M, D).to(DEV)
    with torch.no_grad():
        serving = moe.to_int4(group_size=64)
        y = serving(x)
        _, mask, s = moe.router(x, moe.biases_N)
        layer = momoe_amd.MoMoEInt4.from_momoe(moe.momoe, 64)
        assert torch.equal(layer(x, mask, s)[0], y)
        for W, (q, scale, zero) in zip((moe.momoe.Wl1_ND2H, moe.momoe.Wl2_NHD), ((layer.weights()[i], layer.weights()[i + 1], layer.weights()[4 + i // 2]) for i in (0, 2))):
            v = oracle.int4_weights(q.cpu(), scale.cpu(), zero.cpu(), 64)
            step = scale.cpu().double().repeat_interleave(64, 1)[:, :W.shape[1]]
            # half a step, half a step of a zero that lies between two codes at either end, and the ends: 15 steps of a scale off by 2^-9
            assert ((v - W.detach().cpu().double()).abs() <= step * (0.5 + 0.5 + 15 * 2.0 ** -8)).all()
        other = momoe_amd.MoMoEInt4(D, H, N, K, *_on(_weights((N,), D, H, 64, seed=9)), group_size=64)
        other.load_state_dict(copy.deepcopy(layer.state_dict()))
        for module in (other, copy.deepcopy(layer), copy.deepcopy(layer).to(torch.bfloat16), copy.deepcopy(layer).cpu().to(DEV)):
            assert torch.equal(module(x, mask, s)[0], y)


def test_traced_layers():
    D, H, N, K, group = 96, 64, 4, 2, 32
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, K, *_on(w), group_size=group)
    block = momoe_amd.FeedForwardInt4(D, H, *[t[0] for t in _on(w)], group_size=group)
    args = lambda M: (_x(M, D).view(1, M, D).to(DEV), *[t.to(DEV) for t in make_routing(M, N, K, seed=M)])
    traced, dense = torch.jit.trace(layer, args(10)), torch.jit.trace(block, args(10)[:1])
    for M in (10, 3, 300):
        a = args(M)
        assert all(torch.equal(u, v) for u, v in zip(layer(*a), traced(*a))) and torch.equal(block(a[0]), dense(a[0]))


@pytest.mark.parametrize("M", [1, 100])
def test_weights_past_32_bit_offsets(M):
    """The last of 72 experts, behind 4.5 GiB of others' codes, does what it does alone."""
    N, D, H, group = 72, 8192, 5376, 128
    w = _weights((1,), D, H, group)
    alone = momoe_amd.MoMoEInt4(D, H, 1, 1, *_on(w), group_size=group)
    many = []
    for t in w:
        big = torch.zeros(N, *t.shape[1:], dtype=t.dtype, device=DEV)
        big[-1] = t[0].to(DEV)
        many.append(big)
    last = momoe_amd.MoMoEInt4(D, H, N, 1, *many, group_size=group)
    del many
    x, s = _x(M, D).view(1, M, D).to(DEV), torch.rand(1, M, device=DEV) + 0.5
    mask = torch.zeros(N, M, dtype=torch.int32, device=DEV)
    mask[-1] = 1
    y, sizes = last(x, mask, s.expand(N, M))
    want, _ = alone(x, mask[-1:], s)
    assert sizes[-1] == M and want.norm() > 0
    # (the two may share a contraction among as many wavefronts or not: sums in another order)
    assert (y - want).double().norm() <= 2.0 ** -8 * want.double().norm()


def test_refusals():
    D, H, N, K, M, group = 96, 64, 4, 2, 10, 32
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, K, *_on(w), group_size=group)
    block = momoe_amd.FeedForwardInt4(D, H, *[t[0] for t in _on(w)], group_size=group)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    for a in ((x, mask, s.clone().requires_grad_()), (x.clone().requires_grad_(), mask, s)):
        with pytest.raises(RuntimeError, match="no_grad"):
            layer(*a)
        with torch.no_grad():
            layer(*a)
    with pytest.raises(RuntimeError, match="no_grad"):
        block(x.clone().requires_grad_())
    for a in ((x, mask[:, :9], s), (x, mask, s[:3]), (x, mask, s[:, :9])):
        with pytest.raises(RuntimeError, match="must be"):
            layer(*a)
    for a in ((x[0], mask, s), (x[:, :, :64], mask, s), (x, mask[:3], s)):
        with pytest.raises(AssertionError):
            layer(*a)
    held = layer.Wl1_packed, layer.Wl1_words, layer.Wl2_packed, layer.Wl2_words
    for k in (0, -1):
        with pytest.raises(RuntimeError, match="at least 1"):
            torch.ops.momoe.experts_int4(x, *held, mask, s, k, H, group, False)
    for bad in (x[:, :, :64], x[0, 0, 0]):
        with pytest.raises(AssertionError):
            block(bad)
    held = block.Wl1_packed, block.Wl1_words, block.Wl2_packed, block.Wl2_words
    for h, g in ((32, group), (H, 64), (H, 16), (0, group)):
        with pytest.raises(AssertionError):
            torch.ops.momoe.feed_forward_int4(x, *held, h, g)


@pytest.mark.parametrize("M", [3, 40, 1100])
def test_weights_of_nan_and_infinity_reach_the_results(M):
    """A weight of the first matrix reaches every result, one of the second its column."""
    D, H, N = 288, 160, 2
    g = torch.Generator().manual_seed(4)
    W1, W2 = torch.randn(N, D, 2 * H, generator=g) / D ** 0.5, torch.randn(N, H, D, generator=g) / H ** 0.5
    x = _x(M, D).view(1, M, D).to(DEV)
    mask, s = torch.ones(N, M, dtype=torch.int32, device=DEV), torch.ones(N, M, device=DEV)
    for value in ("nan", "inf", "-inf"):
        for first in (True, False):
            V1, V2 = W1.clone(), W2.clone()
            (V1 if first else V2)[0, 70, 33] = float(value)
            moe = momoe_amd.MoMoE(D, H, N, N, 0, Wl1_ND2H=V1.to(DEV), Wl2_NHD=V2.to(DEV))
            ffn = momoe_amd.FeedForward(D, H, 0, V1[0].to(DEV), V2[0].to(DEV))
            for y in (momoe_amd.MoMoEInt4.from_momoe(moe, 64)(x, mask, s)[0], ffn.to_int4(64)(x)):
                hit = torch.zeros(D, dtype=torch.bool, device=DEV)
                hit[:] = first
                hit[33] = True
                assert not y[..., hit].isfinite().any() and y[..., ~hit].isfinite().all()


def test_pitches_that_are_copied():
    """Rows of x at pitches that the kernels do not take: no multiple of 8, 4 GiB of rows and more, 2^22 elements and more."""
    D, H, N, group = 32, 64, 2, 32
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, 1, *_on(w), group_size=group)
    block = momoe_amd.FeedForwardInt4(D, H, *[t[0] for t in _on(w)], group_size=group)
    for M, width, at in ((70, D + 4, 0), (70, D + 30, 6), (1 << 20, 2080, 2080 - D), (3, (1 << 22) + 8, 8)):
        x = torch.randn(M, D, device=DEV, dtype=torch.bfloat16)
        view = torch.zeros(M, width, device=DEV, dtype=torch.bfloat16)[:, at:at + D]
        view.copy_(x)
        mask = torch.zeros(N, M, dtype=torch.int32, device=DEV)
        mask[torch.arange(M, device=DEV) % N, torch.arange(M, device=DEV)] = 1
        s = torch.rand(N, M, device=DEV)
        assert torch.equal(layer(view.unsqueeze(0), mask, s)[0], layer(x.unsqueeze(0), mask, s)[0]) and torch.equal(block(view), block(x))


@pytest.mark.parametrize("D,H", [(4096, 32), (32, 4096)])
def test_tokens_past_32_bit_offsets(D, H):
    """x, y and ys, or h, of more than 4 GiB: rows at the start, at the end and where offsets pass 2^31 and 2^32.  Experts of such an x take
    tiles of 32 rows."""
    M, N, group = (1 << 19) + 45, 2, 64
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, 1, *_on(w), group_size=group)
    block = momoe_amd.FeedForwardInt4(D, H, *[t[0] for t in _on(w)], group_size=group)
    assert momoe_amd._hip._lib.momoe_int4_tile_rows(M, D, H, N) == 64
    x = torch.randn(1, M, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=torch.bfloat16)
    at = torch.arange(M, device=DEV)
    mask, s = torch.zeros(N, M, dtype=torch.int32, device=DEV), torch.rand(N, M, device=DEV) + 0.5
    mask[at % N, at] = 1
    edge = [e // (c * p) for c in {D, H} for p in (2, 4) for e in (1 << 31, 1 << 32, 1 << 33)]
    rows = torch.cat([torch.arange(max(0, e - 20), min(M, e + 20)) for e in [0, M] + [e for k in (1, 2) for e in (v * k for v in edge) if e < M]]).unique()
    y, sizes = layer(x, mask, s)
    assert torch.equal(sizes, mask.sum(1)) and y.isfinite().all()
    for i in range(N):
        mine = rows[rows % N == i]
        want, off = _block(x[0, mine].cpu().double(), [t[i] for t in w], group)
        sr = s[i, mine].cpu().double()[:, None]
        _check(y[0, mine], sr * want, sr * off + (sr * want).abs() * 8 * E)
    _check(block(x)[0, rows], *_block(x[0, rows].cpu().double(), [t[0] for t in w], group))


def _with_room(n, dtype, value=7):
    """n values and room behind them; how to tell that it keeps its bits."""
    t = torch.full((n + 4096,), value, device=DEV, dtype=dtype)
    return t, lambda: bool((t[n:] == value).all())


def test_laying_weights_out_leaves_what_lies_behind():
    lib, st = momoe_amd._hip._lib, torch.cuda.current_stream().cuda_stream
    for N, R, C, halves, group in ((1, 32, 32, 2, 32), (3, 160, 96, 2, 64), (2, 288, 80, 1, 128), (5, 128, 16, 1, 32)):
        codes, scale, _, _, zero, _ = _on(_weights((N,), R, C // 2, group))
        nb, nw = lib.momoe_int4_weight_bytes(N, R, C), lib.momoe_int4_scale_words(N, R, C, group)
        (packed, same), (words, same_words) = _with_room(nb, torch.uint8), _with_room(nw, torch.int32)
        assert lib.momoe_int4_pack_weights(codes.data_ptr(), scale.data_ptr(), momoe_amd._hip._TYPES[scale.dtype], zero.data_ptr(), N, R, C, halves, group,
                                           packed.data_ptr(), words.data_ptr(), st) == 0
        torch.cuda.synchronize()
        assert same() and same_words()
        want = momoe_amd._hip.int4_pack_weights(codes, scale, zero, halves, group)
        assert torch.equal(packed[:nb], want[0]) and torch.equal(words[:nw], want[1])


@pytest.mark.parametrize("M,D,H", [(1, 96, 64), (16, 160, 2080), (17, 288, 96), (50, 2080, 160), (16, 4096, 1120), (300, 1056, 160), (1000, 288, 160), (2100, 160, 96)])
def test_the_dense_block_leaves_what_lies_behind(M, D, H):
    lib, st, group = momoe_amd._hip._lib, torch.cuda.current_stream().cuda_stream, 64
    w = _weights((), D, H, group)
    block, x = momoe_amd.FeedForwardInt4(D, H, *_on(w), group_size=group), _x(M, D).to(DEV)
    need = lib.momoe_int4_ffn_workspace_bytes(M, D, H)
    (h, h_same), (y, y_same), (ws, ws_same) = _with_room(lib.momoe_int4_h_rows(M, 1) * H, torch.bfloat16), _with_room(M * D, torch.bfloat16), _with_room(need, torch.uint8)
    P = [t.data_ptr() for t in (block.Wl1_packed, block.Wl1_words, block.Wl2_packed, block.Wl2_words)]
    assert lib.momoe_int4_ffn_fwd(x.data_ptr(), D, *P, group, h.data_ptr(), y.data_ptr(), ws.data_ptr() if need else None, need, M, D, H, st) == 0
    torch.cuda.synchronize()
    assert h_same() and y_same() and ws_same() and torch.equal(y[:M * D].view(M, D), block(x))


@pytest.mark.parametrize("M,D,H,N,K,rows", [(1, 96, 64, 4, 2, 32), (7, 288, 160, 8, 2, 32), (40, 96, 160, 2, 1, 32), (7, 288, 160, 8, 2, 64), (100, 1056, 352, 8, 2, 64),
                                            (300, 288, 416, 5, 2, 64), (3000, 160, 96, 3, 1, 64), (20, 1056, 352, 8, 2, 64), (20, 96, 1056, 8, 2, 64)])
def test_the_experts_leave_what_lies_behind(M, D, H, N, K, rows):
    """h with its second half, sums of slices, ys and y; of either height of tiles, whatever suits the sizes."""
    hip, st, group = momoe_amd._hip, torch.cuda.current_stream().cuda_stream, 32
    lib, msum = hip._lib, M * K
    w = _weights((N,), D, H, group)
    layer, x = momoe_amd.MoMoEInt4(D, H, N, K, *_on(w), group_size=group), _x(M, D).to(DEV)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    ib = hip.index_build(mask, K, tile_rows=rows)
    n1, n2 = lib.momoe_int4_slices(msum, N, 2 * H, D, rows), lib.momoe_int4_slices(msum, N, D, H, rows)
    need = n1 * msum * 2 * H * 4 if n1 > 1 else 0
    (h, h_same), (ys, ys_same) = _with_room(lib.momoe_int4_h_rows(msum, N) * H, torch.bfloat16), _with_room(n2 * msum * D, torch.float32)
    (ws, ws_same), (y, y_same) = _with_room(need, torch.uint8), _with_room(M * D, torch.bfloat16)
    P = [t.data_ptr() for t in (layer.Wl1_packed, layer.Wl1_words, layer.Wl2_packed, layer.Wl2_words, ib["idx_Msum"], ib["tile_table"])]
    assert lib.momoe_int4_lin1_swiglu_fwd(x.data_ptr(), D, P[0], P[1], group, P[4], P[5], rows, h.data_ptr(), ws.data_ptr() if need else None, need, M, D, H, N,
                                          msum, st) == 0
    assert lib.momoe_int4_lin2_scale_fwd(h.data_ptr(), P[2], P[3], group, s.data_ptr(), s.stride(0), s.stride(1), P[4], P[5], rows, ys.data_ptr(), M, D, H, N,
                                         msum, st) == 0
    assert lib.momoe_int4_combine(ys.data_ptr(), n2, ib["inv_MK"].data_ptr(), y.data_ptr(), M, D, K, msum, st) == 0
    torch.cuda.synchronize()
    assert h_same() and ys_same() and ws_same() and y_same()
    want, off = torch.zeros(M, D, dtype=torch.float64), torch.zeros(M, D, dtype=torch.float64)
    for i in range(N):
        at = mask[i].cpu().nonzero().flatten()
        if len(at):
            out, d = _block(x[at].cpu().double(), [t[i] for t in w], group, len(at) <= 16 and msum <= 16 * N)
            sr = s[i, at].cpu().double()[:, None]
            want.index_add_(0, at, sr * out)
            off.index_add_(0, at, sr * d + (sr * out).abs() * (K + 2) * 2 * E)
    _check(y[:M * D], want, off)


def test_more_tokens_than_a_launch_has_workgroups():
    """2^24 tokens and more: with a workgroup of 256 for each of them, a launch would have 2^32 threads."""
    M, D, H, N, group = (1 << 24) + 77, 32, 32, 2, 32
    w = _weights((N,), D, H, group)
    layer = momoe_amd.MoMoEInt4(D, H, N, 1, *_on(w), group_size=group)
    x = torch.randn(1, M, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=torch.bfloat16)
    at = torch.arange(M, device=DEV)
    mask, s = torch.zeros(N, M, dtype=torch.int32, device=DEV), torch.rand(N, M, device=DEV) + 0.5
    mask[at % N, at] = 1
    y, _ = layer(x, mask, s)
    assert y.isfinite().all() and (y != 0).any(-1).all()
    rows = torch.cat([torch.arange(e - 40, e + 40) for e in (40, 1 << 22, 1 << 23, 1 << 24, M - 40)])
    for i in range(N):
        mine = rows[rows % N == i]
        want, off = _block(x[0, mine].cpu().double(), [t[i] for t in w], group)
        sr = s[i, mine].cpu().double()[:, None]
        _check(y[0, mine], sr * want, sr * off + (sr * want).abs() * 8 * E)


def test_laying_out_16_gib_of_codes():
    """As many words that 2^32 threads would take one each: the last expert as by itself."""
    N, R, C, group = 520, 4096, 16384, 128
    codes, scale, _, _, zero, _ = _on(_weights((1,), R, C // 2, group))
    many = [torch.zeros(N, *t.shape[1:], dtype=t.dtype, device=DEV) for t in (codes, scale, zero)]
    for big, t in zip(many, (codes, scale, zero)):
        big[0], big[-1] = t[0], t[0]
    assert many[0].numel() > 1 << 34
    packed, words = momoe_amd._hip.int4_pack_weights(*many, 2, group)
    want = momoe_amd._hip.int4_pack_weights(codes, scale, zero, 2, group)
    for got, one in ((packed, want[0]), (words, want[1])):
        assert torch.equal(got.view(N, -1)[0], one) and torch.equal(got.view(N, -1)[-1], one) and not got.view(N, -1)[N // 2].any()
