"""GPU: the experts in 8-bit floating point, step by step against 64 bits, and as a layer."""
import copy

import pytest
import torch

import momoe_amd
import oracle
from helpers import make_routing
from momoe_amd import _hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24


def _x(M, D, dtype=torch.bfloat16, seed=0):
    x = torch.randn(M, D, generator=torch.Generator().manual_seed(seed))
    return (x * torch.exp2(torch.randint(-6, 7, (M, 1), generator=torch.Generator().manual_seed(seed + 1)).float())).to(dtype)


def _weights(N, D, H, seed=0, lift=1.0):
    """(Wl1 e4m3, its scales, Wl2 e4m3, its scales) of N(0, 1) values: scales of any size, powers of two or not."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *size: (32 * torch.randn(*size, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = lambda *size: lift * (0.5 + torch.rand(*size, generator=g)) / 32
    b = oracle.operators.blocks
    return (rand(N, D, 2 * H), scale(N, b(D), 2, b(H)) * 2 / D ** 0.5, rand(N, H, D), scale(N, b(H), b(D)) / H ** 0.5)


def _values(W1, S1, W2, S2):
    H = W2.shape[1]
    return torch.cat([oracle.block_weights(W1[:, :, :H], S1[:, :, 0]), oracle.block_weights(W1[:, :, H:], S1[:, :, 1])], -1), \
        oracle.block_weights(W2, S2)


def _dequantized(q, codes, n):
    KB = q.shape[1] // 128
    v = q.float().cpu().double().view(len(q), KB, 128) * torch.exp2(codes[:, :KB].cpu().double() - 127)[:, :, None]
    return v.reshape(len(q), -1)[:, :n]


# ---- rows ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 128), (57, 328), (200, 96), (5, 2080)])
def test_rows_to_8_bits(rows, cols, dtype):
    """The values themselves: a power of two divides exactly, and what is left is one rounding to nearest even."""
    x = _x(rows, cols, dtype)
    x[0, : cols // 2] = 0
    if dtype != torch.float16 and rows > 2:
        x[1] *= 2.0 ** -115  # below what a scale follows
        x[2] *= 2.0 ** 100
    q, codes = _hip.fp8_quantize_rows(x.to(DEV))
    want, e = oracle.rows_in_8_bits(x)
    KB = q.shape[1] // 128
    assert torch.equal(codes[:, :KB].cpu().to(torch.int64), e + 127)
    got = q.float().cpu().double()
    assert torch.equal(got[:, :cols], want) and (got[:, cols:] == 0).all()


def test_rows_with_a_pitch_and_of_nan():
    x = _x(9, 400).to(DEV)
    q, codes = _hip.fp8_quantize_rows(x[:, 8:136])
    a, b = _hip.fp8_quantize_rows(x[:, 8:136].contiguous())
    assert torch.equal(q.view(torch.uint8), a.view(torch.uint8)) and torch.equal(codes[:, 0], b[:, 0])
    x[2, 300], x[5, 0], x[6, 399] = float("nan"), float("inf"), float("-inf")
    _, codes = _hip.fp8_quantize_rows(x)
    bad = torch.zeros(9, 4, dtype=torch.bool)
    bad[2, 2] = bad[5, 0] = bad[6, 3] = True
    assert torch.equal(codes.cpu() == 255, bad)


@pytest.mark.parametrize("N,D,H", [(1, 32, 32), (3, 160, 96), (2, 288, 416)])
def test_weights_come_back(N, D, H):
    w = _weights(N, D, H)
    layer = momoe_amd.MoMoEFP8(D, H, N, 1, *[t.to(DEV) for t in w])
    for a, b in zip(layer.weights(), w):
        assert a.dtype == b.dtype and torch.equal(a.cpu().float(), b.float())


@pytest.mark.parametrize("N,D,H", [(1, 32, 32), (3, 160, 96), (2, 288, 416)])
def test_weights_quantized(N, D, H):
    """Each 128 x 128 block of each half by the rule for rows."""
    g = torch.Generator().manual_seed(3)
    momoe = momoe_amd.MoMoE(D, H, N, 1, Wl1_ND2H=torch.randn(N, D, 2 * H, generator=g).to(DEV), Wl2_NHD=torch.randn(N, H, D, generator=g).to(DEV))
    with torch.no_grad():
        momoe.Wl2_NHD[0, :, :] = 0
    W1, S1, W2, S2 = [t.cpu() for t in momoe_amd.MoMoEFP8.from_momoe(momoe).weights()]
    src1, src2 = momoe.Wl1_ND2H.detach().cpu().double(), momoe.Wl2_NHD.detach().cpu().double()
    for src, q, scale in ((src1[:, :, :H], W1[:, :, :H], S1[:, :, 0]), (src1[:, :, H:], W1[:, :, H:], S1[:, :, 1]), (src2, W2, S2)):
        R, C = src.shape[1:]
        for i in range(scale.shape[1]):
            for j in range(scale.shape[2]):
                at = (slice(None), slice(128 * i, min(R, 128 * i + 128)), slice(128 * j, min(C, 128 * j + 128)))
                for n in range(N):
                    want, e = oracle.rows_in_8_bits(torch.cat([src[n][at[1:]].reshape(1, -1).amax(1, keepdim=True),
                                                               src[n][at[1:]].reshape(1, -1).amin(1, keepdim=True)], 1))
                    assert scale[n, i, j].double() == 2.0 ** e[0, 0].item()
                    assert torch.equal(q[n][at[1:]].float().double(), oracle.e4m3(src[n][at[1:]] / 2.0 ** e[0, 0].item()))


# ---- the products -------------------------------------------------------------------------------------------------------------
# M, D, H, N, K, Ks, skew: tiles of few rows, of up to 256; widths below, at and past a block; contractions past the blocks that are
# held at a time; experts without a token and with nearly all
SIZES = [
    (1, 32, 32, 2, 1, 0, 0), (1, 256, 128, 8, 8, 0, 0), (7, 96, 160, 4, 2, 0, 0), (50, 288, 416, 5, 2, 1, 0), (33, 2208, 64, 3, 1, 0, 0),
    (64, 64, 2208, 2, 2, 1, 0), (200, 128, 128, 16, 2, 0, 1.5),
    (300, 96, 64, 4, 2, 0, 0), (517, 288, 160, 5, 2, 1, 0), (700, 128, 416, 4, 3, 1, 2.0), (900, 640, 96, 3, 1, 0, 0),
    (150, 8320, 32, 2, 1, 0, 0), (140, 32, 8320, 2, 1, 0, 0), (150, 8192, 384, 2, 1, 0, 0), (200, 384, 1056, 3, 1, 0, 0), (700, 4224, 4192, 3, 2, 0, 0), (130, 7200, 64, 2, 1, 0, 0),
    (60, 128, 8192, 1, 1, 0, 0), (2, 8224, 2112, 12, 3, 0, 0), (90, 1056, 1024, 40, 4, 0, 0), (18, 2080, 160, 1, 1, 0, 0), (300, 128, 96, 40, 2, 0, 2.0),
    (9, 1056, 512, 8, 2, 0, 0), (9000, 64, 1280, 6, 2, 0, 0.5), (7000, 512, 288, 20, 2, 0, 0.5),
]


def _of_experts(mask):
    """(token, expert) of the sorted rows."""
    i, m = torch.nonzero(mask, as_tuple=True)
    return m, i


def _sum_error(terms, a, w, tiles):
    """How far a product of rows a and weights w may be off.  bf16 products in fp32: each of `terms` additions rounds.  8-bit
    products: of eight at a time, what lies 13 binades below the largest is cut off, at most 2^-13 of the largest each."""
    off = 2 * terms * E * (a.abs() @ w.abs())
    if tiles:
        pad = -a.shape[1] % 8
        top = lambda t: torch.nn.functional.pad(t, (0, pad)).abs().view(len(t), -1, 8).amax(-1)
        off = off + 8 * 2.0 ** -13 * (top(a) @ top(w.T).T)
    return off


@pytest.mark.parametrize("M,D,H,N,K,Ks,skew", SIZES)
def test_products(M, D, H, N, K, Ks, skew):
    mask, s = make_routing(M, N, K, Ks, seed=5, skew=skew)
    W1, S1, W2, S2 = _weights(N, D, H)
    V1, V2 = _values(W1, S1, W2, S2)
    tile_rows = _hip.fp8_tile_rows(M * K, D, H, N)
    index = _hip.index_build(mask.to(DEV), K, tile_rows=tile_rows)
    tok, exp = _of_experts(mask)
    assert torch.equal(index["idx_Msum"].cpu().long(), tok)
    xq, xc = _hip.fp8_quantize_rows(_x(M, D).to(DEV))
    p1, p2 = _hip.fp8_pack_weights(W1.to(DEV), 2), _hip.fp8_pack_weights(W2.to(DEV), 1)
    at = index["idx_Msum"], index["tile_table"]
    sd = s.T.contiguous().to(DEV).T
    if tile_rows == 32:  # the products bring their rows to 8 bits themselves
        h32 = _hip.fp8_few_lin1_swiglu_fwd(_x(M, D).to(DEV), p1, S1.to(DEV), *at, H)
        hq, hc = _hip.fp8_quantize_rows(h32)
        ys = _hip.fp8_few_lin2_scale_fwd(h32, p2, S2.to(DEV), sd, *at, D)
    else:
        hq, hc = _hip.fp8_lin1_swiglu_fwd(xq, xc, p1, S1.to(DEV), *at, D, H)
        ys = _hip.fp8_lin2_scale_fwd(hq, hc, p2, S2.to(DEV), sd, *at, D, H)
    assert torch.equal(hq.view(torch.uint8)[:, H:], torch.zeros_like(hq.view(torch.uint8)[:, H:]))
    xv, hv = _dequantized(xq, xc, D)[tok], _dequantized(hq, hc, H)
    codes = hc.cpu().long()[:, :hq.shape[1] // 128].repeat_interleave(128, 1)[:, :H]
    y = _hip.fp8_combine(ys, index["inv_MK"], D).cpu().double()
    tiles = tile_rows == 256
    total, slack = torch.zeros(M, D, dtype=torch.float64), torch.zeros(M, D, dtype=torch.float64)
    for i in range(N):
        r = exp == i
        if not r.any():
            continue
        z, dz = xv[r] @ V1[i], _sum_error(D, xv[r], V1[i], tiles)
        a, b, da, db = z[:, :H], z[:, H:], dz[:, :H], dz[:, H:]
        sig = torch.sigmoid(b)
        h = a * b * sig
        # |d(b sig)/db| <= 1.1; exp and reciprocal of the sigmoid, the products: some 16 + |b| roundings
        dh = da * (b * sig).abs() + (a.abs() + da) * db * 1.1 + h.abs() * (16 + b.abs()) * 2 * E
        # half a step of e4m3, of which the least is 2^-9 of the scale
        unit = torch.exp2(codes[r].double() - 127)
        bound = dh + (h.abs() + dh) * 2.0 ** -4 + unit * 2.0 ** -10
        assert ((hv[r] - h).abs() <= bound).all(), ((hv[r] - h).abs() / bound).max()
        # the scale is the least that will do, with the slack of what it was taken from
        for c0 in range(0, H, 128):
            top, dt = h[:, c0:c0 + 128].abs().amax(1), dh[:, c0:c0 + 128].amax(1)
            u = unit[:, c0]
            assert ((top - dt).clamp_min(2.0 ** -100) <= 448 * u).all() and ((top + dt >= 224 * u) | (u <= 2.0 ** -108)).all()
        # rows of y from the h that the first product left: packets are 15 bits of the largest of eight
        out, do = hv[r] @ V2[i], _sum_error(H, hv[r], V2[i], tiles)
        sr = s[i, tok[r]].double()[:, None]
        total.index_add_(0, tok[r], sr * out)
        grouped = lambda t: t.view(len(t), D // 32, 2, 4, 4).transpose(2, 3).reshape(len(t), D // 8, 8).amax(-1).repeat_interleave(8, 1) \
            .view(len(t), D // 32, 4, 2, 4).transpose(2, 3).reshape(len(t), D)
        slack.index_add_(0, tok[r], sr * do + 2.0 ** -13 * grouped(sr * (out.abs() + do)) + (sr * out).abs() * 4 * K * E)
    slack += total.abs() * 2.0 ** -8 + 1e-37
    assert torch.isfinite(y).all() and ((y - total).abs() <= slack).all(), ((y - total).abs() / slack).max()


@pytest.mark.parametrize("M", [1, 1000])
def test_weights_past_32_bit_offsets(M):
    """The last of 40 experts, behind 5 GiB of others' weights, does what it does alone."""
    N, D, H = 40, 8192, 8192
    w = _weights(1, D, H)
    alone = momoe_amd.MoMoEFP8(D, H, 1, 1, *[t.to(DEV) for t in w])
    many = []
    for t in w:
        big = torch.zeros(N, *t.shape[1:], dtype=t.dtype, device=DEV)
        big[-1] = t[0].to(DEV)
        many.append(big)
    last = momoe_amd.MoMoEFP8(D, H, N, 1, *many)
    del many
    x, s = _x(M, D).view(1, M, D).to(DEV), torch.rand(1, M, device=DEV) + 0.5
    mask = torch.zeros(N, M, dtype=torch.int32, device=DEV)
    mask[-1] = 1
    y, sizes = last(x, mask, s.expand(N, M))
    want, _ = alone(x, mask[-1:], s)
    assert sizes[-1] == M and want.norm() > 0 and torch.equal(y, want)


def _layer(D, H, N, K, seed=0):
    w = _weights(N, D, H, seed)
    return momoe_amd.MoMoEFP8(D, H, N, K, *[t.to(DEV) for t in w]), _values(*w)


def _close(y, ref):
    """Half a step of bf16, and values of h next to a border that fell on its other side: were one in 256 off by a whole step (2^-3
    of itself), 2^-7 of the norm."""
    y = y.detach().cpu().double().reshape(ref.shape)
    assert torch.isfinite(y).all() and (y - ref).norm() <= (2.0 ** -8 + 2.0 ** -7) * ref.norm(), (y - ref).norm() / ref.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16, torch.float64])
@pytest.mark.parametrize("B,S,D,H,N,K,Ks", [(1, 1, 128, 64, 4, 2, 0), (3, 7, 160, 288, 6, 3, 1), (2, 200, 288, 96, 4, 2, 0)])
def test_layer(B, S, D, H, N, K, Ks, dtype):
    layer, (V1, V2) = _layer(D, H, N, K)
    mask, s = make_routing(B * S, N, K, Ks, seed=2)
    x = _x(B * S, D, dtype)
    y, sizes = layer(x.view(B, S, D).to(DEV), mask.to(DEV), s.to(DEV))
    assert y.shape == (B, S, D) and y.dtype == torch.bfloat16 and torch.equal(sizes.cpu(), mask.sum(1))
    src = x.to(torch.bfloat16) if dtype == torch.float64 else x
    _close(y, oracle.experts_fp8(src.double(), V1, V2, mask, s))


@pytest.mark.parametrize("M", [12, 400])
def test_strides_and_places_of_the_arguments(M):
    D, H, N, K = 96, 64, 4, 2
    layer, _ = _layer(D, H, N, K)
    mask, s = make_routing(M, N, K, seed=2)
    x = _x(M, D).view(1, M, D).to(DEV)
    ref, sizes = layer(x, mask.to(DEV), s.to(DEV))
    wide = torch.zeros(1, 2 * M, D + 24, device=DEV, dtype=torch.bfloat16)
    wide[:, ::2, 3:D + 3] = x
    for args in ((wide[:, ::2, 3:D + 3], mask.to(DEV), s.contiguous().to(DEV)), (x, mask.T.contiguous().to(DEV).T, s.to(DEV)),
                 (x, mask.bool().to(DEV), s.double().to(DEV)), (x, mask, s),
                 (x.transpose(1, 2).contiguous().transpose(1, 2), mask.to(DEV), s.repeat(1, 2).to(DEV)[:, :M])):
        y, n = layer(*args)
        assert torch.equal(y, ref) and torch.equal(n, sizes)
    y, n = layer(x.cpu(), mask, s)
    assert y.device.type == "cpu" and torch.equal(y, ref.cpu())
    zero = layer(x[:, :0], mask[:, :0].to(DEV), s[:, :0].to(DEV))
    assert zero[0].shape == (1, 0, D) and zero[1].abs().sum() == 0


@pytest.mark.parametrize("M", [40, 600])
def test_tokens_of_nan_infinity_and_zero(M):
    """They stay with themselves; the others keep their bits."""
    D, H, N, K = 288, 160, 4, 2
    layer, _ = _layer(D, H, N, K)
    mask, s = make_routing(M, N, K, seed=2)
    x = _x(M, D).view(1, M, D).to(DEV)
    ref, _ = layer(x, mask.to(DEV), s.to(DEV))
    bad = x.clone()
    bad[0, 3, 100], bad[0, 17, 200], bad[0, M - 1, 0], bad[0, 20] = float("nan"), float("inf"), float("-inf"), 0
    y, _ = layer(bad, mask.to(DEV), s.to(DEV))
    assert y[0, [3, 17, M - 1]].isnan().all() and (y[0, 20] == 0).all()
    keep = torch.ones(M, dtype=torch.bool)
    keep[[3, 17, 20, M - 1]] = False
    assert torch.equal(y[0, keep.to(DEV)], ref[0, keep.to(DEV)])


@pytest.mark.parametrize("M", [40, 600])
def test_routing_that_is_not_k_of_n(M, monkeypatch):
    """Too few experts: what is missing is absent.  Too many: zeros.  CHECK_ROUTING raises for both."""
    D, H, N, K = 96, 64, 4, 2
    layer, (V1, V2) = _layer(D, H, N, K)
    mask, s = make_routing(M, N, K, seed=2)
    x = _x(M, D)
    few = mask.clone()
    few[:, 5] = 0
    few[mask[:, 6].nonzero()[0], 6] = 0
    y, _ = layer(x.view(1, M, D).to(DEV), few.to(DEV), s.to(DEV))
    _close(y, oracle.experts_fp8(x, V1, V2, few, s))
    assert (y[0, 5] == 0).all()
    many = torch.ones_like(mask)
    assert (layer(x.view(1, M, D).to(DEV), many.to(DEV), s.to(DEV))[0] == 0).all()
    monkeypatch.setattr(momoe_amd.experts, "CHECK_ROUTING", True)
    for m in (few, many):
        with pytest.raises(RuntimeError, match="exactly K"):
            layer(x.view(1, M, D).to(DEV), m.to(DEV), s.to(DEV))


def test_traced_layer():
    layer, _ = _layer(96, 64, 4, 2)
    args = lambda M: (_x(M, 96).view(1, M, 96).to(DEV), *[t.to(DEV) for t in make_routing(M, 4, 2, seed=M)])
    traced = torch.jit.trace(layer, args(10))
    for M in (10, 3, 300):
        a = args(M)
        assert all(torch.equal(u, v) for u, v in zip(layer(*a), traced(*a)))


def test_refusals():
    D, H, N, K, M = 96, 64, 4, 2, 10
    layer, _ = _layer(D, H, N, K)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    for a in ((x, mask, s.clone().requires_grad_()), (x.clone().requires_grad_(), mask, s)):
        with pytest.raises(RuntimeError, match="no_grad"):
            layer(*a)
        with torch.no_grad():
            layer(*a)
    for a in ((x, mask[:3], s), (x, mask[:, :9], s), (x, mask, s[:3]), (x, mask, s[:, :9])):
        with pytest.raises(RuntimeError, match="must be"):
            layer(*a)
    held = layer.Wl1_packed, layer.Wl1_scale_bits, layer.Wl2_packed, layer.Wl2_scale_bits
    for k in (0, -1):
        with pytest.raises(RuntimeError, match="at least 1"):
            torch.ops.momoe.experts_fp8(x, *held, mask, s, k, H, False)
    for bad in (x[0], x[:, :, :64], torch.cat([x, x, x], -1)):
        with pytest.raises(AssertionError):
            layer(bad, mask, s)


def test_state_moves_as_it_is():
    D, H, N, K, M = 96, 160, 4, 2, 30
    layer, _ = _layer(D, H, N, K)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    ref, _ = layer(x, mask, s)
    other, _ = _layer(D, H, N, K, seed=9)
    other.load_state_dict(copy.deepcopy(layer.state_dict()))
    for module in (other, copy.deepcopy(layer), copy.deepcopy(layer).to(torch.bfloat16), copy.deepcopy(layer).cpu().to(DEV)):
        assert torch.equal(module(x, mask, s)[0], ref)
    with pytest.raises(RuntimeError, match="no CPU compute path"):
        copy.deepcopy(layer).cpu()(x, mask, s)


@pytest.mark.parametrize("M", [3, 30, 500])
def test_same_bits_each_time_on_another_stream_and_in_a_graph(M):
    D, H, N, K = 288, 160, 8, 2
    layer, _ = _layer(D, H, N, K)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    ref, _ = layer(x, mask, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            y, _ = layer(x, mask, s)
    torch.cuda.synchronize()
    assert torch.equal(y, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, n = layer(x, mask, s)
    for seed in (5, 6, 7):
        m2, s2 = [t.to(DEV) for t in make_routing(M, N, K, seed=seed)]
        x2 = _x(M, D, seed=seed).view(1, M, D).to(DEV)
        want, sizes = layer(x2, m2, s2)
        x.copy_(x2), mask.copy_(m2), s.copy_(s2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(n, sizes)


def test_trained_with_a_balance_loss_then_served_in_8_bits():
    """The operators together: a step of a `MoE` with its balance loss, its experts then quantized and served."""
    D, H, N, K, Ks, B, S = 160, 96, 8, 3, 1, 2, 60
    g = torch.Generator().manual_seed(9)
    moe = momoe_amd.MoE(D, H, N, K, Ks, balance="sequence", Wg_DN=(torch.randn(D, N, generator=g) / D ** 0.5).to(DEV),
                        Wl1_ND2H=(torch.randn(N, D, 2 * H, generator=g) / D ** 0.5).to(DEV),
                        Wl2_NHD=(torch.randn(N, H, D, generator=g) / H ** 0.5).to(DEV))
    x = torch.randn(B, S, D, generator=g).to(DEV, torch.bfloat16)
    y, loss = moe(x)
    (y.float().pow(2).mean() + 0.01 * loss).backward()
    with torch.no_grad():
        for p in (moe.router.Wg_DN, moe.momoe.Wl1_ND2H, moe.momoe.Wl2_NHD):
            assert torch.isfinite(p.grad).all()
            p.add_(p.grad, alpha=-1e-2)
    served = moe.to_fp8()
    with torch.no_grad():
        _, mask, s = moe.router(x, moe.biases_N)
        before = moe.biases_N.clone()
        got = served(x)
    assert torch.equal(before, served.biases_N)
    W1, S1, W2, S2 = [t.cpu() for t in served.momoe.weights()]
    _close(got, oracle.experts_fp8(x.cpu().view(-1, D), *_values(W1, S1, W2, S2), mask.cpu(), s.cpu()))
    with torch.no_grad():  # and near the layer in bf16: weights, x and h each off by 2^-4 / sqrt(3) of themselves at most
        ref, _ = moe.momoe(x, mask, s)
    assert (got.float() - ref.float()).norm() <= 0.1 * ref.float().norm()
    with pytest.raises(RuntimeError, match="no_grad"):
        served(x)


@pytest.mark.parametrize("bits", [0x7FC00000, 0x7FFFFFFF, -1])
@pytest.mark.parametrize("M", [12, 400])
def test_nan_of_any_bits_in_gate_weights_and_scales(M, bits):
    """A NaN stays one whatever its payload, and stays with the results that it is part of."""
    D, H, N, K, e = 288, 160, 4, 2, 1
    w = [t.to(DEV) for t in _weights(N, D, H)]
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    layer = lambda *held: momoe_amd.MoMoEFP8(D, H, N, K, *held)
    ref, _ = layer(*w)(x, mask, s)
    held = mask[e].bool()
    rows, cols = held[:, None].expand(M, D), torch.arange(D, device=DEV) // 128

    def poisoned(t, at):
        t = t.clone(memory_format=torch.contiguous_format)
        t.view(torch.int32)[at] = bits
        return t

    def check(y, nan):
        assert torch.equal(y[0].isnan(), nan) and torch.equal(y[0][~nan], ref[0][~nan])

    m = held.nonzero()[3, 0]
    check(layer(*w)(x, mask, poisoned(s, (e, m)))[0], (torch.arange(M, device=DEV) == m)[:, None].expand(M, D))
    check(layer(w[0], w[1], w[2], poisoned(w[3], (e, 1, 1)))(x, mask, s)[0], rows & (cols == 1))
    for half in range(2):  # h is brought to 8 bits again: all that follows from it
        check(layer(w[0], poisoned(w[1], (e, 2, half, 1)), w[2], w[3])(x, mask, s)[0], rows)


@pytest.mark.parametrize("byte", [0x7F, 0xFF])
@pytest.mark.parametrize("M", [12, 400])
def test_nan_among_the_weights(M, byte):
    """Of Wl1: all results of the expert's tokens.  Of Wl2: the eight columns that share a packet with its own."""
    D, H, N, K, e = 288, 160, 4, 2, 1
    w = [t.to(DEV) for t in _weights(N, D, H)]
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    ref, _ = momoe_amd.MoMoEFP8(D, H, N, K, *w)(x, mask, s)
    rows, col = mask[e].bool()[:, None].expand(M, D), torch.arange(D, device=DEV)
    for which, at, nan in ((0, (e, 200, 70), rows), (0, (e, 31, H + 150), rows),
                           (2, (e, 150, 201), rows & (col // 32 == 201 // 32) & (col % 16 // 4 == 201 % 16 // 4))):
        bad = [t.clone() for t in w]
        bad[which].view(torch.uint8)[at] = byte
        y, _ = momoe_amd.MoMoEFP8(D, H, N, K, *bad)(x, mask, s)
        assert torch.equal(y[0].isnan(), nan) and torch.equal(y[0][~nan], ref[0][~nan])


@pytest.mark.parametrize("M", [300_000, 540_000])
def test_tokens_past_32_bit_offsets(M):
    """Tokens of 2.3 GiB and of 4.1 GiB in 8 bits: the last of them against 64 bits."""
    D, H = 8192, 32
    layer, (V1, V2) = _layer(D, H, 1, 1)
    x = torch.randn(1, M, D, device=DEV, dtype=torch.bfloat16)
    s = torch.rand(1, M, device=DEV) + 0.5
    mask = torch.ones(1, M, dtype=torch.int32, device=DEV)
    y, sizes = layer(x, mask, s)
    assert sizes.item() == M
    for at in (slice(0, 8), slice(M // 2, M // 2 + 8), slice(M - 8, M)):
        _close(y[0, at], oracle.experts_fp8(x[0, at].cpu().double(), V1, V2, mask[:, at].cpu(), s[:, at].cpu()))


@pytest.mark.parametrize("M,D,H,N,K", [(700, 8224, 288, 3, 2), (600, 160, 8320, 2, 2), (2000, 8224, 64, 40, 2)])
def test_many_rows_in_tiles_of_few(M, D, H, N, K):
    """Contractions past what the tall tiles take: more tiles than experts."""
    assert _hip.fp8_tile_rows(M * K, D, H, N) == 32 and M * K > 32 * N
    test_products(M, D, H, N, K, 0, 0.5)


def test_weights_anywhere_in_memory():
    """Views into one buffer, off the boundaries that the kernels read by."""
    D, H, N, K, M = 96, 64, 4, 2, 30
    w = _weights(N, D, H)
    mask, s = [t.to(DEV) for t in make_routing(M, N, K, seed=2)]
    x = _x(M, D).view(1, M, D).to(DEV)
    ref, _ = momoe_amd.MoMoEFP8(D, H, N, K, *[t.to(DEV) for t in w])(x, mask, s)
    placed = []
    for t in w:
        raw = torch.empty(t.numel() * t.element_size() + 4, dtype=torch.uint8, device=DEV)[4:]
        raw.copy_(t.contiguous().view(torch.uint8).reshape(-1))
        placed.append(raw.view(t.dtype).view(t.shape))
        assert placed[-1].data_ptr() % 16 == 4
    assert torch.equal(momoe_amd.MoMoEFP8(D, H, N, K, *placed)(x, mask, s)[0], ref)
    momoe = momoe_amd.MoMoE(D, H, N, K)
    ref = momoe_amd.MoMoEFP8.from_momoe(momoe).weights()
    for name in ("Wl1_ND2H", "Wl2_NHD"):
        p = getattr(momoe, name)
        off = torch.empty(p.numel() + 2, dtype=p.dtype, device=DEV)[2:].view(p.shape)
        p.data = off.copy_(p.data)
        assert p.data_ptr() % 16 == 4
    for a, b in zip(momoe_amd.MoMoEFP8.from_momoe(momoe).weights(), ref):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("M,D,H", [
    *[(9000, 2080, H) for H in (96, 256, 384, 512, 640)],  # the second product's tiles, of 1 to 5 blocks of its contraction
    *[(9000, D, 1120) for D in (96, 256, 384, 512, 640)],  # the first one's
    (9000, 1120, 1120),
])
def test_tiles_one_behind_the_other(M, D, H):
    """Two tiles and more a workgroup do what they do in calls of fewer tokens, a tile a workgroup: a row's results are its own."""
    N, K = 6, 2
    layer, (V1, V2) = _layer(D, H, N, K)
    mask, s = make_routing(M, N, K, seed=2, skew=0.5)
    x = _x(M, D)
    row_tiles = lambda m: ((m.sum(1) + 255) // 256).sum().item()
    blocks = {"first": -(-H // 128), "second": -(-D // 256)}
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert max(blocks.values()) * row_tiles(mask) > 2 * cus
    assert _hip.fp8_tile_rows(M * K, D, H, N) == _hip.fp8_tile_rows(500 * K, D, H, N) == 256
    y, sizes = layer(x.view(1, M, D).to(DEV), mask.to(DEV), s.to(DEV))
    assert torch.equal(sizes.cpu(), mask.sum(1))
    for at in range(0, M, 500):
        part = slice(at, at + 500)
        assert max(blocks.values()) * row_tiles(mask[:, part]) <= cus
        few, _ = layer(x[part].view(1, -1, D).to(DEV), mask[:, part].contiguous().to(DEV), s[:, part].to(DEV))
        assert torch.equal(few[0], y[0, part])
    at = slice(M - 200, M)
    _close(y[0, at], oracle.experts_fp8(x[at], V1, V2, mask[:, at], s[:, at]))
