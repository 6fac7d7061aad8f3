"""GPU: the dense SwiGLU block, forward and backward, against the formulas in 64 bits."""
import copy

import pytest
import torch

import momoe_amd
import oracle
from gpu_util import gz_and_error, large_gate_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E, B = 2.0 ** -24, 2.0 ** -8  # half a step of fp32, of bf16


def _inputs(M, D, H, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *size: torch.randn(*size, generator=g)
    lift = torch.exp2(torch.randint(-3, 4, (M, 1), generator=g).float())
    return [t.to(torch.bfloat16) for t in (r(M, D) * lift, r(D, 2 * H) * 2 / D ** 0.5, r(H, D) / H ** 0.5, r(M, D))]


def _block(W1, W2, save=0):
    return momoe_amd.FeedForward(W2.shape[1], W2.shape[0], save, Wl1_D2H=W1.to(DEV), Wl2_HD=W2.to(DEV))


def _bounds(x, W1, W2, Gy):
    """[(value, how far it may be off)] of y, Gx, GW1, GW2, the last rounding included.  A sum of n products is off by 2 (n + 8) E of their
    magnitudes at most; h and gz are rounded to bf16 before they are multiplied."""
    x, W1, W2, Gy = [t.double() for t in (x, W1, W2, Gy)]
    H = W2.shape[0]
    sums = lambda a, b: a.abs() @ b.abs() * 2 * (a.shape[1] + 8) * E
    a, b, h, y = oracle.swiglu_block(x, W1, W2)
    d = sums(x, W1)
    da, db = d[:, :H], d[:, H:]
    sig = torch.sigmoid(b)
    silu, slope = b * sig, sig * (1 + b * (1 - sig))
    # |silu'| <= 1.1, |silu''| <= 0.5; exp and reciprocal of the sigmoid, the products: some 16 + |b| roundings
    few = (16 + b.abs()) * 2 * E
    dsilu, dslope = 1.1 * db + silu.abs() * few, 0.5 * db + (slope.abs() + silu.abs() + 1) * few
    rounded = lambda v, dv: dv + (v.abs() + dv) * B
    dh = da * (silu.abs() + dsilu) + a.abs() * dsilu + h.abs() * 8 * E
    # (of up to 16 rows the forward has what the rounding of h leaves, in bf16, too)
    dhy = dh + (h.abs() + dh) * B * B if len(x) <= 16 else rounded(h, dh)
    dh = rounded(h, dh)
    u, du = Gy @ W2.T, sums(Gy, W2.T)
    ga, gb = u * silu, u * a * slope
    dga = rounded(ga, du * (silu.abs() + dsilu) + u.abs() * dsilu + ga.abs() * 8 * E)
    dgb = rounded(gb, (du * (a.abs() + da) + u.abs() * da) * (slope.abs() + dslope) + (u * a).abs() * dslope + gb.abs() * 8 * E)
    gz, dgz = torch.cat([ga, gb], 1), torch.cat([dga, dgb], 1)
    Gx, GW1, GW2 = oracle.swiglu_block_gradients(x, W1, W2, Gy)
    out = [(y, dhy @ W2.abs() + 2 * sums(h.abs() + dhy, W2)), (Gx, dgz @ W1.abs().T + sums(gz.abs() + dgz, W1.T)),
           (GW1, x.abs().T @ dgz + sums(x.T, gz.abs() + dgz)), (GW2, dh.T @ Gy.abs() + sums((h.abs() + dh).T, Gy))]
    return [(v, dv + (v.abs() + dv) * B + 1e-37) for v, dv in out]


def _check(got, bounds):
    for name, t, (v, off) in zip(("y", "Gx", "GW1", "GW2"), got, bounds):
        t = t.detach().cpu().double().reshape(v.shape)
        assert torch.isfinite(t).all() and ((t - v).abs() <= off).all(), (name, ((t - v).abs() / off).max())


def _step(block, x, Gy):
    block.zero_grad()
    x = x.detach().requires_grad_()
    y = block(x)
    y.backward(Gy)
    return y.detach(), x.grad, block.Wl1_D2H.grad, block.Wl2_HD.grad


# M, D, H: one row, ends of groups of 16 and 32 rows, of tiles of 64, 128 and 256; contractions of one, one and a half, two halves of a
# stage, odd and even; columns short of a tile and past it
SIZES = [
    (1, 32, 32), (1, 2048, 96), (3, 96, 2080), (9, 288, 2112), (15, 2080, 64), (16, 64, 64), (17, 160, 32), (31, 32, 288), (33, 288, 96), (64, 128, 128), (65, 96, 64), (128, 96, 64),
    (130, 224, 160), (257, 416, 352), (300, 640, 96), (513, 128, 1056), (700, 1056, 128), (1025, 320, 576), (2000, 96, 32), (5000, 64, 160),
    # large launches: of x W1 and G_y W2^T, of h W2 and gz W1^T; contractions of an odd number of 32
    (8200, 160, 1056), (8200, 1056, 160), (17000, 128, 544),
    # gradients of W1 or of both weights that are large launches
    (40, 1056, 4256), (35, 2080, 4224),
]


@pytest.mark.parametrize("M,D,H", SIZES)
def test_values_and_gradients(M, D, H):
    x, W1, W2, Gy = _inputs(M, D, H)
    bounds = _bounds(x, W1, W2, Gy)
    for save in (0, 50, 100):
        got = _step(_block(W1, W2, save), x.to(DEV), Gy.to(DEV))
        assert all(t.dtype == torch.bfloat16 for t in got)
        _check(got, bounds)
        with torch.no_grad():
            assert torch.equal(_block(W1, W2, save)(x.to(DEV)), got[0])


def test_gradients_by_differences():
    """v = sum(y * G_y) at two points of a line through each input: v(p + d) - v(p - d) = 2 g . d + r, where r, what the definition in 64 bits
    has beyond its own derivative on so long a step, is computed from it.  The left side is off by the bounds of y at the two points
    times |G_y|, the right by those of g times |d|."""
    M, D, H = 64, 96, 64
    x, W1, W2, Gy = _inputs(M, D, H)
    grads = _step(_block(W1, W2), x.to(DEV), Gy.to(DEV))[1:]
    bounds = _bounds(x, W1, W2, Gy)[1:]
    for i, (g, (exact, off)) in enumerate(zip(grads, bounds)):
        step = (g.cpu().float() * ((x, W1, W2)[i].float().norm() / g.float().norm().item())).to(torch.bfloat16)  # as long as the input itself
        value, true, slack, points = [], [], 0.0, []
        for sign in (1, -1):
            p = [x, W1, W2]
            p[i] = (p[i].float() + sign * step.float()).to(torch.bfloat16)
            y = _block(p[1], p[2])(p[0].to(DEV)).cpu().double()
            want, dy = _bounds(*p, Gy)[0]
            value.append((y * Gy.double()).sum().item())
            true.append((want * Gy.double()).sum().item())
            slack += (dy * Gy.double().abs()).sum().item()
            points.append(p[i].double())
        d = points[0] - points[1]
        r = true[0] - true[1] - (exact * d).sum().item()
        slack += (off * d.abs()).sum().item()
        along = (g.cpu().double() * d).sum().item()
        assert slack < 0.3 * abs(along) and abs(value[0] - value[1] - along - r) <= slack, (i, slack, along, r)


@pytest.mark.parametrize("save", [0, 50, 100])
def test_only_the_gradients_that_are_wanted(save):
    M, D, H = 100, 96, 160
    x, W1, W2, Gy = _inputs(M, D, H)
    ref = _step(_block(W1, W2, save), x.to(DEV), Gy.to(DEV))[1:]
    for wanted in range(1, 8):
        block, xd = _block(W1, W2, save), x.to(DEV)
        leaves = [xd, block.Wl1_D2H, block.Wl2_HD]
        for i, t in enumerate(leaves):
            t.requires_grad_(bool(wanted >> i & 1))
        block(xd).backward(Gy.to(DEV))
        for i, (t, r) in enumerate(zip(leaves, ref)):
            assert (t.grad is None) if not wanted >> i & 1 else torch.equal(t.grad, r)


def test_strides_types_shapes_and_places():
    M, D, H = 60, 96, 64
    x, W1, W2, Gy = [t.to(DEV) for t in _inputs(M, D, H)]
    ref = _step(_block(W1, W2), x, Gy)
    wide = torch.zeros(2 * M, D + 24, device=DEV, dtype=torch.bfloat16)
    for at in (0, 3, 8):
        wide[::2, at:at + D] = x
        gwide = torch.zeros_like(wide)
        gwide[::2, at:at + D] = Gy
        got = _step(_block(W1, W2), wide[::2, at:at + D], gwide[::2, at:at + D])
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    for f in (torch.float32, torch.float64):
        y, Gx, G1, G2 = _step(_block(W1, W2), x.to(f), Gy)
        assert y.dtype == torch.bfloat16 and Gx.dtype == f and all(torch.equal(a.to(torch.bfloat16), b) for a, b in zip((y, Gx, G1, G2), ref))
    got = _step(_block(W1, W2), x.view(3, 5, 4, D), Gy.view(3, 5, 4, D))
    assert got[0].shape == got[1].shape == (3, 5, 4, D) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, ref))
    got = _step(_block(W1, W2), x.T.contiguous().T, Gy.T.contiguous().T)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    # a broadcast input: its gradient is the sum over the rows, of bf16 rows
    one = x[:1].detach().requires_grad_()
    _block(W1, W2)(one.expand(M, D)).backward(Gy)
    rows = _step(_block(W1, W2), x[:1].repeat(M, 1), Gy)[1].float()
    assert one.grad.shape == (1, D) and ((one.grad.float() - rows.sum(0)).abs() <= 2 * B * rows.sum(0).abs() + M * B * rows.abs().amax(0)).all()
    # a vector, a tensor on the host, a broadcast gradient, no rows
    assert torch.equal(_block(W1, W2)(x[0]), _block(W1, W2)(x[:1])[0])
    host = x.cpu().requires_grad_()
    y = _block(W1, W2)(host)
    y.backward(Gy.cpu())
    assert y.device.type == "cpu" and torch.equal(y, ref[0].cpu()) and torch.equal(host.grad, ref[1].cpu())
    a = _step(_block(W1, W2), x, torch.ones(1, 1, device=DEV, dtype=torch.bfloat16).expand(M, D))
    b = _step(_block(W1, W2), x, torch.ones(M, D, device=DEV, dtype=torch.bfloat16))
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    for save in (0, 100):
        y, Gx, G1, G2 = _step(_block(W1, W2, save), x[:0], Gy[:0])
        assert y.shape == Gx.shape == (0, D) and (G1 == 0).all() and (G2 == 0).all()


@pytest.mark.parametrize("save", [0, 100])
@pytest.mark.parametrize("M", [40, 600])
def test_rows_of_nan_and_infinity_stay_with_themselves(M, save):
    D, H = 160, 288
    x, W1, W2, Gy = [t.to(DEV) for t in _inputs(M, D, H)]
    ref = _step(_block(W1, W2, save), x, Gy)
    bad, gbad = x.clone(), Gy.clone()
    bad[3, 100], bad[17, 20], bad[M - 1, 0], gbad[20, 5], gbad[M - 2, 0] = float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[[3, 17, 20, M - 1, M - 2]] = False
    got = _step(_block(W1, W2, save), bad, gbad)
    assert torch.equal(got[0][keep], ref[0][keep]) and torch.equal(got[1][keep], ref[1][keep])
    assert not got[0][3].isfinite().any() and not got[1][20].isfinite().any()
    # of the gradient of W2 column d sees G_y[:, d] alone: those without a bad value in it or a bad h
    ok = _step(_block(W1, W2, save), x, gbad)[3]
    cols = torch.ones(D, dtype=torch.bool, device=DEV)
    cols[[5, 0]] = False
    assert torch.equal(ok[:, cols], ref[3][:, cols]) and not ok[:, 5].isfinite().any() and not ok[:, 0].isfinite().any()


def test_few_rows_of_nan_and_infinity():
    """Rows that are two each; an infinite h stays one, and y with it."""
    x, W1, W2, _ = [t.to(DEV) for t in _inputs(9, 96, 64)]
    W2 = W2.abs() + 1
    bad = x.clone()
    bad[2, 5], bad[4] = float("nan"), 3e38
    W1[:, 0], W1[:, 64] = 1, 1  # a and b of column 0 overflow together: h = inf
    y, ref = _block(W1, W2)(bad), _block(W1, W2)(x)
    keep = [0, 1, 3, 5, 6, 7, 8]
    assert torch.equal(y[keep], ref[keep]) and y[2].isnan().all() and not y[4].isfinite().any()
    big = torch.zeros(1, 96, device=DEV, dtype=torch.bfloat16)
    big[0, 0] = 2.0 ** 70
    V1, V2 = torch.zeros(96, 128, device=DEV), torch.ones(64, 96, device=DEV)
    V1[0, 0], V1[0, 64] = 1, 1
    assert (_block(V1, V2)(big) == float("inf")).all()


@pytest.mark.parametrize("M,D,H", [(3, 96, 64), (70, 160, 288), (1100, 96, 64), (40, 1056, 4256)])
def test_gradients_leave_what_lies_behind(M, D, H):
    """The entry points of the backward on buffers with room behind them: the last rows' padding is zeros, and the rest keeps its bits."""
    lib, st, P = momoe_amd._hip._lib, torch.cuda.current_stream().cuda_stream, (M + 31) // 32 * 32
    x, W1, W2, Gy = [t.to(DEV) for t in _inputs(M, D, H)]
    flat = lambda n: torch.full((n + 4096,), 7.0, device=DEV, dtype=torch.bfloat16)
    u = torch.full((lib.momoe_ffn_fragment_floats(M, H) + 1024,), 7.0, device=DEV)
    gz, hT, Gx, G1, G2 = flat(2 * H * P), flat(P * H + 32 * H), flat(M * D), flat(2 * D * H), flat(D * H)
    counts = torch.full((6,), 7, device=DEV, dtype=torch.int32)
    need = lib.momoe_ffn_gradients_workspace_bytes(M, D, H, 1, 1, 1)
    ws = torch.full((need + 64,), 7, device=DEV, dtype=torch.uint8)
    assert lib.momoe_ffn_dgrad_h(Gy.data_ptr(), D, W2.data_ptr(), u.data_ptr(), M, D, H, st) == 0
    assert lib.momoe_ffn_swiglu_bwd(x.data_ptr(), D, W1.data_ptr(), u.data_ptr(), gz.data_ptr(), hT.data_ptr(), counts.data_ptr(), M, M, P, D, H, st) == 0
    assert lib.momoe_ffn_gradients(x.data_ptr(), D, Gy.data_ptr(), D, gz.data_ptr(), hT.data_ptr(), W1.data_ptr(), counts.data_ptr(), Gx.data_ptr(),
                                   G1.data_ptr(), G2.data_ptr(), ws.data_ptr(), need, M, P, D, H, st) == 0
    torch.cuda.synchronize()
    assert counts.tolist() == [0, M, 7, 7, 7, 7] and (ws[need:] == 7).all() and (u[lib.momoe_ffn_fragment_floats(M, H):] == 7).all()
    for t, n in ((gz, 2 * H * P), (hT, P * H), (Gx, M * D), (G1, 2 * D * H), (G2, D * H)):
        assert (t[n:] == 7).all()
    assert (gz[:2 * H * P].view(-1, P, 32)[:, M:] == 0).all() and (hT[:P * H].view(-1, H, 32).transpose(1, 2).reshape(P, H)[M:] == 0).all()
    want = _step(_block(W1, W2), x, Gy)
    got = Gx[:M * D].view(M, D), G1[:2 * D * H].view(D, 2 * H), G2[:D * H].view(H, D)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))


def test_gradients_of_rows_that_share_memory():
    """A gradient or an input that one row, or one value, stands for."""
    x, W1, W2, Gy = [t.to(DEV) for t in _inputs(70, 96, 64)]
    block = _block(W1, W2, 50)
    for a, b in ((x, Gy[:1].expand(70, 96)), (x, Gy[:1, :1].expand(70, 96)), (x[:1].expand(70, 96), Gy)):
        got, want = _step(block, a, b), _step(block, a.contiguous(), b.contiguous())
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_rows_behind_the_last_stay_as_they_are():
    """Results lie in a larger buffer of the allocator's: what is behind them keeps its bits."""
    D, H = 96, 64
    for M in (1, 31, 33, 100):
        x, W1, W2, Gy = [t.to(DEV) for t in _inputs(M, D, H)]
        y = torch.full((M + 40, D), 7.0, device=DEV, dtype=torch.bfloat16)
        ldm = momoe_amd._hip._lib.momoe_ffn_h_rows(M)
        h = torch.full((H // 32, ldm, 32), 7.0, device=DEV, dtype=torch.bfloat16)
        guard = torch.full((4096,), 7.0, device=DEV, dtype=torch.bfloat16)
        lib, st = momoe_amd._hip._lib, torch.cuda.current_stream().cuda_stream
        assert lib.momoe_ffn_lin1_fwd(x.data_ptr(), D, W1.data_ptr(), h.data_ptr(), None, 0, M, ldm, D, H, st) == 0
        ws = torch.empty(max(lib.momoe_ffn_workspace_bytes(M, D, H), 16), dtype=torch.uint8, device=DEV)
        assert lib.momoe_ffn_lin2_fwd(h.data_ptr(), W2.data_ptr(), y.data_ptr(), M, ldm, D, H, ws.data_ptr(), ws.numel(), st) == 0
        torch.cuda.synchronize()
        assert torch.equal(y[:M], _block(W1, W2)(x)) and (y[M:] == 7).all() and (guard == 7).all()


@pytest.mark.parametrize("M,save", [(40, 0), (300, 50), (700, 100)])
def test_streams_and_replayed_graphs(M, save):
    D, H = 160, 288
    ins = [[t.to(DEV) for t in _inputs(M, D, H, seed=i)] for i in range(3)]
    block = _block(ins[0][1], ins[0][2], save)

    def step(x, Gy):
        y = block(x)
        return (y, *torch.autograd.grad(y, (x, block.Wl1_D2H, block.Wl2_HD), Gy))
    leaf = lambda i: (ins[i][0].detach().requires_grad_(), ins[i][3])
    ref = [[t.detach().clone() for t in step(*leaf(i))] for i in range(3)]
    torch.cuda.synchronize()
    streams, out = [torch.cuda.Stream() for _ in ins], []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            out.append([t.detach() for t in step(*leaf(i))])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for u, v in zip(out, ref) for a, b in zip(u, v))
    del out
    x, Gy = leaf(0)
    x = x.detach().clone().requires_grad_()
    Gy = Gy.clone()
    with torch.cuda.stream(streams[0]):
        step(x, Gy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, Gy)
    got = [t.detach() for t in got]
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            x.copy_(ins[i][0])
            Gy.copy_(ins[i][3])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, ref[i]))
        eager = step(*leaf(i))
        assert all(torch.equal(a, b) for a, b in zip(eager, ref[i]))
        torch.cuda.synchronize()


def test_beside_a_mixture():
    """As a model has it: a dense layer, then a mixture, one backward through both; and a step of an optimizer."""
    D, H, N, K, S = 64, 96, 4, 2, 50
    g = torch.Generator().manual_seed(1)
    r = lambda *size: (torch.randn(*size, generator=g) * 0.1).to(DEV)
    dense = momoe_amd.FeedForward(D, H, 100, r(D, 2 * H), r(H, D))
    moe = momoe_amd.MoE(D, H, N, K, 0, Wg_DN=r(D, N), Wl1_ND2H=r(N, D, 2 * H), Wl2_NHD=r(N, H, D))
    x = r(2, S, D).to(torch.bfloat16).requires_grad_()
    mid = x + dense(x)
    mid.retain_grad()
    y = mid + moe(mid)
    y.float().square().sum().backward()
    want = _step(copy.deepcopy(dense), x, mid.grad)
    assert torch.equal(dense.Wl1_D2H.grad, want[2]) and torch.equal(dense.Wl2_HD.grad, want[3])
    assert ((x.grad - (mid.grad.float() + want[1].float())).abs() <= B * (mid.grad.float() + want[1].float()).abs() + 1e-30).all()
    before = dense.Wl1_D2H.detach().clone()
    torch.optim.SGD(dense.parameters(), lr=0.1).step()
    assert not torch.equal(before, dense.Wl1_D2H)
    with torch.no_grad():
        served = dense.to_int4(32)
        y4, ref = served(x), dense(x)
    W = [oracle.int4_weights(*[t.cpu() for t in q], 32) for q in ((w[0], w[1], w[4]) if i == 0 else (w[2], w[3], w[5])
                                                               for i, w in ((0, served.weights()), (1, served.weights())))]
    want4 = oracle.swiglu_block(x.detach().cpu().reshape(-1, D), *W)[3]
    assert (y4.cpu().double().reshape(want4.shape) - want4).norm() <= 2 * B * want4.norm()
    assert (y4 - ref).norm() < 0.5 * ref.norm()


def test_traced_block():
    x, W1, W2, Gy = [t.to(DEV) for t in _inputs(40, 96, 64)]
    block = _block(W1, W2, 50)
    traced = torch.jit.trace(block, (x,))
    for M in (40, 7, 300):
        xs, _, _, g = [t.to(DEV) for t in _inputs(M, 96, 64, seed=M)]
        a, b = _step(block, xs, g), None
        leaf = xs.detach().requires_grad_()
        block.zero_grad()
        y = traced(leaf)
        y.backward(g)
        b = y.detach(), leaf.grad, block.Wl1_D2H.grad, block.Wl2_HD.grad
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_refusals():
    x, W1, W2, Gy = [t.to(DEV) for t in _inputs(10, 96, 64)]
    f = momoe_amd.FeedForwardFunction.apply
    for bad in ((x[:, :64], W1, W2), (x, W1[:64], W2), (x, W1[:, :64], W2), (x, W1, W2[:32]), (x, W1, W2[:, :64]), (x[0, 0], W1, W2), (x, W1, W2.cpu())):
        with pytest.raises(AssertionError):
            f(*bad)
    for bad in ((x, W1[:, :96].contiguous(), W2[:48]), (x[:, :48], W1[:48], W2[:, :48])):
        with pytest.raises(RuntimeError, match="multiples of 32"):
            f(*bad)
    for save in (-1, 101, float("nan")):
        with pytest.raises(RuntimeError, match="save_percent"):
            f(x, W1, W2, save)
    block, leaf = _block(W1, W2), x.clone().requires_grad_()
    y = block(leaf)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, leaf, Gy, create_graph=True)
    huge = torch.empty(1, 1, device=DEV, dtype=torch.bfloat16).expand(1 << 23, 32)
    with pytest.raises(RuntimeError, match="split the batch"):
        _block(torch.zeros(32, 64), torch.zeros(32, 32))(huge)
    with torch.no_grad():
        block.Wl1_D2H.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(Gy)
    for shape in ((10, 96), (2, 5, 96)):
        changed = x.clone().view(shape)
        y = _block(W1, W2)(changed)
        changed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward(Gy.view(shape))


@pytest.mark.parametrize("save", [0, 50, 100])
@pytest.mark.parametrize("M,D,H", [(5, 96, 64), (70, 96, 64), (5100, 224, 1024)])
def test_gradients_of_large_gates(M, D, H, save):
    """G_x and G_W1, of which the slope at the gate is a factor, where it is 1 or 0 and where it is not."""
    x, W1, W2, Gy = large_gate_inputs(M, D, H)
    got = _step(_block(W1, W2, save), x.to(DEV), Gy.to(DEV))
    dx, d1, d2, dy = [t.double() for t in (x, W1, W2, Gy)]
    a, b, _, _ = oracle.swiglu_block(dx, d1, d2)
    u = dy @ d2.T
    gz, dgz = gz_and_error(a, b, u)
    want = oracle.swiglu_block_gradients(dx, d1, d2, dy)
    off = dgz @ d1.abs().T + (gz.abs() + dgz) @ d1.abs().T * 2 * (2 * H + 8) * E, dx.abs().T @ dgz + dx.abs().T @ (gz.abs() + dgz) * 2 * (M + 8) * E
    for name, t, v, o in zip(("Gx", "GW1"), got[1:3], want, off):
        o = o + (v.abs() + o) * B + 1e-37
        t = t.detach().cpu().double()
        assert ((t - v).abs() <= o).all(), (name, ((t - v).abs() / o).max())


@pytest.mark.parametrize("D,H,which", [(32, (1 << 19) + 32, 1), (32, (1 << 20) + 32, 2), ((1 << 20) + 32, 32, 1), ((1 << 20) + 32, 32, 2)])
def test_weights_too_wide_for_their_gradients(D, H, which):
    """Refused before the forward computes; without that gradient, such a block does what any other does."""
    x, W1, W2, Gy = _inputs(3, D, H)
    block, leaf = _block(W1, W2), x.to(DEV).requires_grad_()
    leaves = [leaf, block.Wl1_D2H, block.Wl2_HD]
    block.requires_grad_(False)
    leaves[which].requires_grad_()
    with pytest.raises(RuntimeError, match="1048576"):
        block(leaf)
    with torch.no_grad():
        y = block(leaf)
    leaves[which].requires_grad_(False)
    z = block(leaf)
    z.backward(Gy.to(DEV))
    assert torch.equal(y, z)
    _check((y, leaf.grad), _bounds(x, W1, W2, Gy)[:2])


def test_weights_too_wide():
    W = torch.empty(1, 1, device=DEV, dtype=torch.bfloat16)
    x = W.expand(2, 1 << 22)
    with pytest.raises(RuntimeError, match="4194304"):
        momoe_amd.FeedForwardFunction.apply(x, W.expand(1 << 22, 64), W.expand(32, 1 << 22))


def _check_on_gpu(got, ins):
    """As _check, the 64-bit side on the GPU."""
    for name, t, (v, off) in zip(("y", "Gx", "GW1", "GW2"), got, _bounds(*[t.to(DEV) for t in ins])):
        t = t.detach().double()
        assert torch.isfinite(t).all() and ((t - v).abs() <= off).all(), (name, ((t - v).abs() / off).max())


# M, D, H, of the gradients of W1 and of W2: "small" tiles of 128 x 128; "large" launches of 256 x 256 that are whole because they fill the
# CUs ("whole"), or with scratch for pieces of the tokens, which 300 of them are not cut into ("kept"), or which they are ("cut")
LARGE = [(300, 2048, 5632, "kept", "kept"), (4133, 1056, 4256, "cut", "small"), (4133, 2080, 4224, "cut", "cut"), (4133, 2048, 8192, "whole", "whole"),
         (6049, 1056, 4256, "cut", "small")]


@pytest.mark.parametrize("M,D,H,first,second", LARGE)
def test_large_gradients_of_the_weights(M, D, H, first, second):
    """Many stages, an odd number of groups of 32 rows, a ragged end."""
    lib = momoe_amd._hip._lib
    for kind, X, Y, which, layout in ((first, D, 2 * H, (0, 1, 0), 2), (second, H, D, (0, 0, 1), 0)):
        tiles, need = -(-X // 128) * -(-Y // 128), lib.momoe_ffn_gradients_workspace_bytes(M, D, H, *which)
        assert (tiles <= 512) == (kind == "small")
        if kind != "small":
            assert need == (0 if kind == "whole" else lib.momoe_wgrad_workspace_bytes(1, X, Y, M)) and lib.momoe_wgrad_stage_rows(1, X, Y, M, layout) == 64
        if need:  # pieces of 64 stages of 32 tokens or more, so that the scratch holds them
            stages, parts = -(-X // 256) * -(-Y // 256) * (M // 32 + 1), need // (256 * 256 * 4)
            assert (-(-M // 32) >= 2 * max(64, -(-stages // max(parts, 1)))) == (kind == "cut") or kind == "small"
    ins = _inputs(M, D, H)
    for save in (0, 100):
        _check_on_gpu(_step(_block(ins[1], ins[2], save), ins[0].to(DEV), ins[3].to(DEV)), ins)


@pytest.mark.parametrize("M,D,H", [(33, 288, 96), (1025, 320, 576), (1100, 96, 64), (5000, 64, 160), (17000, 128, 96), (300, 2048, 5632), (4133, 1056, 4256), (4133, 2080, 4224)])
def test_gradients_of_few_rows_among_many(M, D, H):
    """G_y of zeros but for a few rows: the last ones, or 20 either side of where a slice or a piece of the tokens may end.  What they add
    to the gradients of the weights is all there is, and the bounds are as small."""
    ins = [t.to(DEV) for t in _inputs(M, D, H)]
    block, zeros = _block(ins[1], ins[2]), torch.zeros_like(ins[3])
    ends = list(range(64, M, 64)) if D * H < 1 << 20 else list(range(64, M, 64 * 7))
    for lo, hi in [(M - 1, M), (M - M % 32, M), (M - 5, M), (max(0, M - 40), M)] + [(max(0, e - 20), min(M, e + 20)) for e in ends]:
        Gy = zeros.clone()
        Gy[lo:hi] = ins[3][lo:hi]
        some = ins[0][lo:hi], ins[1], ins[2], Gy[lo:hi]
        x, W1, W2, g = [t.double() for t in some]
        got = _step(block, ins[0], Gy)
        for name, t, (v, off) in zip(("GW1", "GW2"), got[2:], _bounds(*some)[2:]):
            assert ((t.double() - v).abs() <= off).all(), (name, lo, hi, ((t.double() - v).abs() / off).max())
            if hi - lo == 1:  # (that it were lost would be seen)
                assert (v.abs() > 2 * off).any()


def _pitches(D):
    """[M, D] views of wider buffers: pitches that are no multiple of 8, of 4 GiB of rows and more, of 2^22 elements and more; with the rows
    at the start, in the middle and at the end of the buffer's."""
    for M, width, at in ((70, D + 4, 0), (70, D + 30, 6), (1 << 20, 2080, 0), (1 << 20, 2080, 2080 - D), (3, (1 << 22) + 8, 8)):
        yield M, torch.zeros(M, width, device=DEV, dtype=torch.bfloat16)[:, at:at + D]


def test_pitches_that_are_copied():
    D, H = 32, 64
    _, W1, W2, _ = _inputs(1, D, H)
    block = _block(W1, W2)
    for M, view in _pitches(D):
        x, Gy = [torch.randn(M, D, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
        want = _step(block, x, Gy)
        view.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(_step(block, view, Gy), want))
        view.copy_(Gy)
        assert all(torch.equal(a, b) for a, b in zip(_step(block, x, view), want))


@pytest.mark.parametrize("save", [0, 100])
@pytest.mark.parametrize("D,H", [(4096, 32), (32, 4096)])
def test_tokens_past_32_bit_offsets(D, H, save):
    """x, y and Gx, or h, gz and what is kept, of more than 4 GiB: rows at the start, at the end and where offsets pass 2^31 and 2^32."""
    M = (1 << 19) + 45
    _, W1, W2, _ = _inputs(1, D, H)
    g = torch.Generator(device=DEV).manual_seed(1)
    x, Gy = [torch.randn(M, D, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    block = _block(W1, W2, save).requires_grad_(False)
    y, Gx = _step(block, x, Gy)[:2]
    edge = [e // (w * p) for w in {D, H, 2 * H} for p in (2, 4) for e in (1 << 31, 1 << 32, 1 << 33)]
    rows = torch.cat([torch.arange(max(0, e - 20), min(M, e + 20)) for e in [0, M] + [e for e in edge if e < M]]).unique().to(DEV)
    _check((y[rows], Gx[rows]), _bounds(x[rows].cpu(), W1, W2, Gy[rows].cpu())[:2])
    with torch.no_grad():
        assert torch.equal(block(x)[rows], y[rows])


@pytest.mark.parametrize("M,D,H", [(1, 96, 64), (16, 2080, 64), (17, 96, 64), (31, 288, 96), (100, 96, 2080), (1250, 224, 2048)])
def test_the_forward_leaves_what_lies_behind(M, D, H):
    """The entry points of the forward on buffers with room behind them, and h of more rows than there are."""
    lib, st = momoe_amd._hip._lib, torch.cuda.current_stream().cuda_stream
    x, W1, W2, _ = [t.to(DEV) for t in _inputs(M, D, H)]
    held, kept = lib.momoe_ffn_h_rows(M), (M + 15) // 16 * 16
    ldm, need = held + 40, lib.momoe_ffn_workspace_bytes(M, D, H)
    h, y = [torch.full((n + 4096,), 7.0, device=DEV, dtype=torch.bfloat16) for n in (H * ldm, M * D)]
    ab = torch.full((lib.momoe_ffn_fragment_floats(M, 2 * H) + 4096,), 7.0, device=DEV)
    ws = torch.full((need + 4096,), 7, device=DEV, dtype=torch.uint8)
    assert lib.momoe_ffn_lin1_fwd(x.data_ptr(), D, W1.data_ptr(), h.data_ptr(), ab.data_ptr(), (M + 31) // 32 * 32, M, ldm, D, H, st) == 0
    assert lib.momoe_ffn_lin2_fwd(h.data_ptr(), W2.data_ptr(), y.data_ptr(), M, ldm, D, H, ws.data_ptr() if need else None, need, st) == 0
    torch.cuda.synchronize()
    assert (h[H * ldm:] == 7).all() and (h[:H * ldm].view(-1, ldm, 32)[:, held:] == 7).all() and (ab[kept * 2 * H:] == 7).all()
    assert (y[M * D:] == 7).all() and (ws[need:] == 7).all() and torch.equal(y[:M * D].view(M, D), _block(W1, W2)(x))
