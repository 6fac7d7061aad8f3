"""CPU: what the blocks with 4-bit weights refuse, before any launch, their sizes, and how weights are quantized."""
import pytest
import torch

import momoe_amd
import oracle
from momoe_amd import _hip
from momoe_amd.int4 import quantize

lib, P = _hip._lib, 4096


def test_sizes():
    assert lib.momoe_int4_weight_bytes(3, 200, 64) == 3 * 4 * 2 * 1024
    assert lib.momoe_int4_weight_bytes(3, 200, 40) == lib.momoe_int4_weight_bytes(0, 1, 16) == -1
    assert [lib.momoe_int4_scale_words(2, 160, 32, g) for g in (32, 64, 128, 16)] == [2 * 32 * 2 * 4, 2 * 32 * 2 * 2, 2 * 32 * 2, -1]
    assert lib.momoe_int4_scale_words(1, 0, 32, 64) == lib.momoe_int4_scale_words(1, 32, 24, 64) == -1
    rows = lib.momoe_int4_tile_rows
    assert rows(0, 64, 64, 8) == rows(1, 0, 64, 8) == rows(1, 64, 0, 8) == rows(1, 64, 64, 0) == 0
    assert rows(8, 2048, 768, 128) == 32 and rows(8000, 2048, 768, 128) == 64 and rows(200, 1024, 1024, 1) == 32 and rows(300, 1024, 1024, 1) == 64
    assert [lib.momoe_int4_h_rows(*n) for n in ((-1, 1), (1, 0), (0, 1), (16, 1), (17, 1), (2048, 128), (2049, 128))] == [-1, -1, 0, 32, 17, 4096, 2049]
    slices = lib.momoe_int4_slices
    assert slices(0, 1, 64, 64, 64) == slices(1, 0, 64, 64, 64) == slices(1, 1, 0, 64, 64) == slices(1, 1, 64, 0, 64) == 0
    assert slices(16, 1, 4096, 11264, 32) == 1 and slices(16, 1, 4096, 11264, 64) > 1 and slices(8000, 128, 1536, 2048, 64) == 1
    assert lib.momoe_int4_ffn_workspace_bytes(0, 64, 64) == -1 and lib.momoe_int4_ffn_workspace_bytes(4, 512, 512) == 0
    n = slices(16, 1, 22528, 4096, 64), slices(16, 1, 4096, 11264, 64)
    assert lib.momoe_int4_ffn_workspace_bytes(16, 4096, 11264) == max(n[0] * 22528, n[1] * 4096) * 16 * 4


def test_refusals_of_the_entry_points():
    w = lambda **c: lib.momoe_int4_pack_weights(*{**dict(W=P, scale=P, t=0, zero=P, N=2, R=64, C=64, halves=2, group=32, packed=P, words=P), **c}.values(), None)
    assert all(w(**{k: None}) == 1 for k in ("W", "scale", "packed", "words")) and all(w(**{k: 0}) == 1 for k in ("N", "R", "C", "halves"))
    assert w(t=1) == w(t=3) == w(halves=3) == w(packed=P + 8) == w(words=P + 4) == w(scale=P + 1) == 1
    assert w(R=48) == w(C=48) == w(group=16) == w(group=0) == w(R=1 << 22) == 2
    one = dict(x=P, ld=64, W=P, S=P, group=32, idx=P, table=P, rows=32, h=P, ws=None, bytes=0, M=16, D=64, H=32, N=8, Msum=32)
    lin1 = lambda **c: lib.momoe_int4_lin1_swiglu_fwd(*{**one, **c}.values(), None)
    assert all(lin1(**{k: None}) == 1 for k in ("x", "W", "S", "idx", "table", "h"))
    assert all(lin1(**{k: 0}) == 1 for k in ("M", "D", "H", "N", "Msum")) and all(lin1(**{k: P + 8}) == 1 for k in ("x", "W", "S", "h"))
    assert lin1(ws=P + 8) == lin1(rows=64, D=1024, ld=1024, N=1, Msum=16) == 1 and lin1(rows=64, M=1 << 21, ld=1024) == 2  # no room for slices; rows past 32 bits
    assert lin1(ld=56) == 1 and lin1(ld=68) == lin1(D=48) == lin1(H=40) == lin1(Msum=1 << 31) == lin1(group=48) == lin1(rows=128) == 2
    two = dict(h=P, W=P, S=P, group=32, s=P, sn=16, sm=1, idx=P, table=P, rows=32, ys=P, M=16, D=64, H=32, N=8, Msum=32)
    lin2 = lambda **c: lib.momoe_int4_lin2_scale_fwd(*{**two, **c}.values(), None)
    assert all(lin2(**{k: None}) == 1 for k in ("h", "W", "S", "s", "idx", "table", "ys"))
    assert all(lin2(**{k: 0}) == 1 for k in ("M", "D", "H", "N", "Msum")) and all(lin2(**{k: P + 8}) == 1 for k in ("h", "W", "S", "ys"))
    assert lin2(D=48) == lin2(H=40) == lin2(group=0) == lin2(rows=0) == 2
    c = lambda **k: lib.momoe_int4_combine(*{**dict(ys=P, slices=1, inv=P, out=P, M=4, D=64, K=2, Msum=8), **k}.values(), None)
    assert all(c(**{k: None}) == 1 for k in ("ys", "inv", "out")) and all(c(**{k: 0}) == 1 for k in ("slices", "M", "D", "K", "Msum"))
    assert c(ys=P + 8) == c(out=P + 8) == 1 and c(D=48) == c(M=1 << 31) == 2
    ffn = dict(x=P, ld=64, W1=P, S1=P, W2=P, S2=P, group=32, h=P, y=P, ws=None, bytes=0, M=16, D=64, H=32)
    f = lambda **k: lib.momoe_int4_ffn_fwd(*{**ffn, **k}.values(), None)
    assert all(f(**{k: None}) == 1 for k in ("x", "W1", "S1", "W2", "S2", "h", "y")) and all(f(**{k: 0}) == 1 for k in ("M", "D", "H"))
    assert all(f(**{k: P + 8}) == 1 for k in ("x", "W1", "S1", "W2", "S2", "h", "y"))
    assert f(ws=P + 8) == f(M=16, D=4096, H=11264, ld=4096) == f(M=16, D=4096, H=11264, ld=4096, ws=P, bytes=64) == 1
    assert f(ld=56) == 1 and f(ld=1 << 22) == f(ld=68) == f(D=48) == f(H=40) == f(group=100) == f(M=1 << 31) == 2


def test_constructor_refusals():
    D, H, N, G = 160, 64, 2, 64
    u8, bf = lambda *s: torch.zeros(*s, dtype=torch.uint8), lambda *s: torch.ones(*s, dtype=torch.bfloat16)
    dense = dict(Wl1_D2H=u8(D // 2, 2 * H), Wl1_scale=bf(3, 2 * H), Wl2_HD=u8(H // 2, D), Wl2_scale=bf(1, D))
    names = dict(Wl1_D2H="Wl1_ND2H", Wl2_HD="Wl2_NHD")
    many = {names.get(k, k): torch.stack([v, v]) for k, v in dense.items()}
    for k, bad in (("Wl1_D2H", u8(D, 2 * H)), ("Wl1_D2H", bf(D // 2, 2 * H)), ("Wl1_scale", bf(2, 2 * H)), ("Wl1_scale", bf(3, 2 * H).float()),
                   ("Wl2_HD", u8(H // 2, H)), ("Wl2_scale", bf(D)), ("Wl1_zero", bf(3, 2 * H)), ("Wl2_zero", u8(2, D))):
        with pytest.raises(AssertionError, match=k[:3]):
            momoe_amd.FeedForwardInt4(D, H, **{**dense, k: bad}, group_size=G)
        with pytest.raises(AssertionError, match=k[:3]):
            momoe_amd.MoMoEInt4(D, H, N, 1, **{**many, names.get(k, k): torch.stack([bad, bad])}, group_size=G)
    for k in (0, 3):
        with pytest.raises(AssertionError, match="num_chosen_experts"):
            momoe_amd.MoMoEInt4(D, H, N, k, **many, group_size=G)
    for d, h, g, what in ((160, 48, G, "multiples of 32"), (0, 64, G, "multiples of 32"), (160, 64, 48, "group_size")):
        with pytest.raises(AssertionError, match=what):
            momoe_amd.FeedForwardInt4(d, h, **dense, group_size=g)
    with pytest.raises(RuntimeError):
        momoe_amd.FeedForwardInt4(D, H, **dense, group_size=G)  # weights on the host: there is no CPU compute path


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(group):
    """Every code is the nearest of its group's 16 values, zero is one of them, and a group of zeros stays zeros."""
    W = torch.randn(2, 160, 24, generator=torch.Generator().manual_seed(0))
    W[0, :, 3] = 0
    W[0, :, 4] = W[0, :, 4].abs()
    W[1, :, 5] = -W[1, :, 5].abs()
    q, scale, zero = quantize(W, group)
    assert q.shape == (2, 80, 24) and scale.shape == zero.shape == (2, -(-160 // group), 24) and zero.max() <= 15
    v = oracle.int4_weights(q, scale, zero, group)
    each = lambda t: t.double().repeat_interleave(group, 1)[:, :160]
    grid = (torch.arange(16).view(16, 1, 1, 1) - each(zero)) * each(scale)
    # the nearest, but for a value half way between two, by fp32's rounding of the quotient
    assert ((v - W.double()).abs() <= (grid - W.double()).abs().amin(0) + each(scale) * 2.0 ** -18).all()
    assert (v[0, :, 3] == 0).all() and (zero[0, :, 4] == 0).all() and (zero[1, :, 5] == 15).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_of_nan_and_infinity(group):
    """A weight that is no number leaves none in its group and column; every other group is as without it."""
    W = torch.randn(2, 160, 24, generator=torch.Generator().manual_seed(1)) * 0.02
    clean = quantize(W, group)
    bad = W.clone()
    where = ((0, 3, 5, "nan"), (0, 159, 7, "inf"), (1, 40, 0, "-inf"), (1, 0, 23, "nan"))
    for n, r, c, v in where:
        bad[n, r, c] = float(v)
    bad[1, 41, 0] = float("inf")
    q, scale, zero = quantize(bad, group)
    assert zero.max() <= 15
    v, hit = oracle.int4_weights(q, scale, zero, group), torch.zeros(2, 160, 24, dtype=torch.bool)
    for n, r, c, _ in where:
        hit[n, r // group * group:(r // group + 1) * group, c] = True
    assert not v[hit].isfinite().any() and torch.equal(v[~hit], oracle.int4_weights(*clean, group)[~hit])
