"""CPU: what the 8-bit experts refuse, before any launch, and their sizes."""
import ctypes

import pytest
import torch

import momoe_amd
from momoe_amd import _hip

lib, P = _hip._lib, 4096
i64 = ctypes.c_int64


def test_sizes():
    assert [lib.momoe_fp8_row_bytes(n) for n in (0, 1, 128, 129, 2048)] == [-1, 128, 128, 256, 2048]
    assert [lib.momoe_fp8_code_bytes(n) for n in (0, 1, 512, 513, 2048)] == [-1, 4, 4, 8, 16]
    assert lib.momoe_fp8_weight_bytes(3, 200, 64) == 3 * 4 * 2 * 2048
    assert lib.momoe_fp8_weight_bytes(3, 200, 40) == lib.momoe_fp8_weight_bytes(0, 1, 16) == -1
    rows = lib.momoe_fp8_tile_rows
    assert rows(0, 64, 64, 8) == rows(1, 0, 64, 8) == rows(1, 64, 0, 8) == rows(1, 64, 64, 0) == 0
    assert [rows(m, 2048, 768, 128) for m in (1, 8, 1000)] == [32] * 3 and rows(65536, 2048, 768, 128) == 256
    assert rows(65536, 8224, 768, 128) == rows(65536, 768, 8224, 128) == 32  # contractions past what a tall tile holds the scales of


def test_refusals_of_the_entry_points():
    q = lambda **c: lib.momoe_fp8_quantize_rows(*{**dict(x=P, t=0, ld=64, rows=4, cols=64, q=P, codes=P), **c}.values(), None)
    assert all(q(**{k: None}) == 1 for k in ("x", "q", "codes"))
    assert q(t=3) == q(ld=56) == q(rows=0) == q(cols=0) == q(x=P + 8) == q(q=P + 4) == q(codes=P + 2) == 1
    assert q(cols=60) == q(ld=68) == q(rows=1 << 31) == 2
    w = lambda **c: lib.momoe_fp8_pack_weights(*{**dict(W=P, quantized=0, N=2, R=64, C=64, halves=2, packed=P, scale=P), **c}.values(), None)
    assert all(w(**{k: None}) == 1 for k in ("W", "packed", "scale"))
    assert w(N=0) == w(R=0) == w(C=0) == w(halves=0) == w(halves=3) == w(W=P + 8) == 1
    assert w(C=48) == w(N=70000) == 2
    one = dict(x=P, xc=P, W=P, S=P, idx=P, table=P, h=P, hc=P, M=16, D=64, H=32, N=8, Msum=32)
    lin1 = lambda **c: lib.momoe_fp8_lin1_swiglu_fwd(*{**one, **c}.values(), None)
    assert all(lin1(**{k: None}) == 1 for k in ("x", "xc", "W", "S", "idx", "table", "h", "hc"))
    assert all(lin1(**{k: 0}) == 1 for k in ("M", "D", "H", "N", "Msum")) and all(lin1(**{k: P + 8}) == 1 for k in ("x", "W", "h"))
    assert lin1(xc=P + 2) == lin1(hc=P + 1) == 1
    assert lin1(D=48) == lin1(H=40) == lin1(Msum=1 << 31) == 2
    assert lin1(M=1 << 21, D=4096, Msum=1 << 22) == 2  # rows past 32-bit offsets
    two = dict(h=P, hc=P, W=P, S=P, s=P, sn=16, sm=1, idx=P, table=P, ys=P, M=16, D=64, H=32, N=8, Msum=32)
    lin2 = lambda **c: lib.momoe_fp8_lin2_scale_fwd(*{**two, **c}.values(), None)
    assert all(lin2(**{k: None}) == 1 for k in ("h", "hc", "W", "S", "s", "idx", "table", "ys"))
    assert all(lin2(**{k: 0}) == 1 for k in ("M", "D", "H", "N", "Msum")) and all(lin2(**{k: P + 8}) == 1 for k in ("h", "W", "ys"))
    assert lin2(hc=P + 2) == 1 and lin2(D=48) == lin2(H=40) == 2
    few1 = dict(x=P, t=0, ld=64, W=P, S=P, idx=P, table=P, h=P, M=16, D=64, H=32, N=8, Msum=32)
    lin1 = lambda **c: lib.momoe_fp8_few_lin1_swiglu_fwd(*{**few1, **c}.values(), None)
    assert all(lin1(**{k: None}) == 1 for k in ("x", "W", "S", "idx", "table", "h"))
    assert all(lin1(**{k: 0}) == 1 for k in ("M", "D", "H", "N", "Msum")) and all(lin1(**{k: P + 8}) == 1 for k in ("x", "W", "h"))
    assert lin1(t=3) == lin1(t=-1) == lin1(ld=56) == 1 and lin1(ld=68) == lin1(D=48) == lin1(H=40) == lin1(Msum=1 << 31) == 2
    few2 = {k: v for k, v in two.items() if k != "hc"}
    lin2 = lambda **c: lib.momoe_fp8_few_lin2_scale_fwd(*{**few2, **c}.values(), None)
    assert all(lin2(**{k: None}) == 1 for k in ("h", "W", "S", "s", "idx", "table", "ys"))
    assert all(lin2(**{k: 0}) == 1 for k in ("M", "D", "H", "N", "Msum")) and all(lin2(**{k: P + 8}) == 1 for k in ("h", "W", "ys"))
    assert lin2(D=48) == lin2(H=40) == 2
    c = lambda **k: lib.momoe_fp8_combine(*{**dict(ys=P, inv=P, out=P, M=4, D=64, K=2, Msum=8), **k}.values(), None)
    assert all(c(**{k: None}) == 1 for k in ("ys", "inv", "out")) and all(c(**{k: 0}) == 1 for k in ("M", "D", "K", "Msum"))
    assert c(ys=P + 8) == c(out=P + 8) == 1 and c(D=48) == c(M=1 << 31) == 2


def test_constructor_refusals():
    e4 = lambda *size: torch.zeros(*size, dtype=torch.float8_e4m3fn)
    good = dict(Wl1_ND2H=e4(2, 160, 128), Wl1_scale=torch.ones(2, 2, 2, 1), Wl2_NHD=e4(2, 64, 160), Wl2_scale=torch.ones(2, 1, 2))
    for name, bad in (("Wl1_ND2H", torch.zeros(2, 160, 128)), ("Wl1_ND2H", e4(2, 160, 64)), ("Wl1_scale", torch.ones(2, 2, 2)),
                      ("Wl1_scale", good["Wl1_scale"].double()), ("Wl2_NHD", e4(2, 160, 64)), ("Wl2_scale", torch.ones(2, 2, 1))):
        with pytest.raises(AssertionError, match=name):
            momoe_amd.MoMoEFP8(160, 64, 2, 1, **{**good, name: bad})
    for k in (0, 3):
        with pytest.raises(AssertionError, match="num_chosen_experts"):
            momoe_amd.MoMoEFP8(160, 64, 2, k, **good)
    with pytest.raises(AssertionError, match="multiples of 32"):
        momoe_amd.MoMoEFP8(160, 48, 2, 1, **good)
    with pytest.raises(RuntimeError, match="no CPU compute path"):
        momoe_amd.MoMoEFP8(160, 64, 2, 1, **good)
