"""CPU: what the balance loss refuses, before any launch."""
import ctypes

import pytest
import torch

import momoe_amd
from momoe_amd import _hip


def test_refusals_of_the_entry_points():
    p, lib = 4096, _hip._lib
    good = dict(logits=p, type=0, ld=64, mask=p, sn=128, sm=1, valid=None, G=2, S=64, N=64, Ks=4, loss=p, counts=p, info=p, ws=p, bytes=1 << 20)

    def fwd(**changed):
        a = {**good, **changed}
        return lib.momoe_balance_fwd(*a.values(), None)

    for name in ("logits", "mask", "loss", "counts", "info", "ws"):
        assert fwd(**{name: None}) == 1
    assert all(fwd(type=t) == 1 for t in (-1, 3))
    assert fwd(ld=63) == fwd(G=0) == fwd(S=0) == fwd(N=0) == fwd(Ks=-1) == fwd(Ks=64) == 1
    assert fwd(ws=p + 8) == fwd(bytes=0) == 1
    assert fwd(N=513, ld=513) == fwd(G=1 << 20, S=1 << 12) == fwd(S=1 << 31) == fwd(G=1, S=(1 << 30) + 1) == 2
    back = dict(logits=p, type=1, ld=64, valid=None, counts=p, info=p, g=p, add=None, out=p, gtype=1, G=2, S=64, N=64, Ks=0)

    def bwd(**changed):
        return lib.momoe_balance_bwd(*{**back, **changed}.values(), None)

    for name in ("logits", "counts", "info", "g", "out"):
        assert bwd(**{name: None}) == 1
    assert bwd(type=7) == bwd(gtype=-1) == bwd(ld=8) == bwd(Ks=64) == 1
    assert bwd(gtype=2) == bwd(N=520, ld=520) == 2  # (the gradient is of the logits' type or bf16)


def test_workspace_is_small():
    ws = _hip._lib.momoe_balance_workspace_bytes
    assert ws(0, 1, 8) == ws(1, 0, 8) == ws(1, 1, 0) == ws(1, 8, 513) == -1
    assert ws(1, 128, 8) == 16
    for G, S, N in ((1, 8192, 128), (8, 8192, 64), (64, 1024, 512), (1, 65536, 512)):
        assert 0 < ws(G, S, N) <= 4 * 512 * N * 3


def test_host_checks():
    with pytest.raises(RuntimeError, match="no CPU compute path"):
        momoe_amd.balance_loss(torch.zeros(4, 8), torch.zeros(8, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="balance must be"):
        momoe_amd.MoE(32, 32, 4, 2, 0, balance="tokens")


def test_refusals_of_the_entry_points_with_another_output():
    """As those without: before any launch."""
    p, lib = 4096, _hip._lib
    good = dict(logits=p, type=0, ld=64, mask=p, sn=128, sm=1, valid=None, G=2, S=64, N=64, Ks=4, loss=p, counts=p, kept=p, info=p, ws=p, bytes=1 << 20)
    kept = lambda **c: lib.momoe_balance_fwd_kept(*{**good, **c}.values(), None)
    assert all(kept(**{k: None}) == 1 for k in ("logits", "mask", "loss", "counts", "info", "ws"))
    assert kept(type=3) == kept(ld=63) == kept(Ks=64) == kept(ws=p + 8) == kept(bytes=0) == 1 and kept(N=513, ld=513) == 2
    gate = dict(x=p, ldx=64, Wg=p, bias=p, M=4, D=64, N=8, K=2, Ks=0, mask=p, s=p, psel=p, ng=p, ks=p, logits=p, ws=p, bytes=1 << 20)
    route = lambda **c: lib.momoe_gate_router_fwd_logits(*{**gate, **c}.values(), None)
    assert all(route(**{k: None}) == 1 for k in ("x", "Wg", "bias", "mask", "s", "psel", "ng", "ks", "ws"))
    assert route(M=0) == route(K=9) == route(ldx=56) == route(x=p + 8) == route(bytes=0) == 1 and route(N=12) == route(ldx=68) == 2
