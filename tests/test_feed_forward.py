"""CPU: what the dense block refuses, before any launch."""
import pytest
import torch

import momoe_amd
from momoe_amd import _hip

lib, P = _hip._lib, 4096


def test_sizes():
    assert [lib.momoe_ffn_fragment_floats(r, 64) for r in (0, 1, 16, 17)] == [0, 1024, 1024, 2048]
    assert lib.momoe_ffn_fragment_floats(-1, 64) == lib.momoe_ffn_fragment_floats(1, 24) == lib.momoe_ffn_fragment_floats(1, 0) == -1


def test_rows_of_h():
    assert [lib.momoe_ffn_h_rows(n) for n in (-1, 0, 1, 16, 17, 100)] == [-1, 0, 2, 32, 17, 100]
    assert lib.momoe_ffn_workspace_bytes(5, 64, 64) == 2 * 5 * 64 * 4 and lib.momoe_ffn_lin1_fwd(P, 64, P, P, None, 0, 16, 31, 64, 32, None) == 1


def _refuses(fn, good, pointers, aligned, optional=()):
    call = lambda **c: fn(*{**good, **c}.values(), None)
    assert all(call(**{k: None}) == 1 for k in pointers) and all(call(**{k: P + 8}) == 1 for k in aligned)
    assert all(call(**{k: 0}) == 1 for k in ("rows", "D", "H")) and call(D=48) == call(H=40) == 2
    assert call(D=1 << 16, H=1 << 16, **{k: 1 << 17 for k in good if k.startswith("ld") and k != "ldm"}) == 2
    return call


def test_refusals_of_the_entry_points():
    sizes, padded = dict(rows=40, ldm=40, D=64, H=32), dict(rows=40, ldm=64, D=64, H=32)
    c = _refuses(lib.momoe_ffn_lin1_fwd, dict(x=P, ldx=64, W=P, h=P, ab=None, ab_rows=0, **sizes), ("x", "W", "h"), ("x", "W", "h"))
    assert c(ldx=56) == c(ldm=39) == c(ab_rows=32) == c(ab=P, ab_rows=-32) == c(ab=P, ab_rows=96) == c(ab=P + 4, ab_rows=32) == 1
    assert c(ldx=68) == c(ab=P, ab_rows=40) == c(ldx=1 << 22) == 2
    room = dict(ws=P, bytes=1 << 40)
    c = _refuses(lib.momoe_ffn_lin2_fwd, dict(h=P, W=P, y=P, **sizes, **room), ("h", "W", "y", "ws"), ("h", "W", "y", "ws"))
    assert c(ldm=39) == c(bytes=-1) == 1 and c(ldm=1 << 31) == 2
    need = lib.momoe_ffn_workspace_bytes(1, 2048, 8192)
    assert need > 0 and c(rows=1, D=2048, H=8192, bytes=need - 4) == c(rows=1, D=2048, H=8192, ws=None, bytes=0) == 1
    assert lib.momoe_ffn_workspace_bytes(0, 64, 64) == lib.momoe_ffn_workspace_bytes(1, 0, 64) == lib.momoe_ffn_workspace_bytes(1, 64, 0) == -1
    c = _refuses(lib.momoe_ffn_dgrad_h, dict(Gy=P, ldgy=64, W=P, u=P, rows=40, D=64, H=32), ("Gy", "W", "u"), ("Gy", "W", "u"))
    assert c(ldgy=56) == 1 and c(ldgy=68) == 2
    c = _refuses(lib.momoe_ffn_swiglu_bwd, dict(x=P, ldx=64, W=P, u=P, gz=P, hT=None, counts=None, tokens=40, **padded), ("x", "W", "u", "gz"), ("x", "W", "u", "gz", "hT"))
    assert c(ldx=56) == c(ldm=63) == c(tokens=39) == 1 and c(ldx=68) == 2
    c = _refuses(lib.momoe_ffn_dgrad_h_saved, dict(Gy=P, ldgy=64, W=P, ab=P, gz=P, hT=None, counts=None, tokens=40, **padded), ("Gy", "W", "ab", "gz"), ("Gy", "W", "ab", "gz", "hT"))
    assert c(ldgy=56) == c(ldm=63) == c(tokens=39) == 1 and c(ldgy=68) == 2
    need = lib.momoe_ffn_gradients_workspace_bytes
    assert all(need(*n, 1, 1, 1) == -1 for n in ((0, 64, 64), (64, 0, 64), (64, 64, 0))) and need(40, 64, 32, 0, 0, 0) == 0
    each = [need(1024, 512, 1024, *w) for w in ((1, 0, 0), (0, 1, 0), (0, 0, 1))]
    assert all(n > 0 for n in each) and need(1024, 512, 1024, 1, 1, 1) == sum(each)
    good = dict(x=P, ldx=64, Gy=P, ldgy=64, gz=P, hT=P, W=P, counts=P, Gx=P, GW1=P, GW2=P, **room, rows=40, ldm=64, D=64, H=32)
    c = _refuses(lib.momoe_ffn_gradients, good, ("x", "Gy", "gz", "hT", "W", "counts", "ws"), ("x", "Gy", "gz", "hT", "W", "Gx", "GW1", "GW2", "ws"))
    assert c(ldx=56) == c(ldgy=56) == c(ldm=63) == c(bytes=-1) == c(rows=-40) == 1
    assert c(rows=1024, ldm=1024, D=512, H=1024, ldx=512, ldgy=512, bytes=sum(each) - 4) == 1
    assert c(ldx=68) == c(ldgy=68) == c(rows=1 << 20, ldm=1 << 20, ldx=2048) == c(rows=1 << 20, ldm=1 << 20, ldgy=2048) == c(ldm=1 << 23) == 2
    for wants, needs in ((("Gx",), ("gz", "W")), (("GW1",), ("x", "gz", "counts")), (("GW2",), ("Gy", "hT", "counts"))):
        one = {**{k: None for k in ("x", "Gy", "gz", "hT", "W", "counts", "Gx", "GW1", "GW2")}, **{k: P for k in wants + needs}}
        assert all(c(**{**one, k: None}) == 1 for k in needs)


def test_module_refusals():
    W1, W2 = torch.zeros(32, 64), torch.zeros(32, 32)
    for save in (-1, 101):
        with pytest.raises(AssertionError, match="save_percent"):
            momoe_amd.FeedForward(32, 32, save, W1, W2)
    with pytest.raises(RuntimeError, match="no CPU compute path"):
        momoe_amd.FeedForward(32, 32, 0, W1, W2)(torch.zeros(4, 32))


def test_gradients_of_weights_that_are_too_wide_are_refused_before_any_is_computed():
    """A gradient of more than 2^20 rows or columns, beside one that could be had."""
    good = dict(x=P, ldx=64, Gy=P, ldgy=64, gz=P, hT=P, W=P, counts=P, Gx=None, GW1=None, GW2=None, ws=P, bytes=1 << 40, rows=40, ldm=64, D=32, H=32)
    c = lambda **k: lib.momoe_ffn_gradients(*{**good, **k}.values(), None)
    for wants, sizes in ((("GW1", "GW2"), dict(H=(1 << 19) + 32)), (("GW1",), dict(H=(1 << 19) + 32)), (("GW2",), dict(H=(1 << 20) + 32)),
                         (("GW1", "GW2"), dict(D=(1 << 20) + 32)), (("Gx", "GW2"), dict(D=(1 << 20) + 32))):
        ld = sizes.get("D", 64)
        assert c(**sizes, **{k: P for k in wants}, ldx=ld, ldgy=ld) == 2, (wants, sizes)
    take, most = lib.momoe_ffn_gradients_take, 1 << 20
    assert take(most, most // 2, 1, 1) == take(most, most, 0, 1) == take(2 * most, 2 * most, 0, 0) == 1
    assert take(most + 32, 32, 1, 0) == take(most + 32, 32, 0, 1) == take(32, most // 2 + 32, 1, 0) == take(32, most + 32, 0, 1) == take(0, 32, 0, 0) == 0


def test_launches_of_2_to_the_32_threads_are_refused():
    n = 1 << 30
    assert lib.momoe_ffn_lin1_fwd(P, 32, P, P, None, 0, n, n, 32, 32, None) == lib.momoe_ffn_lin2_fwd(P, P, P, n, n, 32, 32, None, 0, None) == 2
    assert lib.momoe_ffn_dgrad_h(P, 32, P, P, n, 32, 32, None) == lib.momoe_ffn_swiglu_bwd(P, 32, P, P, P, None, None, n, n, n, 32, 32, None) == 2
    assert lib.momoe_ffn_dgrad_h_saved(P, 32, P, P, P, None, None, n, n, n, 32, 32, None) == 2
    assert lib.momoe_ffn_gradients(None, 0, None, 0, P, None, P, None, P, None, None, None, 0, n, n, 32, 32, None) == 2
