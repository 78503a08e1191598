"""Host side of the group norm and the lateral adapters: what the C entries and the Python functions
refuse before any GPU work, and the workspace sizes (no GPU)."""
import ctypes

import pytest
import torch

OK = 4096  # (an aligned address that is never read: every call here is refused on the host)


@pytest.fixture(scope="module")
def L():
    from unified_fpn import _lib
    return _lib


def _arr(*v):
    return (ctypes.c_void_p * len(v))(*v)


def _px(*v):
    return (ctypes.c_longlong * len(v))(*v)


def _norm(L, **kw):
    """ufpn_group_norm of one map 1 x 64 x 100000 with arguments replaced by name."""
    a = dict(dtype=2, levels=1, x=_arr(OK), y=_arr(OK), weight=None, bias=None, mean=None, rstd=None, N=1, C=64,
             pixels=_px(100000), groups=8, eps=1e-5, act=0, alpha=0.0, ws=OK, ws_bytes=1 << 40)
    a.update(kw)
    return L.lib.ufpn_group_norm(*a.values(), None)


def _norm_bwd(L, **kw):
    a = dict(dtype=2, levels=1, x=_arr(OK), gy=_arr(OK), gx=_arr(OK), weight=None, bias=None, mean=_arr(OK),
             rstd=_arr(OK), gw=None, gb=None, N=1, C=64, pixels=_px(100), groups=8, act=0, alpha=0.0, ws=OK,
             ws_bytes=1 << 40)
    a.update(kw)
    return L.lib.ufpn_group_norm_backward(*a.values(), None)


@pytest.mark.parametrize("call", [_norm, _norm_bwd])
@pytest.mark.parametrize("kw,want", [
    (dict(dtype=99), "UNSUPPORTED"), (dict(levels=0), "INVALID_ARG"), (dict(levels=9), "INVALID_ARG"),
    (dict(x=None), "INVALID_ARG"), (dict(x=_arr(None)), "INVALID_ARG"), (dict(x=_arr(OK + 8)), "ALIGNMENT"),
    (dict(N=0), "INVALID_ARG"), (dict(C=12), "UNSUPPORTED"), (dict(C=2056), "UNSUPPORTED"),
    (dict(groups=0), "INVALID_ARG"), (dict(groups=7), "INVALID_ARG"), (dict(pixels=None), "INVALID_ARG"),
    (dict(pixels=_px(0)), "INVALID_ARG"), (dict(pixels=_px(-4)), "INVALID_ARG"), (dict(act=4), "INVALID_ARG"),
    (dict(pixels=_px(1 << 60)), "INVALID_ARG"), (dict(ws=None), "INVALID_ARG"), (dict(ws_bytes=16), "INVALID_ARG"),
    (dict(ws=OK + 8), "ALIGNMENT")])
def test_group_norm_refusals(L, call, kw, want):
    assert call(L, **kw) == getattr(L, "ERR_" + want), L.lib.ufpn_last_error()


def test_group_norm_refusals_of_one_direction(L):
    assert _norm(L, y=None) == L.ERR_INVALID_ARG
    assert _norm(L, y=_arr(OK + 2)) == L.ERR_ALIGNMENT
    assert _norm(L, mean=_arr(OK)) == L.ERR_INVALID_ARG  # (both statistics or none)
    assert _norm(L, mean=_arr(None), rstd=_arr(OK)) == L.ERR_INVALID_ARG
    assert _norm(L, eps=-1e-5) == L.ERR_INVALID_ARG
    assert _norm(L, eps=float("nan")) == L.ERR_INVALID_ARG
    assert _norm_bwd(L, gy=None) == L.ERR_INVALID_ARG
    assert _norm_bwd(L, mean=None) == L.ERR_INVALID_ARG
    assert _norm_bwd(L, mean=None, rstd=None) == L.ERR_INVALID_ARG
    assert _norm_bwd(L, gx=_arr(OK + 4)) == L.ERR_ALIGNMENT


def test_group_norm_workspace(L):
    size = lambda c=64, g=8, bwd=0, *px: L.lib.ufpn_group_norm_workspace(2, len(px), 2, c, _px(*px), g, bwd)  # noqa: E731
    assert size(64, 8, 0, 100) == 0 and size(64, 8, 0, 100000) > 0  # (small maps need none)
    assert size(64, 8, 1, 100) > 0 and size(64, 8, 1, 100000) > size(64, 8, 0, 100000)
    assert size(64, 8, 0, 1 << 22) < 64 << 20  # (partials, not a copy of the map)
    for bad in ((12, 4, 0, 100), (64, 7, 0, 100), (64, 8, 0, 0), (64, 8, 0), (64, 8, 0, *[4] * 9)):
        assert size(*bad) == 0
    assert L.lib.ufpn_group_norm_workspace(9, 1, 2, 64, _px(4), 8, 0) == 0


def _adapters(L, **kw):
    a = dict(dtype=2, x=OK, w=OK, bias=OK, down=OK, up=OK, index=OK, scales=None, scale=1.0, coarse=None, out=2 * OK,
             hidden=None, N=1, Cin=64, H=4, W=4, rank=8, adapters=2, Hc=0, Wc=0)
    a.update(kw)
    return L.lib.ufpn_lateral_adapters(*a.values(), None)


def _adapters_bwd(L, **kw):
    a = dict(dtype=2, x=OK, w=OK, w_t=None, gout=OK, down=OK, up=OK, index=OK, scales=None, scale=1.0, hidden=OK,
             gx=OK, gdown=OK, gup=OK, N=1, Cin=64, H=4, W=4, rank=8, adapters=2, ws=OK, ws_bytes=1 << 40)
    a.update(kw)
    return L.lib.ufpn_lateral_adapters_backward(*a.values(), None)


@pytest.mark.parametrize("call", [_adapters, _adapters_bwd])
@pytest.mark.parametrize("kw,want", [
    (dict(dtype=0), "UNSUPPORTED"), (dict(dtype=7), "UNSUPPORTED"), (dict(Cin=12), "UNSUPPORTED"),
    (dict(Cin=2056), "UNSUPPORTED"), (dict(rank=0), "UNSUPPORTED"), (dict(rank=65), "UNSUPPORTED"),
    (dict(adapters=65536), "UNSUPPORTED"), (dict(H=1 << 16, W=1 << 15), "UNSUPPORTED"),
    (dict(N=1 << 30, W=8), "UNSUPPORTED"), (dict(N=0), "INVALID_ARG"), (dict(H=-1), "INVALID_ARG"), (dict(adapters=0), "INVALID_ARG"), (dict(x=None), "INVALID_ARG"),
    (dict(w=None), "INVALID_ARG"), (dict(down=None), "INVALID_ARG"), (dict(up=None), "INVALID_ARG"),
    (dict(index=None), "INVALID_ARG"), (dict(x=OK + 2), "ALIGNMENT"), (dict(w=OK + 8), "ALIGNMENT"),
    (dict(down=OK + 2), "ALIGNMENT"), (dict(up=OK + 4), "ALIGNMENT"), (dict(hidden=OK + 2), "ALIGNMENT")])
def test_adapter_refusals(L, call, kw, want):
    assert call(L, **kw) == getattr(L, "ERR_" + want), L.lib.ufpn_last_error()


def test_adapter_refusals_of_one_direction(L):
    assert _adapters(L, bias=None) == L.ERR_INVALID_ARG
    assert _adapters(L, out=None) == L.ERR_INVALID_ARG
    assert _adapters(L, coarse=OK) == L.ERR_INVALID_ARG
    assert _adapters(L, coarse=OK, Hc=5, Wc=2) == L.ERR_INVALID_ARG
    assert _adapters(L, coarse=OK + 2, Hc=2, Wc=2) == L.ERR_ALIGNMENT
    for name in ("gout", "hidden", "gdown", "gup", "ws"):
        assert _adapters_bwd(L, **{name: None}) == L.ERR_INVALID_ARG, name
    assert _adapters_bwd(L, ws_bytes=8) == L.ERR_INVALID_ARG
    assert _adapters_bwd(L, ws=OK + 16) == L.ERR_ALIGNMENT
    assert _adapters_bwd(L, gx=OK + 2) == L.ERR_ALIGNMENT


def test_adapter_workspace(L):
    size = lambda n=2, cin=64, h=8, r=8, k=2, wt=0, dx=1: L.lib.ufpn_lateral_adapters_workspace(2, n, cin, h, h, r, k, wt, dx)  # noqa: E731
    assert size() > size(wt=1) > 0  # (the transposed weights)
    assert size(wt=1) == size(dx=0)
    assert size(n=4) > size()
    for kw in (dict(r=65), dict(r=0), dict(cin=4), dict(k=0), dict(n=0), dict(h=0)):
        assert size(**kw) == 0


def test_python_refuses_cpu_tensors():
    import unified_fpn as U
    x = torch.zeros(1, 64, 4, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        U.fpn_group_norm(x, groups=8)
    with pytest.raises(ValueError, match="activation"):
        U.fpn_group_norm(x, groups=8, activation="gelu")
    with pytest.raises(ValueError, match="eps"):
        U.fpn_group_norm(x, groups=8, eps=-1.0)
    with pytest.raises(ValueError, match="1 to 8"):
        U.fpn_group_norm([])
    with pytest.raises(ValueError, match="CUDA"):
        U.fpn_group_norm_backward(x, x, torch.zeros(1, 8), torch.zeros(1, 8))
    down, up = torch.zeros(1, 4, 64), torch.zeros(1, 256, 4)
    with pytest.raises(ValueError, match="CUDA"):
        U.fpn_lateral_adapters(x, torch.zeros(256, 64), torch.zeros(256), down, up, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="4-D"):
        U.fpn_lateral_adapters(x[0], torch.zeros(256, 64), torch.zeros(256), down, up,
                               torch.zeros(1, dtype=torch.int32))
    for kw in (dict(norm_groups=7), dict(activation="relu"), dict(adapters=1, adapter_rank=65), dict(adapters=-1)):
        with pytest.raises(ValueError):
            U.FPNNeck(**kw)
