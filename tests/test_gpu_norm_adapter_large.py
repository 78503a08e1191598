"""Maps of more than 2^31 values: the last image of three, far behind the 32-bit offsets, against a call with it
alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last


def _map(n, c, h, w, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    t = torch.empty(n, h, w, c, device=dev, dtype=torch.bfloat16)
    for i in range(n):
        t[i].normal_(generator=g)
    return t.permute(0, 3, 1, 2)


def test_group_norm(cuda_device):
    import unified_fpn as U
    x, dy = _map(3, 256, 1700, 1650, cuda_device, 1), _map(3, 256, 1700, 1650, cuda_device, 2)
    assert x.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(3)
    w, b = torch.rand(256, device="cuda", generator=g) + 0.5, torch.randn(256, device="cuda", generator=g)
    y, mean, rstd = U.fpn_group_norm(x, w, b, activation="relu", return_stats=True)
    dx, dw, db = U.fpn_group_norm_backward(x, dy, mean, rstd, w, b, activation="relu")
    dw1, db1 = torch.zeros_like(dw), torch.zeros_like(db)
    for i in range(3):
        one = x[i:i + 1]
        y1, m1, r1 = U.fpn_group_norm(one, w, b, activation="relu", return_stats=True)
        dx1, dwi, dbi = U.fpn_group_norm_backward(one, dy[i:i + 1], m1, r1, w, b, activation="relu")
        # (a segment holds one image in either call: the same cut, the same bits)
        assert torch.equal(y[i:i + 1], y1) and torch.equal(mean[i], m1[0]) and torch.equal(rstd[i], r1[0])
        assert torch.equal(dx[i:i + 1], dx1)
        dw1, db1 = dw1 + dwi, db1 + dbi
    # (the same rows in another order: sums over 8.4e6 terms of order one, some hundred additions' 2^-24 of them)
    for got, want in ((dw, dw1), (db, db1)):
        assert (got - want).abs().max() <= 2.0 ** -24 * 256 * 8.4e6 ** 0.5 * 4
    torch.cuda.synchronize()
    assert U.device_status() == 0


def test_adapters(cuda_device):
    import unified_fpn as U
    x, dy = _map(3, 1024, 820, 900, cuda_device, 4), _map(3, 256, 820, 900, cuda_device, 5)
    assert x.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(6)
    t = lambda *s: (torch.randn(*s, generator=g, device="cuda") / 32).bfloat16()  # noqa: E731
    w, down, up, bias = t(256, 1024), t(2, 8, 1024), t(2, 256, 8), torch.zeros(256, device="cuda")
    coarse = _map(3, 256, 410, 450, cuda_device, 7)
    index = torch.tensor([0, -1, 1], device="cuda")
    out, hidden = U.fpn_lateral_adapters(x, w, bias, down, up, index, coarse=coarse, return_hidden=True)
    one = (x[2:], w, bias, down, up, index[2:])
    out1, hidden1 = U.fpn_lateral_adapters(*one, coarse=coarse[2:], return_hidden=True)
    assert torch.equal(out[2:], out1) and torch.equal(hidden[2:], hidden1)
    dx, gd, gu = U.fpn_lateral_adapters_backward(x, w, dy, down, up, index, hidden)
    dx1, gd1, gu1 = U.fpn_lateral_adapters_backward(x[2:], w, dy[2:], down, up, index[2:], hidden1)
    assert torch.equal(dx[2:], dx1)
    # (the same products cut into other splits: 2^-16 of the gradient's norm covers either cut's accumulation)
    for a, b in ((gd, gd1), (gu, gu1)):
        assert (a[1] - b[1]).norm() <= 2.0 ** -16 * b[1].norm()
    torch.cuda.synchronize()
    assert U.device_status() == 0
