"""The group norm of small maps at every cluster size it takes (1 to 16 blocks a map, shares up to 96 KB of 640-byte
pixels), and the sizes just beyond, where it asks for a workspace."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last


@pytest.mark.parametrize("n,pixels,small", [
    (1, 1, True), (1, 25, True), (1, 51, True), (1, 102, True), (1, 204, True), (1, 409, True), (1, 2448, True),
    (1, 2449, False), (8, 1224, True), (8, 1225, False), (64, 306, True), (64, 307, False), (128, 153, True),
    (129, 3, False)])
def test_cluster_sizes(cuda_device, n, pixels, small):
    import unified_fpn as U
    from unified_fpn import _lib
    c, groups = 320, 32
    need = _lib.lib.ufpn_group_norm_workspace(2, 1, n, c, (ctypes.c_longlong * 1)(pixels), groups, 0)
    assert (need == 0) == small
    g = torch.Generator().manual_seed(pixels)
    x = (torch.randn(n, c, pixels, 1, generator=g) + torch.randn(1, c, 1, 1, generator=g)).bfloat16()
    x = x.to(cuda_device).contiguous(memory_format=CL)
    y, mean, rstd = U.fpn_group_norm(x, groups=groups, return_stats=True)
    xg = x.double().reshape(n, groups, -1)
    m = xg.mean(-1)
    r = ((xg - m[..., None]) ** 2).mean(-1).add(1e-5).rsqrt()
    z = (xg - m[..., None]) * r[..., None]
    # (fp32 sums: some dozens of u = 2^-24 in the mean, relative to the spread, and in rstd; then a rounding to bf16)
    assert ((mean.double() - m).abs() * r).max() <= 2.0 ** -20 and (rstd.double() / r - 1).abs().max() <= 2.0 ** -20
    lim = 2.0 ** -19 * (1 + z.abs())
    assert ((y.double().reshape(z.shape) - z).abs() <= lim + torch.finfo(y.dtype).eps / 2 * (z.abs() + lim)).all()
    torch.cuda.synchronize()
    assert U.device_status() == 0
