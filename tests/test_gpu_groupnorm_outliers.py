"""Group norm where one value lies far from all others, at any pixel: statistics and outputs in units of the
spread.

With u = 2^-24, an outlier D among m values: the spread is at least D / sqrt(m) and the mean D / m.  A thread adds at
most some hundred values of size D / its count and below, in fp32, and the trees over threads and blocks some dozen
more: the mean is off by less than 8 u of the spread (2^-21).  The squares are D^2 and m terms next to nothing: an
addition to what holds D^2 rounds by u of it, up to the small term as a whole, and at these shapes at most 128 follow
one another (pixels of a thread 52, its lanes 8, channels of a lane 64 with one group, else 8, rows of a merge 37):
128 u of the variance, 64 u of rstd (2^-18).  So z = (x - mean) rstd w + b is within 2^-17 |xhat| |w| for rstd, its own
products and the weight's, and 2^-20 (|w| + |b|) for the mean and the sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last


@pytest.mark.parametrize("value", [1e6, -3e4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,c,h,w,groups", [(1, 256, 200, 304, 32), (2, 320, 100, 152, 16), (1, 256, 25, 38, 32),
                                            (3, 64, 7, 9, 8), (2, 1000, 61, 64, 125), (1, 2048, 40, 33, 1)])
def test_one_outlier(cuda_device, dtype, value, n, c, h, w, groups):
    import unified_fpn as U
    g = torch.Generator().manual_seed(c + h)
    base = torch.randn(n, c, h, w, generator=g)
    wt = (torch.rand(c, generator=g) + 0.5).to(cuda_device)
    b = torch.randn(c, generator=g).to(cuda_device)
    every = c // groups
    # (the first pixel of the image; its middle and its last; the first of another block's share)
    for y, x in ((0, 0), (h * w // 2 // w, h * w // 2 % w), (h - 1, w - 1), (h // 3, w // 2), (h // 2, 0)):
        t = base.clone()
        t[:, ::every, y, x] = value
        t = t.to(dtype).to(cuda_device).contiguous(memory_format=CL)
        out, mean, rstd = U.fpn_group_norm(t, wt, b, groups=groups, return_stats=True)
        xg = t.double().reshape(n, groups, -1)
        m = xg.mean(-1)
        r = ((xg - m[..., None]) ** 2).mean(-1).add(1e-5).rsqrt()
        assert ((mean.double() - m).abs() * r).max() <= 2.0 ** -21, (y, x)
        assert (rstd.double() / r - 1).abs().max() <= 2.0 ** -18, (y, x)
        xh = ((xg - m[..., None]) * r[..., None]).reshape(t.shape)
        ref = xh * wt.double().view(1, -1, 1, 1) + b.double().view(1, -1, 1, 1)
        wa, ba = wt.double().view(1, -1, 1, 1), b.double().abs().view(1, -1, 1, 1)
        lim = 2.0 ** -17 * xh.abs() * wa + 2.0 ** -20 * (wa + ba)
        lim = lim + torch.finfo(dtype).eps / 2 * (ref.abs() + lim)
        assert ((out.double() - ref).abs() <= lim).all(), (y, x)
    torch.cuda.synchronize()
    assert U.device_status() == 0
