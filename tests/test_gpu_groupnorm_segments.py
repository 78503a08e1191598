"""Group norm over more segments than the statistics may run ahead of the application (seven images of 35 MB, a
segment each, in either direction), with gradients whose group means matter.

dy = p + q xhat + noise with p and q of order one, other ones for every image and group: both sums that the
backward takes back out of dx are as large as the gradient itself, and another segment's would show.  Bounds element by
element: every fp32 term of dx carries at most 2^-18 of itself (its products, the statistics' 2^-20 and the swish's
2^-21 (1 + |z|)), the group means 2^-18 of the mean absolute term, and the result half a step of the map's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "swish"])
@pytest.mark.parametrize("dtype,c", [(torch.bfloat16, 256), (torch.float16, 256), (torch.float32, 128)])
def test_seven_segments(cuda_device, dtype, c, act):
    import unified_fpn as U
    n, h, w, groups = 7, 250, 274, 16
    g = torch.Generator(device="cuda").manual_seed(c)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    spread, offset = rand(n, 1, groups, 1).exp(), 3 * rand(n, 1, groups, 1)
    x = (rand(n, h * w, groups, c // groups) * spread + offset).to(dtype)
    x = x.view(n, h, w, c).permute(0, 3, 1, 2)
    wt, b = torch.rand(c, generator=g, device="cuda") + 0.5, rand(c) * 0.3
    dy = torch.empty_like(x)
    p, q = rand(n, groups, 1), rand(n, groups, 1)

    def image(i):
        """xhat, z, rstd of image i in 64 bits, [groups, values]."""
        v = x[i].double().reshape(groups, -1)
        d = v - v.mean(1, keepdim=True)
        r = (d * d).mean(1, keepdim=True).add(1e-5).rsqrt()
        wg, bg = (t.double().view(groups, -1, 1).expand(groups, c // groups, h * w).reshape(groups, -1) for t in (wt, b))
        return d * r, d * r * wg + bg, r, wg
    for i in range(n):
        xh = image(i)[0]
        dy[i] = (p[i] + q[i] * xh + rand(*xh.shape)).reshape(c, h, w).to(dtype)
    y, mean, rstd = U.fpn_group_norm(x, wt, b, groups=groups, activation=act, return_stats=True)
    dx, dw, db = U.fpn_group_norm_backward(x, dy, mean, rstd, wt, b, activation=act)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    sums = torch.zeros(4, c, device="cuda", dtype=torch.float64)
    for i in range(n):
        xh, z, r, wg = image(i)
        sig = torch.sigmoid(z)
        val = z * sig if act else z
        lim = 2.0 ** -18 * (1 + xh.abs()) * (wg + 1) * (1 + z.abs() if act else 1)
        assert ((y[i].double().reshape(groups, -1) - val).abs() <= lim + half * (val.abs() + lim) + tiny).all(), i
        slope = sig * (1 + z * (1 - sig)) if act else torch.ones_like(z)
        dz = dy[i].double().reshape(groups, -1) * slope
        err = 2.0 ** -18 * dy[i].double().abs().reshape(groups, -1) * (1 + z.abs())  # of dz
        t = wg * dz
        m1, m2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
        a1, a2 = (wg * (dz.abs() + err)).mean(1, keepdim=True), (wg * (dz.abs() + err) * xh.abs()).mean(1, keepdim=True)
        want = r * (t - m1 - xh * m2)
        lim = r * (wg * err + 2.0 ** -18 * (t.abs() + a1 + (1 + xh.abs()) * a2)
                   + (wg * err).mean(1, keepdim=True) + xh.abs() * (wg * err * xh.abs()).mean(1, keepdim=True))
        got = dx[i].double().reshape(groups, -1)
        assert ((got - want).abs() <= lim + half * (want.abs() + lim) + tiny).all(), i
        # the bound sees the means: without them most values would be off
        if dtype is not torch.bfloat16:
            assert ((got - r * t).abs() > lim + half * (want.abs() + lim)).double().mean() > 0.9
        per_c = lambda v: v.reshape(c, -1).sum(1)  # noqa: E731
        sums += torch.stack([per_c(dz * xh), per_c(dz), per_c((dz.abs() + err) * (1 + xh.abs())), per_c(dz.abs() + err)])
    # (the sums' own terms as above; 64 u for some dozens of additions in sequence and the trees)
    assert ((dw.double() - sums[0]).abs() <= 2.0 ** -17 * sums[2]).all()
    assert ((db.double() - sums[1]).abs() <= 2.0 ** -17 * sums[3]).all()
    # again, and in place: the same bits
    dx2, dw2, db2 = U.fpn_group_norm_backward(x, dy, mean, rstd, wt, b, activation=act)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)
    assert torch.equal(U.fpn_group_norm(x, wt, b, groups=groups, activation=act, out=x), y)
    torch.cuda.synchronize()
    assert U.device_status() == 0
