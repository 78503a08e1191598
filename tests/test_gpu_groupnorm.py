"""Group norm with an activation (forward, backward) against its definition in 64 bits.

Tolerances are counted, not fitted.  A result is an fp32 computation rounded once to the map's
type: half a step of that type (finfo.eps / 2, relative) plus the fp32 part.  With u = 2^-24, S =
1 + max |x| rstd |w| + |b| bounds every intermediate: x - mean carries u |x| for the stored mean
and u for itself, the mean and rstd a few u each (their sums are trees of at most some dozens of
sequential fp32 additions), the swish of 16-bit maps 2^-21 (1 + |z|) for its approximate exponential and
reciprocal: 16 u S = 2^-20 S covers their sum for values, and each gradient factor below says what it multiplies.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last
ACTS = [None, "relu", "leaky_relu", "swish"]


def _act(z, act, alpha):
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky_relu":
        return torch.where(z > 0, z, alpha * z)
    if act == "swish":
        return z * torch.sigmoid(z)
    return z


def _slope(z, act, alpha):
    if act == "relu":
        return (z > 0).double()
    if act == "leaky_relu":
        return torch.where(z > 0, 1.0, alpha).double()
    if act == "swish":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _ref(x, w, b, groups, eps=1e-5, act=None, alpha=0.01, dy=None):
    """The definition on the input's device in 64 bits."""
    n, c, h, wd = x.shape
    xg = x.double().reshape(n, groups, -1)
    mean = xg.mean(-1)
    rstd = ((xg - mean[..., None]) ** 2).mean(-1).add(eps).rsqrt()
    xh = ((xg - mean[..., None]) * rstd[..., None]).reshape(n, c, h, wd)
    wt = torch.ones(c, device=x.device).double() if w is None else w.double()
    bs = torch.zeros(c, device=x.device).double() if b is None else b.double()
    z = xh * wt.view(1, -1, 1, 1) + bs.view(1, -1, 1, 1)
    r = {"y": _act(z, act, alpha), "z": z, "mean": mean, "rstd": rstd, "xh": xh}
    if dy is not None:
        dz = dy.double() * _slope(z, act, alpha)
        wdz = dz * wt.view(1, -1, 1, 1)
        a1 = wdz.reshape(n, groups, -1).mean(-1, keepdim=True)
        a2 = (wdz * xh).reshape(n, groups, -1).mean(-1, keepdim=True)
        r["dx"] = ((wdz.reshape(n, groups, -1) - a1 - xh.reshape(n, groups, -1) * a2)
                   * rstd[..., None]).reshape(n, c, h, wd)
        r["dw"], r["db"] = (dz * xh).sum((0, 2, 3)), dz.sum((0, 2, 3))
        r["abs_dw"], r["abs_db"] = (dz * xh).abs().sum((0, 2, 3)), dz.abs().sum((0, 2, 3))
    return r


def _scale(x, r, w, b):
    """S of the module's comment."""
    wm = 1.0 if w is None else w.abs().max().item()
    bm = 0.0 if b is None else b.abs().max().item()
    return 1 + x.double().abs().max().item() * r["rstd"].max().item() * wm + bm


def _check(got, ref, atol, what):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # half a subnormal step
    err = (got.double() - ref).abs()
    lim = half * (ref.abs() + atol) + atol + tiny
    bad = err > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {(err / lim).max().item():.3g} of the bound"


def _inputs(n, c, h, w, dtype, dev, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, c, h, w, generator=g) + offset * torch.randn(1, c, 1, 1, generator=g)).to(dtype)
    wt = torch.rand(c, generator=g) + 0.5
    b = torch.randn(c, generator=g) * 0.3
    dy = torch.randn(n, c, h, w, generator=g).to(dtype)
    cl = lambda t: t.to(dev).contiguous(memory_format=CL)  # noqa: E731
    return cl(x), wt.to(dev), b.to(dev), cl(dy)


SHAPES = [(1, 256, 25, 38, 32), (2, 256, 1, 1, 32), (3, 320, 7, 11, 16), (2, 40, 5, 3, 8), (1, 8, 33, 1, 1),
          (2, 24, 9, 9, 24), (1, 2048, 3, 5, 1), (2, 1000, 4, 4, 125), (5, 64, 2, 2, 2), (1, 256, 131, 97, 32),
          (2, 256, 16, 24, 256), (2, 2048, 2, 3, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(cuda_device, dtype, shape):
    import unified_fpn as U
    n, c, h, w, groups = shape
    x, wt, b, _ = _inputs(n, c, h, w, dtype, cuda_device, c + h)
    act = ACTS[(c // 8 + h) % 4]
    y, mean, rstd = U.fpn_group_norm(x, wt, b, groups=groups, activation=act, alpha=0.2, return_stats=True)
    r = _ref(x, wt, b, groups, act=act, alpha=0.2)
    s = _scale(x, r, wt, b)
    assert y.dtype == dtype and y.is_contiguous(memory_format=CL)
    _check(y, r["y"], 2.0 ** -20 * s, "y")
    _check(mean, r["mean"], 2.0 ** -22 * x.abs().max().item(), "mean")
    # (rstd: its relative error is half the variance's, whose squares and means carry some u each,
    # and the mean's error enters squared; exact for a constant group: var = 0)
    _check(rstd / r["rstd"], torch.ones_like(r["rstd"]), 2.0 ** -20, "rstd")
    y2 = U.fpn_group_norm(x, wt, b, groups=groups, activation=act, alpha=0.2)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_activations_and_defaults(cuda_device, dtype, act):
    import unified_fpn as U
    x, _, b, _ = _inputs(2, 96, 10, 13, dtype, cuda_device, 5)
    y = U.fpn_group_norm(x, None, b, groups=12, eps=1e-3, activation=act)
    r = _ref(x, None, b, 12, eps=1e-3, act=act)
    _check(y, r["y"], 2.0 ** -20 * _scale(x, r, None, b), "y")
    y = U.fpn_group_norm(x, groups=12, eps=1e-3, activation=act)
    r = _ref(x, None, None, 12, eps=1e-3, act=act)
    _check(y, r["y"], 2.0 ** -20 * _scale(x, r, None, None), "y")


def test_large_offset_and_constant_groups(cuda_device):
    """A mean 4 000 times the spread costs no more than the mean's own rounding; a constant group
    normalises to exactly the bias."""
    import unified_fpn as U
    x, wt, b, _ = _inputs(2, 64, 40, 30, torch.float32, cuda_device, 9)
    x = (x * 0.25 + 1000).contiguous(memory_format=CL)
    y, mean, rstd = U.fpn_group_norm(x, wt, b, groups=8, return_stats=True)
    r = _ref(x, wt, b, 8)
    _check(y, r["y"], 2.0 ** -20 * _scale(x, r, wt, b), "y")
    _check(rstd / r["rstd"], torch.ones_like(r["rstd"]), 2.0 ** -20, "rstd")
    x[:, :8] = 3.0
    y = U.fpn_group_norm(x, wt, b, groups=8)
    assert torch.equal(y[:, :8], b[:8].view(1, 8, 1, 1).expand(2, 8, 40, 30))


def test_non_finite_values_stay_in_their_group(cuda_device):
    import unified_fpn as U
    x, wt, b, _ = _inputs(2, 64, 12, 9, torch.bfloat16, cuda_device, 11)
    clean = U.fpn_group_norm(x, wt, b, groups=8)
    x[0, 3, 4, 4] = float("nan")
    x[1, 20, 0, 0] = float("inf")
    y = U.fpn_group_norm(x, wt, b, groups=8)
    bad = torch.zeros(2, 64, dtype=torch.bool, device=cuda_device)
    bad[0, :8] = True
    bad[1, 16:24] = True
    assert torch.isnan(y.float()[bad]).all()
    assert torch.equal(y.permute(0, 2, 3, 1)[:, :, :][~bad[:, None, None, :].expand(2, 12, 9, 64)],
                       clean.permute(0, 2, 3, 1)[~bad[:, None, None, :].expand(2, 12, 9, 64)])


def test_layouts_in_place_and_many_images(cuda_device):
    import unified_fpn as U
    x, wt, b, _ = _inputs(3, 64, 6, 7, torch.float16, cuda_device, 13)
    y = U.fpn_group_norm(x, wt, b, groups=4, activation="relu")
    assert torch.equal(U.fpn_group_norm(x.contiguous(), wt, b, groups=4, activation="relu"), y)
    wide = torch.zeros(3, 128, 6, 7, device=cuda_device, dtype=torch.float16).contiguous(memory_format=CL)
    wide[:, :64] = x
    assert torch.equal(U.fpn_group_norm(wide[:, :64], wt.double(), b.half().float(), groups=4), U.fpn_group_norm(
        x, wt, b.half(), groups=4))
    z = x.clone(memory_format=torch.preserve_format)
    assert U.fpn_group_norm(z, wt, b, groups=4, activation="relu", out=z) is z
    assert torch.equal(z, y)
    x, wt, b, _ = _inputs(700, 32, 3, 2, torch.float32, cuda_device, 14)
    y = U.fpn_group_norm(x, wt, b, groups=4)
    r = _ref(x, wt, b, 4)
    _check(y, r["y"], 2.0 ** -20 * _scale(x, r, wt, b), "y")


PYRAMID = [(40, 61), (20, 31), (10, 16), (5, 8), (3, 4), (1, 1), (2, 1), (1, 2)]


@pytest.mark.parametrize("per_level", [False, True])
def test_pyramid_in_one_call_equals_single_maps(cuda_device, per_level):
    import unified_fpn as U
    xs, dys, ws, bs = [], [], [], []
    for i, (h, w) in enumerate(PYRAMID):
        x, wt, b, dy = _inputs(2, 64, h, w, torch.bfloat16, cuda_device, 20 + i)
        xs.append(x), dys.append(dy), ws.append(wt), bs.append(b)
    w, b = (ws, bs) if per_level else (ws[0], bs[0])
    ys, means, rstds = U.fpn_group_norm(xs, w, b, groups=8, activation="swish", return_stats=True)
    dxs, dw, db = U.fpn_group_norm_backward(xs, dys, means, rstds, w, b, activation="swish")
    tot_w = tot_b = 0
    for i, x in enumerate(xs):
        wi, bi = ws[i if per_level else 0], bs[i if per_level else 0]
        r = _ref(x, wi, bi, 8, act="swish", dy=dys[i])
        s = _scale(x, r, wi, bi)
        _check(ys[i], r["y"], 2.0 ** -20 * s, f"y {i}")
        _check_dx(dxs[i], r, s, wi, dys[i])
        if per_level:
            _check_sums(dw[i], db[i], r, s)
        else:
            tot_w, tot_b = tot_w + r["dw"], tot_b + r["db"]
    if not per_level:
        lim = sum(_ref(x, ws[0], bs[0], 8, act="swish", dy=d)["abs_dw"] for x, d in zip(xs, dys))
        assert ((dw.double() - tot_w).abs() <= 2.0 ** -16 * lim).all()
        assert (db.double() - tot_b).abs().max() <= 2.0 ** -16 * lim.max()


def _check_dx(dx, r, s, w, dy, what="dx"):
    # dz carries |dy| (16 u S + 2^-21) from z and the sigmoid; dx multiplies it by rstd |w| (1 + |xhat|)
    # once for itself and once more through each mean
    wm = 1.0 if w is None else w.abs().max().item()
    xm = 1 + r["xh"].abs().max().item()
    atol = 2.0 ** -19 * s * r["rstd"].max().item() * wm * max(wm, 1) * dy.double().abs().max().item() * xm * xm
    _check(dx, r["dx"], atol, what)


def _check_sums(dw, db, r, s):
    # every term: dz's error and xhat's, 32 u S relative to |dy xhat| at most; the sum's own
    # additions (some dozens in sequence, then a tree) stay below 64 u of the absolute sum
    lim = 2.0 ** -18 * (1 + s)
    assert ((dw.double() - r["dw"]).abs() <= lim * (r["abs_dw"] + r["abs_db"])).all()
    assert ((db.double() - r["db"]).abs() <= lim * r["abs_db"] + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(cuda_device, dtype, shape):
    import unified_fpn as U
    n, c, h, w, groups = shape
    x, wt, b, dy = _inputs(n, c, h, w, dtype, cuda_device, c + h + 1)
    act = ACTS[(c // 8 + h + 1) % 4]
    r = _ref(x, wt, b, groups, act=act)
    s = _scale(x, r, wt, b)
    # no gradient where z is within its own error of an activation's kink
    dy = torch.where(r["z"].abs() < 2.0 ** -18 * s, 0.0, dy.float()).to(dtype).contiguous(memory_format=CL)
    r = _ref(x, wt, b, groups, act=act, dy=dy)
    _, mean, rstd = U.fpn_group_norm(x, wt, b, groups=groups, activation=act, return_stats=True)
    dx, dw, db = U.fpn_group_norm_backward(x, dy, mean, rstd, wt, b, activation=act)
    assert dx.dtype == dtype and dx.is_contiguous(memory_format=CL) and dw.dtype == torch.float32
    _check_dx(dx, r, s, wt, dy)
    _check_sums(dw, db, r, s)
    none, dw2, db2 = U.fpn_group_norm_backward(x, dy, mean, rstd, wt, b, activation=act, need_input_grad=False)
    assert none is None and torch.equal(dw, dw2) and torch.equal(db, db2)


def test_backward_without_weights_and_one_value_groups(cuda_device):
    """Groups of one value: xhat = 0 and every gradient of x is exactly 0."""
    import unified_fpn as U
    x, _, _, dy = _inputs(3, 16, 1, 1, torch.float32, cuda_device, 31)
    _, mean, rstd = U.fpn_group_norm(x, groups=16, return_stats=True)
    dx, dw, db = U.fpn_group_norm_backward(x, dy, mean, rstd)
    assert torch.equal(dx, torch.zeros_like(dx)) and torch.equal(dw, torch.zeros_like(dw))
    torch.testing.assert_close(db, dy.sum((0, 2, 3)), rtol=2.0 ** -22, atol=2.0 ** -22)


def test_backward_against_differences(cuda_device):
    """<dx, d> against central differences of the forward kernel's own outputs (fp32): truncation
    h^2 / 6 of a third derivative of order one, noise 2^-23 sqrt(values) / h."""
    import unified_fpn as U
    x, wt, b, dy = _inputs(2, 32, 9, 8, torch.float32, cuda_device, 37)
    g = torch.Generator().manual_seed(38)
    d = torch.randn(x.shape, generator=g).to(cuda_device)
    h = 2.0 ** -7

    def loss(t, w_, b_):
        return (U.fpn_group_norm(t.contiguous(memory_format=CL), w_, b_, groups=4, activation="swish").double()
                * dy.double()).sum().item()
    _, mean, rstd = U.fpn_group_norm(x, wt, b, groups=4, activation="swish", return_stats=True)
    dx, dw, db = U.fpn_group_norm_backward(x, dy, mean, rstd, wt, b, activation="swish")
    norm = (dx.double() ** 2).sum().sqrt().item() * (d.double() ** 2).sum().sqrt().item()
    num = (loss(x + h * d, wt, b) - loss(x - h * d, wt, b)) / (2 * h)
    assert abs(num - (dx.double() * d.double()).sum().item()) <= 2e-3 * norm
    dwv = torch.randn(32, generator=g).to(cuda_device)
    num = (loss(x, wt + h * dwv, b) - loss(x, wt - h * dwv, b)) / (2 * h)
    assert abs(num - (dw.double() * dwv.double()).sum().item()) <= 2e-3 * dw.norm().item() * dwv.norm().item()
    num = (loss(x, wt, b + h * dwv) - loss(x, wt, b - h * dwv)) / (2 * h)
    assert abs(num - (db.double() * dwv.double()).sum().item()) <= 2e-3 * db.norm().item() * dwv.norm().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_batches_larger_than_the_cache(cuda_device, dtype):
    """Several launches per call: images split over runs, forward and backward, the sums over all."""
    import unified_fpn as U
    n = 5 if dtype == torch.bfloat16 else 3
    g = torch.Generator(device="cuda").manual_seed(41)
    xs = [torch.randn(n, h, w, 256, device="cuda", generator=g).to(dtype).permute(0, 3, 1, 2)
          for h, w in [(200, 150), (100, 75)]]
    dys = [torch.randn(x.permute(0, 2, 3, 1).shape, device="cuda", generator=g).to(dtype).permute(0, 3, 1, 2)
           for x in xs]
    wt, b = torch.rand(256, device="cuda", generator=g) + 0.5, torch.randn(256, device="cuda", generator=g)
    ys, m, rs = U.fpn_group_norm(xs, wt, b, activation="swish", return_stats=True)
    dxs, dw, db = U.fpn_group_norm_backward(xs, dys, m, rs, wt, b, activation="swish")
    dw64 = db64 = lw = lb = 0
    for i, x in enumerate(xs):
        r = _ref(x, wt, b, 32, act="swish", dy=dys[i])
        s = _scale(x, r, wt, b)
        _check(ys[i], r["y"], 2.0 ** -20 * s, "y")
        _check_dx(dxs[i], r, s, wt, dys[i])
        dw64, db64, lw, lb = dw64 + r["dw"], db64 + r["db"], lw + r["abs_dw"], lb + r["abs_db"]
    lim = 2.0 ** -18 * (1 + s)
    assert ((dw.double() - dw64).abs() <= lim * (lw + lb)).all() and ((db.double() - db64).abs() <= lim * lb).all()


def test_streams_and_graph_replay(cuda_device):
    """The call on a side stream, two at once, and captured into a graph that is replayed on new
    values: the same bits each time."""
    import unified_fpn as U
    x, wt, b, dy = _inputs(2, 256, 33, 21, torch.bfloat16, cuda_device, 51)
    x2 = _inputs(2, 256, 33, 21, torch.bfloat16, cuda_device, 52)[0]

    def step(t):
        y, m, r = U.fpn_group_norm(t, wt, b, activation="swish", return_stats=True)
        return (y, *U.fpn_group_norm_backward(t, dy, m, r, wt, b, activation="swish"))
    want, want2 = step(x), step(x2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, t in zip(streams, (x, x2)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(t))
    torch.cuda.synchronize()
    for a, e in zip(got[0] + got[1], want + want2):
        assert torch.equal(a, e)
    static = x.clone(memory_format=torch.preserve_format)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for t, e in ((x2, want2), (x, want)):
        static.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, q in zip(out, e):
            assert torch.equal(a, q)


def test_refusals(cuda_device):
    import unified_fpn as U
    x, wt, b, dy = _inputs(2, 64, 4, 4, torch.bfloat16, cuda_device, 61)
    _, mean, rstd = U.fpn_group_norm(x, wt, b, groups=8, return_stats=True)
    bad = [lambda: U.fpn_group_norm(x, wt, b, groups=7), lambda: U.fpn_group_norm(x, wt[:-1], b, groups=8),
           lambda: U.fpn_group_norm(x, wt, b.cpu(), groups=8), lambda: U.fpn_group_norm(x.cpu(), groups=8),
           lambda: U.fpn_group_norm(x[:, :60], groups=4), lambda: U.fpn_group_norm(x, groups=8, activation="gelu"),
           lambda: U.fpn_group_norm(x, groups=8, eps=-1.0), lambda: U.fpn_group_norm([x] * 9, groups=8),
           lambda: U.fpn_group_norm([], groups=8), lambda: U.fpn_group_norm([x, x.float()], groups=8),
           lambda: U.fpn_group_norm(x[:0], groups=8), lambda: U.fpn_group_norm(x, [wt, wt], b, groups=8),
           lambda: U.fpn_group_norm(x, groups=8, out=x.float()), lambda: U.fpn_group_norm(x[0], groups=8),
           lambda: U.fpn_group_norm(x, groups=8, eps=float("nan")),
           lambda: U.fpn_group_norm_backward(x, dy.float(), mean, rstd, wt, b),
           lambda: U.fpn_group_norm_backward(x, dy[:1], mean, rstd, wt, b),
           lambda: U.fpn_group_norm_backward(x, dy, mean[:1], rstd, wt, b),
           lambda: U.fpn_group_norm_backward(x, dy, mean, rstd.double(), wt, b)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        U.fpn_group_norm(x.double(), groups=8)
    # a map whose storage starts off a 16-byte boundary
    flat = torch.zeros(x.numel() + 1, device=cuda_device, dtype=torch.bfloat16)[1:]
    shifted = flat.view(2, 4, 4, 64).permute(0, 3, 1, 2)
    with pytest.raises(U.UFPNError):
        U.fpn_group_norm(shifted, groups=8)
    torch.cuda.synchronize()
