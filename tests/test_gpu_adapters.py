"""Lateral convs with a low-rank adapter per image (forward, backward) against 64 bits.

Tolerances are counted.  With u = 2^-24: an fp32 sum of K products is within K u of the sum of
their absolute values (any order); h keeps 2^-22 of itself (parts of 8 or 11 bits, the last one
rounded to half a step; fp16 loses what is below 2^-24, 2^-25 absolute); a 16-bit result is rounded
once, finfo.eps / 2 of its value.  The bounds use the absolute sums, element by element.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last


def _make(n, cin, h, w, rank, count, dtype, dev, seed, index=None):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, scale=1.0, cl=False):
        v = (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)
        return v.contiguous(memory_format=CL) if cl else v
    s = {"x": t(n, cin, h, w, cl=True), "w": t(256, cin, scale=(2 / cin) ** 0.5),
         "b": torch.randn(256, generator=g).to(dev), "down": t(count, rank, cin, scale=cin ** -0.5),
         "up": t(count, 256, rank, scale=0.5), "dy": t(n, 256, h, w, cl=True),
         "scales": (torch.rand(count, generator=g) + 0.5).to(dev)}
    if index is None:
        index = torch.randint(-1, count, (n,), generator=g)
    s["index"] = torch.as_tensor(index, dtype=torch.int32).to(dev)
    return s


def _px(t):
    """[N, C, H, W] -> [N, pixels, C] in 64 bits."""
    return t.double().permute(0, 2, 3, 1).flatten(1, 2)


def _ref(s, scale=1.0, coarse=None):
    """Values and the bounds of their fp32 parts."""
    x, dy, w = _px(s["x"]), _px(s["dy"]), s["w"].double()
    n, p, cin = x.shape
    count, rank = s["down"].shape[:2]
    u = 2.0 ** -24
    fp16 = s["x"].dtype == torch.float16
    hrel, habs = 2.0 ** -22, (2.0 ** -25 if fp16 else 0.0)
    out = x @ w.t() + s["b"].double()
    out_lim = (cin + 8) * u * (x.abs() @ w.abs().t() + s["b"].double().abs())
    dx, dx_lim = dy @ w, 264 * u * (dy.abs() @ w.abs())
    gd, gu = torch.zeros_like(s["down"], dtype=torch.float64), torch.zeros_like(s["up"], dtype=torch.float64)
    gd_lim, gu_lim = torch.zeros_like(gd), torch.zeros_like(gu)
    for i, a in enumerate(s["index"].tolist()):
        if not 0 <= a < count:
            continue
        sc = scale * (s["scales"][a].item() if s["scales"] is not None else 1.0)
        d, up = s["down"][a].double(), s["up"][a].double()
        h = sc * (x[i] @ d.t())
        h_lim = abs(sc) * (cin + 4) * u * (x[i].abs() @ d.abs().t()) + hrel * h.abs() + habs
        out[i] += h @ up.t()
        out_lim[i] += h_lim @ up.abs().t() + (2 * rank + 8) * u * (h.abs() @ up.abs().t())
        dh = sc * (dy[i] @ up)
        dh_lim = abs(sc) * 264 * u * (dy[i].abs() @ up.abs()) + hrel * dh.abs() + habs
        dx[i] += dh @ d
        dx_lim[i] += dh_lim @ d.abs() + (2 * rank + 8) * u * (dh.abs() @ d.abs())
        gd[a] += dh.t() @ x[i]
        gd_lim[a] += dh_lim.t() @ x[i].abs() + (2 * p + n + 8) * u * (dh.abs().t() @ x[i].abs())
        gu[a] += dy[i].t() @ h
        gu_lim[a] += dy[i].abs().t() @ h_lim + (2 * p + n + 8) * u * (dy[i].abs().t() @ h.abs())
    if coarse is not None:
        hh, ww = s["x"].shape[2:]
        up = torch.nn.functional.interpolate(coarse.double(), size=(hh, ww), mode="bilinear", align_corners=False)
        out += _px(up)
        # bilinear weights are rounded to the 16-bit type when the add runs on the tensor cores: half
        # a step of each of the four taps; and their fp32 positions 2^-18 of a pixel at these sizes
        out_lim += (torch.finfo(s["x"].dtype).eps / 2 + 2.0 ** -16) * _px(
            torch.nn.functional.max_pool2d(torch.nn.functional.interpolate(
                coarse.double().abs(), size=(hh, ww), mode="nearest"), 5, 1, 2)) * 2
    back = lambda t: t.unflatten(1, s["x"].shape[2:]).permute(0, 3, 1, 2)  # noqa: E731
    return {"out": back(out), "out_lim": back(out_lim), "dx": back(dx), "dx_lim": back(dx_lim),
            "gd": gd, "gd_lim": gd_lim, "gu": gu, "gu_lim": gu_lim}


def _check(got, ref, lim, what):
    f = torch.finfo(got.dtype)
    lim = lim + f.eps / 2 * (ref.abs() + lim) + f.smallest_normal * f.eps
    err = (got.double() - ref).abs()
    bad = ~(err <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(err / lim).max().item():.3g} of the bound"


SHAPES = [  # n, cin, h, w, rank, adapters
    (1, 8, 1, 1, 1, 1), (3, 64, 5, 7, 16, 2), (2, 256, 16, 17, 16, 3), (4, 96, 11, 13, 4, 2), (2, 320, 1, 129, 20, 5),
    (5, 512, 7, 7, 32, 4), (2, 1024, 9, 14, 64, 2), (1, 2048, 25, 38, 8, 1), (2, 200, 30, 9, 33, 3),
    (70, 256, 1, 1, 8, 9), (3, 72, 1, 2, 7, 40), (2, 136, 40, 61, 48, 2),
    (3, 64, 150, 152, 16, 3), (7, 320, 70, 64, 32, 2)]  # (several tiles per block, some without an adapter)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(cuda_device, dtype, shape):
    import unified_fpn as U
    n, cin, h, w, rank, count = shape
    s = _make(n, cin, h, w, rank, count, dtype, cuda_device, sum(shape))
    ops = (s["down"], s["up"], s["index"])
    out, hidden = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], *ops, scale=s["scales"], return_hidden=True)
    dx, gd, gu = U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], *ops, hidden, scale=s["scales"])
    torch.cuda.synchronize()
    assert U.device_status() == 0
    r = _ref(s)
    assert out.dtype == dtype and out.is_contiguous(memory_format=CL)
    _check(out, r["out"], r["out_lim"], "out")
    _check(dx, r["dx"], r["dx_lim"], "dx")
    _check(gd, r["gd"], r["gd_lim"], "ddown")
    _check(gu, r["gu"], r["gu_lim"], "dup")
    assert torch.equal(out, U.fpn_lateral_adapters(s["x"], s["w"], s["b"], *ops, scale=s["scales"]))
    # adapters' gradients alone, and again: the same bits
    none, gd2, gu2 = U.fpn_lateral_adapters_backward(s["x"], None, s["dy"], *ops, hidden, scale=s["scales"],
                                                     need_input_grad=False)
    assert none is None and torch.equal(gd, gd2) and torch.equal(gu, gu2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("maps", [((20, 31), (10, 16)), ((25, 38), (25, 38)), ((13, 21), (7, 11)), ((1, 1), (1, 1)),
                                  ((40, 6), (13, 3)), ((100, 152), (50, 76))])
def test_top_down_add(cuda_device, dtype, maps):
    import unified_fpn as U
    (h, w), (hc, wc) = maps
    s = _make(3, 128, h, w, 16, 2, dtype, cuda_device, h + wc, index=[1, -1, 0])
    s["scales"] = None
    g = torch.Generator().manual_seed(9)
    coarse = torch.randn(3, 256, hc, wc, generator=g).to(dtype).to(cuda_device).contiguous(memory_format=CL)
    out = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], s["down"], s["up"], s["index"], scale=0.75, coarse=coarse)
    torch.cuda.synchronize()
    assert U.device_status() == 0
    r = _ref(s, scale=0.75, coarse=coarse)
    _check(out, r["out"], r["out_lim"], "out")


def test_images_without_an_adapter_equal_the_plain_lateral(cuda_device):
    """index outside 0 .. L - 1 (either sign, 64-bit ones too): the lateral's values, zero h, and no
    share in any gradient."""
    import unified_fpn as U
    s = _make(5, 256, 12, 19, 16, 3, torch.bfloat16, cuda_device, 3, index=[-1, 3, -7, 2 ** 31 - 1, -2 ** 31])
    ops = (s["down"], s["up"])
    out, hid = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], *ops, s["index"], return_hidden=True)
    plain = U.fpn_lateral_conv(s["x"], s["w"], s["b"])
    assert torch.equal(out, plain) and not hid.any()
    wide = torch.tensor([2 ** 32, 2 ** 32 + 1, -2 ** 40, 3, -1], device=cuda_device)
    assert torch.equal(U.fpn_lateral_adapters(s["x"], s["w"], s["b"], *ops, wide), plain)
    dx, gd, gu = U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], *ops, s["index"], hid)
    assert not gd.any() and not gu.any()
    assert torch.equal(dx, U.fpn_lateral_conv_backward(s["x"], s["w"], s["dy"])[0])


def test_one_adapter_for_all_and_unused_ones(cuda_device):
    """The same index for every image (their gradients add), unused adapters keep zeros, and
    non-finite values of an unused adapter stay out of everything."""
    import unified_fpn as U
    s = _make(6, 128, 9, 10, 12, 4, torch.bfloat16, cuda_device, 4, index=[2] * 6)
    s["down"][[0, 1, 3]] = float("nan")
    s["up"][[0, 1, 3]] = float("inf")
    ops = (s["down"], s["up"], s["index"])
    out, hid = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], *ops, scale=s["scales"], return_hidden=True)
    dx, gd, gu = U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], *ops, hid, scale=s["scales"])
    r = _ref(s)
    for got, k in ((out, "out"), (dx, "dx"), (gd, "gd"), (gu, "gu")):
        _check(got, r[k], r[k + "_lim"], k)
    assert not gd[[0, 1, 3]].any() and not gu[[0, 1, 3]].any()


def test_layouts_dtypes_and_transposed_weight(cuda_device):
    import unified_fpn as U
    s = _make(2, 136, 10, 11, 16, 2, torch.float16, cuda_device, 5, index=[1, 0])
    ops = (s["down"], s["up"], s["index"])
    want, hid = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], *ops, scale=2.0, return_hidden=True)
    nchw = U.fpn_lateral_adapters(s["x"].contiguous(), s["w"].float().view(256, 136, 1, 1), s["b"].double(),
                                  s["down"].float(), s["up"].transpose(1, 2).contiguous().transpose(1, 2),
                                  s["index"].long(), scale=torch.full((2,), 2.0, device=cuda_device))
    assert torch.equal(nchw, want)
    dx = U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], *ops, hid, scale=2.0)[0]
    wt = torch.zeros(256, 256, device=cuda_device, dtype=torch.float16)
    wt[:136] = s["w"].t()
    assert torch.equal(U.fpn_lateral_adapters_backward(s["x"], None, s["dy"], *ops, hid, scale=2.0, weight_t=wt)[0], dx)


def test_fp16_hidden_beyond_its_range(cuda_device):
    """h of 100 000 does not fit fp16; its two parts carry it."""
    import unified_fpn as U
    s = _make(1, 64, 4, 4, 16, 1, torch.float16, cuda_device, 6, index=[0])
    s["x"].fill_(1.0)
    s["down"].fill_(0.0)
    s["down"][0, 0, 0] = 1.0
    s["up"].fill_(2.0 ** -10)
    s["scales"] = None
    out = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], s["down"], s["up"], s["index"], scale=100000.0)
    r = _ref(s, scale=100000.0)
    _check(out, r["out"], r["out_lim"], "out")


def test_gradients_against_differences(cuda_device):
    """Central differences in the adapters' own values: the output is linear in ``up`` and in ``down``,
    so only its rounding to fp16 (2^-11 of its size, averaged over the pixels) enters."""
    import unified_fpn as U
    s = _make(2, 64, 16, 16, 8, 2, torch.float16, cuda_device, 8, index=[1, 1])
    args = (s["x"], s["w"], s["b"])
    _, hid = U.fpn_lateral_adapters(*args, s["down"], s["up"], s["index"], return_hidden=True)
    _, gd, gu = U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], s["down"], s["up"], s["index"], hid)

    def loss(down, up):
        return (U.fpn_lateral_adapters(*args, down, up, s["index"]).double() * s["dy"].double()).sum().item()
    g = torch.Generator().manual_seed(1)
    for name, grad in (("down", gd), ("up", gu)):
        # a step that is exact in fp16: multiples of 1/16 added to values kept to multiples of 1/64
        d = torch.randint(-2, 3, s[name].shape, generator=g).to(cuda_device).half() / 16
        base = (s[name] * 64).round() / 64
        p = {"down": s["down"], "up": s["up"]}
        _, hid = U.fpn_lateral_adapters(*args, **{**p, name: base}, index=s["index"], return_hidden=True)
        r = U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], p["down"] if name == "up" else base,
                                            p["up"] if name == "down" else base, s["index"], hid)
        grad = r[1] if name == "down" else r[2]
        num = (loss(**{**p, name: base + d}) - loss(**{**p, name: base - d})) / 2
        # 2 x 256 x 256 outputs of size up to 16, each off by at most 2^-11 of it on either side, their
        # signs independent: 6 standard deviations of the sum
        lim = 6 * 2.0 ** -11 * 16 * s["dy"].double().norm().item()
        assert abs(num - (grad.double() * d.double()).sum().item()) <= lim, name


def test_streams_and_graph_replay(cuda_device):
    import unified_fpn as U
    s = _make(4, 512, 14, 15, 16, 3, torch.bfloat16, cuda_device, 11, index=[0, 2, -1, 2])
    idx2 = torch.tensor([1, -1, 0, 0], device=cuda_device, dtype=torch.int32)

    def step(index):
        out, hid = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], s["down"], s["up"], index, scale=s["scales"],
                                          return_hidden=True)
        return (out, *U.fpn_lateral_adapters_backward(s["x"], s["w"], s["dy"], s["down"], s["up"], index, hid,
                                                      scale=s["scales"]))
    want, want2 = step(s["index"]), step(idx2)
    got = []
    for i in (s["index"], idx2):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(step(i))
    torch.cuda.synchronize()
    for a, e in zip(got[0] + got[1], want + want2):
        assert torch.equal(a, e)
    static = s["index"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i, e in ((idx2, want2), (s["index"], want)):
        static.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        for a, q in zip(outs, e):
            assert torch.equal(a, q)
    assert U.device_status() == 0


def test_refusals(cuda_device):
    import unified_fpn as U
    s = _make(2, 64, 4, 4, 8, 2, torch.bfloat16, cuda_device, 12, index=[0, 1])
    x, w, b, d, u, i, dy = (s[k] for k in ("x", "w", "b", "down", "up", "index", "dy"))
    _, hid = U.fpn_lateral_adapters(x, w, b, d, u, i, return_hidden=True)
    f, g = U.fpn_lateral_adapters, U.fpn_lateral_adapters_backward
    big = torch.zeros(2, 65, 64, device=cuda_device, dtype=torch.bfloat16)
    bad = [lambda: f(x[:, :60], w, b, d, u, i), lambda: f(x[:0], w, b, d, u, i[:0]), lambda: f(x, w[:128], b, d, u, i),
           lambda: f(x, w, b[:-1], d, u, i), lambda: f(x, w, b, d[:, :, :32], u, i), lambda: f(x, w, b, d, u[:1], i),
           lambda: f(x, w, b, d, u, i[:1]), lambda: f(x, w, b, d, u, i.float()), lambda: f(x, w, b, d, u, i.cpu()),
           lambda: f(x.cpu(), w, b, d, u, i), lambda: f(x, w, b, d, u, i, scale=torch.ones(3, device=cuda_device)),
           lambda: f(x, w, b, big, torch.zeros(2, 256, 65, device=cuda_device), i),
           lambda: f(x, w, b, d, u, i, coarse=dy.float()), lambda: f(x, w, b, d, u, i, coarse=dy[:1]),
           lambda: f(x, w, b, d[0], u, i), lambda: f(x[0], w, b, d, u, i),
           lambda: g(x, w, dy.half(), d, u, i, hid), lambda: g(x, w, dy[:1], d, u, i, hid),
           lambda: g(x, w, dy, d, u, i, hid[:1]), lambda: g(x, None, dy, d, u, i, hid),
           lambda: g(x, None, dy, d, u, i, hid, weight_t=w)]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {k} was not refused")
    with pytest.raises(TypeError):
        f(x.float(), w, b, d, u, i)
    with pytest.raises(U.UFPNError):  # a coarse map larger than the output
        f(x, w, b, d, u, i, coarse=torch.zeros(2, 256, 5, 5, device=cuda_device, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    assert U.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,size", [
    ((1, 1032, 17, 23, 64, 3), (9, 12)),   # four tiles, k in quarters: 17 k-blocks, the last one of 8 channels
    ((2, 2040, 13, 29, 33, 2), (7, 15)),   # six tiles in eighths
    ((2, 520, 40, 41, 9, 2), (20, 21)),    # 26 tiles in halves, ranks that are no whole vectors
    ((37, 712, 3, 43, 40, 5), (2, 43)),    # 74 tiles in halves, one of a single pixel an image
    ((37, 264, 3, 43, 40, 5), (2, 43)),    # too few k-blocks to split
    ((3, 1024, 1, 1, 1, 2), (1, 1))])
def test_few_tiles_split_over_k(cuda_device, dtype, shape, size):
    import unified_fpn as U
    n, cin, h, w, rank, count = shape
    s = _make(n, cin, h, w, rank, count, dtype, cuda_device, sum(shape))
    g = torch.Generator().manual_seed(h)
    coarse = torch.randn(n, 256, *size, generator=g).to(dtype).to(cuda_device).contiguous(memory_format=CL)
    out, hidden = U.fpn_lateral_adapters(s["x"], s["w"], s["b"], s["down"], s["up"], s["index"], scale=s["scales"],
                                         coarse=coarse, return_hidden=True)
    torch.cuda.synchronize()
    assert U.device_status() == 0
    r = _ref(s, coarse=coarse)
    _check(out, r["out"], r["out_lim"], "out")
    # the hidden values: their parts' sum
    hid = hidden.double().sum(3).flatten(1, 2)
    for i, a in enumerate(s["index"].tolist()):
        if not 0 <= a < count:
            assert not hid[i].any()
            continue
        x, d, sc = _px(s["x"])[i], s["down"][a].double(), s["scales"][a].double()
        want = sc * (x @ d.t())
        lim = sc * (cin + 4) * 2.0 ** -24 * (x.abs() @ d.abs().t()) + 2.0 ** -22 * want.abs() + 2.0 ** -25
        assert ((hid[i, :, :rank] - want).abs() <= lim).all()
        assert not hid[i, :, rank:].any()
    # one image of the batch alone (another split): the same within the bounds; NaN stays in its image
    x = s["x"].clone(memory_format=torch.preserve_format)
    x[0] = float("nan")
    other = U.fpn_lateral_adapters(x, s["w"], s["b"], s["down"], s["up"], s["index"], scale=s["scales"], coarse=coarse)
    assert other[0].isnan().all() and torch.equal(other[1:], out[1:])


@pytest.mark.parametrize("h,w", [(3, 5), (130, 120)])  # (split over k, and not)
def test_hidden_values_beyond_the_16_bit_range(cuda_device, h, w):
    """fp16: h = 102 400 (above 65 504) still counts in full; beyond both parts' range the result is not finite
    rather than a wrong number.  bf16: infinities stay infinities."""
    import unified_fpn as U
    dev, cin = cuda_device, 512
    x = torch.ones(2, cin, h, w, device=dev, dtype=torch.float16).contiguous(memory_format=CL)
    wt, b = torch.zeros(256, cin, device=dev, dtype=torch.float16), torch.zeros(256, device=dev)
    down = torch.full((2, 1, cin), 200.0, device=dev, dtype=torch.float16)
    down[1] = 800.0
    up = torch.full((2, 256, 1), 2.0 ** -10, device=dev, dtype=torch.float16)
    index = torch.tensor([0, 1], device=dev)
    out, hid = U.fpn_lateral_adapters(x, wt, b, down, up, index, return_hidden=True)
    assert (out[0] == 100.0).all() and (hid[0].float().sum(2)[..., 0] == 102400.0).all()
    assert not hid[1].float().sum(2)[..., 0].isfinite().any()
    gd, gu = U.fpn_lateral_adapters_backward(x, None, torch.ones_like(out), down, up, index, hid,
                                             need_input_grad=False)[1:]
    assert (gu[0] == 102400.0 * h * w).all() and not gu[1].isfinite().any()
    assert gd[0].isfinite().all()
    xb = x.bfloat16().contiguous(memory_format=CL)
    xb[1, 0, 0, 0] = float("inf")
    out, hid = U.fpn_lateral_adapters(xb, wt.bfloat16(), b, down.bfloat16(), up.bfloat16(), index, return_hidden=True)
    assert (hid[1, 0, 0].float().sum(0)[0] == float("inf")) and hid[0].isfinite().all()
    assert out[0].isfinite().all() and out[1, :, 1:].isfinite().all()
