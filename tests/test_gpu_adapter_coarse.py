"""The top-down add of the adapters' lateral in each of its forms: the bilinear weights beside the output's own
rounding, and values of ``coarse`` that are not finite, which reach the pixels that use them and no others.

Pixels beside those may be computed in another form than without them.  Both forms round the same sum once, in
fp32 before that: with A the sum of the products' absolute values and M the largest of coarse, either is within
(K + 2 R + 16) 2^-24 A and 4 x 2^-17 M (two-part weights) of it, and the results within a 16-bit step more."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last
MAPS = [  # h, w, hc, wc, cin
    (32, 48, 16, 24, 64), (64, 96, 8, 24, 128), (101, 67, 51, 34, 64), (150, 160, 50, 54, 320), (48, 64, 47, 63, 64),
    (200, 304, 100, 152, 256),                         # on the tensor cores, exact weights and others
    (100, 152, 50, 76, 64), (40, 30, 40, 30, 64), (129, 40, 43, 40, 192), (40, 6, 13, 3, 64),  # other boxes
    (13, 21, 7, 11, 1024), (12, 14, 12, 14, 512), (9, 30, 3, 10, 2048), (1, 1, 1, 1, 512)]  # split over k


def _source(out, size, dev):
    return ((torch.arange(out, device=dev, dtype=torch.float64) + 0.5) * (size / out) - 0.5).clamp(0, size - 1)


def _weights(out, size, dev):
    """[out, size] in 64 bits."""
    return (1 - (_source(out, size, dev)[:, None] - torch.arange(size, device=dev)).abs()).clamp(min=0)


def _inputs(dev, dtype, maps, rank, zero=False, n=2):
    h, w, hc, wc, cin = maps
    g = torch.Generator().manual_seed(h + w + rank)

    def t(*shape, size=1.0):
        return (torch.randn(*shape, generator=g) * (0.0 if zero else size)).to(dtype).to(dev)
    x = t(n, cin, h, w).contiguous(memory_format=CL)
    args = (x, t(256, cin, size=cin ** -0.5), torch.zeros(256, device=dev), t(2, rank, cin, size=cin ** -0.5),
            t(2, 256, rank, size=0.3), torch.tensor([1, -1][:n], device=dev))
    coarse = torch.randn(n, 256, hc, wc, generator=g).to(dtype).to(dev).contiguous(memory_format=CL)
    return args, coarse


def _beside(out, clean, args, coarse, keep):
    """Whether ``out`` is ``clean`` at ``keep``, but for another order of the sums."""
    x, w, _, down, up, _ = (a.double().abs() for a in args)
    px = x.permute(0, 2, 3, 1)
    a = (px @ w.t()).max() + (px @ down[1].t() @ up[1].t()).max()
    limit = 2 * (x.shape[1] + 2 * down.shape[1] + 16) * 2.0 ** -24 * a + 2.0 ** -14 * coarse.abs().max()
    limit = limit + torch.finfo(clean.dtype).eps * (clean.double().abs() + limit)
    return bool(((out.double() - clean.double()).abs() <= limit)[keep].all())


@pytest.mark.parametrize("rank", [4, 32, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("maps", MAPS)
def test_weights(cuda_device, dtype, maps, rank):
    import unified_fpn as U
    h, w, hc, wc, _ = maps
    args, coarse = _inputs(cuda_device, dtype, maps, rank, zero=True)
    out = U.fpn_lateral_adapters(*args, coarse=coarse)
    ref = _weights(h, hc, cuda_device) @ coarse.double() @ _weights(w, wc, cuda_device).t()
    # A weight has 16 bits and more (2^-17 of it lost); fp32 positions up to 151 are 3 x 2^-24 of them off,
    # 2^-15, on either axis, each times a difference of taps.  With M the largest value: 2^-17 M + 2 x 2^-15 x 2 M.
    limit = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -12.9 * coarse.abs().max().item()
    assert ((out.double() - ref).abs() <= limit).all()
    # the weights sum to 1 within 2^-15: nearer to 1 than to its neighbours
    ones = U.fpn_lateral_adapters(*args, coarse=torch.ones_like(coarse))
    assert (ones == 1).all()
    torch.cuda.synchronize()
    assert U.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("maps", MAPS)
def test_values_that_are_not_finite(cuda_device, dtype, maps):
    import unified_fpn as U
    h, w, hc, wc, _ = maps
    inf = float("inf")
    # (image, channel, row, column, value); the last two meet in one channel
    spots = [(0, 5, hc // 2, wc // 2, inf), (0, 200, 0, 0, float("nan")), (1, 64, hc - 1, wc - 1, -inf),
             (1, 255, hc // 3, wc - 1, inf), (1, 7, 0, wc // 2, inf), (1, 7, 0, min(wc // 2 + 1, wc - 1), -inf)]
    for rank in (4, 64):
        args, coarse = _inputs(cuda_device, dtype, maps, rank)
        clean, finite = U.fpn_lateral_adapters(*args, coarse=coarse), coarse.clone()
        must = torch.zeros(clean.shape, dtype=torch.bool, device=cuda_device)
        may = must.clone()
        sy, sx = _source(h, hc, cuda_device), _source(w, wc, cuda_device)
        for n, c, r, q, v in spots:
            coarse[n, c, r, q] = v
            dy, dx = (sy - r).abs()[:, None], (sx - q).abs()[None, :]
            # (fp32 positions are up to 2^-15 off: a weight below that may be 0, one of 0 be that)
            must[n, c] |= (dy < 1 - 1e-4) & (dx < 1 - 1e-4)
            may[n, c] |= (dy < 1 + 1e-4) & (dx < 1 + 1e-4)
        for _ in range(2):
            out = U.fpn_lateral_adapters(*args, coarse=coarse)
            assert not out[must].isfinite().any()
            assert _beside(out, clean, args, finite, ~may)
    torch.cuda.synchronize()
    assert U.device_status() == 0


def test_many_tiles_with_and_without(cuda_device):
    """Several tiles a block, the values in some of them only; with h, which is stored twice there."""
    import unified_fpn as U
    maps = (208, 304, 104, 152, 64)
    args, coarse = _inputs(cuda_device, torch.bfloat16, maps, 16)
    clean, hidden = U.fpn_lateral_adapters(*args, coarse=coarse, return_hidden=True)
    g = torch.Generator().manual_seed(1)
    pick = (torch.rand(2, 1, 104, 152, generator=g) < 2e-4).expand(2, 256, 104, 152).to(cuda_device)
    dirty = torch.where(pick, torch.full_like(coarse, float("inf")), coarse).contiguous(memory_format=CL)
    out, hidden2 = U.fpn_lateral_adapters(*args, coarse=dirty, return_hidden=True)
    used = (_weights(208, 104, cuda_device) @ pick.double() @ _weights(304, 152, cuda_device).t()) > 0
    assert pick.any() and not out[used].isfinite().any() and torch.equal(hidden, hidden2)
    assert _beside(out, clean, args, coarse, ~used)
    torch.cuda.synchronize()
    assert U.device_status() == 0


def test_graph_replay_and_streams(cuda_device):
    """A captured call on coarse maps that come and go with such values, and two calls at once."""
    import unified_fpn as U
    args, coarse = _inputs(cuda_device, torch.bfloat16, (101, 67, 51, 34, 64), 16)
    dirty = coarse.clone(memory_format=torch.preserve_format)
    dirty[:, 3, 20, 20] = float("nan")
    want = [U.fpn_lateral_adapters(*args, coarse=c) for c in (coarse, dirty)]
    assert not want[1].isfinite().all() and want[0].isfinite().all()
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))  # noqa: E731
    static = coarse.clone(memory_format=torch.preserve_format)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = U.fpn_lateral_adapters(*args, coarse=static)
    for k in (1, 0, 1, 1, 0):
        static.copy_((coarse, dirty)[k])
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want[k]), k
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    got = []
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((k, U.fpn_lateral_adapters(*args, coarse=(coarse, dirty)[k])))
    torch.cuda.synchronize()
    assert all(same(o, want[k]) for k, o in got)
    assert U.device_status() == 0
