"""The adapters' fp32 gradients for fp16 operands of every size, small ones above all: ``up`` starts at zero
in training, so that the gradient at the hidden values (dh = scale dy up) is far below fp16's steps.

The bound is relative to the gradient's norm and knows no absolute floor.  A tensor-core accumulation
rounds each of its steps towards zero, by up to 2^-23 of the accumulator: 16 steps make dh or h (K = 256), at
most 64 of a split's k-steps one accumulator of the gradient, so 2^-19 + 2^-17; the parts of dh and h keep
2^-22, the fp32 sums over splits less.  Together below 2^-16."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last
LIMIT = 2.0 ** -16


def _run(dev, dtype, dy_size, up_size, x_size, down_size, rank=16, n=2, cin=256, h=33, w=31):
    import unified_fpn as U
    g = torch.Generator().manual_seed(rank + h)

    def t(*shape, size):
        return (torch.randn(*shape, generator=g) * size).to(dtype).to(dev)
    x, dy = (t(n, c, h, w, size=s).contiguous(memory_format=CL) for c, s in ((cin, x_size), (256, dy_size)))
    down, up = t(2, rank, cin, size=down_size), t(2, 256, rank, size=up_size)
    weight, bias = t(256, cin, size=cin ** -0.5), torch.zeros(256, device=dev)
    index = torch.tensor([1] * n, device=dev)
    _, hidden = U.fpn_lateral_adapters(x, weight, bias, down, up, index, scale=1.5, return_hidden=True)
    _, gd, gu = U.fpn_lateral_adapters_backward(x, weight, dy, down, up, index, hidden, scale=1.5)
    torch.cuda.synchronize()
    assert U.device_status() == 0
    px = lambda v: v.double().permute(0, 2, 3, 1).flatten(0, 2)  # noqa: E731
    want_gd = (1.5 * px(dy) @ up[1].double()).t() @ px(x)
    want_gu = px(dy).t() @ (1.5 * px(x) @ down[1].double().t())
    assert not gd[0].any() and not gu[0].any()
    largest = (1.5 * px(x) @ down[1].double().t()).abs().max().item()
    return [((a[1].double() - b).norm() / b.norm()).item() for a, b in ((gd, want_gd), (gu, want_gu))] + [largest]


@pytest.mark.parametrize("rank", [3, 16, 33, 64])
@pytest.mark.parametrize("dy_size,up_size", [
    (2.0 ** -7, 2.0 ** -7), (2.0 ** -10, 2.0 ** -10), (2.0 ** -13, 2.0 ** -13), (2.0 ** -16, 2.0 ** -13),
    (1e-4, 1e-4), (3e-5, 1e-4), (2.0 ** -14, 2.0 ** -17), (2.0 ** 4, 2.0 ** -20), (2.0 ** 9, 1.0)])
def test_down_gradient_of_small_and_large_dh(cuda_device, dy_size, up_size, rank):
    """dh from 1.6e-9 to 1e5 (root mean squares; the table of sizes is theirs)."""
    for dtype in (torch.float16, torch.bfloat16):
        gd, _, _ = _run(cuda_device, dtype, dy_size, up_size, 1.0, 1 / 16, rank=rank)
        assert gd <= LIMIT, (dtype, gd)


@pytest.mark.parametrize("h,w", [(33, 31), (3, 5)])  # (K = 512: few tiles are split over k)
@pytest.mark.parametrize("x_size,down_size", [
    (2.0 ** -7, 2.0 ** -7), (2.0 ** -10, 2.0 ** -8), (2.0 ** -12, 2.0 ** -9), (1.0, 2.0 ** -20), (2.0 ** 6, 2.0 ** 3),
    (2.0 ** 8, 2.0 ** 3)])
def test_up_gradient_of_small_and_large_h(cuda_device, x_size, down_size, h, w):
    """h from 1e-5 to 7e4 (root mean squares).  fp16 parts end at 2 x 65504: a value beyond leaves no finite number."""
    for dtype in (torch.float16, torch.bfloat16):
        _, gu, largest = _run(cuda_device, dtype, 1.0, 0.1, x_size, down_size, cin=512, h=h, w=w)
        if dtype is torch.float16 and largest > 131008:
            assert not gu < float("inf")
        else:
            assert gu <= LIMIT, (dtype, gu)


def test_two_part_hidden_of_the_c_entries(cuda_device):
    """ufpn_lateral_adapters and its backward take fp16 h in two parts, as before: values of ordinary size give
    the three parts' gradient."""
    import unified_fpn as U
    from unified_fpn import _lib
    dev, n, cin, h, w, rank = cuda_device, 2, 64, 9, 10, 12
    g = torch.Generator().manual_seed(3)
    t = lambda *s: torch.randn(*s, generator=g).half().to(dev)  # noqa: E731
    x, dy = t(n, cin, h, w).contiguous(memory_format=CL), t(n, 256, h, w).contiguous(memory_format=CL)
    down, up, weight, bias = t(1, rank, cin), t(1, 256, rank), t(256, cin), torch.zeros(256, device=dev)
    index = torch.zeros(n, device=dev, dtype=torch.int32)
    want, hid3 = U.fpn_lateral_adapters(x, weight, bias, down, up, index, return_hidden=True)
    want_gx, want_gd, want_gu = U.fpn_lateral_adapters_backward(x, weight, dy, down, up, index, hid3)
    hid2 = torch.full((n, h, w, 2, 16), 7.0, device=dev, dtype=torch.float16)
    out, gx = torch.empty_like(want), torch.empty_like(want_gx)
    gd, gu = torch.empty_like(want_gd), torch.empty_like(want_gu)
    st = torch.cuda.current_stream().cuda_stream
    p = lambda v: v.data_ptr()  # noqa: E731
    assert _lib.lib.ufpn_lateral_adapters(1, p(x), p(weight), p(bias), p(down), p(up), p(index), None, 1.0, None, p(out),
                                          p(hid2), n, cin, h, w, rank, 1, 0, 0, st) == 0
    need = _lib.lib.ufpn_lateral_adapters_workspace(1, n, cin, h, w, rank, 1, 0, 1)
    work = torch.empty(need, device=dev, dtype=torch.uint8)
    assert _lib.lib.ufpn_lateral_adapters_backward(1, p(x), p(weight), None, p(dy), p(down), p(up), p(index), None, 1.0,
                                                   p(hid2), p(gx), p(gd), p(gu), n, cin, h, w, rank, 1, p(work), need,
                                                   st) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(hid2, hid3[:, :, :, :2])
    assert torch.equal(gx, want_gx) and torch.equal(gd, want_gd)
    assert ((gu - want_gu).norm() / want_gu.norm()).item() <= 2.0 ** -20
