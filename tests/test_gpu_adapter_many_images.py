"""The adapters' gradients over more images than one launch takes (their partial sums stay below 256 MB), and over
more than 1024 images of an adapter: against the sums of calls with parts of the batch."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,cin,h,w,rank", [(260, 2048, 40, 52, 64), (2300, 64, 3, 5, 4)])
def test_gradients_of_the_parts_add_up(cuda_device, dtype, n, cin, h, w, rank):
    import unified_fpn as U
    g = torch.Generator(device="cuda").manual_seed(n)
    t = lambda *s: torch.empty(s, device="cuda", dtype=dtype).normal_(generator=g)  # noqa: E731
    x, dy = t(n, h, w, cin).permute(0, 3, 1, 2), t(n, h, w, 256).permute(0, 3, 1, 2)
    down, up = t(3, rank, cin) / cin ** 0.5, t(3, 256, rank) / 16
    weight, bias = t(256, cin) / cin ** 0.5, torch.zeros(256, device="cuda")
    index = torch.randint(-1, 2, (n,), generator=g, device="cuda", dtype=torch.int32)  # (adapter 2: no image)

    def grads(k0, k1):
        args = (down, up, index[k0:k1])
        hidden = U.fpn_lateral_adapters(x[k0:k1], weight, bias, *args, return_hidden=True)[1]
        return U.fpn_lateral_adapters_backward(x[k0:k1], None, dy[k0:k1], *args, hidden, need_input_grad=False)[1:]
    whole = grads(0, n)
    cuts = [0, n // 3, n // 2 + 7, n]
    parts = [grads(a, b) for a, b in zip(cuts, cuts[1:])]
    for k in range(2):
        want = sum(p[k].double() for p in parts)
        assert not whole[k][2].any() and want[:2].any()
        # (other cuts of the same products: at most 64 steps of 2^-23 an accumulation, 2^-16 for both sides)
        assert (whole[k].double() - want).norm() <= 2.0 ** -16 * want.norm()
    assert all(torch.equal(a, b) for a, b in zip(whole, grads(0, n)))
    torch.cuda.synchronize()
    assert U.device_status() == 0
