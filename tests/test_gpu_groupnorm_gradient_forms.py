import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight", ["none", "shared", "each"])
@pytest.mark.parametrize("bias", ["none", "shared", "each"])
def test_gradients_of_shared_missing_and_separate_parameters(cuda_device, weight, bias):
    """One vector, the sum over the maps, for a parameter that is shared or None; else one per map."""
    import unified_fpn as U
    g = torch.Generator().manual_seed(3)
    t = lambda *s: torch.randn(*s, generator=g).to(cuda_device)  # noqa: E731
    xs = [t(2, 32, h, w).contiguous(memory_format=torch.channels_last) for h, w in ((9, 7), (5, 4), (1, 1))]
    dys = [t(*x.shape).contiguous(memory_format=torch.channels_last) for x in xs]
    form = {"none": lambda: None, "shared": lambda: t(32), "each": lambda: [t(32) for _ in xs]}
    w, b = form[weight](), form[bias]()
    each = lambda p, i: p[i] if isinstance(p, list) else p  # noqa: E731
    _, mean, rstd = U.fpn_group_norm(xs, w, b, groups=4, activation="swish", return_stats=True)
    _, gw, gb = U.fpn_group_norm_backward(xs, dys, mean, rstd, w, b, activation="swish")
    single = [U.fpn_group_norm_backward(xs[i], dys[i], mean[i], rstd[i], each(w, i), each(b, i), activation="swish")[1:]
              for i in range(3)]
    for got, kind, k in ((gw, weight, 0), (gb, bias, 1)):
        want = torch.stack([s[k] for s in single])
        if kind == "each":
            assert isinstance(got, list) and len(got) == 3
            got = torch.stack(got)
        else:
            assert isinstance(got, torch.Tensor) and got.shape == (32,)
            want = want.sum(0)
        # (the same terms in another order: 64 additions' u of at most 158 terms of size 30)
        assert got.dtype == torch.float32 and (got - want).abs().max() <= 2.0 ** -24 * 64 * 158 * 30
