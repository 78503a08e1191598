import pytest
import torch

pytestmark = pytest.mark.gpu
CL = torch.channels_last
CHANS = (64, 96, 128, 256)


@pytest.mark.parametrize("norm", [None, 16])
def test_a_neck_with_adapters_graphed_without_an_index(cuda_device, norm):
    """The plain step's outputs and gradients, bit for bit; the adapters get none, as in eager calls."""
    import unified_fpn as U
    kw = dict(norm_groups=norm, adapters=2, adapter_rank=8, seed=3)
    graphed, eager = (U.FPNNeck(CHANS, **kw).to(cuda_device) for _ in range(2))

    def data(seed):
        g = torch.Generator().manual_seed(seed)
        t = lambda *s: torch.randn(*s, generator=g).bfloat16().to(cuda_device).contiguous(memory_format=CL)  # noqa: E731
        sizes = [(24, 32), (12, 16), (6, 8), (3, 4)]
        return ([t(2, c, h, w).requires_grad_() for c, (h, w) in zip(CHANS, sizes)],
                [t(2, 256, h, w) for h, w in sizes + [(2, 2)]])
    run = graphed.make_graphed(data(1)[0])
    for seed in (2, 3):
        got = []
        for call, neck in ((run, graphed), (eager, eager)):
            x, grads = data(seed)
            neck.zero_grad(set_to_none=True)
            outs = call(x)
            torch.autograd.backward(outs, grads)
            got.append([o.detach().clone() for o in outs] + [t.grad.clone() for t in x]
                       + [p.grad.clone() for k, p in neck.named_parameters() if not k.startswith("adapter")])
            assert all(p.grad is None for k, p in neck.named_parameters() if k.startswith("adapter"))
            del outs
        assert all(torch.equal(a, b) for a, b in zip(*got))
    torch.cuda.synchronize()
    assert U.device_status() == 0
