import pytest
import torch

pytestmark = pytest.mark.gpu
CHANS = (64, 96, 128, 256)


@pytest.mark.parametrize("norm,index", [(16, None), (None, [0, -1]), (16, [1, 0])])
def test_second_derivatives_are_refused(cuda_device, norm, index):
    """The norm's and the adapters' gradients are not differentiable: a loss of them raises instead of leaving its
    share out."""
    import unified_fpn as U
    neck = U.FPNNeck(CHANS, norm_groups=norm, adapters=2, adapter_rank=4).to(cuda_device)
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(2, c, s, s, generator=g).bfloat16().to(cuda_device).requires_grad_()
         for c, s in zip(CHANS, (16, 8, 4, 2))]
    idx = None if index is None else torch.tensor(index, device=cuda_device)
    outs = neck(x, idx)
    grads = torch.autograd.grad([o.float().square().sum() for o in outs], x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable|does not require grad"):
        sum(v.float().square().sum() for v in grads).backward()
