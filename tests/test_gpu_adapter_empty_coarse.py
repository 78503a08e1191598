import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [(0, 4), (4, 0), (0, 0)])
def test_an_empty_coarse_map_is_refused(cuda_device, size):
    """(its address is NULL, which the library takes for "no top-down add")"""
    import unified_fpn as U
    t = lambda *s: torch.zeros(*s, device=cuda_device, dtype=torch.bfloat16)  # noqa: E731
    args = (t(1, 64, 4, 4), t(256, 64), torch.zeros(256, device=cuda_device), t(1, 8, 64), t(1, 256, 8),
            torch.zeros(1, device=cuda_device, dtype=torch.int32))
    with pytest.raises(ValueError, match="empty"):
        U.fpn_lateral_adapters(*args, coarse=t(1, 256, *size))
