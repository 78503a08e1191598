"""UnifiedFPN.set_group_norm while forwards run on other streams than its caller's."""
import pytest
import torch

from oracle import fpn_oracle as O

pytestmark = pytest.mark.gpu
CL = torch.channels_last
CHANS = (64, 96, 128, 256)
SIZES = [(40, 48), (20, 24), (10, 12), (5, 6)]


def _setup(dev):
    import unified_fpn as U
    fpn = U.UnifiedFPN(device=dev)
    w = O.make_weights(CHANS, seed=4, bias_scale=0.1)
    fpn.initialize_weights(w.lat_w, w.lat_b, w.out_w, w.out_b)
    g = torch.Generator().manual_seed(5)
    feats = [torch.randn(2, c, h, s, generator=g).bfloat16().contiguous(memory_format=CL)
             for c, (h, s) in zip(CHANS, SIZES)]
    norms = [([torch.rand(256, generator=g) + 0.5 for _ in range(4)], [torch.randn(256, generator=g) for _ in range(4)])
             for _ in range(2)]
    want = []
    x = [f.to(dev) for f in feats]
    for weights, biases in norms:
        fpn.set_group_norm(weights, biases, groups=16, activation="swish")
        want.append([o.clone() for o in fpn(x, return_p6=True)])
    fpn.set_group_norm(None)
    torch.cuda.synchronize()
    return U, fpn, feats, x, [[[t.to(dev) for t in ts] for ts in pair] for pair in norms], want


def _fill(dev):
    """What a freed block of the vectors' sizes would be handed to next."""
    return [torch.full((k,), float("nan"), device=dev) for k in (256, 1024, 2048) for _ in range(32)]


def test_parameters_set_on_a_busy_stream(cuda_device):
    U, fpn, _, x, norms, want = _setup(cuda_device)
    setter, runner = torch.cuda.Stream(cuda_device), torch.cuda.Stream(cuda_device)
    for k in (0, 1, 0):
        with torch.cuda.stream(setter):
            torch.cuda._sleep(20_000_000)  # (about 10 ms)
            fpn.set_group_norm(*norms[k], groups=16, activation="swish")
        with torch.cuda.stream(runner):
            got = fpn(x, return_p6=True)
        runner.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k])), k
    assert U.device_status() == 0


def test_host_pipeline_across_new_parameters(cuda_device):
    """Batches submitted before set_group_norm come out with the old vectors, later ones with the new, and none
    with memory that was released in between."""
    U, fpn, feats, _, norms, want = _setup(cuda_device)
    pinned = [f.pin_memory() for f in feats]
    pipe = U.HostPipeline(fpn, pinned, depth=2)
    sent, keep = [], []
    for k in (0, 1, 0, 1):
        fpn.set_group_norm(*norms[k], groups=16, activation="swish")
        keep.append(_fill(cuda_device))
        for _ in range(3):
            out = pipe.host_buffers()
            pipe.submit(pinned, out)
            sent.append((k, out))
    fpn.set_group_norm(None)
    keep.append(_fill(cuda_device))
    pipe.synchronize()
    for k, out in sent:
        assert all(torch.equal(a, b.cpu()) for a, b in zip(out, want[k])), k
    assert U.device_status() == 0


def test_vectors_keep_their_address(cuda_device):
    """(a graph captured from a forward reads them at replay)"""
    U, fpn, _, x, norms, want = _setup(cuda_device)
    fpn.set_group_norm(*norms[0], groups=16, activation="swish")
    before = [t.data_ptr() for ts in fpn._norm[:2] for t in ts]
    assert all(torch.equal(a, b) for a, b in zip(fpn(x, return_p6=True), want[0]))
    fpn.set_group_norm(None)
    fpn.set_group_norm(norms[1][0], norms[1][1], groups=16, activation="swish")
    assert [t.data_ptr() for ts in fpn._norm[:2] for t in ts] == before
    assert all(torch.equal(a, b) for a, b in zip(fpn(x, return_p6=True), want[1]))
