"""The neck with a group norm behind its 3x3s and an adapter per image on its laterals, as they are
used together: training (eager and as CUDA graphs) and serving, against autograd through the CPU
oracle's convs.

Inputs and weights are rounded to the kernels' 16-bit type first.  The bounds are those of the
neck's own gradient tests (16-bit maps between the kernels): the norm and the adapters add two more
16-bit maps to each chain of four."""
import pytest
import torch
import torch.nn.functional as F

from oracle import fpn_oracle as O

pytestmark = pytest.mark.gpu
CL = torch.channels_last
CHANS = (64, 96, 128, 256)
SIZES = [(40, 48), (20, 24), (10, 12), (5, 6)]
INDEX = [1, -1, 0, 1]


def _neck(U, dev, **kw):
    neck = U.FPNNeck(CHANS, seed=3, **kw)
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for name, p in neck.named_parameters():
            if name.startswith(("lateral_b", "output_b", "norm_b")):
                p.copy_(torch.randn(p.shape, generator=g) * 0.2)
            elif name.startswith("norm_w"):
                p.copy_(torch.rand(p.shape, generator=g) + 0.5)
            elif name.startswith("adapter_up"):
                p.copy_(torch.randn(p.shape, generator=g) * 0.2)
            if name.startswith(("lateral_w", "output_w", "adapter")):
                p.copy_(p.to(torch.bfloat16).float())
    return neck.to(dev)


def _data(dev, seed=11):
    g = torch.Generator().manual_seed(seed)
    feats = [torch.randn(4, c, h, w, generator=g).to(torch.bfloat16) for c, (h, w) in zip(CHANS, SIZES)]
    grads = [torch.randn(4, 256, h, w, generator=g).to(torch.bfloat16) for h, w in SIZES + [(3, 3)]]
    return feats, grads


def _oracle(neck, feats, index):
    """The same neck on the CPU in 64 bits from the module's parameters; (outputs, leaves by name)."""
    leaves = {k: p.detach().cpu().double().requires_grad_() for k, p in neck.named_parameters()}
    x = [f.double().requires_grad_() for f in feats]
    m = [None] * 4
    for l in (3, 2, 1, 0):
        v = F.conv2d(x[l], leaves[f"lateral_w.{l}"][:, :, None, None], leaves[f"lateral_b.{l}"])
        if index is not None:
            down, up = leaves[f"adapter_down.{l}"], leaves[f"adapter_up.{l}"]
            parts = []
            for n, a in enumerate(index):
                t = v[n:n + 1]
                if a >= 0:
                    h = F.conv2d(x[l][n:n + 1], down[a][:, :, None, None]) * neck.adapter_scale
                    t = t + F.conv2d(h, up[a][:, :, None, None])
                parts.append(t)
            v = torch.cat(parts)
        if l < 3:
            v = v + F.interpolate(m[l + 1], size=SIZES[l], mode="bilinear", align_corners=False)
        m[l] = v
    outs = [F.conv2d(m[l], leaves[f"output_w.{l}"], leaves[f"output_b.{l}"], padding=1) for l in range(4)]
    if neck.norm_groups is not None:
        outs = [F.group_norm(o, neck.norm_groups, leaves[f"norm_w.{l}"], leaves[f"norm_b.{l}"], neck.eps)
                for l, o in enumerate(outs)]
        if neck.activation == "swish":
            outs = [F.silu(o) for o in outs]
    return outs + [outs[3][:, :, ::2, ::2]], x, leaves


@pytest.mark.parametrize("norm,adapters", [(32, True), (8, False), (None, True)])
def test_training_against_autograd(cuda_device, norm, adapters):
    import unified_fpn as U
    neck = _neck(U, cuda_device, norm_groups=norm, activation="swish" if norm else None, adapters=2,
                 adapter_rank=12, adapter_scale=0.5)
    feats, grads = _data(cuda_device)
    index = torch.tensor(INDEX, device=cuda_device) if adapters else None
    x = [f.to(cuda_device).contiguous(memory_format=CL).requires_grad_() for f in feats]
    outs = neck(x, index)
    torch.autograd.backward(outs, [g.to(cuda_device).contiguous(memory_format=CL) for g in grads])
    torch.cuda.synchronize()
    assert U.device_status() == 0
    ref, xr, leaves = _oracle(neck, feats, INDEX if adapters else None)
    torch.autograd.backward(ref, [g.double() for g in grads])
    for k, (o, r) in enumerate(zip(outs, ref)):
        O.check_close(o.detach().float().cpu(), r.detach().float(), "bf16")
        assert o.is_contiguous(memory_format=CL), k
    for l in range(4):
        O.check_close(x[l].grad.float().cpu(), xr[l].grad.float(), "grad16", tol=2e-2)
    for name, p in neck.named_parameters():
        want = leaves[name].grad
        if want is None:
            assert p.grad is None, name
            continue
        assert p.grad.dtype == torch.float32 and p.grad.shape == p.shape
        O.check_close(p.grad.cpu(), want.float(), "grad16", tol=2e-2)


def test_adapters_and_norms_alone(cuda_device):
    """Frozen convs and backbone: the same adapter and norm gradients, and none elsewhere."""
    import unified_fpn as U
    feats, grads = _data(cuda_device)
    index = torch.tensor(INDEX, device=cuda_device)
    g = [v.to(cuda_device).contiguous(memory_format=CL) for v in grads]
    res = []
    for frozen in (False, True):
        neck = _neck(U, cuda_device, norm_groups=32, activation="relu", adapters=2, adapter_rank=8)
        if frozen:
            for name, p in neck.named_parameters():
                p.requires_grad_(name.startswith(("adapter", "norm")))
        x = [f.to(cuda_device).contiguous(memory_format=CL).requires_grad_(not frozen) for f in feats]
        torch.autograd.backward(neck(x, index), g)
        res.append({k: p.grad for k, p in neck.named_parameters()})
        assert all((p.grad is not None) == p.requires_grad for p in neck.parameters())
    for k, v in res[1].items():
        if v is not None:
            # (the 3x3's input gradient comes from the same kernel either way)
            assert torch.equal(v, res[0][k]), k


def test_without_an_index_the_neck_is_the_plain_one(cuda_device):
    import unified_fpn as U
    feats, _ = _data(cuda_device)
    x = [f.to(cuda_device).contiguous(memory_format=CL) for f in feats]
    plain, adapted = _neck(U, cuda_device), _neck(U, cuda_device, adapters=2)
    with torch.no_grad():
        for a, b in zip(plain(x), adapted(x)):
            assert torch.equal(a, b)
        none = adapted(x, torch.full((4,), -1, device=cuda_device))
    for a, b in zip(plain(x), none):
        # (per-level kernels instead of the grouped laterals: one 16-bit rounding of M apart)
        O.check_close(b.float().cpu(), a.detach().float().cpu(), "bf16")
    with pytest.raises(ValueError):
        plain(x, torch.zeros(4, device=cuda_device, dtype=torch.int64))
    for kw in ({"norm_groups": 7}, {"activation": "relu"}, {"adapters": 1, "adapter_rank": 65}, {"adapters": -1},
               {"norm_groups": 8, "activation": "gelu"}):
        with pytest.raises(ValueError):
            U.FPNNeck(CHANS, **kw)


def test_serving_engine_with_the_trained_norm(cuda_device):
    """UnifiedFPN.set_group_norm gives the module's inference outputs bit for bit, in either layout, into
    given outputs, quantised, and goes away again."""
    import unified_fpn as U
    neck = _neck(U, cuda_device, norm_groups=32, activation="relu")
    feats, _ = _data(cuda_device)
    x = [f.to(cuda_device).contiguous(memory_format=CL) for f in feats]
    with torch.no_grad():
        want = neck(x)
    fpn = U.UnifiedFPN(device=cuda_device)
    fpn.initialize_weights(*[[p.detach() for p in ps] for ps in (neck.lateral_w, neck.lateral_b, neck.output_w,
                                                                   neck.output_b)])
    raw = fpn(x, return_p6=True)
    fpn.set_group_norm(list(neck.norm_w), list(neck.norm_b), groups=32, activation="relu")
    for _ in range(3):  # (direct, captured, replayed)
        got = fpn(x, return_p6=True)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    out = [torch.empty_like(o) for o in want]
    assert fpn(x, return_p6=True, out=out)[4] is out[4]
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert len(fpn(x)) == 4
    nchw = fpn([t.contiguous() for t in x], return_p6=True)
    for a, b in zip(nchw, want):
        assert a.is_contiguous()
        O.check_close(a.float().cpu(), b.float().cpu(), "bf16")
    for (q, sc), o in zip(fpn(x, output_fp8=True), want):
        q2, sc2 = U.quantize_fp8(o, per_image=True)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(sc, sc2)
    fpn.set_group_norm(None)
    for a, b in zip(fpn(x, return_p6=True), raw):
        assert torch.equal(a, b)
    for bad in (lambda: fpn.set_group_norm(list(neck.norm_w)[:3]), lambda: fpn.set_group_norm(list(neck.norm_w), groups=7),
                lambda: fpn.set_group_norm(list(neck.norm_w), activation="gelu"),
                lambda: fpn.set_group_norm(list(neck.norm_w), eps=-1)):
        with pytest.raises(ValueError):
            bad()


def test_graphed_steps_with_changing_indices(cuda_device):
    """make_graphed with an adapter index: replays on other indices and features give the eager
    step's outputs and gradients bit for bit."""
    import unified_fpn as U
    kw = dict(norm_groups=32, activation="swish", adapters=3, adapter_rank=8)
    neck, eager = _neck(U, cuda_device, **kw), _neck(U, cuda_device, **kw)
    feats, grads = _data(cuda_device)
    g = [v.to(cuda_device).contiguous(memory_format=CL) for v in grads]
    x = [f.to(cuda_device).contiguous(memory_format=CL).requires_grad_() for f in feats]
    run = neck.make_graphed(x, torch.tensor(INDEX, device=cuda_device, dtype=torch.int32))
    for seed, index in ((11, INDEX), (12, [2, 2, -1, 0]), (13, [-1, -1, -1, -1])):
        idx = torch.tensor(index, device=cuda_device, dtype=torch.int32)
        f2, _ = _data(cuda_device, seed)
        xs = [[f.to(cuda_device).contiguous(memory_format=CL).requires_grad_() for f in f2] for _ in range(2)]
        got = []
        for fn, mod, xx in ((run, neck, xs[0]), (eager, eager, xs[1])):
            mod.zero_grad(set_to_none=True)
            outs = fn(xx, idx)
            torch.autograd.backward(outs, g)
            got.append([o.detach().clone() for o in outs] + [t.grad.clone() for t in xx]
                       + [p.grad.clone() for p in mod.parameters()])
            del outs
        for k, (a, b) in enumerate(zip(*got)):
            assert torch.equal(a, b), (seed, k)
    torch.cuda.synchronize()
    assert U.device_status() == 0


def test_calls_at_once_on_two_streams(cuda_device):
    """Norms of maps of both forms and adapters of both, running on two streams together: the results of the
    same calls one after the other, bit for bit."""
    import unified_fpn as U
    g = torch.Generator().manual_seed(5)

    def t(*shape):
        return torch.randn(*shape, generator=g).to(torch.bfloat16).to(cuda_device)
    maps = [t(2, 256, 120, 160).contiguous(memory_format=CL), t(1, 256, 9, 11).contiguous(memory_format=CL)]
    x = [t(2, 256, 120, 160).contiguous(memory_format=CL), t(2, 1024, 12, 13).contiguous(memory_format=CL)]
    w, down, up = [t(256, v.shape[1]) for v in x], [t(2, 8, v.shape[1]) for v in x], t(2, 256, 8)
    b, index = torch.zeros(256, device=cuda_device), torch.tensor([1, 0], device=cuda_device)

    def calls(k):
        out = list(U.fpn_group_norm(maps[k], groups=32, activation="swish", return_stats=True))
        out.append(U.fpn_group_norm_backward(maps[k], maps[k], out[1], out[2], activation="swish")[0])
        o, h = U.fpn_lateral_adapters(x[k], w[k], b, down[k], up, index, return_hidden=True)
        return out + [o, *U.fpn_lateral_adapters_backward(x[k], w[k], o, down[k], up, index, h)]
    want = [calls(0), calls(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device), torch.cuda.Stream(cuda_device)]
    got = [[], []]
    for _ in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(calls(k))
    torch.cuda.synchronize()
    assert U.device_status() == 0
    for k in range(2):
        for run in got[k]:
            assert all(torch.equal(a, v) for a, v in zip(run, want[k]))


@pytest.mark.parametrize("adapters", [True, False])
def test_losses_of_some_outputs(cuda_device, adapters):
    """A loss of P3 and P6 alone whose gradients are broadcast scalars (stride 0); the others' are missing."""
    import unified_fpn as U
    neck = _neck(U, cuda_device, norm_groups=16 if not adapters else None,
                 activation="swish" if not adapters else None, adapters=2, adapter_rank=4)
    feats, _ = _data(cuda_device)
    index = torch.tensor(INDEX, device=cuda_device) if adapters else None
    x = [f.to(cuda_device).contiguous(memory_format=CL).requires_grad_() for f in feats]
    outs = neck(x, index)
    (outs[1].sum() + 2.0 * outs[4].sum()).backward()
    ref, xr, leaves = _oracle(neck, feats, INDEX if adapters else None)
    (ref[1].sum() + 2.0 * ref[4].sum()).backward()
    for l in range(1, 4):
        O.check_close(x[l].grad.float().cpu(), xr[l].grad.float(), "grad16", tol=2e-2)
    assert not x[0].grad.any()
    for name, p in neck.named_parameters():
        want = leaves[name].grad
        if want is None or name.endswith(".0"):
            assert p.grad is None or not p.grad.any(), name
        else:
            O.check_close(p.grad.cpu(), want.float(), "grad16", tol=2e-2)
