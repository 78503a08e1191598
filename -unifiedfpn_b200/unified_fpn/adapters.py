"""Lateral 1x1 convs with a low-rank adapter per image, forward and backward.

One batch serves images of many requests: they share the lateral's weights, and image n adds its
own adapter a = index[n] of rank R (none where index[n] is outside 0 .. L - 1):

    h   = scale * conv1x1(x, down[a])                                   (R channels)
    out = conv1x1(x, weight) + bias + conv1x1(h, up[a]) [+ bilinear(coarse)]

Both functions run on the tensors' device and torch's current stream, in one pass over the map for
the shared projection and every adapter, and never block the host: ``index`` is read on the device.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .groupnorm import _on_device, _stream
from .ops import _DT

_CL = torch.channels_last
MAX_RANK = 64
_PARTS = 3  # 16-bit values that make up one of h


def _cl(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous(memory_format=_CL) else t.contiguous(memory_format=_CL)


def _operand(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if t.dtype is not dtype:
        t = t.detach().to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _check(x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, index: torch.Tensor, scale):
    """The checks of both directions; (down, up, index, scales or None, scale) as the library takes them."""
    if not isinstance(x, torch.Tensor) or x.dim() != 4:
        raise ValueError("input must be 4-D [N, C, H, W]")
    for t in (x, down, up, index):
        if not t.is_cuda:
            raise ValueError("all tensors must be CUDA tensors")
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float16:
        raise TypeError(f"unsupported dtype {x.dtype}: expected float16 or bfloat16")
    if x.numel() == 0:
        raise ValueError("input must not be empty")
    n, cin = x.shape[:2]
    if cin % 8 or cin > 2048:
        raise ValueError("input channels must be a multiple of 8, at most 2048")
    if down.dim() != 3 or down.shape[2] != cin or down.shape[0] < 1:
        raise ValueError("down must be [adapters, rank, Cin]")
    count, rank = down.shape[:2]
    if not 1 <= rank <= MAX_RANK:
        raise ValueError(f"adapters have rank 1 to {MAX_RANK}")
    if tuple(up.shape) != (count, 256, rank):
        raise ValueError("up must be [adapters, 256, rank]")
    if index.dim() != 1 or index.shape[0] != n or index.dtype not in (torch.int32, torch.int64):
        raise ValueError("index must be one int32 or int64 per image")
    if down.device != x.device or up.device != x.device or index.device != x.device:
        raise ValueError("all tensors must be on the input's device")
    if index.dtype is not torch.int32:
        # (clamped: a value beyond 32 bits must stay "no adapter")
        index = index.clamp(-1, count).to(torch.int32)
    scales = None
    if isinstance(scale, torch.Tensor):
        if not scale.is_cuda or scale.numel() != count or scale.device != x.device:
            raise ValueError("scale must be one number or one value per adapter on the input's device")
        scales = scale
        if scales.dtype is not torch.float32 or not scales.is_contiguous():
            scales = scales.detach().reshape(-1).to(torch.float32).contiguous()
        scale = 1.0
    return (_operand(down, x.dtype), _operand(up, x.dtype), index if index.is_contiguous() else index.contiguous(),
            scales, float(scale))


def _weight(weight: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    cin = x.shape[1]
    if weight.shape[0] != 256 or weight.numel() != 256 * cin:
        raise ValueError("weight must be [256, Cin] or [256, Cin, 1, 1]")
    if weight.device != x.device:
        raise ValueError("all tensors must be on the input's device")
    return _operand(weight, x.dtype)


def fpn_lateral_adapters(input: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, down: torch.Tensor,
                         up: torch.Tensor, index: torch.Tensor, scale=1.0, coarse: torch.Tensor | None = None,
                         return_hidden: bool = False):
    """:func:`fpn_lateral_conv` (16-bit, channels_last, 256 outputs) with one low-rank adapter per
    image, optionally with the fused top-down add of ``coarse``.

    ``down`` [L, R, Cin] and ``up`` [L, 256, R]: the adapters, R 1 to 64 (used in the input's dtype);
    ``index``: one integer per image on the device, values outside 0 .. L - 1 (-1 by convention) run
    without an adapter; ``scale``: a number, or [L] on the device.  ``weight`` [256, Cin] or [256,
    Cin, 1, 1], ``bias`` [256], Cin a multiple of 8, at most 2048.  Sums are fp32 and rounded once;
    h is carried in 16-bit parts of 22 bits and more together, of which fp16 loses what is below 2^-25 (up
    to 2^-25 * sum_r |up| in the output, whose own steps end at 2^-24); the bilinear weights are fp32 or have 16
    bits and more.  Values of ``coarse`` that are not finite reach the pixels that use them alone (a call
    that meets any takes up to twice as long).  With ``return_hidden`` also returns
    h in parts (opaque, [N, H, W, 3, R rounded up to 8]; fp16: what is below 2^-36 is lost) for
    :func:`fpn_lateral_adapters_backward`."""
    down, up, index, scales, scale = _check(input, down, up, index, scale)
    x = _cl(input)
    n, cin, h, w = x.shape
    dev = x.device
    wt = _weight(weight, x)
    if bias.numel() != 256 or bias.device != dev:
        raise ValueError("bias must have 256 values on the input's device")
    b = _operand(bias, torch.float32)
    hc = wc = 0
    if coarse is not None:
        if coarse.dtype is not x.dtype or coarse.dim() != 4 or coarse.shape[0] != n or coarse.shape[1] != 256 \
                or coarse.device != dev:
            raise ValueError("coarse must match the output's dtype, device, batch and channels")
        if coarse.numel() == 0:
            raise ValueError("coarse must not be empty")
        coarse = _cl(coarse)
        hc, wc = coarse.shape[2:]
    count, rank = down.shape[:2]
    # (channels_last; torch.empty with the memory format takes a microsecond more)
    out = torch.empty_strided((n, 256, h, w), (h * w * 256, 1, w * 256, 256), dtype=x.dtype, device=dev)
    hidden = torch.empty((n, h, w, _PARTS, (rank + 7) // 8 * 8), dtype=x.dtype,
                         device=dev) if return_hidden else None

    check(_on_device(
        dev, lib.ufpn_lateral_adapters_parts, _DT[x.dtype], x.data_ptr(), wt.data_ptr(), b.data_ptr(), down.data_ptr(),
        up.data_ptr(), index.data_ptr(), None if scales is None else scales.data_ptr(), scale,
        None if coarse is None else coarse.data_ptr(), out.data_ptr(), None if hidden is None else hidden.data_ptr(),
        _PARTS, n, cin, h, w, rank, count, hc, wc, _stream(dev)), "ufpn_lateral_adapters")
    return (out, hidden) if return_hidden else out


def fpn_lateral_adapters_backward(input: torch.Tensor, weight: torch.Tensor | None, grad_output: torch.Tensor,
                                  down: torch.Tensor, up: torch.Tensor, index: torch.Tensor,
                                  hidden: torch.Tensor, scale=1.0, need_input_grad: bool = True,
                                  weight_t: torch.Tensor | None = None):
    """Gradients of :func:`fpn_lateral_adapters` given ``hidden`` from its forward: ``(grad_input,
    grad_down [L, R, Cin] fp32, grad_up [L, 256, R] fp32)``; grad_input is None without
    ``need_input_grad`` (``weight`` may then be None).  An adapter without images gets zeros.
    ``weight_t``: the weights transposed for the input gradient, as
    :func:`fpn_lateral_conv_backward` takes them (``weight`` is then not read).  The shared weight's
    and bias's gradients are :func:`fpn_lateral_conv_backward`'s, the coarse map's
    :func:`fpn_upsample_add_backward`'s.  Deterministic (every sum in a fixed order).  fp16: dh = scale *
    grad_output up[a] enters grad_down to 22 bits and more, of which what is below 2^-47 is lost, and
    grad_input (steps of 2^-24) without what is below 2^-25 of it."""
    down, up, index, scales, scale = _check(input, down, up, index, scale)
    x = _cl(input)
    n, cin, h, w = x.shape
    dev = x.device
    if grad_output.dtype is not x.dtype or tuple(grad_output.shape) != (n, 256, h, w) or grad_output.device != dev:
        raise ValueError("grad_output must be [N, 256, H, W] in the input's dtype")
    g = _cl(grad_output)
    count, rank = down.shape[:2]
    if hidden.dtype is not x.dtype or tuple(hidden.shape) != (n, h, w, _PARTS, (rank + 7) // 8 * 8) \
            or hidden.device != dev or not hidden.is_contiguous():
        raise ValueError("hidden must be what the forward returned")
    wt = wtt = None
    if need_input_grad:
        if weight_t is not None:
            if weight_t.dtype is not x.dtype or tuple(weight_t.shape) != ((cin + 255) // 256 * 256, 256) \
                    or weight_t.device != dev:
                raise ValueError("weight_t must be [ceil(Cin/256)*256, 256] in the input's dtype")
            wtt = _operand(weight_t, x.dtype)
        elif weight is None:
            raise ValueError("the input gradient needs weight or weight_t")
        else:
            wt = _weight(weight, x)
    gx = torch.empty_like(x, memory_format=_CL) if need_input_grad else None
    gdown = torch.empty((count, rank, cin), device=dev, dtype=torch.float32)
    gup = torch.empty((count, 256, rank), device=dev, dtype=torch.float32)
    code = _DT[x.dtype]

    need = _on_device(dev, lib.ufpn_lateral_adapters_workspace, code, n, cin, h, w, rank, count, wtt is not None,
                      need_input_grad)
    work = torch.empty(need, device=dev, dtype=torch.uint8)
    check(_on_device(
        dev, lib.ufpn_lateral_adapters_backward_parts, code, x.data_ptr(), None if wt is None else wt.data_ptr(),
        None if wtt is None else wtt.data_ptr(), g.data_ptr(), down.data_ptr(), up.data_ptr(), index.data_ptr(),
        None if scales is None else scales.data_ptr(), scale, hidden.data_ptr(), _PARTS,
        None if gx is None else gx.data_ptr(),
        gdown.data_ptr(), gup.data_ptr(), n, cin, h, w, rank, count, work.data_ptr(), need, _stream(dev)),
        "ufpn_lateral_adapters_backward")
    return gx, gdown, gup
