"""Group norm with an activation on channels-last maps, forward and backward.

    xhat = (x - mean) * rstd   (mean, biased variance per image and group of C / groups channels)
    y    = act(xhat * weight[c] + bias[c])

The norm that a neck's 3x3 outputs take when its batch per GPU is too small for BatchNorm; next
to :func:`fold_batch_norm`, which folds frozen statistics into the conv.  Every function takes one
map or the list of a pyramid's maps (one batch size and channel count; each map has its own
statistics) in one library call, on the tensors' device and torch's current stream; nothing
blocks the host.
"""
from __future__ import annotations

import ctypes
import functools
from array import array
from typing import Sequence

import torch

from . import _lib
from ._lib import check, lib
from .ops import _ACTIVATIONS, _DT

_CL = torch.channels_last
MAX_LEVELS = 8


@functools.lru_cache(maxsize=256)
def _workspace_bytes(dev: torch.device, code: int, n: int, c: int, pixels: tuple, groups: int, backward: int) -> int:
    # (the plan follows the device's SM count)
    return _on_device(dev, lib.ufpn_group_norm_workspace, code, len(pixels), n, c,
                      (ctypes.c_longlong * len(pixels))(*pixels), groups, backward)


def _table(*lists):
    """The lists' entries (tensors as addresses, None as 0, integers) as one array of 64-bit words, and the
    address of each list (None for a list that is None).  The array must outlive the call."""
    words, at = array("Q"), []
    for entries in lists:
        at.append(None if entries is None else len(words))
        if entries is not None:
            words.extend([t if type(t) is int else 0 if t is None else t.data_ptr() for t in entries])
    base = words.buffer_info()[0]
    return words, [None if k is None else base + 8 * k for k in at]


def _stream(dev: torch.device) -> int:
    """Handle of torch's current stream on ``dev`` (the Stream object that
    ``torch.cuda.current_stream`` makes costs 2 us a call)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _on_device(dev: torch.device, fn, *args) -> int:
    """``fn(*args)`` with ``dev`` as the current CUDA device."""
    if dev.index == torch._C._cuda_getDevice():
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _levels(input, what: str = "input"):
    """(maps as channels_last, was a single tensor) after the checks that need no other argument."""
    single = isinstance(input, torch.Tensor)
    xs = [input] if single else list(input)
    if not 1 <= len(xs) <= MAX_LEVELS:
        raise ValueError(f"{what} must be one map or a list of 1 to {MAX_LEVELS} maps")
    x0 = xs[0]
    for t in xs:
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{what} must be 4-D [N, C, H, W]")
        if not t.is_cuda:
            raise ValueError("all tensors must be CUDA tensors")
        if t.dtype is not x0.dtype or t.device != x0.device or t.shape[:2] != x0.shape[:2]:
            raise ValueError(f"the maps of {what} must share dtype, device, batch and channels")
        if t.numel() == 0:
            raise ValueError(f"{what} must not be empty")
    if x0.dtype not in _DT:
        raise TypeError(f"unsupported dtype {x0.dtype}: expected float32, float16 or bfloat16")
    return [t if t.is_contiguous(memory_format=_CL) else t.contiguous(memory_format=_CL) for t in xs], single


def _params(p, what: str, n: int, c: int, dev: torch.device):
    """Per-level fp32 vectors of a weight or bias argument (None, one vector or one per level)."""
    if p is None:
        return None, True
    shared = isinstance(p, torch.Tensor)
    ps = [p] * n if shared else list(p)
    if len(ps) != n:
        raise ValueError(f"{what} must be one vector or one per map")
    out = []
    for t in ps[:1] if shared else ps:
        if t is not None:
            if t.numel() != c or t.device != dev:
                raise ValueError(f"{what} needs {c} values on the maps' device")
            if t.dtype is not torch.float32 or not t.is_contiguous() or t.dim() != 1:
                t = t.detach().reshape(-1).to(torch.float32).contiguous()
        out.append(t)
    return (out * n if shared else out), shared


def _check_groups(c: int, groups: int):
    if c % 8 or c > 2048:
        raise ValueError("channels must be a multiple of 8, at most 2048")
    if groups < 1 or c % groups:
        raise ValueError("groups must divide the channels")


def fpn_group_norm(input: torch.Tensor | Sequence[torch.Tensor], weight=None, bias=None, groups: int = 32,
                   eps: float = 1e-5, activation: str | None = None, alpha: float = 0.01,
                   return_stats: bool = False, out=None):
    """Group norm with an activation of a map [N, C, H, W] or of a list of maps (channels_last;
    other layouts are converted; bf16, fp16 or fp32, computed in fp32).

    ``weight`` / ``bias``: [C] (any float dtype), shared by the maps, or one per map; None = 1 / 0.
    C a multiple of 8, at most 2048; ``groups`` any divisor of it.  ``activation``: None, "relu",
    "leaky_relu" (negative slope ``alpha``) or "swish", as :func:`fpn_conv3x3`.  ``out``: maps to
    write (channels_last, like the inputs; a map may be its own input, but overlap no other).  Returns the
    channels_last output(s); with ``return_stats`` also ``mean`` and ``rstd`` (fp32 [N, groups], per
    map) for :func:`fpn_group_norm_backward`."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    xs, single = _levels(input)
    n, c = xs[0].shape[:2]
    _check_groups(c, groups)
    dev = xs[0].device
    ws, _ = _params(weight, "weight", len(xs), c, dev)
    bs, _ = _params(bias, "bias", len(xs), c, dev)
    if out is None:
        ys = [torch.empty_like(t, memory_format=_CL) for t in xs]
    else:
        ys = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(ys) != len(xs) or any(
                y.shape != x.shape or y.dtype is not x.dtype or y.device != dev
                or not y.is_contiguous(memory_format=_CL) for x, y in zip(xs, ys)):
            raise ValueError("out must be channels_last maps like the inputs")
    means = rstds = None
    if return_stats:
        stats = torch.empty((2 * len(xs), n, groups), device=dev, dtype=torch.float32).unbind()
        means, rstds = list(stats[:len(xs)]), list(stats[len(xs):])
    code = _DT[xs[0].dtype]
    pixels = tuple([t.shape[2] * t.shape[3] for t in xs])
    need = _workspace_bytes(dev, code, n, c, pixels, groups, 0)
    work = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
    words, (px, xp, yp, wp, bp, mp, rp) = _table(pixels, xs, ys, ws, bs, means, rstds)
    check(_on_device(
        dev, lib.ufpn_group_norm, code, len(xs), xp, yp, wp, bp, mp, rp, n, c, px, groups, eps,
        _ACTIVATIONS[activation], alpha, work.data_ptr() if need else None, need, _stream(dev)), "ufpn_group_norm")
    if single:
        return (ys[0], means[0], rstds[0]) if return_stats else ys[0]
    return (ys, means, rstds) if return_stats else ys


def fpn_group_norm_backward(input, grad_output, mean, rstd, weight=None, bias=None,
                            activation: str | None = None, alpha: float = 0.01,
                            need_input_grad: bool = True):
    """Gradients of :func:`fpn_group_norm` with the ``mean`` and ``rstd`` that it returned:
    ``(grad_input, grad_weight, grad_bias)``; grad_input like the input(s) (None without
    ``need_input_grad``), the other two fp32 [C] -- summed over the maps where ``weight`` (for grad_weight)
    or ``bias`` (for grad_bias) is shared or None, else a list with one per map.  ``grad_output``: the
    shapes and dtype of the outputs.
    Deterministic (every sum in a fixed order)."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    xs, single = _levels(input)
    gs, _ = _levels(grad_output, "grad_output")
    if len(gs) != len(xs):
        raise ValueError("grad_output must have the input's shapes, dtype and device")
    for g, x in zip(gs, xs):
        if g.shape != x.shape or g.dtype is not x.dtype or g.device != x.device:
            raise ValueError("grad_output must have the input's shapes, dtype and device")
    n, c = xs[0].shape[:2]
    dev = xs[0].device
    means = [mean] if isinstance(mean, torch.Tensor) else list(mean)
    rstds = [rstd] if isinstance(rstd, torch.Tensor) else list(rstd)
    groups = means[0].shape[-1] if means and means[0].dim() == 2 else 0
    _check_groups(c, groups)
    for ts, what in ((means, "mean"), (rstds, "rstd")):
        ok = len(ts) == len(xs)
        for k, t in enumerate(ts):
            ok = ok and t.shape == (n, groups) and t.dtype is torch.float32 and t.device == dev
            if ok and not t.is_contiguous():
                ts[k] = t.contiguous()
        if not ok:
            raise ValueError(f"{what} must be fp32 [N, groups] per map on the maps' device")
    ws, shared_w = _params(weight, "weight", len(xs), c, dev)
    bs, shared_b = _params(bias, "bias", len(xs), c, dev)
    shared = shared_w and shared_b
    gxs = [torch.empty_like(t, memory_format=_CL) for t in xs] if need_input_grad else None
    rows = 1 if shared else len(xs)
    gwb = torch.empty((2 * rows, c), device=dev, dtype=torch.float32).unbind()
    gw, gb = list(gwb[:rows]), list(gwb[rows:])
    pad = [None] * (len(xs) - rows)
    code = _DT[xs[0].dtype]
    pixels = tuple([t.shape[2] * t.shape[3] for t in xs])
    need = _workspace_bytes(dev, code, n, c, pixels, groups, 1)
    work = torch.empty(need, device=dev, dtype=torch.uint8)
    words, (px, xp, gp, gxp, wp, bp, mp, rp, gwp, gbp) = _table(pixels, xs, gs, gxs, ws, bs, means, rstds, gw + pad,
                                                                gb + pad)
    check(_on_device(
        dev, lib.ufpn_group_norm_backward, code, len(xs), xp, gp, gxp, wp, bp, mp, rp, gwp, gbp, n, c, px, groups,
        _ACTIVATIONS[activation], alpha, work.data_ptr(), need, _stream(dev)), "ufpn_group_norm_backward")
    if single or shared:
        return (gxs[0] if single and gxs else gxs), gw[0], gb[0]
    # a parameter shared by the maps (or None) beside one that is not: its gradient is the sum over the maps
    return gxs, torch.stack(gw).sum(0) if shared_w else gw, torch.stack(gb).sum(0) if shared_b else gb
