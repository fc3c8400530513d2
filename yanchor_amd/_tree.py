"""Arguments that the operators over drafted trees share."""
from __future__ import annotations

import torch

MAX_NODES = 64


def device_of(first, *rest):
    """The ROCm device that all of the tensors (or None) share."""
    dev = first.device
    if dev.type != "cuda":
        raise ValueError(f"yanchor_amd kernels take ROCm device tensors (got a tensor on {dev})")
    for t in rest:
        if t is not None and t.device != dev:
            if t.device.type != "cuda":
                raise ValueError(f"yanchor_amd kernels take ROCm device tensors (got a tensor on {t.device})")
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def ints(t, dtype, device, name, size=None):
    """``t`` as a contiguous 1-D integer tensor of ``dtype`` on the device."""
    if t.ndim != 1 or (t.dtype != dtype and t.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"{name} must be a 1-D integer tensor")
    if size is not None and t.shape[0] != size:
        raise ValueError(f"{name} must hold {size} entries, got {t.shape[0]}")
    if t.dtype != dtype or t.device != device:
        t = t.to(device=device, dtype=dtype)
    return t if t.is_contiguous() else t.contiguous()


def offsets(cu_seqlens, total, device, most=None):
    """cu_seqlens as int32 on the device.  Offsets that come from the host are
    checked; those on the device are not read back, and the kernels clamp them
    to the packed rows."""
    if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a 1-D offset vector")
    if not cu_seqlens.is_cuda:
        h = cu_seqlens.tolist()
        if h[0] != 0 or h[-1] > total or any(b < a for a, b in zip(h, h[1:])):
            raise ValueError("cu_seqlens must be non-decreasing offsets from 0 within the packed rows")
        if most is not None and any(b - a > most for a, b in zip(h, h[1:])):
            raise ValueError(f"a request may have at most {most} nodes")
    return ints(cu_seqlens, torch.int32, device, "cu_seqlens")


def nodes(parents, cu_seqlens, max_nodes, total, device):
    """(parents or None, cu_seqlens, max_nodes) of a packed set of trees."""
    most = MAX_NODES if max_nodes is None else int(max_nodes)
    if not 1 <= most <= MAX_NODES:
        raise ValueError(f"max_nodes must be 1 to {MAX_NODES}")
    cu = offsets(cu_seqlens, total, device, most)
    if parents is not None:
        parents = ints(parents, torch.int32, device, "parents", total)
    return parents, cu, most
