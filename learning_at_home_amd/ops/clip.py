"""Global gradient norm over many tensors, clipping, and the clipped SGD step.

    norm, scale = grad_clip_scale(grads, max_norm)      # on the GPU, no host read
    master_sgd_step_(params, masters, grads, lr=lr, grad_scale=scale)

or, for an optimizer that knows nothing of it, clip_grad_norm_(grads, max_norm)
in place. On a GPU a few launches serve all tensors (clip.hip); on the CPU, and
for tensors the kernels do not take (not contiguous), plain torch.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _C, HAS_HIP


def _listed(tensors) -> list:
    if isinstance(tensors, torch.Tensor):
        tensors = [tensors]
    tensors = list(tensors)
    if not tensors:
        raise ValueError("no tensors")
    return tensors


def _check_distinct(tensors, name) -> None:
    """Those that are written: on a GPU by many blocks at once."""
    at = [t.data_ptr() for t in tensors if t.numel() and t.device.type != "meta"]
    if len(set(at)) < len(at):
        raise ValueError(f"the same tensor twice among the {name}")


@torch.no_grad()
def grad_clip_scale(tensors: Sequence[torch.Tensor], max_norm: float,
                    eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(norm, scale), two fp32 numbers on the tensors' device: the 2-norm of all
    tensors together, and min(1, max_norm / (norm + eps)). A gradient that is
    not finite makes a norm that is not (scale 0 for infinity, not-a-number for
    one). The norm is this process's own: steps here wait for no other rank."""
    tensors = _listed(tensors)
    if not max_norm > 0:
        raise ValueError(f"max_norm must be positive, got {max_norm}")
    if HAS_HIP and tensors[0].is_cuda:
        got = _C.grad_norm(tensors, max_norm, eps) or _C.grad_norm([t.contiguous() for t in tensors], max_norm, eps)
        if got:
            return tuple(got)
    if any(t.device != tensors[0].device for t in tensors):
        raise ValueError("all tensors must be on one device")
    norm = torch.stack([t.double().square().sum() for t in tensors]).sum().sqrt()
    return norm.float(), (max_norm / (norm + eps)).clamp(max=1.0).float()


@torch.no_grad()
def clip_grad_norm_(tensors: Sequence[torch.Tensor], max_norm: float,
                    eps: float = 1e-6) -> torch.Tensor:
    """Scales the tensors in place to a common 2-norm of at most max_norm, and
    returns the norm they had, on their device. No tensor may be there twice."""
    tensors = _listed(tensors)
    if not (HAS_HIP and tensors[0].is_cuda):  # where the kernels check the same
        _check_distinct(tensors, "tensors")
    norm, scale = grad_clip_scale(tensors, max_norm, eps)
    if not (HAS_HIP and tensors[0].is_cuda and _C.grad_scale_(tensors, scale)):
        for t in tensors:
            t.mul_(scale)
    return norm


@torch.no_grad()
def master_sgd_step_(params: Sequence[torch.Tensor], masters: Sequence[torch.Tensor],
                     grads: Sequence[torch.Tensor], lr: float, momentum: float = 0.0,
                     weight_decay: float = 0.0,
                     momentum_bufs: Optional[Sequence[torch.Tensor]] = None,
                     grad_scale: Optional[torch.Tensor] = None) -> None:
    """One SGD step of fp32 masters, all tensors at once:

        u = grad_scale * g + weight_decay * m
        b = momentum * b + u, u = b          (with momentum_bufs)
        m -= lr * u;  p = m rounded to p's type

    No parameter, master or buffer may be there twice."""
    params, masters, grads = list(params), list(masters), list(grads)
    bufs = list(momentum_bufs) if momentum_bufs is not None else []
    if not len(params) == len(masters) == len(grads) or (bufs and len(bufs) != len(params)):
        raise ValueError("params, masters, grads and momentum_bufs must go together")
    if momentum and not bufs:
        raise ValueError("momentum needs momentum_bufs")
    if not params:
        return
    if isinstance(grad_scale, torch.Tensor) and (grad_scale.numel() != 1 or (
            params[0].is_cuda and grad_scale.device != params[0].device)):
        raise ValueError(f"grad_scale must be one number on the params' device, got {tuple(grad_scale.shape)} "
                         f"on {grad_scale.device}")
    if HAS_HIP and params[0].is_cuda:  # with the same checks
        if _C.master_sgd_(params, masters, grads, bufs, grad_scale, lr, momentum, weight_decay):
            return
    else:
        if any(m.dtype != torch.float32 for m in masters + bufs):
            raise ValueError("masters and momentum_bufs must be fp32")
        if any(p.shape != m.shape or p.shape != g.shape for p, m, g in zip(params, masters, grads)):
            raise ValueError("params, masters and grads must have the same shapes")
        if any(p.shape != b.shape for p, b in zip(params, bufs)):
            raise ValueError("momentum_bufs must have the shapes of the params")
        for name, ts in (("params", params), ("masters", masters), ("momentum_bufs", bufs)):
            _check_distinct(ts, name)
    for i in range(len(params)):
        b = bufs[i : i + 1]
        if HAS_HIP and params[i].is_cuda and _C.master_sgd_(params[i : i + 1], masters[i : i + 1], grads[i : i + 1],
                                                           b, grad_scale, lr, momentum, weight_decay):
            continue
        u = grads[i].float()
        if grad_scale is not None:
            u = u * grad_scale
        if weight_decay:
            u = u + weight_decay * masters[i]
        if b:
            u = b[0].mul_(momentum).add_(u)
        masters[i].add_(u, alpha=-lr)
        params[i].copy_(masters[i])
