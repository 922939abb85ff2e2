"""Experts without capacity: rows sorted by expert, products over ragged groups.

The capacity layout (functional.dispatch / batched_ffn) gives every expert C
rows, drops what does not fit and multiplies what stays empty. Here the rows of
one expert stand together, as many as it was chosen for, and the products take
the groups as they are:

    layout = ragged_layout(topk_idx, E)            # on the GPU, no host read
    rows = ragged_gather(tokens, layout)           # [T, D] -> [T*k, D]
    y = ragged_ffn(rows, layout.offsets, stack)    # or grouped_linear(...)
    out = ragged_combine(y, layout, topk_w)        # [T*k, D] -> [T, D]

Nothing waits for the host, so a forward, a backward or a single decoded token
can be captured in a graph. The kernels' gradients cannot be differentiated
again: that raises an error. Slots whose id is no expert (padding, experts that
left) have no row; rows from offsets[E] on belong to nobody: products give
zeros there, and weights get nothing from them.

On a GPU the kernels are ragged_layout.hip and ragged_gemm.hip (bf16, N and K
multiples of 8); on the CPU plain torch with the same meaning.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from . import _C, HAS_HIP

_PLAIN, _GELU, _GELU_DER = 0, 1, 2  # epilogues of ragged_gemm.hip


class RaggedLayout(NamedTuple):
    """offsets [E + 1] int32: expert e has rows offsets[e] .. offsets[e + 1].
    order [T * k] int32: the slot t * k + j of each row, -1 from offsets[E] on.
    rows [T, k] int32: the row of each slot, -1 where it has none."""

    offsets: torch.Tensor
    order: torch.Tensor
    rows: torch.Tensor


def ragged_layout(topk_idx: torch.Tensor, num_experts: int) -> RaggedLayout:
    """Rows of each expert from the router's choice topk_idx [T, k] (int32 or
    int64): slots sorted by expert, and by slot within one. Ids outside
    [0, num_experts) choose nobody."""
    if topk_idx.is_cuda and HAS_HIP:
        return RaggedLayout(*_C.ragged_layout(topk_idx, num_experts))
    if topk_idx.dim() != 2 or topk_idx.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"topk_idx must be [T, k] int32 or int64, got "
                         f"{tuple(topk_idx.shape)} {topk_idx.dtype}")
    if not 1 <= num_experts <= 4096:
        raise ValueError(f"1 to 4096 experts, got {num_experts}")
    flat = topk_idx.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < num_experts), flat, num_experts)
    order = torch.argsort(key, stable=True)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.bincount(key, minlength=num_experts + 1)[:num_experts]
    offsets = F.pad(torch.cumsum(counts, 0), (1, 0))
    return RaggedLayout(offsets.int(), torch.where(key[order] < num_experts, order, -1).int(),
                        torch.where(key < num_experts, rows, -1).int().view(topk_idx.shape))


class _Refuse(torch.autograd.Function):
    """A gradient as it is. The kernels know nothing of the tensors `of` that it depends on, so
    a second derivative would silently lack this path: it raises an error instead."""

    @staticmethod
    def forward(ctx, grad, *of):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("the ragged operators are differentiable once on the GPU")


def _once(grad, *of):
    return _Refuse.apply(grad, *of) if torch.is_grad_enabled() and grad is not None else grad


class _GatherHip(torch.autograd.Function):
    """Rows by the kernels of the capacity layout, all in one group: their number is their slot."""

    @staticmethod
    def forward(ctx, x, rows, order):
        ctx.save_for_backward(rows)
        return _C.dispatch_gather(x, order.unsqueeze(0), rows.shape[1])[0]

    @staticmethod
    def backward(ctx, d):
        rows, = ctx.saved_tensors
        return _once(_C.dispatch_bwd(d.unsqueeze(0), torch.zeros_like(rows), rows, rows.shape[0]), d), None, None


class _CombineHip(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, rows, order, w, least):
        out = _C.combine_fwd(y.unsqueeze(0), torch.zeros_like(rows), rows, w, least)
        ctx.save_for_backward(y, out, rows, order, w)
        ctx.least = least
        return out

    @staticmethod
    def backward(ctx, d):
        y, out, rows, order, w = ctx.saved_tensors
        dy, dw = _C.combine_bwd(d, y.unsqueeze(0), out, torch.zeros_like(rows), rows, w, order.unsqueeze(0), ctx.least)
        return _once(dy[0], w, d), None, None, _once(dw, y, w, d), None


def _check_layout(layout, t, name):
    """The layout's parts go together, and with t: the kernels take rows and slots from them."""
    rows, order = layout.rows, layout.order
    if rows.dtype != torch.int32 or order.dtype != torch.int32:
        raise ValueError(f"the layout's order and rows must be int32, got {order.dtype} and {rows.dtype}")
    if rows.dim() != 2 or order.shape != (rows.numel(),):
        raise ValueError(f"the layout must have rows [T, k] and order [T * k], got {tuple(rows.shape)} "
                         f"and {tuple(order.shape)}")
    if not t.device == rows.device == order.device:
        raise ValueError(f"{name} and the layout must be on one device")


def _check_gpu_rows(t, name, rows=0):
    if t.dtype != torch.bfloat16:
        raise ValueError(f"the GPU kernels take bf16, got {name} in {t.dtype}")
    if t.shape[1] % 8:
        raise ValueError(f"{name} must have a multiple of 8 columns (16-byte rows), got {tuple(t.shape)}")
    if max(t.shape[0], rows) >= 1 << 26:  # a wave each, and 2^32 threads a launch
        raise ValueError(f"below 2^26 tokens and rows, got {t.shape[0]} and {rows}")


def ragged_gather(x: torch.Tensor, layout: RaggedLayout) -> torch.Tensor:
    """x [T, D] -> the layout's rows [T * k, D]; rows of nobody are zeros. On a
    GPU: bf16, D a multiple of 8, below 2^26 rows."""
    from .functional import dispatch

    _check_layout(layout, x, "x")
    T, k = layout.rows.shape
    if x.dim() != 2 or x.shape[0] != T:
        raise ValueError(f"x must be [{T}, D], a row for each token of the layout, got {tuple(x.shape)}")
    if x.is_cuda and HAS_HIP:
        _check_gpu_rows(x, "x", layout.order.numel())
        return _GatherHip.apply(_ready(x), layout.rows, layout.order)
    one = torch.zeros_like(layout.rows)  # all rows in one group: their number is their slot
    return dispatch(x, one, layout.rows, layout.order.unsqueeze(0), k)[0]


def ragged_ungather(y: torch.Tensor, layout: RaggedLayout) -> torch.Tensor:
    """y [T * k, D] -> [T * k, D], row of slot t * k + j at its place again (each
    slot's own row, not summed); zeros for slots that have none. On a GPU: bf16, D
    a multiple of 8."""
    weights = torch.ones(layout.rows.numel(), 1, device=y.device, dtype=torch.float32)
    rows = layout.rows.reshape(-1, 1)
    return ragged_combine(y, RaggedLayout(layout.offsets, layout.order, rows), weights)


def ragged_combine(y: torch.Tensor, layout: RaggedLayout, weights: torch.Tensor,
                   min_mass: float = 0.0) -> torch.Tensor:
    """y [T * k, D] -> [T, D], each token's rows by its weights [T, k], which are
    normalised over the slots that have a row: divided by their sum, or by
    min_mass where that is larger (the bound on 1 / sum that functional.combine
    has behind a capacity, 0.2). A sum of zero or less gives zeros. On a GPU: y
    bf16, D a multiple of 8, weights fp32, below 2^26 rows."""
    from .functional import combine

    if not min_mass >= 0:
        raise ValueError(f"min_mass must not be negative, got {min_mass}")
    least = max(min_mass, torch.finfo(torch.float32).tiny)  # the smallest normal number's inverse is finite
    _check_layout(layout, y, "y")
    if y.dim() != 2 or y.shape[0] != layout.order.numel():
        raise ValueError(f"y must be [{layout.order.numel()}, D], the layout's rows, got {tuple(y.shape)}")
    if weights.shape != layout.rows.shape:
        raise ValueError(f"weights must be {tuple(layout.rows.shape)}, one for each slot, got {tuple(weights.shape)}")
    if weights.device != y.device:
        raise ValueError("y, weights and the layout must be on one device")
    if y.is_cuda and HAS_HIP:
        _check_gpu_rows(y, "y")
        if weights.dtype != torch.float32:
            raise ValueError(f"weights must be fp32, got {weights.dtype}")
        return _CombineHip.apply(_ready(y), layout.rows, layout.order, weights, least)
    one = torch.zeros_like(layout.rows)
    return combine(y.unsqueeze(0), one, layout.rows, weights, layout.order.unsqueeze(0), least)


# ---------------------------------------------------------------------------
# one product
# ---------------------------------------------------------------------------
def _check_product(x, weight, offsets, bias, activation):
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2]:
        raise ValueError(f"x must be [R, K] and weight [E, N, K], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if offsets.dtype != torch.int32 or offsets.shape != (weight.shape[0] + 1,):
        raise ValueError(f"offsets must be [E + 1] int32, got {tuple(offsets.shape)} {offsets.dtype}")
    if bias is not None and bias.shape != weight.shape[:2]:
        raise ValueError(f"bias must be [E, N], got {tuple(bias.shape)}")
    if activation not in (None, "gelu"):
        raise ValueError(f"activation must be None or 'gelu', got {activation!r}")
    if len({t.device for t in (x, weight, offsets, bias) if t is not None}) > 1:
        raise ValueError("x, weight, offsets and bias must be on one device")
    if x.dtype != weight.dtype:
        raise ValueError(f"x and weight must have one type, got {x.dtype} and {weight.dtype}")


def _check_gpu_product(x, weight):
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError(f"the GPU kernels take bf16, got {x.dtype} and {weight.dtype}")
    if weight.shape[0] == 0 or weight[0].numel() == 0:
        raise ValueError(f"weight must not be empty, got {tuple(weight.shape)}")
    if weight.shape[1] % 8 or weight.shape[2] % 8:
        raise ValueError(f"N and K must be multiples of 8 (16-byte rows), got {tuple(weight.shape)}")
    if weight[0].numel() >= 1 << 30 or max(weight.shape[1:]) >= 1 << 21:
        raise ValueError(f"one expert's weight must have below 2^30 numbers, and N and K be below "
                         f"2^21, got {tuple(weight.shape)}")


def _ready(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, from a multiple of 16 bytes on: what the kernels load."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                   bias: Optional[torch.Tensor] = None,
                   activation: Optional[str] = None) -> torch.Tensor:
    """y[r] = act(weight[e] @ x[r] + bias[e]) for the rows offsets[e] <= r < offsets[e + 1].

    x [R, K]; weight [E, N, K]; offsets [E + 1] int32, ascending from 0, at most
    R (a RaggedLayout's, or any other groups); bias [E, N]; activation None or
    "gelu" (its tanh form). Returns [R, N], zeros from row offsets[E] on.
    Differentiable in x, weight and bias; a group without rows has zero weight
    gradients. Sums are fp32; y, dx and dW are rounded once (with gelu its slope
    is kept in fp16, and the gradient at its input is rounded to bf16 between the
    products, not for the bias's sums). On a GPU: bf16,
    at most 4096 groups, N and K multiples of 8 below 2^21, N * K below 2^30.
    Differentiable once, backwards: on a GPU forward-mode derivatives and a
    backward pass with create_graph=True are refused. As with other operators, a backward pass is captured into
    a graph with torch.autograd.grad or with no eager graph of the leaves alive."""
    if x.is_cuda and HAS_HIP:  # checks, gradients and all: bindings.cpp
        return _C.grouped_linear(x, weight, offsets, bias, activation)
    _check_product(x, weight, offsets, bias, activation)
    return _grouped_linear_torch(x, weight, offsets, bias, activation == "gelu")


def _grouped_linear_torch(x, weight, offsets, bias, gelu):
    at = offsets.tolist()
    parts = []
    wide = torch.promote_types(x.dtype, torch.float32)  # sums, bias and gelu; rounded once
    for e, (lo, hi) in enumerate(zip(at[:-1], at[1:])):
        h = x[lo:hi].to(wide) @ weight[e].to(wide).t()
        if bias is not None:
            h = h + bias[e].to(wide)
        parts.append((F.gelu(h, approximate="tanh") if gelu else h).to(x.dtype))
    parts.append(x.new_zeros(x.shape[0] - at[-1], weight.shape[1]))
    return torch.cat(parts)


# ---------------------------------------------------------------------------
# an expert stack's FFN
# ---------------------------------------------------------------------------
class _RaggedFFNHip(torch.autograd.Function):
    """Both products of a stack's experts; weight gradients go into the stack's
    main_grad buffers, as functional._BatchedFFNHip has them."""

    @staticmethod
    def forward(ctx, x, offsets, stack):
        der = torch.empty(x.shape[0], stack.ffn_dim, dtype=torch.float16, device=x.device)
        h = _C.ragged_nt(x, stack.W1c, offsets, stack.b1_f32, der, _GELU_DER)
        y = _C.ragged_nt(h, stack.W2c, offsets, stack.b2_f32, None, _PLAIN)
        ctx.save_for_backward(x, offsets, der, h)
        ctx.stack = stack
        return y

    @staticmethod
    def backward(ctx, dy):
        from .functional import _wait_pending_opt

        x, offsets, der, h = ctx.saved_tensors
        stack = ctx.stack
        _check_stack(stack)
        _wait_pending_opt(stack)
        dy = _ready(dy)
        dh = _C.ragged_nn(dy, stack.W2c, offsets, der)  # at gelu's input, rounded to bf16 for the next two
        # products, and for b1's sums, which ride in one of them (as the capacity layout has them)
        dx = _C.ragged_nn(dh, stack.W1c, offsets) if ctx.needs_input_grad[0] else None
        acc = stack.grad_ready
        _C.ragged_tn(dh, x, offsets, stack.main_grad_W1, stack.main_grad_b1, acc)
        _C.ragged_tn(dy, h, offsets, stack.main_grad_W2, stack.main_grad_b2, acc)
        stack.grad_ready = True
        return _once(dx, x, dy), None, None


def _check_stack(stack):
    if getattr(stack, "_fused_sr_opt", None) is not None:
        raise RuntimeError("the fused dW + SGD backward is for capacity buffers: construct "
                           "FusedExpertSGD(fused_backward=False) for ragged rows")


def ragged_ffn(x: torch.Tensor, offsets: torch.Tensor, stack) -> torch.Tensor:
    """Each expert's FFN over its rows: x [R, d] -> [R, d], gelu between the two
    products. `stack`: a parallel.ExpertStack. On a GPU its weight gradients go
    to main_grad_* when x has a gradient (one backward writes, further ones of a
    step add)."""
    if x.dim() != 2 or x.shape[1] != stack.d_model:
        raise ValueError(f"x must be [R, {stack.d_model}], got {tuple(x.shape)}")
    if offsets.dtype != torch.int32 or offsets.shape != (stack.num_local + 1,):
        raise ValueError(f"offsets must be [{stack.num_local + 1}] int32, got "
                         f"{tuple(offsets.shape)} {offsets.dtype}")
    if x.is_cuda and HAS_HIP:
        from .functional import _wait_pending_opt

        if not stack._gpu_state_ready:
            raise RuntimeError("call the stack's init_gpu_state() first")
        _check_gpu_product(x, stack.W1c)
        x, offsets = _ready(x), offsets.contiguous()
        _wait_pending_opt(stack)
        if torch.is_grad_enabled() and x.requires_grad:
            _check_stack(stack)
            return _RaggedFFNHip.apply(x, offsets, stack)
        h = _C.ragged_nt(x, stack.W1c, offsets, stack.b1_f32, None, _GELU)
        return _C.ragged_nt(h, stack.W2c, offsets, stack.b2_f32, None, _PLAIN)
    h = _grouped_linear_torch(x.float(), stack.W1.float(), offsets, stack.W1_bias, True)
    return _grouped_linear_torch(h, stack.W2.float(), offsets, stack.W2_bias, False).to(x.dtype)
