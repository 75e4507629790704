"""The gated norm between the state space scan and the output projection of a Mamba-2 style block.

``gated_norm_fn`` normalises groups of adjacent columns (RMS or layer norm)
with an optional SiLU gate before or after the norm, forward and backward, in
hand-written sm_100a kernels (cc1d_gated_norm_fwd / cc1d_gated_norm_bwd).
The reference package has no counterpart; its path ends at the conv.
"""

from __future__ import annotations

import math

import torch

from . import _ops

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _rows(t):
    """(..., dim) as (rows, dim) with unit stride over dim; a copy only when its strides need one."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


class _GatedNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, z, eps, group_size, layer, gate_first):
        x2, z2 = _rows(x), None if z is None else _rows(z)
        w, b = weight.contiguous(), None if bias is None else bias.contiguous()
        M, dim = x2.shape
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = [None, None]
        if any(ctx.needs_input_grad[:4]):
            shape = (M, dim // group_size)
            stats = [torch.empty(shape, dtype=torch.float32, device=x.device) if want else None for want in (layer, True)]
        _ops.norm_fwd(x2, z2, w, b, eps, group_size, layer, gate_first, y.view(M, dim), *stats)
        ctx.save_for_backward(x2, z2, w, b, *stats)
        ctx.how = eps, group_size, layer, gate_first
        ctx.shapes = x.shape, None if z is None else z.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_norm_fn has no second derivative (backward with create_graph=True)")
        x, z, w, b, mean, rstd = ctx.saved_tensors
        eps, group_size, layer, gate_first = ctx.how
        dy = _rows(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dz = None if z is None else torch.empty(z.shape, dtype=z.dtype, device=z.device)
        dw = torch.empty_like(w)
        db = None if b is None else torch.empty_like(b)
        _ops.norm_bwd(x, z, w, b, dy, mean, rstd, eps, group_size, layer, gate_first, dx, dz, dw, db)
        return dx.view(ctx.shapes[0]), dw, db, None if dz is None else dz.view(ctx.shapes[1]), None, None, None, None


def gated_norm_fn(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    eps: float = 1e-5,
    group_size: int | None = None,
    kind: str = "rms",
    gate_first: bool = True,
) -> torch.Tensor:
    """
    x: (..., dim) fp16 / bf16 / fp32
    weight, bias: (dim,), x.dtype or float32 (both the same); bias may be None
    z: (..., dim) like x, or None -- the gate: the norm is taken of x * silu(z) with
        gate_first, else its result is multiplied by silu(z)
    group_size: columns per group, a divisor of dim; dim when None
    kind: "rms" (no mean taken) or "layer"

    Returns y like x (contiguous).  Statistics and sums are in float32.  Differentiable
    in x, weight, bias and z; the sums of the weight's and bias's gradients are taken in
    a fixed order (bitwise reproducible).
    """
    if kind not in ("rms", "layer"):
        raise NotImplementedError(f"kind must be 'rms' or 'layer' (got {kind!r})")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"unsupported dtype {x.dtype}; only fp16/bf16/fp32 are supported")
    if x.dim() < 1:
        raise ValueError("x must be (..., dim)")
    dim = x.shape[-1]
    if weight.dtype not in (x.dtype, torch.float32):
        raise NotImplementedError(f"weight.dtype ({weight.dtype}) must be x.dtype ({x.dtype}) or float32")
    if bias is not None and bias.dtype != weight.dtype:
        raise NotImplementedError(f"bias.dtype ({bias.dtype}) must match weight.dtype ({weight.dtype})")
    if weight.shape != (dim,) or (bias is not None and bias.shape != (dim,)):
        raise ValueError(f"weight and bias must be ({dim},)")
    if z is not None:
        if z.dtype != x.dtype:
            raise NotImplementedError(f"z.dtype ({z.dtype}) must match x.dtype ({x.dtype})")
        if z.shape != x.shape:
            raise ValueError(f"z shape {tuple(z.shape)} != x shape {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("z", z)):
        if t is not None and t.device != x.device:
            raise NotImplementedError(f"{name}.device ({t.device}) must match x.device ({x.device})")
    if group_size is None:
        group_size = max(dim, 1)
    if group_size < 1 or dim % group_size != 0:
        raise ValueError(f"dim ({dim}) must be a multiple of group_size ({group_size})")
    return _GatedNormFn.apply(x, weight, bias, z, float(eps), int(group_size), kind == "layer", bool(gate_first))
