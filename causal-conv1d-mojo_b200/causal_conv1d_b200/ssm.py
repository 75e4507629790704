"""The selective state space scan that follows the causal conv in a Mamba-2 style block.

Per sequence and head, with a (headdim, dstate) state S, a step length
dt' = softplus(dt + dt_bias) and the head's rate A < 0:

    S_t = exp(dt' * A) * S_{t-1} + dt' * outer(x_t, B_t)
    y_t = S_t @ C_t + D * x_t

``state_space_scan`` runs it over whole prompts (a batch of equal lengths, or
prompts packed one behind the other), ``state_space_update`` advances a pool
of states by one token.  x, B and C are what ``causal_conv1d_fn`` /
``causal_conv1d_update`` return, split by channels; slices of that tensor are
read in place.  Hand-written sm_100a kernels (cc1d_scan, cc1d_scan_update);
no CPU fallback.  Forward only (prefill and decoding): inputs that require
grad are refused.  The reference package has no counterpart; its path ends at
the conv.
"""

from __future__ import annotations

import torch

from . import _ops

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_MAX_STATE = 256


def _check_types(x, dt, A, B, C, D, dt_bias, state, state_name):
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"unsupported dtype {x.dtype}; only fp16/bf16/fp32 are supported")
    for name, t in (("B", B), ("C", C)):
        if t.dtype != x.dtype:
            raise NotImplementedError(f"{name}.dtype ({t.dtype}) must match x.dtype ({x.dtype})")
    for name, t in (("dt", dt), (state_name, state)):
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise NotImplementedError(f"{name}.dtype ({t.dtype}) must be x.dtype ({x.dtype}) or float32")
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None and t.dtype != torch.float32:
            raise NotImplementedError(f"{name} must be float32, got {t.dtype}")


def _check_device(x, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != x.device:
            raise NotImplementedError(f"{name}.device ({t.device}) must match x.device ({x.device})")


def _check_heads(H, A, D, dt_bias, G, N):
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None and t.shape != (H,):
            raise ValueError(f"{name} must be ({H},), got {tuple(t.shape)}")
    if G < 1 or H % G != 0:
        raise ValueError(f"nheads ({H}) must be a multiple of ngroups ({G})")
    if N > _MAX_STATE:
        raise NotImplementedError(f"dstate must be at most {_MAX_STATE} (got {N})")


def _refuse_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} is forward only: detach its inputs or call it under torch.no_grad()")


def _index(name, t, x, shape):
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} != expected {shape}")
    if t.dtype != torch.int32:
        raise ValueError(f"{name}.dtype must be int32 (got {t.dtype})")
    if t.device != x.device:
        raise ValueError(f"{name}.device ({t.device}) must match x.device ({x.device})")
    return t if t.is_contiguous() else t.contiguous()


def _flat(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def state_space_scan(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    initial_states: torch.Tensor | None = None,
    return_final_states: bool = False,
    cu_seqlens: torch.Tensor | None = None,
    max_seqlen: int | None = None,
):
    """
    x: (batch, seqlen, nheads, headdim); any strides
    dt: (batch, seqlen, nheads), x.dtype or float32; the step length is
        dt + dt_bias, through softplus with dt_softplus, and must not be negative
        (a step of 0, e.g. from dt = -inf with dt_softplus, leaves the state alone)
    A: (nheads,) float32, negative; D, dt_bias: (nheads,) float32 or None
    B, C: (batch, seqlen, ngroups, dstate), head h reads group h // (nheads // ngroups);
        dstate <= 256
    initial_states: (num_seqs, nheads, headdim, dstate), float32 or x.dtype, or None
    cu_seqlens: (num_seqs + 1,) int32 on the device, non-decreasing: sequence i is
        tokens [cu_seqlens[i], cu_seqlens[i+1]) of the single batch row.  Sequences may
        be empty; y is 0 for tokens outside all of them.  Without it every batch row
        is a sequence (num_seqs = batch).
    max_seqlen: the longest sequence's length if the caller knows it (with cu_seqlens;
        it only helps to divide the work, and must not be too small to be useful)

    Returns y (batch, seqlen, nheads, headdim) in x.dtype, or (y, final_states) with
    final_states (num_seqs, nheads, headdim, dstate) in float32.

    bf16 and fp16 prompts run on the tensor cores; the state is kept in fp32 between
    blocks of tokens.  There a non-finite x, B, C or dt can reach earlier tokens of its own
    sequence within its block of 128 tokens (not other sequences), and fp16 state values
    beyond 65504 overflow in y (not in the state).
    """
    if x.dim() != 4 or dt.dim() != 3 or B.dim() != 4 or C.dim() != 4:
        raise ValueError("x must be (batch, seqlen, nheads, headdim), dt (batch, seqlen, nheads), "
                         "B and C (batch, seqlen, ngroups, dstate)")
    _check_types(x, dt, A, B, C, D, dt_bias, initial_states, "initial_states")
    batch, seqlen, H, P = x.shape
    G, N = B.shape[2], B.shape[3]
    if dt.shape != (batch, seqlen, H):
        raise ValueError(f"dt must be {(batch, seqlen, H)}, got {tuple(dt.shape)}")
    if B.shape != (batch, seqlen, G, N) or C.shape != B.shape:
        raise ValueError(f"B and C must be ({batch}, {seqlen}, ngroups, dstate), got {tuple(B.shape)} and {tuple(C.shape)}")
    _check_heads(H, A, D, dt_bias, G, N)
    _check_device(x, dt=dt, A=A, B=B, C=C, D=D, dt_bias=dt_bias, initial_states=initial_states)
    nseq = batch
    if cu_seqlens is not None:
        if batch != 1:
            raise ValueError(f"cu_seqlens needs batch == 1 (got {batch})")
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            raise ValueError(f"cu_seqlens must be (num_seqs + 1,), got {tuple(cu_seqlens.shape)}")
        cu_seqlens = _index("cu_seqlens", cu_seqlens, x, tuple(cu_seqlens.shape))
        nseq = cu_seqlens.shape[0] - 1
    if initial_states is not None:
        if initial_states.shape != (nseq, H, P, N):
            raise ValueError(f"initial_states must be {(nseq, H, P, N)}, got {tuple(initial_states.shape)}")
        if initial_states.stride(3) != 1 or initial_states.stride(2) != N:
            initial_states = initial_states.contiguous()
    if max_seqlen is not None and max_seqlen < 0:
        raise ValueError(f"max_seqlen must not be negative (got {max_seqlen})")
    _refuse_grad("state_space_scan", x, dt, A, B, C, D, dt_bias, initial_states)
    y = torch.empty(batch, seqlen, H, P, dtype=x.dtype, device=x.device)
    fs = torch.empty(nseq, H, P, N, dtype=torch.float32, device=x.device) if return_final_states else None
    _ops.scan(x, dt, _flat(A), B, C, _flat(D), _flat(dt_bias), dt_softplus, initial_states, cu_seqlens,
              int(max_seqlen or 0), y, fs)
    return (y, fs) if return_final_states else y


def state_space_update(
    x: torch.Tensor,
    state: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    state_indices: torch.Tensor | None = None,
    out_state_indices: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token per batch row.

    x: (batch, nheads, headdim); dt: (batch, nheads), x.dtype or float32
    state: (batch_or_pool_size, nheads, headdim, dstate), float32 or x.dtype, unit
        stride over dstate; mutated in place.  The step is computed in float32 either way;
        with a 16-bit state each step rounds it once more.
    A, D, dt_bias: (nheads,) float32; B, C: (batch, ngroups, dstate)
    state_indices: (batch,) int32 or None -- the state row that batch row b reads; an
        index outside the pool (such as -1) zeroes y[b] and writes no state.
    out_state_indices: (batch,) int32 or None -- the row that receives the new state
        (the one that was read, when None); an index outside the pool drops it.  No two
        batch rows may write the same row, or one write what another reads.

    Returns y (batch, nheads, headdim).
    """
    if x.dim() != 3 or dt.dim() != 2 or B.dim() != 3 or C.dim() != 3 or state.dim() != 4:
        raise ValueError("x must be (batch, nheads, headdim), dt (batch, nheads), B and C (batch, ngroups, dstate), "
                         "state (rows, nheads, headdim, dstate)")
    _check_types(x, dt, A, B, C, D, dt_bias, state, "state")
    batch, H, P = x.shape
    G, N = B.shape[1], B.shape[2]
    if dt.shape != (batch, H):
        raise ValueError(f"dt must be {(batch, H)}, got {tuple(dt.shape)}")
    if B.shape != (batch, G, N) or C.shape != B.shape:
        raise ValueError(f"B and C must be ({batch}, ngroups, dstate), got {tuple(B.shape)} and {tuple(C.shape)}")
    _check_heads(H, A, D, dt_bias, G, N)
    rows = state.shape[0]
    if state.shape != (rows, H, P, N):
        raise ValueError(f"state shape {tuple(state.shape)}: expected (*, {H}, {P}, {N})")
    if state_indices is None and rows != batch:
        raise ValueError(f"state shape {tuple(state.shape)} != expected {(batch, H, P, N)}")
    if N > 1 and state.stride(3) != 1:
        raise ValueError("state must have unit stride over dstate")
    _check_device(x, dt=dt, A=A, B=B, C=C, D=D, dt_bias=dt_bias, state=state)
    state_indices = _index("state_indices", state_indices, x, (batch,))
    out_state_indices = _index("out_state_indices", out_state_indices, x, (batch,))
    _refuse_grad("state_space_update", x, state, dt, A, B, C, D, dt_bias)
    y = torch.empty(batch, H, P, dtype=x.dtype, device=x.device)
    _ops.scan_update(x, state, dt, _flat(A), B, C, _flat(D), _flat(dt_bias), dt_softplus, state_indices,
                     out_state_indices, y)
    return y
