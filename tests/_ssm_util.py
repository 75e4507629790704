"""Inputs and 64-bit references of the state space scan tests."""

from __future__ import annotations

import math

import torch

# Unit roundoffs: the largest relative error of one rounding to the type.
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def scan_inputs(rows, L, H, P, G, N, dtype, seed=0, device="cuda", sliced=True, step=(1e-3, 1e-1)):
    """x, dt, A, B, C, D, dt_bias as a block has them: x, B and C slices of one tensor, rates in
    [1, 16], steps around [1e-3, 1e-1] before the data moves them."""
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=device)

    width = H * P + 2 * G * N
    xbc = torch.nn.functional.silu(randn(rows, L, width)).to(dtype)
    if not sliced:  # contiguous pieces of their own
        x, B, C = (t.contiguous() for t in xbc.split([H * P, G * N, G * N], -1))
    else:
        x, B, C = xbc.split([H * P, G * N, G * N], -1)
    A = -(1 + 15 * torch.rand(H, generator=g, device=device))
    lo, hi = math.log(step[0]), math.log(step[1])
    s = torch.exp(lo + torch.rand(H, generator=g, device=device) * (hi - lo))
    bias = s + torch.log(-torch.expm1(-s))
    return dict(x=x.unflatten(-1, (H, P)), dt=(0.5 * randn(rows, L, H)).to(dtype), A=A, B=B.unflatten(-1, (G, N)),
                C=C.unflatten(-1, (G, N)), D=1 + 0.1 * randn(H), dt_bias=bias)


def _recurrence(x, dt, A, B, C, D, S):
    """One sequence, (L, H, P) and so on, float64, dt final."""
    y = torch.empty_like(x)
    for t in range(x.shape[0]):
        S = S * torch.exp(dt[t] * A)[:, None, None] + (dt[t][:, None] * x[t])[:, :, None] * B[t][:, None, :]
        y[t] = (S * C[t][:, None, :]).sum(-1) + D[:, None] * x[t]
    return y, S


def scan_reference(x, dt, A, B, C, D=None, dt_bias=None, dt_softplus=True, initial_states=None, ranges=None):
    """y, final states and, for error bounds, the same sums with every term's magnitude: (y, S, |y|, |S|)."""
    rows, L, H, P = x.shape
    N = B.shape[-1]
    R = H // B.shape[2]
    step = dt.double()
    if dt_bias is not None:
        step = step + dt_bias.double()
    if dt_softplus:
        step = torch.nn.functional.softplus(step, threshold=50)
    Ad = A.double()
    Dd = D.double() if D is not None else torch.zeros(H, dtype=torch.float64, device=x.device)
    xd = x.double()
    Bd, Cd = (v.double().repeat_interleave(R, 2) for v in (B, C))
    if ranges is None:
        ranges = [(b, 0, L) for b in range(rows)]
    y, my = torch.zeros_like(xd), torch.zeros_like(xd)
    finals, mfinals = [], []
    for i, (b, t0, t1) in enumerate(ranges):
        S0 = torch.zeros(H, P, N, dtype=torch.float64, device=x.device) if initial_states is None else initial_states[i].double()
        s = (b, slice(t0, t1))
        y[s], S = _recurrence(xd[s], step[s], Ad, Bd[s], Cd[s], Dd, S0)
        my[s], mS = _recurrence(xd[s].abs(), step[s], Ad, Bd[s].abs(), Cd[s].abs(), Dd.abs(), S0.abs())
        finals.append(S)
        mfinals.append(mS)
    shape = (0, H, P, N)
    stack = lambda v: torch.stack(v) if v else torch.zeros(shape, dtype=torch.float64, device=x.device)  # noqa: E731
    return y, stack(finals), my, stack(mfinals)


def scan_bounds(y, S, my, mS, dtype, L, N, x, C):
    """Elementwise error bounds of y and the final state.

    Every product and sum in fp32 (unit e = 2^-24) with at most six roundings per token of a
    term's way (step length, its product with the rate, the exponential at two units, the decay's
    product, the sum), and the sum over N: (6 L + N + 16) e of the sum of the terms' magnitudes.
    In 16 bits a term of y may besides be rounded once (unit u) as an operand of a matrix
    product, and y is rounded to its type.  A 16-bit operand below fp16's normal range is off by
    2^-25 at most, for each of up to 128 tokens' x and N values of C.  The final state has no
    16-bit rounding.
    """
    e, u = 2.0 ** -24, UNIT[dtype]
    c = (6 * L + N + 16) * e
    by = c * my + u * y.abs() * (1 + 2 * u) + 1e-30
    if dtype != torch.float32:
        by = by + u * my
    if dtype == torch.float16 and x.numel():
        by = by + 2.0 ** -25 * (1 + 128 * x.double().abs().max() + N * C.double().abs().max())
    return by, c * mS + 1e-30


def check_scan(got, final, ref, dtype, L, N, x, C):
    y, S, my, mS = ref
    by, bS = scan_bounds(y, S, my, mS, dtype, L, N, x, C)
    assert torch.isfinite(got).all()
    over = (got.double() - y).abs() - by
    assert not (over > 0).any(), f"y: {int((over > 0).sum())} values beyond the bound, worst by {over.max().item():.3e}"
    if final is not None:
        assert final.dtype == torch.float32 and torch.isfinite(final).all()
        over = (final.double() - S).abs() - bS
        assert not (over > 0).any(), f"final: {int((over > 0).sum())} beyond the bound, worst by {over.max().item():.3e}"
        if S.norm() > 0:
            # Independent roundings add up like a random walk: far below the bound above, and above
            # what a state summed from operands of under 20 bits would reach.
            rel = ((final.double() - S).norm() / S.norm()).item()
            assert rel < 4e-6, f"final: relative error {rel:.2e}"
