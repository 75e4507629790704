"""The gated norm, forward and backward, against its formulas in 64 bits and against differences.

Bounds.  All sums and products are in fp32 (unit e = 2^-24); a sum over a group of n columns is
within (n / 32 + 16) e of the sum of its terms' magnitudes (a thread's own columns, then a tree),
SiLU within 8 e relative, and every output is rounded once to its type (unit u).  With
k = (n / 32 + 64) e for a whole chain of such steps, an output is checked against
k * (its terms' magnitudes) + u * |its value|.
"""

from __future__ import annotations

import pytest
import torch

from _ssm_util import UNIT
from causal_conv1d_b200.norm import gated_norm_fn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(M, dim, dtype, gate, bias, wdtype=None, seed=0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=DEV)

    wdtype = wdtype or dtype
    return dict(x=(randn(M, dim) + mean).to(dtype), weight=(1 + 0.2 * randn(dim)).to(wdtype),
                bias=(0.2 * randn(dim)).to(wdtype) if bias else None, z=randn(M, dim).to(dtype) if gate else None,
                dy=randn(M, dim).to(dtype))


def _formulas(v, group, kind, gate_first, eps):
    """Outputs in 64 bits and the magnitudes their error bounds scale with."""
    M, dim = v["x"].shape
    sh = (M, dim // group, group)
    x, dy, w = v["x"].double().view(sh), v["dy"].double().view(sh), v["weight"].double().view(sh[1:])
    b = v["bias"].double().view(sh[1:]) if v["bias"] is not None else torch.zeros_like(w)
    z = v["z"].double().view(sh) if v["z"] is not None else None
    s = z * torch.sigmoid(z) if z is not None else None
    ds = torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z))) if z is not None else None
    dsm = torch.sigmoid(z) * (1 + z.abs()) if z is not None else None
    u = x * s if z is not None and gate_first else x
    mu = u.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(u[..., :1])
    mmu = u.abs().mean(-1, keepdim=True) if kind == "layer" else mu
    r = (u - mu).pow(2).mean(-1, keepdim=True).add(eps).rsqrt()
    h = (u - mu) * r
    mh = (u.abs() + mmu) * r * (1 + h.abs().clamp(max=1)) + h.abs()
    o, mo = h * w + b, mh * w.abs() + b.abs()
    post = z is not None and not gate_first
    out = {"y": (o * s, mo * s.abs()) if post else (o, mo)}
    d, md = (dy * s, (dy * s).abs()) if post else (dy, dy.abs())
    out["dweight"] = ((d * h).sum(0).flatten(), (md * mh).sum(0).flatten())
    out["dbias"] = (d.sum(0).flatten(), md.sum(0).flatten())
    g, mg = d * w, md * w.abs()
    c1, m1 = (g * h).mean(-1, keepdim=True), (mg * mh).mean(-1, keepdim=True)
    c2, m2 = g.mean(-1, keepdim=True), mg.mean(-1, keepdim=True)
    du = r * (g - h * c1 - (c2 if kind == "layer" else 0))
    mdu = r * (mg + mh * m1 + (m2 if kind == "layer" else 0)) * (1 + mmu * r)
    if z is None:
        out["dx"] = (du, mdu)
    elif gate_first:
        out["dx"], out["dz"] = (du * s, mdu * s.abs()), (du * x * ds, mdu * x.abs() * dsm)
    else:
        out["dx"], out["dz"] = (du, mdu), (dy * o * ds, dy.abs() * mo * dsm)
    return {k: (a.reshape(M, dim) if k not in ("dweight", "dbias") else a,
                m.reshape(M, dim) if k not in ("dweight", "dbias") else m) for k, (a, m) in out.items()}


def _run(v, group, kind, gate_first, eps):
    leaves = {k: v[k].detach().requires_grad_() for k in ("x", "weight", "bias", "z") if v[k] is not None}
    y = gated_norm_fn(leaves["x"], leaves["weight"], leaves.get("bias"), z=leaves.get("z"), eps=eps, group_size=group,
                      kind=kind, gate_first=gate_first)
    grads = torch.autograd.grad(y, list(leaves.values()), v["dy"])
    return {"y": y.detach(), **{"d" + k: t for k, t in zip(leaves, grads)}}


def _check(v, group, kind, gate_first, eps=1e-5):
    got = _run(v, group, kind, gate_first, eps)
    ref = _formulas(v, group, kind, gate_first, eps)
    M = v["x"].shape[0]
    k = (group / 32 + 64) * 2.0 ** -24
    for name, t in got.items():
        want, mag = ref[name]
        over_rows = name in ("dweight", "dbias")
        c = k + (M + 16) * 2.0 ** -24 if over_rows else k
        u = UNIT[t.dtype]
        assert torch.isfinite(t).all(), name
        over = (t.double() - want).abs() - (c * mag + u * want.abs() * (1 + u) + 2.0 ** -25 * (t.dtype == FP16) + 1e-30)
        assert not (over > 0).any(), f"{name}: {int((over > 0).sum())} beyond the bound, worst by {over.max().item():.3e}"
    return got


@pytest.mark.parametrize("dtype", [BF, FP16, F32])
@pytest.mark.parametrize("kind,gate,gate_first,bias", [
    ("rms", False, True, False), ("rms", True, True, False), ("rms", True, False, True), ("layer", False, True, True),
    ("layer", True, True, True), ("layer", True, False, False),
])
@pytest.mark.parametrize("M,dim,group", [
    (1, 64, 64), (5, 1, 1), (7, 1001, 1001), (3, 5120, 5120), (300, 96, 32), (33, 640, 640), (4, 5120, 640),
    (2, 8200, 8200),
])
def test_norm_matches_formulas(dtype, kind, gate, gate_first, bias, M, dim, group):
    if group == 1 and kind == "layer":
        pytest.skip("a group of one column has no variance: its gradient is 0 times 1/sqrt(eps)")
    v = _inputs(M, dim, dtype, gate, bias, seed=M + dim)
    _check(v, group, kind, gate_first)


@pytest.mark.parametrize("dtype,dim", [(BF, 40000), (F32, 33000), (F32, 16384), (BF, 4099)])
@pytest.mark.parametrize("gate,gate_first,kind", [(True, True, "rms"), (True, False, "layer"), (False, True, "layer")])
def test_norm_wide_rows(dtype, dim, gate, gate_first, kind):
    _check(_inputs(6, dim, dtype, gate, True, seed=dim), dim, kind, gate_first)


@pytest.mark.parametrize("rows", [1500, 5000])
def test_norm_many_rows_and_fp32_weight(rows):
    """More rows than teams; weights and their gradients in fp32 next to bf16 data."""
    v = _inputs(rows, 512, BF, True, True, wdtype=F32, seed=rows)
    got = _check(v, 512, "rms", True)
    assert got["dweight"].dtype == F32
    again = _run(v, 512, "rms", True, 1e-5)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype,rows,dim,group,wdtype", [(BF, 2500, 5120, 5120, None), (FP16, 1900, 2056, 2056, F32),
                                                        (F32, 2000, 2048, 2048, None), (BF, 1801, 3200, 1600, None)])
@pytest.mark.parametrize("kind,gate,gate_first,bias", [
    ("rms", False, True, False), ("rms", True, True, False), ("layer", True, False, True), ("layer", False, True, True),
])
def test_norm_many_wide_rows(dtype, rows, dim, group, wdtype, kind, gate, gate_first, bias):
    """Several rows per block, so that they come through shared memory; rows that do not divide evenly."""
    _check(_inputs(rows, dim, dtype, gate, bias, wdtype=wdtype, seed=dim), group, kind, gate_first)


def test_norm_large_mean():
    """A layer norm of values far from zero: the variance is that of the centred values."""
    _check(_inputs(9, 1024, F32, False, True, seed=1, mean=300.0), 1024, "layer", True)


def test_norm_layouts_and_shapes():
    """Rows with a pitch of their own, odd offsets, more than two axes, expanded gradients."""
    M, dim = 6, 256
    v = _inputs(M, dim, BF, True, False, seed=2)
    want = _run(v, dim, "rms", True, 1e-5)
    for off in (8, 1):  # aligned and not
        wide = {k: torch.zeros(M, dim + 24, dtype=BF, device=DEV) for k in ("x", "z", "dy")}
        for k, t in wide.items():
            t[:, off:off + dim] = v[k]
        got = _run({**v, **{k: t[:, off:off + dim] for k, t in wide.items()}}, dim, "rms", True, 1e-5)
        for k in want:
            torch.testing.assert_close(got[k].float(), want[k].float(), rtol=2.0 ** -7, atol=1e-5)
    t = {k: v[k].view(2, 3, dim) for k in ("x", "z")}
    y = gated_norm_fn(t["x"], v["weight"], z=t["z"])
    assert torch.equal(y.view(M, dim), want["y"])
    x = t["x"].transpose(0, 1).detach().requires_grad_()  # rows out of order
    y = gated_norm_fn(x, v["weight"], z=t["z"].transpose(0, 1))
    assert torch.equal(y.transpose(0, 1).reshape(M, dim), want["y"])
    y.sum().backward()
    ones = _run({**v, "dy": torch.ones_like(v["dy"])}, dim, "rms", True, 1e-5)
    assert torch.equal(x.grad.transpose(0, 1).reshape(M, dim), ones["dx"])


def test_norm_zero_rows_and_zero_columns():
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    y = gated_norm_fn(x, w)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert (w.grad == 0).all() and x.grad.shape == (0, 64)
    assert gated_norm_fn(torch.zeros(3, 0, device=DEV), torch.zeros(0, device=DEV)).shape == (3, 0)
    # A row of zeros: 0 / sqrt(eps), and a gradient of w / sqrt(eps).
    x = torch.zeros(2, 64, device=DEV, requires_grad=True)
    y = gated_norm_fn(x, w)
    assert (y == 0).all()
    y.sum().backward()
    torch.testing.assert_close(x.grad, torch.full_like(x, 1e-5 ** -0.5))


@pytest.mark.parametrize("kind,gate,gate_first,bias", [("rms", True, True, False), ("layer", True, False, True),
                                                       ("layer", False, True, True)])
def test_norm_gradients_against_differences(kind, gate, gate_first, bias):
    """<gradient, direction> against the central difference of the kernel's own forward, in fp32.
    The difference is off by h^2 / 6 times the third derivative (values near 1: about 1e-4 of it at
    h = 1e-2) and by the forward's rounding over h (2^-22 * sqrt(values) / h); both under 2e-3."""
    v = _inputs(4, 128, F32, gate, bias, seed=5)
    got = _run(v, 64, kind, gate_first, 1e-5)
    h = 1e-2

    def loss(changed):
        q = {**v, **changed}
        y = gated_norm_fn(q["x"], q["weight"], q["bias"], z=q["z"], group_size=64, kind=kind, gate_first=gate_first)
        return (y.double() * v["dy"].double()).sum()

    g = torch.Generator(device=DEV).manual_seed(11)
    for name in ("x", "weight", "bias", "z"):
        if v[name] is None:
            continue
        way = torch.randn(v[name].shape, generator=g, device=DEV)
        way = way / way.norm()
        diff = ((loss({name: v[name] + h * way}) - loss({name: v[name] - h * way})) / (2 * h)).item()
        exact = (got["d" + name].double() * way.double()).sum().item()
        scale = got["d" + name].double().norm().item()
        assert abs(diff - exact) <= 2e-3 * max(1.0, scale), (name, diff, exact)


def test_norm_stream_graph_and_compile():
    v = _inputs(40, 512, BF, True, False, seed=3)
    want = gated_norm_fn(v["x"], v["weight"], z=v["z"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_norm_fn(v["x"], v["weight"], z=v["z"])
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gated_norm_fn(v["x"], v["weight"], z=v["z"])
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    fn = torch.compile(lambda x, w, z: gated_norm_fn(x, w, z=z), fullgraph=True, backend="aot_eager")
    x = v["x"].detach().requires_grad_()
    w = v["weight"].detach().requires_grad_()
    y = fn(x, w, v["z"])
    assert torch.equal(y, want)
    dx, dw = torch.autograd.grad(y, [x, w], v["dy"])
    ref = _run(v, 512, "rms", True, 1e-5)
    assert torch.equal(dx, ref["dx"]) and torch.equal(dw, ref["dweight"])
