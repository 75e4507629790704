"""The state-space operators that follow the causal conv in a Mamba-2 style block, as measured work.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as a call of
this library:

* the selective state space scan over whole prompts,
* its form for single tokens, on a pool of states,
* the gated norm behind it, forward alone and forward with backward.

Sizes: the library's 2.7B-like block (conv channels 5376 = 80 heads of 64, and B and C of 128), its
packed prefill of 65536 fp16 tokens in 32 sequences, its fp32 case of (2, 512) tokens, its decode
batch of 256 rows on a pool of 512, and generic small and odd ones.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64  # tokens per block of the plain scan


def _product():
    """The package's folder has no module name of its own: it goes on the path, as for any user."""
    folder = os.path.join(os.getcwd(), "causal-conv1d-mojo_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from causal_conv1d_b200 import norm, ssm

    return ssm, norm


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # A batch of eight prompts through the 2.7B-like block: what a prefill server or an
        # evaluation runs, with the final states that the decode steps go on from.
        dict(name="scan_prompts", op="scan", dtype="bf16", batch=8, seqlen=2048, heads=80, headdim=64, groups=1,
             dstate=128, packed=False, init=False, final=True),
        # One long document, prefilled in pieces: few independent rows, a long axis, a state to start from.
        dict(name="scan_document", op="scan", dtype="bf16", batch=1, seqlen=16384, heads=80, headdim=64, groups=1,
             dstate=128, packed=False, init=True, final=True),
        # Packed prefill of 32 prompts of different lengths, the largest call.
        dict(name="scan_packed", op="scan", dtype="fp16", batch=32, seqlen=65536, heads=60, headdim=64, groups=1,
             dstate=128, packed=True, init=False, final=True),
        # The next turn of four chats: a few tokens, an odd length, states from before.
        dict(name="scan_turn", op="scan", dtype="bf16", batch=4, seqlen=37, heads=80, headdim=64, groups=1,
             dstate=128, packed=False, init=True, final=True),
        # The small fp32 layer that a study or a unit test runs.
        dict(name="scan_fp32", op="scan", dtype="fp32", batch=2, seqlen=512, heads=4, headdim=16, groups=1,
             dstate=16, packed=False, init=False, final=True),
        # A decode step of a full serving batch on a pool of 512 states.
        dict(name="update_pool", op="update", dtype="bf16", state="fp32", batch=256, rows=512, heads=80, headdim=64,
             groups=1, dstate=128, idle=0),
        # A decode step of one user: latency.
        dict(name="update_one", op="update", dtype="bf16", state="fp32", batch=1, rows=2, heads=80, headdim=64,
             groups=1, dstate=128, idle=0),
        # An odd batch with two idle slots (index -1), several groups, states kept in 16 bits.
        dict(name="update_odd", op="update", dtype="fp16", state="fp16", batch=17, rows=40, heads=24, headdim=64,
             groups=4, dstate=64, idle=2),
        # The gated RMS norm of the same prefill, inference.
        dict(name="norm_prompts", op="norm", dtype="bf16", rows=16384, dim=5120, group=5120, kind="rms", gate=True,
             gate_first=True, bias=False, train=False),
        # The same in training: forward, then the gradients of input, gate and weight.
        dict(name="norm_train", op="norm", dtype="bf16", rows=16384, dim=5120, group=5120, kind="rms", gate=True,
             gate_first=True, bias=False, train=True),
        # A layer norm of odd sizes in fp32 with its bias, trained.
        dict(name="norm_layer", op="norm", dtype="fp32", rows=1000, dim=1001, group=1001, kind="layer", gate=False,
             gate_first=True, bias=True, train=True),
        # The gated norm of one token: latency.
        dict(name="norm_token", op="norm", dtype="bf16", rows=1, dim=5120, group=640, kind="rms", gate=True,
             gate_first=True, bias=False, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "update", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    groups = rng.choice([1, 1, 2, 4])
    heads = groups * _log(rng, 1, 80 // groups)
    headdim = rng.choice([16, 32, 64, 64, 64, 80, 128])
    dstate = rng.choice([16, 32, 64, 128, 128, 128, 96])
    if op == "scan":
        packed = rng.random() < 0.4
        most = 65536 * 60 * 64 * 128 // (heads * headdim * dstate)  # tokens that cost as much as the largest case
        if dtype == "fp32":
            most //= 8
        tokens = _log(rng, 1, max(1, min(65536, most)))
        batch = min(tokens, _log(rng, 1, 32)) if packed else _log(rng, 1, 8)
        seqlen = tokens if packed else max(1, tokens // batch)
        return dict(op=op, dtype=dtype, batch=batch, seqlen=seqlen, heads=heads, headdim=headdim, groups=groups,
                    dstate=dstate, packed=packed, init=rng.random() < 0.5, final=rng.random() < 0.7)
    if op == "update":
        batch = _log(rng, 1, min(256, 256 * 80 * 64 * 128 // (heads * headdim * dstate)))
        idle = rng.choice([0, 0, 1]) if batch > 1 else 0
        return dict(op=op, dtype=dtype, state=rng.choice(["fp32", dtype]), batch=batch, rows=2 * batch + rng.randint(0, 5),
                    heads=heads, headdim=headdim, groups=groups, dstate=dstate, idle=idle)
    parts = rng.choice([1, 1, 1, 2, 8])
    dim = parts * _log(rng, max(1, 32 // parts), 8192 // parts)
    rows = _log(rng, 1, max(1, min(65536, 16384 * 5120 // dim // (2 if dtype == "fp32" else 1))))
    gate = rng.random() < 0.6
    kind = rng.choice(["rms", "layer"])
    return dict(op=op, dtype=dtype, rows=rows, dim=dim, group=dim // parts, kind=kind, gate=gate,
                gate_first=rng.random() < 0.6, bias=kind == "layer" and parts == 1, train=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _silu(t):
    return t * torch.sigmoid(t)


def _heads(case, g):
    """Per-head parameters as such a block has them: decay rates in [1, 16], steps that start between 1e-3 and 1e-1."""
    H = case["heads"]
    A = -(1 + 15 * torch.rand(H, generator=g, device=DEV))
    step = torch.exp(math.log(1e-3) + torch.rand(H, generator=g, device=DEV) * math.log(100.0))
    dt_bias = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias) == step
    D = 1 + 0.1 * torch.randn(H, generator=g, device=DEV)
    return A, dt_bias, D


def _lengths(case, g):
    """Ragged lengths, at least one token each, that sum to the packed batch's tokens."""
    n, total = case["batch"], case["seqlen"]
    share = (0.1 + torch.rand(n, generator=g, device=DEV)).double()
    cut = torch.floor(torch.cumsum(share, 0) / share.sum() * (total - n)).long()
    cut[-1] = total - n
    cu = torch.zeros(n + 1, dtype=torch.int64, device=DEV)
    cu[1:] = cut + torch.arange(1, n + 1, device=DEV)
    return cu.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt_ = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"] == "scan":
        H, P, G, N = case["heads"], case["headdim"], case["groups"], case["dstate"]
        n, L = case["batch"], case["seqlen"]
        rows = 1 if case["packed"] else n
        A, dt_bias, D = _heads(case, g)
        # x, B and C are slices of the conv's output, as the block has them.
        xbc = _silu(randn(rows, L, H * P + 2 * G * N)).to(dt_)
        state = dict(
            op="scan", x=xbc[..., :H * P].unflatten(-1, (H, P)),
            B=xbc[..., H * P:H * P + G * N].unflatten(-1, (G, N)), C=xbc[..., H * P + G * N:].unflatten(-1, (G, N)),
            dt=(0.5 * randn(rows, L, H)).to(dt_), A=A, dt_bias=dt_bias, D=D, final=case["final"], cu=None, longest=None,
            init=0.3 * randn(n, H, P, N) if case["init"] else None)
        if case["packed"]:
            state["cu"] = _lengths(case, g)
            state["longest"] = int((state["cu"][1:] - state["cu"][:-1]).max())
        return state
    if case["op"] == "update":
        H, P, G, N = case["heads"], case["headdim"], case["groups"], case["dstate"]
        b, rows = case["batch"], case["rows"]
        A, dt_bias, D = _heads(case, g)
        xbc = _silu(randn(b, H * P + 2 * G * N)).to(dt_)
        order = torch.randperm(rows, generator=g, device=DEV).to(torch.int32)
        read, write = order[:b].clone(), order[b:2 * b].clone()
        if case["idle"]:
            read[torch.arange(case["idle"], device=DEV) * (b // case["idle"])] = -1
        return dict(
            op="update", x=xbc[:, :H * P].unflatten(-1, (H, P)), B=xbc[:, H * P:H * P + G * N].unflatten(-1, (G, N)),
            C=xbc[:, H * P + G * N:].unflatten(-1, (G, N)), dt=(0.5 * randn(b, H)).to(dt_), A=A, dt_bias=dt_bias, D=D,
            # The new states go to rows of their own (the old ones stay, as for a checkpoint to roll back to).
            pool=(0.3 * randn(rows, H, P, N)).to(DTYPES[case["state"]]), read=read, write=write)
    M, dim = case["rows"], case["dim"]
    state = dict(op="norm", x=randn(M, dim).to(dt_), weight=(1 + 0.1 * randn(dim)).to(dt_),
                 bias=(0.1 * randn(dim)).to(dt_) if case["bias"] else None,
                 z=randn(M, dim).to(dt_) if case["gate"] else None, group=case["group"], kind=case["kind"],
                 gate_first=case["gate_first"], train=case["train"], eps=1e-5)
    if case["train"]:
        state["dy"] = randn(M, dim).to(dt_)
        for k in ("x", "weight", "bias", "z"):
            if state[k] is not None:
                state[k].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _softplus(t):
    return torch.where(t > 20, t, torch.log1p(torch.exp(torch.clamp(t, max=20))))


def _plain_scan_rows(x, dt, A, B, C, D, init):
    """(b, l, h, p) and so on, all fp32, dt final: y and the last state, by blocks of CHUNK tokens."""
    b, l, H, P = x.shape
    G, N = B.shape[2:]
    R, Q = H // G, CHUNK
    nc = -(-l // Q)

    def blocks(t):
        return torch.cat([t, t.new_zeros(b, nc * Q - l, *t.shape[2:])], 1).unflatten(1, (nc, Q))

    xs, ds = blocks(x).unflatten(3, (G, R)), blocks(dt)
    Bs, Cs = blocks(B), blocks(C)
    cum = torch.cumsum(ds * A, 2)  # b c q h
    ds, cg = ds.unflatten(3, (G, R)), cum.unflatten(3, (G, R))
    ci = cg.permute(0, 1, 3, 4, 2)  # b c g r q
    gap = ci.unsqueeze(-1) - ci.unsqueeze(-2)
    lower = torch.ones(Q, Q, dtype=torch.bool, device=x.device).tril()
    mix = torch.exp(gap.masked_fill_(~lower, float("-inf")))
    mix *= torch.einsum("bcign,bcjgn->bcgij", Cs, Bs).unsqueeze(3)
    mix *= ds.permute(0, 1, 3, 4, 2).unsqueeze(-2)
    y = torch.einsum("bcgrij,bcjgrp->bcigrp", mix, xs)
    del mix, gap
    to_end = torch.exp(cg[:, :, -1:] - cg) * ds
    add = torch.einsum("bcjgn,bcjgrp->bcgrpn", Bs, xs * to_end.unsqueeze(-1)).flatten(2, 3)  # b c h p n
    first = x.new_zeros(b, 1, H, P, N) if init is None else init.unsqueeze(1)
    add = torch.cat([first, add], 1)
    total = torch.cat([cum.new_zeros(b, 1, H), torch.cumsum(cum[:, :, -1], 1)], 1).transpose(1, 2)  # b h c+1
    hop = total.unsqueeze(-1) - total.unsqueeze(-2)
    hop = torch.exp(hop.masked_fill_(~torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=x.device).tril(), float("-inf")))
    states = torch.einsum("bhcz,bzhpn->bchpn", hop, add)
    del add
    y += torch.einsum("bcign,bcgrpn->bcigrp", Cs, states[:, :-1].unflatten(2, (G, R))) * torch.exp(cg).unsqueeze(-1)
    y = y.flatten(3, 4).flatten(1, 2)[:, :l] + x * D[:, None]
    return y, states[:, -1]


def _plain_scan(s):
    x, dt, B, C = (s[k].float() for k in ("x", "dt", "B", "C"))
    dt = _softplus(dt + s["dt_bias"])
    if s["cu"] is None:
        y, last = _plain_scan_rows(x, dt, s["A"], B, C, s["D"], s["init"])
    else:  # each sequence in a row of its own, filled up with steps of length zero
        cu = s["cu"].long()
        at = cu[:-1, None] + torch.arange(s["longest"], device=cu.device)
        there = at < cu[1:, None]
        at = torch.where(there, at, 0)
        y, last = _plain_scan_rows(x[0][at], dt[0][at] * there.unsqueeze(-1), s["A"], B[0][at], C[0][at], s["D"], s["init"])
        y = y[there].unsqueeze(0)
    y = y.to(s["x"].dtype)
    return dict(y=y, final=last) if s["final"] else dict(y=y)


def _plain_update(s):
    x, dt, B, C = (s[k].float() for k in ("x", "dt", "B", "C"))
    R = x.shape[1] // B.shape[1]
    dt = _softplus(dt + s["dt_bias"])
    B, C = B.repeat_interleave(R, 1), C.repeat_interleave(R, 1)
    live = s["read"] >= 0
    old = s["pool"][s["read"].clamp(min=0).long()].float()
    new = old * torch.exp(dt * s["A"])[..., None, None] + (dt[..., None] * x)[..., None] * B[:, :, None, :]
    y = (new * C[:, :, None, :]).sum(-1) + x * s["D"][:, None]
    y = torch.where(live[:, None, None], y, 0.0)
    to = s["write"].long()
    s["pool"][to] = torch.where(live[:, None, None, None], new.to(s["pool"].dtype), s["pool"][to])
    return dict(y=y.to(s["x"].dtype), pool=s["pool"])


def _norm_parts(s, f):
    """Forward values in the arithmetic type that `f` casts to; (rows, parts, group) shapes."""
    shape = (s["x"].shape[0], -1, s["group"])
    x = f(s["x"].detach()).view(shape)
    w = f(s["weight"].detach()).view(shape[1:])
    z = None if s["z"] is None else f(s["z"].detach()).view(shape)
    u = x * _silu(z) if z is not None and s["gate_first"] else x
    mean = u.mean(-1, keepdim=True) if s["kind"] == "layer" else 0
    rstd = 1 / torch.sqrt(((u - mean) ** 2).mean(-1, keepdim=True) + s["eps"])
    hat = (u - mean) * rstd
    out = hat * w
    if s["bias"] is not None:
        out = out + f(s["bias"].detach()).view(shape[1:])
    y = out * _silu(z) if z is not None and not s["gate_first"] else out
    return x, w, z, rstd, hat, out, y


def _norm(s, f):
    """The gated norm, and with `train` the gradients of its inputs from the formulas."""
    x, w, z, rstd, hat, out, y = _norm_parts(s, f)
    if not s["train"]:
        return dict(y=y.flatten(1))
    dy = f(s["dy"]).view(y.shape)
    got = dict(y=y.flatten(1))
    if z is not None:
        sig = torch.sigmoid(z)
        dsilu = sig * (1 + z * (1 - sig))
        if not s["gate_first"]:
            got["dz"] = (dy * out * dsilu).flatten(1)
            dy = dy * z * sig
    got["dweight"] = (dy * hat).sum(0).flatten()
    if s["bias"] is not None:
        got["dbias"] = dy.sum(0).flatten()
    dh = dy * w
    back = dh - hat * (dh * hat).mean(-1, keepdim=True)
    if s["kind"] == "layer":
        back = back - dh.mean(-1, keepdim=True)
    du = back * rstd
    if z is not None and s["gate_first"]:
        got["dz"] = (du * x * dsilu).flatten(1)
        du = du * z * sig
    got["dx"] = du.flatten(1)
    return got


def _plain_norm(s):
    like = dict(y="x", dx="x", dz="z", dweight="weight", dbias="bias")
    return {k: v.to(s[like[k]].dtype) for k, v in _norm(s, torch.Tensor.float).items()}


# ---------------------------------------------------------------------------
# The library's operators
# ---------------------------------------------------------------------------

def _own_scan(s):
    ssm, _ = _product()
    out = ssm.state_space_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"], dt_softplus=True,
                               initial_states=s["init"], return_final_states=s["final"], cu_seqlens=s["cu"],
                               max_seqlen=s["longest"])
    return dict(y=out[0], final=out[1]) if s["final"] else dict(y=out)


def _own_update(s):
    ssm, _ = _product()
    y = ssm.state_space_update(s["x"], s["pool"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"],
                               dt_softplus=True, state_indices=s["read"], out_state_indices=s["write"])
    return dict(y=y, pool=s["pool"])


def _own_norm(s):
    _, norm = _product()
    y = norm.gated_norm_fn(s["x"], s["weight"], s["bias"], z=s["z"], eps=s["eps"], group_size=s["group"], kind=s["kind"],
                           gate_first=s["gate_first"])
    if not s["train"]:
        return dict(y=y)
    names = [k for k in ("x", "weight", "bias", "z") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return dict(y=y.detach(), **{"d" + k: v for k, v in zip(names, grads)})


def run(state):
    if own:
        return {"scan": _own_scan, "update": _own_update, "norm": _own_norm}[state["op"]](state)
    with torch.no_grad():
        return {"scan": _plain_scan, "update": _plain_update, "norm": _plain_norm}[state["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its exact results
# ---------------------------------------------------------------------------

def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    e = size[case["dtype"]]
    if case["op"] == "scan":
        H, P, G, N, n = case["heads"], case["headdim"], case["groups"], case["dstate"], case["batch"]
        tokens = case["seqlen"] * (1 if case["packed"] else n)
        data = tokens * (2 * H * P + 2 * G * N + H) * e
        states = n * H * P * N * 4 * (int(case["init"]) + int(case["final"]))
        # Per token, head and state element: decay, add the outer product, read out.
        return dict(bytes=data + states + 12 * H, flops=5.0 * tokens * H * P * N)
    if case["op"] == "update":
        H, P, G, N, b = case["heads"], case["headdim"], case["groups"], case["dstate"], case["batch"]
        live = b - case["idle"]
        return dict(bytes=live * H * P * N * size[case["state"]] * 2 + b * (2 * H * P + 2 * G * N + H) * e + 12 * H + 8 * b,
                    flops=5.0 * live * H * P * N)
    cells = case["rows"] * case["dim"]
    arrays = 2 + int(case["gate"])
    flops = 8 + 6 * int(case["gate"])
    if case["train"]:  # x and the gate are needed again, and dy; dx and dz are written
        arrays += 3 + 2 * int(case["gate"])
        flops *= 3
    return dict(bytes=cells * arrays * e + case["dim"] * e * (2 if case["bias"] else 1) * (2 if case["train"] else 1),
                flops=float(flops * cells))


def _exact_scan(s):
    """The recurrence, token by token, in 64 bits."""
    A, D, bias = (s[k].double() for k in ("A", "D", "dt_bias"))
    x, B, C = s["x"], s["B"], s["C"]
    dt = torch.nn.functional.softplus(s["dt"].double() + bias, threshold=50)
    H, P = x.shape[2:]
    G, N = B.shape[2:]
    if s["cu"] is None:
        begin = torch.arange(x.shape[0], device=x.device) * x.shape[1]
        end = begin + x.shape[1]
    else:
        begin, end = s["cu"][:-1].long(), s["cu"][1:].long()
    x, B, C, dt = x.flatten(0, 1), B.flatten(0, 1), C.flatten(0, 1), dt.flatten(0, 1)
    y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    n = len(begin)
    S = torch.zeros(n, H, P, N, dtype=torch.float64, device=x.device) if s["init"] is None else s["init"].double()
    for t in range(int((end - begin).max())):
        seqs = torch.nonzero(begin + t < end)[:, 0] if s["cu"] is not None else slice(None)
        at = (begin + t)[seqs]
        step = dt[at]
        xt = x[at].double()
        Bt, Ct = (v[at].double().repeat_interleave(H // G, 1) for v in (B, C))
        new = S[seqs] if s["cu"] is not None else S
        new = new * torch.exp(step * A)[..., None, None]
        new += (step[..., None] * xt)[..., None] * Bt[:, :, None]
        y[at] = torch.matmul(new, Ct[..., None])[..., 0] + D[:, None] * xt
        if s["cu"] is not None:
            S[seqs] = new
        else:
            S = new
    y = y.view(s["x"].shape)
    return dict(y=y, final=S) if s["final"] else dict(y=y)


def _exact_update(s):
    """One step per live slot, in 64 bits; rows that no slot writes stay as they are."""
    pool = s["pool"].double()
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device=pool.device)
    A, D, bias = (s[k].double() for k in ("A", "D", "dt_bias"))
    R = s["x"].shape[1] // s["B"].shape[1]
    old = pool.clone()
    for i, (r, w) in enumerate(zip(s["read"].tolist(), s["write"].tolist())):
        if r < 0:
            continue
        step = torch.nn.functional.softplus(s["dt"][i].double() + bias, threshold=50)
        xi = s["x"][i].double()
        Bi, Ci = (s[k][i].double().repeat_interleave(R, 0) for k in ("B", "C"))
        S = old[r] * torch.exp(step * A)[:, None, None] + torch.einsum("h,hp,hn->hpn", step, xi, Bi)
        y[i] = torch.einsum("hpn,hn->hp", S, Ci) + D[:, None] * xi
        pool[w] = S
    return dict(y=y, pool=pool)


def _exact_norm(s):
    """The definition in 64 bits, its gradients by automatic differentiation."""
    leaf = {k: s[k].detach().double().requires_grad_(s["train"]) for k in ("x", "weight", "bias", "z") if s[k] is not None}
    x = leaf["x"]
    u = x * torch.nn.functional.silu(leaf["z"]) if "z" in leaf and s["gate_first"] else x
    v = u.unflatten(-1, (-1, s["group"]))
    if s["kind"] == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + s["eps"])
    y = v.flatten(-2) * leaf["weight"]
    if "bias" in leaf:
        y = y + leaf["bias"]
    if "z" in leaf and not s["gate_first"]:
        y = y * torch.nn.functional.silu(leaf["z"])
    if not s["train"]:
        return dict(y=y)
    grads = torch.autograd.grad(y, list(leaf.values()), s["dy"].double())
    return dict(y=y.detach(), **{"d" + k: v for k, v in zip(leaf, grads)})


def exact(case, seed):
    if case["op"] == "scan" and not case["packed"] and case["seqlen"] > 40000:
        return None
    s = prepare(case, seed)
    if s["op"] == "scan":
        with torch.no_grad():
            return _exact_scan(s)
    if s["op"] == "update":
        return _exact_update(s)
    return _exact_norm(s)
