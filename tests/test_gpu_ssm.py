"""The state space scan and its single-token step against the recurrence in 64 bits
(bounds: tests/_ssm_util.py)."""

from __future__ import annotations

import pytest
import torch

from _ssm_util import UNIT, check_scan, scan_inputs, scan_reference
from causal_conv1d_b200.ssm import state_space_scan, state_space_update

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def _init(n, H, P, N, dtype=F32, seed=9):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (0.3 * torch.randn(n, H, P, N, generator=g, device=DEV)).to(dtype)


@pytest.mark.parametrize("dtype", [BF, FP16, F32])
@pytest.mark.parametrize("B,L,H,P,G,N,init", [
    (1, 1, 2, 64, 1, 128, True),      # one token
    (2, 2, 3, 64, 1, 128, False),     # an odd number of heads
    (1, 127, 2, 64, 1, 128, True),    # around a block of 128 tokens
    (1, 128, 2, 64, 1, 128, True),
    (1, 129, 2, 64, 1, 128, False),
    (2, 300, 6, 64, 2, 128, True),    # odd heads per group
    (1, 700, 4, 64, 4, 128, True),    # one head per group
    (2, 260, 3, 128, 1, 128, True),   # wide heads
    (1, 200, 4, 80, 2, 96, True),     # sizes between the tiles
    (2, 150, 5, 32, 5, 64, True),
    (1, 140, 4, 16, 1, 16, False),
    (1, 133, 2, 8, 1, 8, True),
    (1, 70, 2, 7, 1, 5, True),        # odd sizes
    (1, 70, 1, 64, 1, 256, True),     # the largest state
    (1, 40, 2, 200, 1, 130, True),
    (3, 20, 2, 1, 1, 1, True),
])
def test_scan_matches_recurrence(dtype, B, L, H, P, G, N, init):
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=L + H)
    s0 = _init(B, H, P, N) if init else None
    y, fs = state_space_scan(**v, dt_softplus=True, initial_states=s0, return_final_states=True)
    assert y.dtype == dtype and y.shape == v["x"].shape and y.is_contiguous()
    ref = scan_reference(**v, initial_states=s0)
    check_scan(y, fs, ref, dtype, L, N, v["x"], v["C"])
    # Without the final states: the same y, within the same bound.
    y2 = state_space_scan(**v, dt_softplus=True, initial_states=s0)
    check_scan(y2, None, ref, dtype, L, N, v["x"], v["C"])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_optional_inputs_and_types(dtype):
    """No D, no bias, no softplus; dt in fp32; states in the data's type."""
    B, L, H, P, G, N = 2, 150, 4, 64, 1, 128
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=5)
    dt = torch.rand(B, L, H, device=DEV) * 0.1
    s0 = _init(B, H, P, N, dtype)
    y, fs = state_space_scan(v["x"], dt, v["A"], v["B"], v["C"], initial_states=s0, return_final_states=True)
    ref = scan_reference(v["x"], dt, v["A"], v["B"], v["C"], dt_softplus=False, initial_states=s0)
    check_scan(y, fs, ref, dtype, L, N, v["x"], v["C"])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["contiguous", "odd_offset", "transposed", "head_major"])
def test_scan_layouts(dtype, layout):
    B, L, H, P, G, N = 2, 140, 4, 64, 2, 64
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=3, sliced=False)
    ref = scan_reference(**v)
    if layout == "odd_offset":  # not aligned to 16 bytes
        for k in "xBC":
            t = v[k]
            wide = torch.zeros(*t.shape[:2], t.shape[2] * t.shape[3] + 3, dtype=t.dtype, device=DEV)
            wide[..., 1:-2] = t.flatten(2)
            v[k] = wide[..., 1:-2].unflatten(-1, t.shape[2:])
    elif layout == "transposed":  # the token axis has unit stride
        for k in "xBC":
            v[k] = v[k].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
        v["dt"] = v["dt"].transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "head_major":
        for k in "xBC":
            v[k] = v[k].transpose(1, 2).contiguous().transpose(1, 2)
    y, fs = state_space_scan(**v, dt_softplus=True, return_final_states=True)
    check_scan(y, fs, ref, dtype, L, N, v["x"], v["C"])


@pytest.mark.parametrize("dtype", [BF, FP16, F32])
@pytest.mark.parametrize("lens,lead,tail,known", [
    ([5, 0, 130, 1, 256, 0], 0, 0, True),   # empty sequences, one token, whole blocks
    ([0, 0], 4, 0, False),                  # nothing but empty ones
    ([300, 17, 128], 3, 9, False),          # tokens outside every sequence
    ([1] * 40, 0, 0, True),                 # more sequences than a warp counts at once
    ([900], 0, 5, True),
])
def test_scan_packed(dtype, lens, lead, tail, known):
    H, P, G, N = 4, 64, 2, 128
    total = lead + sum(lens) + tail
    v = scan_inputs(1, total, H, P, G, N, dtype, seed=total)
    cu = torch.tensor([lead] + [lead + sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device=DEV)
    ranges = [(0, int(a), int(b)) for a, b in zip(cu[:-1], cu[1:])]
    s0 = _init(len(lens), H, P, N)
    ref = scan_reference(**v, initial_states=s0, ranges=ranges)
    y, fs = state_space_scan(**v, dt_softplus=True, initial_states=s0, return_final_states=True, cu_seqlens=cu,
                             max_seqlen=max(lens) if known else None)
    check_scan(y, fs, ref, dtype, max(lens), N, v["x"], v["C"])
    for i, n in enumerate(lens):
        if n == 0:
            assert torch.equal(fs[i], s0[i])
    inside = torch.zeros(total, dtype=torch.bool)
    inside[lead:lead + sum(lens)] = True
    assert (y[0][~inside.to(DEV)] == 0).all()


@pytest.mark.parametrize("dtype", [BF, FP16, F32])
def test_scan_nan_stays_in_its_sequence(dtype):
    """Inf and NaN in one packed sequence, and in tokens outside all, reach no other sequence."""
    lens, lead = [70, 100, 50], 6
    H, P, G, N = 2, 64, 1, 128
    total = lead + sum(lens) + 7
    v = scan_inputs(1, total, H, P, G, N, dtype, seed=8)
    cu = torch.tensor([lead, lead + 70, lead + 170, lead + 220], dtype=torch.int32, device=DEV)
    want, wantf = state_space_scan(**v, dt_softplus=True, cu_seqlens=cu, return_final_states=True)
    bad = {k: t.clone() for k, t in v.items()}
    for k, val in (("x", float("nan")), ("B", float("inf")), ("C", float("nan")), ("dt", float("nan"))):
        bad[k][0, :lead] = val
        bad[k][0, lead + 70:lead + 170] = val
        bad[k][0, lead + 220:] = val
    y, fs = state_space_scan(**bad, dt_softplus=True, cu_seqlens=cu, return_final_states=True)
    for s in (slice(lead, lead + 70), slice(lead + 170, lead + 220)):
        assert torch.equal(y[0, s], want[0, s])
    assert torch.equal(fs[0], wantf[0]) and torch.equal(fs[2], wantf[2])
    assert torch.isnan(y[0, lead + 70:lead + 170]).all()
    assert (y[0, :lead] == 0).all() and (y[0, lead + 220:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_masked_steps(dtype):
    """dt = -inf (or the type's lowest value) with softplus is a step of length zero: the state passes unchanged."""
    B, L, H, P, G, N = 1, 200, 2, 64, 1, 128
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=2)
    v["dt"][:, 30:90] = float("-inf")
    v["dt"][:, 150:] = torch.finfo(dtype).min
    s0 = _init(B, H, P, N)
    y, fs = state_space_scan(**v, dt_softplus=True, initial_states=s0, return_final_states=True)
    check_scan(y, fs, scan_reference(**v, initial_states=s0), dtype, L, N, v["x"], v["C"])
    v["dt"][:] = float("-inf")
    _, fs = state_space_scan(**v, dt_softplus=True, initial_states=s0, return_final_states=True)
    assert torch.equal(fs, s0)


@pytest.mark.parametrize("dtype", [BF, FP16, F32])
def test_scan_strong_decay(dtype):
    """Steps long enough that a state is forgotten within a few tokens, and steps that forget nothing."""
    B, L, H, P, G, N = 1, 300, 4, 64, 1, 64
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=4, step=(1.0, 4.0))
    y, fs = state_space_scan(**v, dt_softplus=True, return_final_states=True)
    check_scan(y, fs, scan_reference(**v), dtype, L, N, v["x"], v["C"])
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=4, step=(1e-6, 1e-5))
    y, fs = state_space_scan(**v, dt_softplus=True, return_final_states=True)
    check_scan(y, fs, scan_reference(**v), dtype, L, N, v["x"], v["C"])


@pytest.mark.parametrize("dtype,L,H", [(BF, 5000, 2), (FP16, 3001, 3), (F32, 2500, 2)])
def test_scan_long_rows_are_split_and_joined(dtype, L, H):
    """Few rows and a long axis: the sequence is worked on in parallel pieces."""
    v = scan_inputs(1, L, H, 64, 1, 128, dtype, seed=6)
    s0 = _init(1, H, 64, 128)
    y, fs = state_space_scan(**v, dt_softplus=True, initial_states=s0, return_final_states=True)
    check_scan(y, fs, scan_reference(**v, initial_states=s0), dtype, L, 128, v["x"], v["C"])
    cu = torch.tensor([0, L - 1100, L - 1099, L], dtype=torch.int32, device=DEV)
    ranges = [(0, 0, L - 1100), (0, L - 1100, L - 1099), (0, L - 1099, L)]
    s3 = _init(3, H, 64, 128)
    y, fs = state_space_scan(**v, dt_softplus=True, initial_states=s3, return_final_states=True, cu_seqlens=cu)
    check_scan(y, fs, scan_reference(**v, initial_states=s3, ranges=ranges), dtype, L, 128, v["x"], v["C"])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_offsets_past_32_bits(dtype):
    """Token strides that carry the last rows past 2^31 elements."""
    L, H, P, N = 9, 2, 64, 128
    v = scan_inputs(1, L, H, P, 1, N, dtype, seed=1)
    pitch = (2 ** 31 // (L - 2) + 64) // 64 * 64
    big = torch.empty(pitch * (L - 1) + H * P, dtype=dtype, device=DEV)
    far = big.as_strided((1, L, H, P), (pitch * L, pitch, P, 1))
    far.copy_(v["x"])
    want, wf = state_space_scan(**v, dt_softplus=True, return_final_states=True)
    got, gf = state_space_scan(**{**v, "x": far}, dt_softplus=True, return_final_states=True)
    assert torch.equal(got, want) and torch.equal(gf, wf)


def test_scan_empty_calls():
    v = scan_inputs(2, 0, 2, 64, 1, 128, BF)
    s0 = _init(2, 2, 64, 128)
    y, fs = state_space_scan(**v, dt_softplus=True, initial_states=s0, return_final_states=True)
    assert y.shape == (2, 0, 2, 64) and torch.equal(fs, s0)
    _, fs = state_space_scan(**v, return_final_states=True)
    assert (fs == 0).all()
    v = scan_inputs(0, 5, 2, 64, 1, 128, BF)
    y, fs = state_space_scan(**v, return_final_states=True)
    assert y.shape == (0, 5, 2, 64) and fs.shape == (0, 2, 64, 128)
    v = scan_inputs(1, 5, 2, 64, 1, 128, BF)
    y, fs = state_space_scan(**v, return_final_states=True, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=DEV))
    assert (y == 0).all() and fs.shape == (0, 2, 64, 128)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_repeats_bitwise_on_any_stream_and_in_graphs(dtype):
    v = scan_inputs(2, 400, 6, 64, 2, 128, dtype, seed=12)
    kw = dict(dt_softplus=True, return_final_states=True)
    y, fs = state_space_scan(**v, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, fs2 = state_space_scan(**v, **kw)
    side.synchronize()
    assert torch.equal(y, y2) and torch.equal(fs, fs2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y3, fs3 = state_space_scan(**v, **kw)
    y3.zero_()
    fs3.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y3) and torch.equal(fs, fs3)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_then_tokens_is_one_scan(dtype):
    """A prompt in two pieces, the second token by token from the first one's state."""
    B, L, cut, H, P, G, N = 2, 150, 141, 4, 64, 2, 128
    v = scan_inputs(B, L, H, P, G, N, dtype, seed=7)
    ref = scan_reference(**v)
    per = ("x", "dt", "B", "C")
    head = {k: (t[:, :cut] if k in per else t) for k, t in v.items()}
    y, state = state_space_scan(**head, dt_softplus=True, return_final_states=True)
    ys = [y]
    for t in range(cut, L):
        tok = {k: (u[:, t] if k in per else u) for k, u in v.items()}
        ys.append(state_space_update(state=state, **tok, dt_softplus=True).unsqueeze(1))
    check_scan(torch.cat(ys, 1), state, ref, dtype, L, N, v["x"], v["C"])


# ---- single tokens ----

def _update_reference(v, state, read, write):
    """Per batch row in 64 bits; y's bound needs the terms' magnitudes."""
    H = v["x"].shape[1]
    R = H // v["B"].shape[1]
    step = torch.nn.functional.softplus(v["dt"].double() + v["dt_bias"].double(), threshold=50)
    x = v["x"].double()
    B, C = (v[k].double().repeat_interleave(R, 1) for k in "BC")
    old, new = state.double(), state.double()
    y, my = torch.zeros_like(x), torch.zeros_like(x)
    mag = new.abs()
    for i in range(x.shape[0]):
        r = read[i] if read is not None else i
        if not 0 <= r < state.shape[0]:
            continue
        dec = torch.exp(step[i] * v["A"].double())[:, None, None]
        add = (step[i][:, None] * x[i])[:, :, None] * B[i][:, None]
        S, m = old[r] * dec + add, old[r].abs() * dec + add.abs()
        y[i] = (S * C[i][:, None]).sum(-1) + v["D"].double()[:, None] * x[i]
        my[i] = (m * C[i].abs()[:, None]).sum(-1) + (v["D"].double()[:, None] * x[i]).abs()
        w = write[i] if write is not None else r
        if 0 <= w < state.shape[0]:
            new[w] = S
            mag[w] = m
    return y, new, my, mag


@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (BF, BF), (FP16, F32), (FP16, FP16), (F32, F32)])
@pytest.mark.parametrize("b,H,P,G,N,mode", [
    (1, 2, 64, 1, 128, "rows"),
    (5, 4, 64, 2, 128, "pool"),
    (300, 6, 64, 1, 128, "pool"),
    (3, 3, 80, 3, 96, "copy"),
    (4, 4, 16, 1, 16, "copy"),
    (2, 2, 7, 1, 5, "pool"),
    (2, 1, 33, 1, 256, "rows"),
    (6, 2, 64, 1, 64, "strided"),
    (40, 24, 64, 4, 64, "idle"),
])
def test_update_matches_recurrence(dtype, sdtype, b, H, P, G, N, mode):
    g = torch.Generator(device=DEV).manual_seed(b + P)
    v = {k: (t[:, 0] if k in ("x", "dt", "B", "C") else t) for k, t in scan_inputs(b, 1, H, P, G, N, dtype, seed=b).items()}
    rows = b if mode == "rows" else 2 * b + 3
    state = (0.3 * torch.randn(rows, H, P, N, generator=g, device=DEV)).to(sdtype)
    if mode == "strided":  # a pool with a row pitch of its own and padded state rows
        wide = torch.zeros(rows, H, P + 1, N + 3, dtype=sdtype, device=DEV)
        wide[:, :, :P, :N] = state
        state = wide[:, :, :P, :N]
    read = write = None
    if mode != "rows":
        order = torch.randperm(rows, generator=g, device=DEV).to(torch.int32)
        read = order[:b].clone()
        if mode == "copy":
            write = order[b:2 * b].clone()
            write[0] = -1
        if mode == "idle":
            read[::3] = -1
            read[1] = rows
    before = state.clone()
    y = state_space_update(state=state, **v, dt_softplus=True, state_indices=read, out_state_indices=write)
    to_list = lambda t: None if t is None else t.tolist()  # noqa: E731
    ry, rs, my, ms = _update_reference(v, before, to_list(read), to_list(write))
    e, u, us = 2.0 ** -24, UNIT[dtype], UNIT[sdtype]
    c = (N + 24) * e
    assert not ((y.double() - ry).abs() > c * my + u * ry.abs() * (1 + u) + 2.0 ** -25).any()
    tol = c * ms + (us * rs.abs() * (1 + us) + 2.0 ** -25 if sdtype != F32 else 0)
    assert not ((state.double() - rs).abs() > tol).any()
    # Rows that nothing wrote keep their bits.
    written = set((write if write is not None else read).tolist()) if read is not None else set(range(b))
    if mode == "idle":
        assert (y[::3] == 0).all() and (y[1] == 0).all()
    for r in range(rows):
        if r not in written:
            assert torch.equal(state[r], before[r])


def test_update_on_another_stream_and_in_a_graph():
    v = {k: (t[:, 0] if k in ("x", "dt", "B", "C") else t) for k, t in scan_inputs(8, 1, 4, 64, 1, 128, BF, seed=3).items()}
    start = _init(8, 4, 64, 128)
    s1, s2, s3 = start.clone(), start.clone(), start.clone()
    y1 = state_space_update(state=s1, **v, dt_softplus=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = state_space_update(state=s2, **v, dt_softplus=True)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y3 = state_space_update(state=s3, **v, dt_softplus=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y1, y2) and torch.equal(s1, s2)
    assert torch.equal(y1, y3) and torch.equal(s1, s3)


def test_scan_and_update_compile():
    v = scan_inputs(1, 20, 2, 64, 1, 128, BF, seed=1)
    want, wf = state_space_scan(**v, dt_softplus=True, return_final_states=True)
    fn = torch.compile(lambda kw: state_space_scan(**kw, dt_softplus=True, return_final_states=True), fullgraph=True,
                       backend="eager")
    got, gf = fn(v)
    assert torch.equal(got, want) and torch.equal(gf, wf)
