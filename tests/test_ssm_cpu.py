"""Refusals of the state space and norm entry points, and their C ABI, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from _ssm_util import scan_inputs, scan_reference
from causal_conv1d_b200 import _lib
from causal_conv1d_b200.norm import gated_norm_fn
from causal_conv1d_b200.ssm import state_space_scan, state_space_update


def _scan(**change):
    v = scan_inputs(2, 6, 4, 8, 2, 16, torch.float32, device="cpu")
    v.update(change)
    return state_space_scan(**v)


def _token(**change):
    v = {k: (t[:, 0] if k in ("x", "dt", "B", "C") else t)
         for k, t in scan_inputs(2, 1, 4, 8, 2, 16, torch.float32, device="cpu").items()}
    v["state"] = torch.zeros(2, 4, 8, 16)
    v.update(change)
    return state_space_update(**v)


@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(2, 6, 32)), ValueError, "x must be"),
    (dict(x=torch.zeros(2, 6, 4, 8, dtype=torch.float64)), NotImplementedError, "unsupported dtype"),
    (dict(x=torch.zeros(2, 6, 4, 8, dtype=torch.bfloat16)), NotImplementedError, "B.dtype"),
    (dict(dt=torch.zeros(2, 6, 4, dtype=torch.bfloat16)), NotImplementedError, "dt.dtype"),
    (dict(A=torch.zeros(4, dtype=torch.float64)), NotImplementedError, "A must be float32"),
    (dict(A=torch.zeros(3)), ValueError, r"A must be \(4,\)"),
    (dict(D=torch.zeros(4, 8)), ValueError, "D must be"),
    (dict(dt=torch.zeros(2, 5, 4)), ValueError, "dt must be"),
    (dict(C=torch.zeros(2, 6, 2, 8)), ValueError, "B and C must be"),
    (dict(B=torch.zeros(2, 6, 3, 16), C=torch.zeros(2, 6, 3, 16)), ValueError, "multiple of ngroups"),
    (dict(B=torch.zeros(2, 6, 1, 257), C=torch.zeros(2, 6, 1, 257)), NotImplementedError, "dstate must be at most"),
    (dict(initial_states=torch.zeros(1, 4, 8, 16)), ValueError, "initial_states must be"),
    (dict(initial_states=torch.zeros(2, 4, 8, 16, dtype=torch.float16)), NotImplementedError, "initial_states.dtype"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError, "batch == 1"),
    (dict(max_seqlen=-1), ValueError, "max_seqlen"),
    (dict(x=torch.zeros(2, 6, 4, 8, requires_grad=True)), NotImplementedError, "forward only"),
])
def test_scan_refuses(change, error, match):
    with pytest.raises(error, match=match):
        _scan(**change)


def test_scan_refuses_bad_sequence_tables():
    v = scan_inputs(1, 6, 4, 8, 2, 16, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="int32"):
        state_space_scan(**v, cu_seqlens=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="num_seqs"):
        state_space_scan(**v, cu_seqlens=torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="initial_states must be"):
        state_space_scan(**v, cu_seqlens=torch.zeros(3, dtype=torch.int32), initial_states=torch.zeros(1, 4, 8, 16))


@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(2, 32)), ValueError, "x must be"),
    (dict(state=torch.zeros(3, 4, 8, 16)), ValueError, "state shape"),
    (dict(state=torch.zeros(2, 4, 8, 15)), ValueError, "state shape"),
    (dict(state=torch.zeros(2, 4, 16, 8).transpose(2, 3)), ValueError, "unit stride"),
    (dict(state=torch.zeros(2, 4, 8, 16, dtype=torch.bfloat16)), NotImplementedError, "state.dtype"),
    (dict(state_indices=torch.zeros(2, dtype=torch.int64)), ValueError, "state_indices.dtype"),
    (dict(state_indices=torch.zeros(3, dtype=torch.int32)), ValueError, "state_indices shape"),
    (dict(out_state_indices=torch.zeros(2, dtype=torch.int64)), ValueError, "out_state_indices.dtype"),
    (dict(dt=torch.zeros(2, 3)), ValueError, "dt must be"),
    (dict(dt_bias=torch.zeros(5)), ValueError, "dt_bias must be"),
    (dict(x=torch.zeros(2, 4, 8, requires_grad=True)), NotImplementedError, "forward only"),
])
def test_update_refuses(change, error, match):
    with pytest.raises(error, match=match):
        _token(**change)


@pytest.mark.parametrize("kw,error,match", [
    (dict(kind="batch"), NotImplementedError, "kind must be"),
    (dict(x=torch.zeros(3, 8, dtype=torch.float64)), NotImplementedError, "unsupported dtype"),
    (dict(weight=torch.zeros(7)), ValueError, r"must be \(8,\)"),
    (dict(weight=torch.zeros(8, dtype=torch.float16)), NotImplementedError, "weight.dtype"),
    (dict(bias=torch.zeros(8, dtype=torch.float16)), NotImplementedError, "bias.dtype"),
    (dict(z=torch.zeros(3, 4)), ValueError, "z shape"),
    (dict(z=torch.zeros(3, 8, dtype=torch.bfloat16)), NotImplementedError, "z.dtype"),
    (dict(group_size=3), ValueError, "multiple of group_size"),
    (dict(group_size=0), ValueError, "multiple of group_size"),
])
def test_norm_refuses(kw, error, match):
    v = dict(x=torch.zeros(3, 8), weight=torch.ones(8))
    v.update(kw)
    with pytest.raises(error, match=match):
        gated_norm_fn(**v)


def test_no_cpu_fallback():
    with torch.no_grad():
        for call in (_scan, _token, lambda: gated_norm_fn(torch.zeros(3, 8), torch.ones(8))):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call()


def test_c_entries_refuse_without_gpu():
    lib = _lib.load()
    n = ctypes.c_size_t(7)
    for fn in (lib.cc1d_scan, lib.cc1d_scan_update, lib.cc1d_gated_norm_fwd, lib.cc1d_gated_norm_bwd):
        assert fn(None, None) == _lib.CC1D_ERR_INVALID_ARGUMENT
        assert b"NULL" in lib.cc1d_last_error()
    p = _lib.ScanParams()
    p.dtype = p.dt_dtype = p.init_dtype = 1
    p.batch, p.seqlen, p.nheads, p.headdim, p.ngroups, p.dstate = 1, 8, 4, 64, 3, 128
    assert lib.cc1d_scan(ctypes.byref(p), None) == _lib.CC1D_ERR_INVALID_ARGUMENT
    assert b"multiple of ngroups" in lib.cc1d_last_error()
    p.ngroups, p.dstate = 2, 300
    assert lib.cc1d_scan(ctypes.byref(p), None) == _lib.CC1D_ERR_UNSUPPORTED
    p.dstate, p.dt_dtype = 128, 0
    assert lib.cc1d_scan(ctypes.byref(p), None) == _lib.CC1D_ERR_UNSUPPORTED
    p.dt_dtype = 2
    assert lib.cc1d_scan(ctypes.byref(p), None) == _lib.CC1D_ERR_INVALID_ARGUMENT  # no tensors
    p.batch = 0
    assert lib.cc1d_scan(ctypes.byref(p), None) == _lib.CC1D_OK
    assert lib.cc1d_scan_workspace_size(ctypes.byref(p), ctypes.byref(n)) == _lib.CC1D_OK and n.value == 0
    u = _lib.ScanUpdateParams()
    u.dtype = u.dt_dtype = u.state_dtype = 2
    u.batch, u.nheads, u.headdim, u.ngroups, u.dstate = -1, 2, 8, 1, 16
    assert lib.cc1d_scan_update(ctypes.byref(u), None) == _lib.CC1D_ERR_INVALID_ARGUMENT
    u.batch = 0
    assert lib.cc1d_scan_update(ctypes.byref(u), None) == _lib.CC1D_OK
    q = _lib.GatedNormParams()
    q.dtype = q.weight_dtype = 1
    q.rows, q.dim, q.group_size = 4, 8, 3
    assert lib.cc1d_gated_norm_fwd(ctypes.byref(q), None) == _lib.CC1D_ERR_INVALID_ARGUMENT
    assert b"group_size" in lib.cc1d_last_error()
    q.rows = 0
    assert lib.cc1d_gated_norm_fwd(ctypes.byref(q), None) == _lib.CC1D_OK


def test_new_struct_layouts_match_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"cc1d_scan_params": _lib.ScanParams, "cc1d_scan_update_params": _lib.ScanUpdateParams,
               "cc1d_gated_norm_params": _lib.GatedNormParams}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "cc1d.h"', "int main(void) {"]
    for c, cls in structs.items():
        lines.append(f'  printf("{c} sizeof %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run([cc, f"-I{Path(__file__).resolve().parent.parent / 'include'}", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        c, f, v = line.split()
        want = ctypes.sizeof(structs[c]) if f == "sizeof" else getattr(structs[c], f).offset
        assert int(v) == want, (c, f)


def test_reference_of_the_tests_on_a_case_by_hand():
    """One head, one state value: S_t = S_{t-1} / 2 + x_t, y_t = 3 S_t."""
    one = torch.ones(1, 3, 1, 1)
    x = torch.tensor([1.0, 2.0, 4.0]).view(1, 3, 1, 1)
    y, S, _, _ = scan_reference(x, torch.ones(1, 3, 1), torch.tensor([-0.6931471805599453]), one, 3 * one, dt_softplus=False)
    assert torch.allclose(y.flatten(), torch.tensor([3.0, 7.5, 15.75], dtype=torch.float64), rtol=1e-7)
    assert torch.allclose(S.flatten(), torch.tensor([5.25], dtype=torch.float64), rtol=1e-7)
