"""The example block: a prompt continued token by token, and packed prompts, against one prompt.

The three ways differ in where bf16 roundings of intermediate values fall (the conv's output and
the scan's y are the same values, rounded alike, but the library GEMM of one token or of a packed
row may sum in another order, which moves a bf16 value by one unit, 2^-8 relative, here and
there).  An output is a sum over the inner size of such values, so relative to its norm it moves
by a few times 2^-9 at most; 2^-6 leaves room, and a wrong state or a mixed-up head gives
differences near 1.
"""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "state_space_block.py"
    spec = importlib.util.spec_from_file_location("state_space_block", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("sizes", [dict(), dict(hidden=256, heads=6, headdim=32, groups=2, dstate=64, width=3)])
def test_prompt_tokens_and_packed_agree(example, sizes):
    got = example.main(**sizes)
    assert _rel(got["stepped"], got["whole"]) < 2 ** -6
    assert _rel(got["packed"], got["whole"]) < 2 ** -6
    assert _rel(got["state"], got["last"]) < 2 ** -6
    assert _rel(got["packed_last"], got["last"]) < 2 ** -6


def test_step_on_pool_slots(example):
    """Rows of a larger cache, with an idle slot."""
    block = example.Block(hidden=256, heads=4, headdim=64, groups=1, dstate=128)
    with torch.no_grad():
        hidden = torch.randn(3, 40, 256, device="cuda").bfloat16()
        _, conv, state = block.prompt(hidden)
        pool_conv, pool = torch.zeros(8, *conv.shape[1:], dtype=conv.dtype, device="cuda"), torch.zeros(8, *state.shape[1:], device="cuda")
        rows = torch.tensor([6, 1, 3], dtype=torch.int32, device="cuda")
        pool_conv[rows.long()], pool[rows.long()] = conv, state
        token = torch.randn(4, 256, device="cuda").bfloat16()
        slots = torch.cat([rows, torch.tensor([-1], dtype=torch.int32, device="cuda")])
        got = block.step(token, pool_conv, pool, slots)
        want = block.step(token[:3], conv, state)
    assert _rel(got[:3], want) < 2 ** -6
    assert torch.isfinite(got).all()
    assert _rel(pool[rows.long()], state) < 2 ** -6
    assert (pool[[0, 2, 4, 5, 7]] == 0).all()
