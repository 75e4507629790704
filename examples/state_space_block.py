"""A Mamba-2 style block on this library: prompts, packed prompts, then token by token.

    hidden -> in_proj -> [z | x B C | dt];  x, B, C <- conv + SiLU;  y <- state space scan;
    y <- RMS norm of y * silu(z);  out <- out_proj(y)

``Block.prompt`` runs whole prompts: the in_proj product of x, B and C with the conv in its
epilogue (bf16), the scan, the gated norm.  ``Block.packed`` does the same for prompts of
different lengths, packed one behind the other.  ``Block.step`` advances by one token, from the
conv and scan states that the prompts left in the caches.

    python examples/state_space_block.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "causal-conv1d-mojo_b200"))

from causal_conv1d_b200 import causal_conv1d_fn, causal_conv1d_update, causal_conv1d_varlen_states  # noqa: E402
from causal_conv1d_b200.fused import in_proj_causal_conv1d  # noqa: E402
from causal_conv1d_b200.norm import gated_norm_fn  # noqa: E402
from causal_conv1d_b200.ssm import state_space_scan, state_space_update  # noqa: E402


class Block:
    def __init__(self, hidden=2560, heads=80, headdim=64, groups=1, dstate=128, width=4, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.headdim, self.groups, self.dstate, self.width = heads, headdim, groups, dstate, width
        self.inner, self.channels = heads * headdim, heads * headdim + 2 * groups * dstate

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) / cols ** 0.5).bfloat16()

        self.w_z, self.w_xbc, self.w_dt = weight(self.inner, hidden), weight(self.channels, hidden), weight(heads, hidden)
        self.w_out = weight(hidden, self.inner)
        self.conv_w = (torch.rand(self.channels, width, generator=g, device=device) - 0.5).bfloat16()
        self.conv_b = (torch.rand(self.channels, generator=g, device=device) - 0.5).bfloat16()
        self.A = -(1 + 15 * torch.rand(heads, generator=g, device=device))
        self.D = torch.ones(heads, device=device)
        step = torch.exp(torch.rand(heads, generator=g, device=device) * 4.6 - 6.9)  # 1e-3 .. 1e-1
        self.dt_bias = step + torch.log(-torch.expm1(-step))
        self.norm_w = torch.ones(self.inner, device=device, dtype=torch.bfloat16)

    def _split(self, xbc):
        """x, B and C as heads and groups: slices of the conv's output, read in place."""
        n = self.groups * self.dstate
        x, B, C = xbc.split([self.inner, n, n], -1)
        return (x.unflatten(-1, (self.heads, self.headdim)), B.unflatten(-1, (self.groups, self.dstate)),
                C.unflatten(-1, (self.groups, self.dstate)))

    def _out(self, y, z):
        return F.linear(gated_norm_fn(y.flatten(-2), self.norm_w, z=z), self.w_out)

    def prompt(self, hidden):
        """hidden (batch, seqlen, hidden) -> out, conv state (batch, channels, width - 1), scan state (fp32)."""
        xbc, conv_state = in_proj_causal_conv1d(hidden, self.w_xbc, self.conv_w, self.conv_b, activation="silu",
                                                return_final_states=True)
        x, B, C = self._split(xbc.transpose(1, 2))
        y, state = state_space_scan(x, F.linear(hidden, self.w_dt), self.A, B, C, D=self.D, dt_bias=self.dt_bias,
                                    dt_softplus=True, return_final_states=True)
        return self._out(y, F.linear(hidden, self.w_z)), conv_state, state

    def packed(self, hidden, lengths):
        """hidden (1, sum of lengths, hidden): prompts one behind the other; states per prompt."""
        cu = torch.tensor([0, *lengths], device=hidden.device).cumsum(0).to(torch.int32)
        seq_idx = torch.repeat_interleave(torch.arange(len(lengths), device=hidden.device, dtype=torch.int32),
                                          torch.tensor(lengths, device=hidden.device))[None]
        xbc = F.linear(hidden, self.w_xbc)
        conv_state = causal_conv1d_varlen_states(xbc[0], cu, self.width - 1)
        xbc = causal_conv1d_fn(xbc.transpose(1, 2), self.conv_w, self.conv_b, seq_idx=seq_idx, activation="silu")
        x, B, C = self._split(xbc.transpose(1, 2))
        y, state = state_space_scan(x, F.linear(hidden, self.w_dt), self.A, B, C, D=self.D, dt_bias=self.dt_bias,
                                    dt_softplus=True, return_final_states=True, cu_seqlens=cu, max_seqlen=max(lengths))
        return self._out(y, F.linear(hidden, self.w_z)), conv_state, state

    def step(self, hidden, conv_state, state, slots=None):
        """hidden (batch, hidden): one token each; the caches' rows `slots` are advanced in place."""
        xbc = causal_conv1d_update(F.linear(hidden, self.w_xbc), conv_state, self.conv_w, self.conv_b, activation="silu",
                                   conv_state_indices=slots)
        x, B, C = self._split(xbc)
        y = state_space_update(x, state, F.linear(hidden, self.w_dt), self.A, B, C, D=self.D, dt_bias=self.dt_bias,
                               dt_softplus=True, state_indices=slots)
        return self._out(y, F.linear(hidden, self.w_z))


@torch.no_grad()
def main(batch=2, seqlen=200, new=4, **sizes):
    """A prompt, then `new` tokens one by one; against the same tokens as one prompt and as packed prompts."""
    block = Block(**sizes)
    hidden = torch.randn(batch, seqlen + new, block.w_out.shape[0], device="cuda").bfloat16()
    whole, _, last = block.prompt(hidden)
    out, conv_state, state = block.prompt(hidden[:, :seqlen].contiguous())
    outs = [out]
    for t in range(seqlen, seqlen + new):
        outs.append(block.step(hidden[:, t], conv_state, state)[:, None])
    stepped = torch.cat(outs, 1)
    packed, _, packed_last = block.packed(hidden.reshape(1, -1, hidden.shape[-1]), [seqlen + new] * batch)
    return {"whole": whole, "stepped": stepped, "packed": packed.view_as(whole), "last": last, "state": state,
            "packed_last": packed_last}


if __name__ == "__main__":
    got = main()
    for name in ("stepped", "packed"):
        d = (got[name].float() - got["whole"].float()).norm() / got["whole"].float().norm()
        print(f"{name}: relative difference to one prompt {d.item():.2e}")
