"""A Mamba-1 style mixer on this package: in_proj -> causal conv + SiLU -> x_proj -> dt_proj ->
state-space scan with gate -> out_proj, trained, prefilled with packed prompts and decoded.

    python examples/mamba_mixer.py

1. Trains the mixer for a few steps to give one batch back delayed (`causal_conv1d_fn` and `ssm_scan`
   through autograd).
2. Serves three requests: `slot_maps_from_lengths` lays their prompts out in one packed row and gives
   each a state slot; one prefill leaves every request's conv and scan state in its slot; decode steps
   (`causal_conv1d_update`, `ssm_update`) continue all of them at once.
3. Checks the served outputs against the mixer run over each whole sequence.
"""

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "causal-conv1d-triton_b200"))
from causal_conv1d_b200 import (causal_conv1d_fn, causal_conv1d_update, slot_maps_from_lengths,  # noqa: E402
                                ssm_scan, ssm_update)


class Mixer(torch.nn.Module):
    def __init__(self, model=256, inner=512, state=16, width=4, rank=16, dtype=torch.bfloat16):
        super().__init__()
        self.inner, self.state, self.width, self.rank = inner, state, width, rank
        self.in_proj = torch.nn.Linear(model, 2 * inner, bias=False, dtype=dtype)
        self.conv_w = torch.nn.Parameter(torch.randn(inner, width) / width**0.5)
        self.conv_b = torch.nn.Parameter(torch.zeros(inner))
        self.x_proj = torch.nn.Linear(inner, rank + 2 * state, bias=False, dtype=dtype)
        self.dt_proj = torch.nn.Linear(rank, inner, bias=False, dtype=dtype)
        step = torch.exp(torch.empty(inner).uniform_(-6.9, -2.3))
        self.dt_bias = torch.nn.Parameter(step + torch.log(-torch.expm1(-step)))  # softplus gives back the step
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1, state + 1).float()).repeat(inner, 1))
        self.D = torch.nn.Parameter(torch.ones(inner))
        self.out_proj = torch.nn.Linear(inner, model, bias=False, dtype=dtype)

    def _gates(self, x):
        """dt, B, C of the convolved x; B and C stay slices of the projection."""
        p = self.x_proj(x)
        low, B, C = p.split([self.rank, self.state, self.state], -1)
        return self.dt_proj(low), B, C

    def forward(self, u, seq_idx=None, ssm_state=None, slots=None):
        """u (batch, seqlen, model); returns (out, the convolution's input)."""
        x, z = self.in_proj(u).chunk(2, -1)
        c = causal_conv1d_fn(x, self.conv_w, self.conv_b, seq_idx=seq_idx, activation="silu")
        dt, B, C = self._gates(c)
        y = ssm_scan(c, dt, -torch.exp(self.A_log), B, C, D=self.D, z=z, dt_bias=self.dt_bias, dt_softplus=True,
                     seq_idx=seq_idx, ssm_state=ssm_state, ssm_state_indices=slots)
        return self.out_proj(y), x

    def step(self, u, conv_state, ssm_state, slots):
        """One token of every request: u (batch, model)."""
        x, z = self.in_proj(u).chunk(2, -1)
        c = causal_conv1d_update(x, conv_state, self.conv_w, self.conv_b, activation="silu", conv_state_indices=slots)
        dt, B, C = self._gates(c)
        y = ssm_update(c, ssm_state, dt, -torch.exp(self.A_log), B, C, D=self.D, z=z, dt_bias=self.dt_bias,
                       dt_softplus=True, ssm_state_indices=slots)
        return self.out_proj(y)


def train(mixer, steps=40, batch=4, seqlen=128, delay=5):
    opt = torch.optim.AdamW(mixer.parameters(), lr=2e-3, weight_decay=0.0)
    u = torch.randn(batch, seqlen, 256, device="cuda", dtype=torch.bfloat16)
    losses = []
    for _ in range(steps):
        out, _ = mixer(u)
        loss = F.mse_loss(out[:, delay:].float(), u[:, :-delay].float())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def serve(mixer, prompts, new_tokens):
    """prompts: (length, model) of each request; new_tokens (steps, requests, model), given so that the
    result can be checked. Returns each request's outputs over its prompt and new tokens."""
    n, dev = len(prompts), prompts[0].device
    conv_state = torch.zeros(8, mixer.width - 1, mixer.inner, device=dev, dtype=torch.bfloat16)
    ssm_state = torch.zeros(8, mixer.inner, mixer.state, device=dev)
    lengths = torch.tensor([p.shape[0] for p in prompts], device=dev, dtype=torch.int32)
    row = torch.zeros(1, 256, 256, device=dev, dtype=torch.bfloat16)  # one packed row, padded to a fixed length
    row[0, :int(lengths.sum())] = torch.cat(prompts)

    maps = slot_maps_from_lengths(lengths, row.shape[1], width=mixer.width,
                                  slots=torch.full((n,), -1, device=dev, dtype=torch.int32),
                                  free_slots=torch.tensor([6, 2, 5, 0], device=dev, dtype=torch.int32))
    out, x = mixer(row, maps.seq_idx, ssm_state, maps.slots)
    # The convolution's state of each request: its last inputs, zero before its first.
    tail = x[0][maps.tail_rows.clamp_min(0)] * (maps.tail_rows >= 0)[..., None]
    conv_state[maps.slots.long()] = tail
    served = [[out[0, a:b]] for a, b in zip(maps.cu_seqlens[:-1].tolist(), maps.cu_seqlens[1:].tolist())]
    for u in new_tokens:
        y = mixer.step(u, conv_state, ssm_state, maps.slots)
        for i in range(n):
            served[i].append(y[i:i + 1])
    return [torch.cat(s) for s in served]


def main():
    torch.manual_seed(0)
    mixer = Mixer().cuda()
    losses = train(mixer)
    print(f"training: loss {losses[0]:.3f} -> {losses[-1]:.3f} in {len(losses)} steps")
    prompts = [torch.randn(k, 256, device="cuda", dtype=torch.bfloat16) for k in (70, 2, 131)]
    new = torch.randn(12, 3, 256, device="cuda", dtype=torch.bfloat16)
    served = serve(mixer, prompts, new)
    worst = 0.0
    for i, p in enumerate(prompts):
        with torch.no_grad():
            whole, _ = mixer(torch.cat([p, new[:, i]])[None])
        worst = max(worst, ((served[i] - whole[0]).float().norm() / whole.float().norm()).item())
    print(f"serving: packed prompts and {len(new)} decode steps of {len(prompts)} requests, {worst:.1e} from the whole sequences")
    return losses, worst


if __name__ == "__main__":
    main()
