"""The state-space recurrence in 64 bits, one token after another: what the kernels are held to.

Tolerances. The kernels compute in fp32. A decay has a relative error below 2^-22 (the exponential,
its argument's rounding), a product or sum 2^-24, and the step size (softplus, measured against 64
bits) below 2^-21; an error made in one token is carried on by decays of at most 1, so a state T
tokens on is off by at most T such errors, about 4e-7 T of its size, and a gradient, a chain back
through the states of a chain, by twice that. Sums over states, channels and CTAs add less than 32
roundings more. Hence an fp32 value may be off by 1e-6 (T + 32) of the largest value of its tensor. A 16-bit
output is that value rounded once: half a unit in the last place more, 2^-9 (bf16) or 2^-11 (fp16)
of the value itself, twice that allowed here for values that the fp32 error moves across a rounding
boundary.
"""

import torch
import torch.nn.functional as F

ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-10}


def per_channel(v, dim):
    """B or C of one token, (batch, [groups,] n) -> (batch, dim, n)."""
    return v.unsqueeze(1).expand(-1, dim, -1) if v.ndim == 2 else v.repeat_interleave(dim // v.shape[1], 1)


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, seq_idx=None, initial_states=None):
    """(out, h after every token); differentiable, every operand in the dtype given."""
    batch, seqlen, dim = x.shape
    h = initial_states if initial_states is not None else x.new_zeros(batch, dim, A.shape[1])
    raw = dt if dt_bias is None else dt + dt_bias
    delta = F.softplus(raw, threshold=40) if dt_softplus else raw
    outs, states = [], []
    for t in range(seqlen):
        step = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * x[:, t]).unsqueeze(-1) * per_channel(B[:, t], dim)
        if seq_idx is not None:
            fresh = (seq_idx[:, t] != seq_idx[:, t - 1]) if t else torch.zeros_like(seq_idx[:, 0], dtype=torch.bool)
            alone = (delta[:, t] * x[:, t]).unsqueeze(-1) * per_channel(B[:, t], dim)
            step = torch.where(fresh[:, None, None], alone, step)
            step = torch.where((seq_idx[:, t] < 0)[:, None, None], torch.zeros_like(step), step)
        h = step
        y = (h * per_channel(C[:, t], dim)).sum(-1)
        if D is not None:
            y = y + D * x[:, t]
        if z is not None:
            y = y * F.silu(z[:, t])
        if seq_idx is not None:
            y = torch.where((seq_idx[:, t] < 0)[:, None], torch.zeros_like(y), y)
        outs.append(y)
        states.append(h)
    return torch.stack(outs, 1), torch.stack(states, 1)


def assert_near(actual, expected, tokens, what=""):
    assert actual.shape == expected.shape, f"{what}: {tuple(actual.shape)} is not {tuple(expected.shape)}"
    if expected.numel() == 0:
        return
    e, a = expected.detach().double(), actual.detach().double()
    bound = 1e-6 * (tokens + 32) * e.abs().max() + ROUND[actual.dtype] * e.abs()
    off = (a - e).abs() - bound
    assert not torch.isnan(a).any(), f"{what}: NaN"
    assert (off <= 0).all(), f"{what}: off by up to {(a - e).abs().max():.3g}, {off.max():.3g} over the bound"


def case(seed, batch, seqlen, dim, dstate, groups=0, dtype=torch.float32, device="cpu", D=True, z=True, bias=True,
         init=False, lengths=None):
    """Operands as a layer has them; groups 0: B and C without a group dimension. lengths: the packed
    sequences of each row, negative for padding."""
    g = torch.Generator().manual_seed(seed)

    def n(*shape):
        return torch.randn(*shape, generator=g)

    ops = dict(x=F.silu(n(batch, seqlen, dim)), dt=0.5 * n(batch, seqlen, dim),
               A=-torch.arange(1, dstate + 1).float() * torch.exp(0.1 * n(dim, dstate)),
               B=n(batch, seqlen, *([groups] if groups else []), dstate),
               C=n(batch, seqlen, *([groups] if groups else []), dstate),
               D=n(dim) if D else None, z=n(batch, seqlen, dim) if z else None,
               dt_bias=(-3.0 + n(dim)) if bias else None)
    ops = {k: v if v is None else v.to(dtype if k in ("x", "dt", "B", "C", "z") else torch.float32).to(device)
           for k, v in ops.items()}
    if not bias:
        ops["dt"] = (ops["dt"].float().abs() * 0.1).to(dtype)
    ops["initial_states"] = n(batch, dim, dstate).to(device) if init else None
    ops["seq_idx"] = None
    if lengths is not None:
        rows = []
        for row in lengths:
            ids, i = [], 0
            for k in row:
                ids += [i if k > 0 else -1] * abs(k)
                i += k > 0
            assert len(ids) == seqlen
            rows.append(ids)
        ops["seq_idx"] = torch.tensor(rows, dtype=torch.int32, device=device)
    return ops


def wide(ops):
    return {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in ops.items()}
