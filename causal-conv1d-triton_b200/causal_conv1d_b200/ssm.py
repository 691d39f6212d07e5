"""The state-space operators of a Mamba-style layer, which follow its causal convolution: the
input-dependent recurrence over a sequence, its single-token form against kept states, and the maps
that a serving step needs from its requests' lengths.

For each batch row, channel d and state n, with delta = softplus(dt + dt_bias) (or dt + dt_bias):

    h[t] = exp(delta[t] A[d, n]) h[t-1] + delta[t] x[t] B[t, n]
    out[t] = (sum_n C[t, n] h[t] + D[d] x[t]) silu(z[t])

The reference has the convolution alone; its README names the layer that calls it
(causal-conv1d-triton README.md:3-4). Layouts, names and conventions are the convolution's:
(batch, seqlen, dim) with channel stride 1 and any other strides, `seq_idx` for packed rows, states
in and out, `*_update` with slot indices for decoding. fp32/fp16/bf16 inputs; all arithmetic, h and
every sum are fp32. The kernels (csrc/cc1d_ssm_*.cu, csrc/cc1d_slot_maps.cu) are behind the C ABI of
include/causal_conv1d_b200.h and run on torch's current stream.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from ._native import check, tex
from .causal_conv1d import _FLOAT, _as_float, _channels_contiguous

MAX_STATE = 64


def _check_operands(x, dt, A, B, C, D, z, dt_bias):
    """Shapes, devices and types common to the scan (3-D x) and the update (after its reshape)."""
    assert x.ndim == 3, "x must be (batch, seqlen, dim)"
    batch, seqlen, dim = x.shape
    assert dt.shape == x.shape, "dt must have the shape of x"
    assert z is None or z.shape == x.shape, "z must have the shape of x"
    assert A.ndim == 2 and A.shape[0] == dim and A.shape[1] >= 1, "A must be (dim, dstate)"
    dstate = A.shape[1]
    assert dstate <= MAX_STATE, f"dstate must be at most {MAX_STATE}"
    assert B.shape == C.shape and B.ndim in (3, 4), "B and C must be (batch, seqlen, [groups,] dstate)"
    assert B.shape[:2] == (batch, seqlen) and B.shape[-1] == dstate, "B and C must be (batch, seqlen, [groups,] dstate)"
    assert B.ndim == 3 or (B.shape[2] >= 1 and dim % B.shape[2] == 0), "dim must be a multiple of the groups of B and C"
    assert D is None or D.shape == (dim,), "D must be (dim,)"
    assert dt_bias is None or dt_bias.shape == (dim,), "dt_bias must be (dim,)"
    for t in (dt, A, B, C, D, z, dt_bias):
        assert t is None or t.device == x.device, "all operands must be on x's device"
    if x.dtype not in _FLOAT:
        raise TypeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    for t in (dt, B, C, z):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"dt, B, C and z must have x's dtype {x.dtype}, got {t.dtype}")
    for t in (A, D, dt_bias):
        if t is not None and not t.is_floating_point():
            raise TypeError(f"A, D and dt_bias must be floating point, got {t.dtype}")
    assert x.is_cuda, "x must be on a CUDA device"


def _vector(t: Tensor | None) -> Tensor | None:
    return None if t is None else _as_float(t.contiguous())


def ssm_scan(
    x: Tensor,
    dt: Tensor,
    A: Tensor,
    B: Tensor,
    C: Tensor,
    D: Tensor | None = None,
    z: Tensor | None = None,
    dt_bias: Tensor | None = None,
    dt_softplus: bool = False,
    seq_idx: Tensor | None = None,
    initial_states: Tensor | None = None,
    return_final_states: bool = False,
    ssm_state: Tensor | None = None,
    ssm_state_indices: Tensor | None = None,
) -> Tensor | tuple[Tensor, Tensor]:
    """The input-dependent state-space recurrence over a sequence (module docstring).

    x, dt, z: (batch, seqlen, dim), one dtype, contiguous along dim (copied otherwise); z gates the
        output with silu(z)
    A: (dim, dstate), usually negative; dstate 1..64
    B, C: (batch, seqlen, dstate), or (batch, seqlen, groups, dstate) where channel d uses group
        d // (dim // groups); x's dtype, contiguous along dstate
    D, dt_bias: (dim,); dt_softplus: delta = softplus(dt + dt_bias) instead of dt + dt_bias
    seq_idx: (batch, seqlen) integer sequence ids for packed sequences, as for causal_conv1d_fn: h
        starts from zero where the id changes; positions with negative ids are padding, and give
        zero outputs and gradients whatever they hold. initial_states count as part of
        seq_idx[:, 0]'s sequence. Cannot be combined with return_final_states
    initial_states: (batch, dim, dstate), h before x[:, 0]
    return_final_states: also return h after the last token, fp32; supports grad
    ssm_state, ssm_state_indices: with seq_idx, a (n_slots, dim, dstate) buffer that gets each
        packed sequence's last h, at slot ssm_state_indices[b, id] ((batch, n_seqs), or (n_seqs,)
        for one row); ids without an entry and negative slots are skipped. Not differentiable

    Returns out of x's shape and dtype, or (out, final_states). Every floating input but ssm_state
    gets a gradient; the gradients are deterministic. The forward keeps h before every 16th token
    for the backward (4 * dstate / 16 bytes per element of x, dstate rounded up to 16, 32 or 64).
    """
    _check_operands(x, dt, A, B, C, D, z, dt_bias)
    batch, seqlen, dim = x.shape
    dstate = A.shape[1]
    if seq_idx is not None:
        assert not return_final_states, "cannot return final states if seq_idx is not None"
        assert seq_idx.shape == (batch, seqlen), "seq_idx must be (batch, seqlen)"
        assert seq_idx.device == x.device, "all operands must be on x's device"
        seq_idx = seq_idx.to(torch.int32).contiguous()
    if initial_states is not None:
        assert initial_states.shape == (batch, dim, dstate), "initial_states must be (batch, dim, dstate)"
        assert initial_states.device == x.device, "all operands must be on x's device"
        if not initial_states.is_floating_point():
            raise TypeError(f"initial_states must be floating point, got {initial_states.dtype}")
    if ssm_state is not None:
        assert seq_idx is not None and ssm_state_indices is not None, "ssm_state requires seq_idx and ssm_state_indices"
        ssm_state_indices = _check_cache(ssm_state, ssm_state_indices, x, dstate)
        if ssm_state_indices.ndim == 1:
            assert batch == 1, "ssm_state_indices must be (batch, n_seqs)"
        else:
            assert ssm_state_indices.ndim == 2 and ssm_state_indices.shape[0] == batch, (
                "ssm_state_indices must be (batch, n_seqs)")
    else:
        assert ssm_state_indices is None, "ssm_state_indices requires ssm_state"

    x, dt, B, C = (_channels_contiguous(t) for t in (x, dt, B, C))
    z = _channels_contiguous(z) if z is not None else None
    A, D, dt_bias, initial_states = _vector(A), _vector(D), _vector(dt_bias), _vector(initial_states)
    needs_grad = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, dt, A, B, C, D, z, dt_bias, initial_states))
    if needs_grad:
        assert ssm_state is None, "ssm_state is not differentiable: call under torch.no_grad()"
        res = tex.ssm_fn(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), seq_idx, initial_states,
                         bool(return_final_states))
        return (res[0], res[1]) if return_final_states else res[0]
    rc, out, final, _ = tex.ssm_fwd(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), seq_idx, initial_states,
                                    bool(return_final_states), False, ssm_state, ssm_state_indices)
    if rc:
        check(rc, "ssm_scan")
    return (out, final) if return_final_states else out


def _check_cache(ssm_state, indices, x, dstate):
    assert ssm_state.ndim == 3 and ssm_state.shape[1:] == (x.shape[-1], dstate), "ssm_state must be (n_slots, dim, dstate)"
    assert ssm_state.device == x.device, "all operands must be on x's device"
    assert ssm_state.is_contiguous(), "ssm_state must be contiguous (it is updated in place)"
    if ssm_state.dtype not in _FLOAT:
        raise TypeError(f"ssm_state must be float32, float16 or bfloat16, got {ssm_state.dtype}")
    return None if indices is None else indices.to(device=x.device, dtype=torch.int32).contiguous()


def ssm_update(
    x: Tensor,
    ssm_state: Tensor,
    dt: Tensor,
    A: Tensor,
    B: Tensor,
    C: Tensor,
    D: Tensor | None = None,
    z: Tensor | None = None,
    dt_bias: Tensor | None = None,
    dt_softplus: bool = False,
    ssm_state_indices: Tensor | None = None,
) -> Tensor:
    """Decode step: run new tokens through the recurrence, continuing from `ssm_state`.

    x, dt, z: (batch, dim) for one new token per batch entry, or (batch, seqlen, dim) for several
    ssm_state: (n_slots, dim, dstate), h before x; updated in place to h after it. fp32 keeps what the
        forward computes; a 16-bit state is rounded once per call
    B, C: (batch, [groups,] dstate), or (batch, seqlen, [groups,] dstate) for several tokens
    A, D, dt_bias, dt_softplus: as for ssm_scan
    ssm_state_indices: optional (batch,) integer slot of each batch entry in ssm_state, no two alike;
        a negative slot leaves that entry's output unwritten and its state untouched

    Returns the output, shaped like x, in x's dtype. Not differentiable (inference only).
    """
    squeeze = x.ndim == 2
    if squeeze:
        x, dt, B, C = (t.unsqueeze(1) for t in (x, dt, B, C))
        z = z.unsqueeze(1) if z is not None else None
    assert x.ndim == 3, "x must be (batch, dim) or (batch, seqlen, dim)"
    _check_operands(x, dt, A, B, C, D, z, dt_bias)
    indices = _check_cache(ssm_state, ssm_state_indices, x, A.shape[1])
    if indices is None:
        assert ssm_state.shape[0] >= x.shape[0], "ssm_state has fewer slots than x has rows"
    else:
        assert indices.shape == (x.shape[0],), "ssm_state_indices must be (batch,)"
    x, dt, B, C = (_channels_contiguous(t) for t in (x, dt, B, C))
    z = _channels_contiguous(z) if z is not None else None
    rc, out = tex.ssm_update(x, ssm_state, dt, _vector(A), B, C, _vector(D), z, _vector(dt_bias), bool(dt_softplus),
                             indices)
    if rc:
        check(rc, "ssm_update")
    return out.squeeze(1) if squeeze else out


class SlotMaps(NamedTuple):
    """What slot_maps_from_lengths returns; int32, on the device of the lengths."""

    cu_seqlens: Tensor  # (n + 1,): request r is tokens [cu[r], cu[r + 1]) of the packed row
    seq_idx: Tensor     # (1, seqlen): each token's request, -1 past the last one
    positions: Tensor   # (1, seqlen): its position in the request, counted from past_lengths; -1 past the last
    tail_rows: Tensor   # (n, width - 1): rows of each request's last width - 1 tokens, -1 before its first
    slots: Tensor | None  # (n,): each request's state slot (None without `slots`)
    n_taken: Tensor     # (1,): how many requests needed a new slot


def slot_maps_from_lengths(
    lengths: Tensor,
    seqlen: int,
    width: int = 1,
    slots: Tensor | None = None,
    free_slots: Tensor | None = None,
    past_lengths: Tensor | None = None,
) -> SlotMaps:
    """The maps of a serving step, built on the device from its requests' lengths without a
    synchronisation: one launch up to 4096 requests, two above.

    lengths: (n,) new tokens of each request, 0 for none; they lie one after another in a packed row
    seqlen: tokens of the packed row; what the lengths leave over is padding, and requests are cut at it
    width: of the convolution whose state rows `tail_rows` gives
    slots: (n,) state slot of each request, negative for none yet; a request with tokens and no slot
        takes the next of free_slots, in request order (-1 once they are used up: n_taken tells)
    past_lengths: (n,) tokens that each request had before this step

    seq_idx goes to causal_conv1d_fn and ssm_scan, slots to ssm_scan(ssm_state_indices=) and the
    updates, tail_rows picks the convolution's states out of its input.
    """
    assert lengths.ndim == 1, "lengths must be (n,)"
    assert width >= 1 and seqlen >= 0, "width must be at least 1 and seqlen at least 0"
    assert slots is not None or free_slots is None, "free_slots requires slots"

    def ints(t, shape, what):
        if t is None:
            return None
        assert t.ndim == 1 and (shape is None or t.shape == shape), f"{what} must be (n,)"
        assert t.device == lengths.device, f"{what} must be on the device of lengths"
        if t.is_floating_point():
            raise TypeError(f"{what} must be integer, got {t.dtype}")
        return t.to(torch.int32).contiguous()

    n = lengths.shape
    args = (ints(lengths, n, "lengths"), seqlen, width, ints(past_lengths, n, "past_lengths"), ints(slots, n, "slots"),
            ints(free_slots, None, "free_slots"))
    assert lengths.is_cuda, "lengths must be on a CUDA device"
    rc, *maps = tex.slot_maps(*args)
    if rc:
        check(rc, "slot_maps_from_lengths")
    return SlotMaps(*maps)
