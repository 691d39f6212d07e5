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
every sum are fp32. Integer tensors of other types are converted to int32, which their values have to
fit. The kernels (csrc/cc1d_ssm_*.cu, csrc/cc1d_slot_maps.cu) are behind the C ABI of
include/causal_conv1d_b200.h and run on torch's current stream. The argument checks and the autograd
Function are C++ (csrc/cc1d_torch_ssm.cpp): AssertionError for shapes and devices, TypeError for
element types, NotImplementedError for forward-mode derivatives (tensors with a tangent), CausalConv1dError
for a failing library call.
"""

from __future__ import annotations

from typing import NamedTuple

from torch import Tensor

from ._native import tex


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
        for one row); ids without an entry and negative slots are skipped. The buffer is written and
        not read: every sequence but a row's first starts from zero, also where its slot holds a state,
        so a request that continues does not belong in a packed row (give it a row of its own with
        initial_states=ssm_state[slot], or take its tokens through ssm_update). An id must not come
        back later in its row and no two sequences may share a slot: which one's h stays is not
        defined. Not differentiable

    Returns out of x's shape and dtype, or (out, final_states). Every floating input but ssm_state
    gets a gradient; the gradients are deterministic, and not differentiable themselves. The forward keeps h before every 16th token
    for the backward (4 * dstate / 16 bytes per element of x, dstate rounded up to 16, 32 or 64).
    """
    return tex.ssm_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, seq_idx, initial_states, return_final_states,
                        ssm_state, ssm_state_indices)


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
    return tex.ssm_update(x, ssm_state, dt, A, B, C, D, z, dt_bias, dt_softplus, ssm_state_indices)


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
        takes the next of free_slots, in request order (-1 once they are used up: n_taken tells). It
        takes it by its length, also where the cut at seqlen leaves none of its tokens in the row: no
        scan then writes the slot, which still holds its last owner's state
    past_lengths: (n,) tokens that each request had before this step

    seq_idx goes to causal_conv1d_fn and ssm_scan, slots to ssm_scan(ssm_state_indices=) and the
    updates, tail_rows picks the convolution's states out of its input. causal_conv1d_fn and ssm_scan
    start every request of a packed row from zero: a row for them holds new requests alone, and a request
    with past_lengths > 0 continues through the updates or through initial_states in a row of its own.
    """
    return SlotMaps._make(tex.slot_maps(lengths, seqlen, width, slots, free_slots, past_lengths))
