"""The state-space scan, its single-token form and the slot maps on the GPU, against the 64-bit
restatement (tests/_ssm_ref.py, which states how the tolerances follow from the arithmetic)."""

import ctypes

import pytest
import torch

import _ssm_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
GRADS = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_states")


def to_dev(ops):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in ops.items()}


def check_scan(ops, softplus=True, final=True, seed=7):
    """Outputs, final states and every gradient of ssm_scan against the restatement."""
    from causal_conv1d_b200 import ssm_scan

    final = final and ops["seq_idx"] is None
    g = torch.Generator().manual_seed(seed)
    dout = torch.randn(ops["x"].shape, generator=g).to(ops["x"].dtype).to(DEV)
    dfin = torch.randn(ops["x"].shape[0], ops["x"].shape[2], ops["A"].shape[1], generator=g).to(DEV)
    mine, want = to_dev(ops), ref.wide(to_dev(ops))
    names = [k for k in GRADS if ops[k] is not None]
    for d in (mine, want):
        for k in names:
            d[k] = d[k].detach().clone().requires_grad_(True) if d[k].is_contiguous() else d[k].detach().requires_grad_(True)
    res = ssm_scan(**mine, dt_softplus=softplus, return_final_states=final)
    out, fin = res if final else (res, None)
    wout, wh = ref.scan(**want, dt_softplus=softplus)
    T = ops["x"].shape[1]
    assert out.dtype == ops["x"].dtype
    ref.assert_near(out, wout, T, "out")
    got_out, got_in = [out], [dout]
    exp_out, exp_in = [wout], [dout.double()]
    if final:
        assert fin.dtype == F32
        ref.assert_near(fin, wh[:, -1], T, "final_states")
        got_out, got_in = [out, fin], [dout, dfin]
        exp_out, exp_in = [wout, wh[:, -1]], [dout.double(), dfin.double()]
    got = torch.autograd.grad(got_out, [mine[k] for k in names], got_in)
    exp = torch.autograd.grad(exp_out, [want[k] for k in names], exp_in)
    for k, a, e in zip(names, got, exp):
        assert a.dtype == ops[k].dtype, k
        ref.assert_near(a, e, T, "d" + k)
    with torch.no_grad():  # the form without a backward gives the same bits
        again = ssm_scan(**{k: v.detach() if torch.is_tensor(v) else v for k, v in mine.items()}, dt_softplus=softplus,
                         return_final_states=final)
    assert torch.equal(again[0] if final else again, out.detach())
    if final:
        assert torch.equal(again[1], fin.detach())


@pytest.mark.parametrize("batch, seqlen, dim, dstate, groups, dtype, kw", [
    (1, 1, 1, 1, 0, F32, {}),
    (2, 1, 64, 16, 0, BF16, dict(init=True)),
    (1, 2, 5, 3, 1, F32, dict(D=False)),
    (2, 15, 8, 4, 2, F16, dict(z=False)),
    (1, 16, 128, 16, 0, BF16, {}),
    (3, 17, 33, 16, 3, F32, dict(init=True, bias=False)),
    (2, 31, 40, 12, 1, BF16, dict(D=False, z=False, bias=False)),
    (1, 33, 130, 16, 0, F16, dict(init=True)),
    (2, 70, 64, 17, 4, F32, dict(init=True)),
    (1, 48, 72, 32, 0, BF16, {}),
    (2, 37, 20, 33, 5, F32, {}),
    (1, 65, 96, 64, 2, F16, dict(init=True)),
    (1, 40, 257, 64, 0, F32, dict(z=False)),
    (5, 64, 516, 16, 3, BF16, dict(init=True)),
])
def test_scan_and_gradients(batch, seqlen, dim, dstate, groups, dtype, kw):
    check_scan(ref.case(seqlen * 31 + dim, batch, seqlen, dim, dstate, groups, dtype, **kw))


@pytest.mark.parametrize("softplus", [False, True])
def test_plain_steps(softplus):
    """Without softplus the step is dt + dt_bias as given, negative ones among them."""
    ops = ref.case(3, 2, 20, 24, 16)
    if not softplus:
        ops["dt"], ops["dt_bias"] = 0.02 * ops["dt"], 0.02 * ops["dt_bias"]
    check_scan(ops, softplus=softplus)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim, dstate, groups", [(32, 16, 0), (40, 20, 2)])
@pytest.mark.parametrize("init", [False, True])
def test_packed(dtype, dim, dstate, groups, init):
    """Sequences that start inside, at and just past the 16- and 32-token tiles, single tokens, padding
    between and around them, a row that is padding alone."""
    check_scan(ref.case(11, 4, 67, dim, dstate, groups, dtype, init=init, lengths=[
        [67], [1, 15, 16, 1, -3, 31], [-2, 30, -1, 1, 33], [-67]]))


def pieces(ops, backward):
    """How many pieces the sequence is cut in, from the workspace that they need (cc1d_ssm_api.cu)."""
    from causal_conv1d_b200 import _native

    b, t, d = ops["x"].shape
    n, groups = ops["A"].shape[1], ops["B"].shape[2] if ops["B"].ndim == 4 else 1
    floats = _native.lib.cc1d_ssm_workspace_bytes(b, t, d, n, groups, _native.DTYPE_CODE[ops["x"].dtype], int(backward)) // 4
    wide = 16 if n <= 16 else 32 if n <= 32 else 64  # states as the kernels hold them
    piece = 3 * b * d * wide
    if not backward:
        return max(1, floats // piece)
    blocks = -(-(d // groups) // (1024 // wide))
    floats -= b * t * groups * blocks * 2 * wide
    part = b * d * wide + 2 * b * d
    return 1 if floats == part else floats // (part + piece)


@pytest.mark.parametrize("kw", [dict(init=True), dict(lengths=[[300, 1, 255, -44, 424, -7, 469]])])
@pytest.mark.parametrize("dim, dstate, dtype", [(24, 16, F32), (8, 40, F32), (64, 16, BF16)])
def test_sequence_in_pieces(dim, dstate, dtype, kw):
    """Few rows and channels: the sequence is cut, and states and gradients pass between pieces."""
    ops = ref.case(5, 1, 1500, dim, dstate, 0, dtype, **kw)
    assert pieces(ops, False) > 2 and pieces(ops, True) > 2
    check_scan(ops)


def test_one_group_does_not_reach_another():
    """Infinities in one group's channels stay out of the other's, whose last block of channels is not full,
    also where a gradient passes between pieces."""
    from causal_conv1d_b200 import ssm_scan

    for seqlen in (40, 1200):
        ops = to_dev(ref.case(83, 1, seqlen, 48, 16, 2))
        names = ("x", "dt", "B", "C", "z")

        def run(dout):
            o = {k: v.clone().requires_grad_(True) if k in names else v for k, v in ops.items()}
            return torch.autograd.grad(ssm_scan(**o, dt_softplus=True), [o[k] for k in names], dout)

        dout = torch.randn(1, seqlen, 48, device=DEV)
        clean = run(dout)
        dout[..., 24:] = float("inf")
        for k, a, e in zip(names, run(dout), clean):
            half = (slice(None), slice(None), slice(0, 1)) if k in "BC" else (Ellipsis, slice(0, 24))
            assert torch.equal(a[half], e[half]), k


def test_gradients_match_differences():
    """The derivative along a direction in every input, by central differences of the 64-bit form."""
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(17, 2, 24, 24, 16, 2, init=True))
    names = [k for k in GRADS if ops[k] is not None]
    mine = {k: v.clone().requires_grad_(True) if k in names else v for k, v in ops.items()}
    g = torch.Generator().manual_seed(1)
    w = torch.randn(ops["x"].shape, generator=g).to(DEV)
    grads = torch.autograd.grad(ssm_scan(**mine, dt_softplus=True), [mine[k] for k in names], w)
    base = ref.wide(ops)
    for k, d in zip(names, grads):
        v = torch.randn(ops[k].shape, generator=g).to(DEV).double()

        def f(e):
            return (ref.scan(**{**base, k: base[k] + e * v}, dt_softplus=True)[0] * w.double()).sum()

        # Central differences at 1e-5 in 64 bits: 1e-10 of cut-off and rounding; the rest is the gradient's own error.
        want = (f(1e-5) - f(-1e-5)) / 2e-5
        scale = (d.double() * v).abs().sum()
        assert ((d.double() * v).sum() - want).abs() <= 1e-6 * 56 * scale, k


def test_values_at_padding_do_not_matter():
    """NaN and infinities in padded places, and in a sequence next to others, stay where they are."""
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(23, 2, 50, 40, 16, lengths=[[10, -5, 35], [-20, 20, -10]]))
    names = [k for k in GRADS if ops[k] is not None]
    dout = torch.randn(2, 50, 40, device=DEV)

    def run(o, d):
        o = {k: v.clone().requires_grad_(True) if k in names else v for k, v in o.items()}
        out = ssm_scan(**o, dt_softplus=True)
        return (out, *torch.autograd.grad(out, [o[k] for k in names], d))

    clean = run(ops, dout)
    off = ops["seq_idx"] < 0
    for bad in (float("nan"), float("inf"), torch.finfo(F32).min):
        dirty = {k: v.clone() if torch.is_tensor(v) else v for k, v in ops.items()}
        for k in ("x", "dt", "B", "C", "z"):
            dirty[k][off] = bad
        d = dout.clone()
        d[off] = bad
        for a, e in zip(run(dirty, d), clean):
            assert torch.equal(a, e)
    assert (clean[0][off] == 0).all() and (clean[1][off] == 0).all()

    # An overflowing first sequence leaves the second one's outputs and token gradients alone.
    dirty = {k: v.clone() if torch.is_tensor(v) else v for k, v in ops.items()}
    dirty["x"][0, :10] = float("inf")
    got = run(dirty, dout)
    assert torch.equal(got[0][0, 10:], clean[0][0, 10:])
    for k, a, e in zip(names, got[1:], clean[1:]):
        if k in ("x", "dt", "B", "C", "z"):
            assert torch.equal(a[0, 10:], e[0, 10:]), k


def test_decay_extremes():
    """Steps whose decay underflows to 0, steps of 0 (decay 1, no input), and a large softplus argument."""
    ops = ref.case(29, 1, 20, 16, 16)
    ops["dt_bias"] = None
    ops["dt"] = torch.tensor([0.0, 1.0, 30.0, 200.0]).repeat(4)[None, None].expand(1, 20, 16).contiguous()
    check_scan(ops, softplus=False)
    ops["dt"] = torch.tensor([-80.0, -15.0, 21.0, 90.0]).repeat(4)[None, None].expand(1, 20, 16).contiguous()
    check_scan(ops, softplus=True)


def test_packed_states_go_to_slots():
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(31, 2, 60, 24, 16, dtype=BF16, lengths=[[20, 1, -4, 35], [-10, 32, 18]]))
    _, h = ref.scan(**ref.wide(ops), dt_softplus=True)
    for dtype in (F32, BF16):
        cache = torch.full((9, 24, 16), 7.0, device=DEV, dtype=dtype)
        slots = torch.tensor([[4, 0, 8], [-1, 2, 5]], device=DEV)  # the second row has two sequences: 5 is not used
        with torch.no_grad():
            out = ssm_scan(**ops, dt_softplus=True, ssm_state=cache, ssm_state_indices=slots)
            assert torch.equal(out, ssm_scan(**ops, dt_softplus=True))
        for slot, (b, t) in {4: (0, 19), 0: (0, 20), 8: (0, 59), 2: (1, 59)}.items():
            ref.assert_near(cache[slot], h[b, t], 60, f"slot {slot}")
        for slot in (1, 3, 5, 6, 7):
            assert (cache[slot] == 7).all()
    # Ids without an entry and slots outside the buffer are skipped.
    cache = torch.full((3, 24, 16), 7.0, device=DEV)
    with torch.no_grad():
        ssm_scan(**ops, dt_softplus=True, ssm_state=cache, ssm_state_indices=torch.tensor([[3], [1]], device=DEV))
    assert (cache[0] == 7).all() and (cache[2] == 7).all()
    ref.assert_near(cache[1], h[1, 41], 60)
    with pytest.raises(AssertionError):
        ops["x"].requires_grad_(True)
        ssm_scan(**ops, ssm_state=cache, ssm_state_indices=slots)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_and_alignment(dtype):
    """Operands as slices of wider projections at odd offsets, transposed and expanded ones."""
    from causal_conv1d_b200 import ssm_scan

    base = to_dev(ref.case(37, 2, 33, 48, 16, dtype=dtype))
    plain = ssm_scan(**base, dt_softplus=True)

    def slice_of(t, offset, extra):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + extra, device=DEV, dtype=t.dtype)
        wide[..., offset:offset + t.shape[-1]] = t
        return wide[..., offset:offset + t.shape[-1]]

    for offset in (1, 4, 8):
        ops = {k: slice_of(v, offset, 24) if k in ("x", "dt", "B", "C", "z") else v for k, v in base.items()}
        assert torch.equal(ssm_scan(**ops, dt_softplus=True), plain)
        check_scan(ops)
    ops = {k: v.transpose(0, 1).contiguous().transpose(0, 1) if k in ("x", "dt", "z") else v for k, v in base.items()}
    ops["B"] = base["B"].transpose(1, 2).contiguous().transpose(1, 2)  # not contiguous along dstate
    assert torch.equal(ssm_scan(**ops, dt_softplus=True), plain)
    # B shared by the batch through a zero stride; a gradient without a channel stride of 1.
    ops = {k: v.clone().requires_grad_(True) if k in ("x", "B") else v for k, v in base.items()}
    one = ops["B"][:1]
    out = ssm_scan(**{**ops, "B": one.expand(2, -1, -1)}, dt_softplus=True)
    dout = torch.randn(2, 48, 33, device=DEV, dtype=dtype).transpose(1, 2)
    (got,) = torch.autograd.grad(out, [ops["B"]], dout)
    want = ref.wide({k: v.detach() if torch.is_tensor(v) else v for k, v in base.items()})
    wb = want["B"][:1].clone().requires_grad_(True)
    wout, _ = ref.scan(**{**want, "B": wb.expand(2, -1, -1)}, dt_softplus=True)
    (exp,) = torch.autograd.grad(wout, [wb], dout.double())
    # Two rounded rows added: twice the rounding of one.
    off = (got[:1].double() - exp).abs()
    assert (off <= 1e-6 * 65 * exp.abs().max() + 3 * ref.ROUND[dtype] * exp.abs().max()).all()
    assert (got[1] == 0).all()


def test_only_some_inputs_need_gradients():
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(41, 2, 20, 24, 16, init=True))
    full = {k: v.clone().requires_grad_(True) if k in GRADS else v for k, v in ops.items()}
    w = torch.randn(2, 20, 24, device=DEV)
    out, fin = ssm_scan(**full, dt_softplus=True, return_final_states=True)
    everything = dict(zip(GRADS, torch.autograd.grad([out], [full[k] for k in GRADS], [w])))  # nothing comes back from fin
    for k in GRADS:
        some = dict(ops, **{k: ops[k].clone().requires_grad_(True)})
        (g,) = torch.autograd.grad(ssm_scan(**some, dt_softplus=True), [some[k]], w)
        assert torch.equal(g, everything[k]), k


def test_parameter_types():
    """A, D, dt_bias and the initial states in 16 bits and in 64."""
    for dtype in (BF16, torch.float64):
        ops = ref.case(43, 2, 18, 24, 16, init=True)
        for k in ("A", "D", "dt_bias", "initial_states"):
            ops[k] = ops[k].to(BF16).to(dtype)
        if dtype == BF16:
            check_scan(ops)
        else:
            from causal_conv1d_b200 import ssm_scan

            o = to_dev(ops)
            o["A"].requires_grad_(True)
            out = ssm_scan(**o, dt_softplus=True)
            (g,) = torch.autograd.grad(out.sum(), [o["A"]])
            assert g.dtype == torch.float64
            ref.assert_near(out, ref.scan(**ref.wide(to_dev(ops)), dt_softplus=True)[0], 18)


def test_nothing_to_do():
    from causal_conv1d_b200 import ssm_scan, ssm_update

    for shape in ((2, 0, 8), (0, 5, 8), (2, 5, 0)):
        ops = to_dev(ref.case(1, *shape, 4, init=True))
        ops = {k: v.requires_grad_(True) if k in GRADS else v for k, v in ops.items()}
        out, fin = ssm_scan(**ops, return_final_states=True)
        assert out.shape == shape
        if shape[1] == 0:
            assert torch.equal(fin, ops["initial_states"])
        grads = torch.autograd.grad([out, fin], [ops[k] for k in GRADS], [torch.ones_like(out), torch.ones_like(fin)])
        for k, g in zip(GRADS, grads):
            assert g.shape == ops[k].shape
            assert (g == (1 if k == "initial_states" and shape[1] == 0 else 0)).all() or shape[0] == 0 or shape[2] == 0
    ops = to_dev(ref.case(1, 2, 0, 8, 4))
    state = torch.ones(2, 8, 4, device=DEV)
    ops.pop("seq_idx"), ops.pop("initial_states")
    assert ssm_update(ssm_state=state, **ops).shape == (2, 0, 8) and (state == 1).all()


def test_same_bits_twice_and_on_another_stream():
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(47, 2, 700, 96, 16, dtype=BF16))
    names = [k for k in GRADS if ops[k] is not None]
    dout = torch.randn(2, 700, 96, device=DEV).to(BF16)

    def run():
        o = {k: v.clone().requires_grad_(True) if k in names else v for k, v in ops.items()}
        out = ssm_scan(**o, dt_softplus=True)
        return (out, *torch.autograd.grad(out, [o[k] for k in names], dout))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, e in zip(second, first):
        assert torch.equal(a, e)


def test_second_derivatives_are_refused():
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(79, 1, 8, 16, 4))
    ops["x"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradients of its gradients"):
        torch.autograd.grad(ssm_scan(**ops).sum(), ops["x"], create_graph=True)


def test_scan_in_a_graph():
    """A captured forward and backward, in one piece and in several, replayed on new inputs."""
    from causal_conv1d_b200 import ssm_scan

    for seqlen in (40, 1000):
        ops = to_dev(ref.case(89, 1, seqlen, 64, 16, dtype=BF16, init=True))
        names = [k for k in GRADS if ops[k] is not None]
        dout = torch.randn(1, seqlen, 64, device=DEV).to(BF16)
        leaves = {k: ops[k].clone().requires_grad_(True) for k in names}

        def step():
            out, fin = ssm_scan(**{**ops, **leaves}, dt_softplus=True, return_final_states=True)
            return (out, fin, *torch.autograd.grad([out], list(leaves.values()), [dout]))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        with torch.no_grad():
            leaves["x"].copy_(torch.randn(1, seqlen, 64, device=DEV).to(BF16))
            dout.copy_(torch.randn(1, seqlen, 64, device=DEV).to(BF16))
        graph.replay()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e)


def test_many_rows():
    """More batch rows than a grid's second and third dimensions hold."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(97, 70000, 2, 8, 4))
    out, fin = ssm_scan(**ops, dt_softplus=True, return_final_states=True)
    wout, wh = ref.scan(**ref.wide(ops), dt_softplus=True)
    ref.assert_near(out, wout, 2)
    ref.assert_near(fin, wh[:, -1], 2)
    state = torch.zeros(70000, 8, 4, device=DEV)
    assert torch.equal(ssm_update(ssm_state=state, dt_softplus=True, **token_ops(ops, slice(0, 2))), out)
    assert torch.equal(state, fin)


def token_ops(ops, t):
    return {k: v[:, t] if k in ("x", "dt", "B", "C", "z") and v is not None else v for k, v in ops.items()
            if k not in ("seq_idx", "initial_states")}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim, dstate, groups", [(64, 16, 0), (33, 5, 3), (40, 64, 2), (24, 30, 1)])
def test_decode_steps_equal_scan(dtype, dim, dstate, groups):
    """Token by token, then several at a time: the scan's outputs and states, bit for bit."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(53, 3, 12, dim, dstate, groups, dtype, init=True))
    full, final = ssm_scan(**ops, dt_softplus=True, return_final_states=True)
    state = ops["initial_states"].clone()
    outs = [ssm_update(ssm_state=state, dt_softplus=True, **token_ops(ops, t)) for t in range(12)]
    assert torch.equal(torch.stack(outs, 1), full) and torch.equal(state, final)
    state = ops["initial_states"].clone()
    outs = [ssm_update(ssm_state=state, dt_softplus=True, **token_ops(ops, slice(t, t + 5))) for t in (0, 5, 10)]
    assert torch.equal(torch.cat(outs, 1), full) and torch.equal(state, final)


@pytest.mark.parametrize("state_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dstate", [16, 7])
def test_update_slots(state_dtype, dstate):
    from causal_conv1d_b200 import ssm_update

    ops = to_dev(ref.case(59, 5, 1, 40, dstate, dtype=BF16, D=False))
    state0 = torch.randn(8, 40, dstate, device=DEV).to(state_dtype)
    slots = torch.tensor([6, -1, 0, 3, 9], device=DEV)  # one padded entry, one slot outside the buffer
    state = state0.clone()
    out = ssm_update(ssm_state=state, dt_softplus=True, ssm_state_indices=slots, **token_ops(ops, 0))
    want = ref.wide(ops)
    for i, s in ((0, 6), (2, 0), (3, 3)):
        one = {k: v[i:i + 1] if k in ("x", "dt", "B", "C", "z") else v for k, v in want.items()}
        one["initial_states"] = state0[s:s + 1].double()
        wout, wh = ref.scan(**one, dt_softplus=True)
        ref.assert_near(out[i:i + 1], wout[:, 0], 1, "out")
        ref.assert_near(state[s], wh[0, 0], 1, "state")
    for s in (1, 2, 4, 5, 7):
        assert torch.equal(state[s], state0[s])


def test_update_misaligned_state_and_offsets_past_32_bits():
    from causal_conv1d_b200 import ssm_update

    ops = token_ops(to_dev(ref.case(61, 2, 1, 2048, 16, dtype=BF16)), 0)
    flat = torch.randn(2 * 2048 * 16 + 1, device=DEV)
    a, b = flat[:-1].clone().view(2, 2048, 16), flat.clone()[1:].view(2, 2048, 16)
    b.copy_(a)
    assert b.data_ptr() % 16 != 0
    oa, ob = (ssm_update(ssm_state=s, dt_softplus=True, **ops) for s in (a, b))
    assert torch.equal(oa, ob) and torch.equal(a, b)
    # 2.3e9 states of 16 bits: slots whose element offsets pass 2^31.
    big = torch.zeros(70000, 2048, 16, device=DEV, dtype=BF16)
    big[66000], big[69999] = flat[:-1].view(2, 2048, 16).to(BF16)
    small = torch.stack([big[66000], big[69999]])
    ob = ssm_update(ssm_state=big, dt_softplus=True, ssm_state_indices=torch.tensor([66000, 69999], device=DEV), **ops)
    oa = ssm_update(ssm_state=small, dt_softplus=True, **ops)
    assert torch.equal(oa, ob) and torch.equal(big[66000], small[0]) and torch.equal(big[69999], small[1])


def test_scan_strides_past_32_bits():
    """Tokens 2^30 elements apart: the last ones lie past 2^31."""
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(67, 1, 3, 16, 4, dtype=BF16))
    far = torch.zeros(2**31 + 64, device=DEV, dtype=BF16)
    x = far.as_strided((1, 3, 16), (0, 2**30, 1))
    x.copy_(ops["x"])
    assert torch.equal(ssm_scan(**{**ops, "x": x}, dt_softplus=True), ssm_scan(**ops, dt_softplus=True))


def test_update_in_a_graph():
    from causal_conv1d_b200 import ssm_update

    ops = token_ops(to_dev(ref.case(71, 4, 1, 64, 16, dtype=BF16)), 0)
    state = torch.randn(4, 64, 16, device=DEV)
    eager = state.clone()
    want = [ssm_update(ssm_state=eager, dt_softplus=True, **ops) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    warm = state.clone()
    with torch.cuda.stream(side):
        ssm_update(ssm_state=warm, dt_softplus=True, **ops)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ssm_update(ssm_state=state, dt_softplus=True, **ops)
    for w in want:
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(state, eager)


def test_c_abi_through_ctypes():
    """The header's structures as the package's ctypes binding lays them out."""
    from causal_conv1d_b200 import _native as n
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(73, 2, 40, 24, 16, 2, BF16, init=True))
    want, final = ssm_scan(**ops, dt_softplus=True, return_final_states=True)
    q = n.SsmProblem(batch=2, seqlen=40, dim=24, dstate=16, groups=2, x_dtype=2, dt_softplus=1)
    for k in ("x", "dt", "z"):
        setattr(q, k, n.Tokens(ops[k].data_ptr(), ops[k].stride(0), ops[k].stride(1), 0))
    for k in ("B", "C"):
        setattr(q, k, n.Tokens(ops[k].data_ptr(), *ops[k].stride()[:3]))
    for k in ("A", "D", "dt_bias", "initial_states"):
        setattr(q, k, n.Param(ops[k].data_ptr(), 0))
    out, fin = torch.empty_like(want), torch.empty_like(final)
    size = n.lib.cc1d_ssm_workspace_bytes(2, 40, 24, 16, 2, 2, 0)
    ws = torch.empty(max(1, size), device=DEV, dtype=torch.uint8)
    stream = torch.cuda.current_stream().cuda_stream
    n.check(n.lib.cc1d_ssm_fwd(ctypes.byref(q), out.data_ptr(), fin.data_ptr(), None, None, 0, 0, None, 0,
                               ws.data_ptr(), size, stream), "cc1d_ssm_fwd")
    assert torch.equal(out, want) and torch.equal(fin, final)


def maps_by_hand(lengths, seqlen, width, slots, free, past):
    cu, seq, pos, tail = [0], [-1] * seqlen, [-1] * seqlen, []
    out, taken = [], 0
    for r, k in enumerate(lengths):
        k = max(k, 0)
        start, end = cu[-1], min(seqlen, cu[-1] + k)
        for i in range(start, end):
            seq[i], pos[i] = r, i - start + (past[r] if past else 0)
        tail.append([i if i >= start else -1 for i in range(end - width + 1, end)])
        if slots is not None:
            if slots[r] < 0 and k > 0:
                out.append(free[taken] if taken < len(free) else -1)
                taken += 1
            else:
                out.append(slots[r])
        cu.append(end)
    return cu, [seq], [pos], tail, out if slots is not None else None, [taken]


@pytest.mark.parametrize("n, seqlen, width, most", [
    (0, 10, 4, 1), (1, 1, 1, 1), (1, 0, 4, 5), (3, 17, 4, 9), (7, 1030, 8, 200), (40, 200, 2, 12), (257, 2048, 4, 9),
    (4096, 9000, 4, 4), (4097, 9000, 3, 4), (5000, 4000, 2, 3),
])
@pytest.mark.parametrize("with_slots", [False, True])
def test_slot_maps(n, seqlen, width, most, with_slots):
    from causal_conv1d_b200 import slot_maps_from_lengths

    g = torch.Generator().manual_seed(n + seqlen)
    lengths = torch.randint(-1, most + 1, (n,), generator=g, dtype=torch.int32)  # zero and negative ones among them
    slots = free = past = None
    if with_slots:
        slots = torch.where(torch.rand(n, generator=g) < 0.5, torch.arange(n), -1)
        free = torch.arange(n, n + n // 3)  # fewer than are wanted
        past = torch.randint(0, 99, (n,), generator=g)
    got = slot_maps_from_lengths(lengths.to(DEV), seqlen, width, *(t.to(DEV) if t is not None else None for t in (slots, free, past)))
    want = maps_by_hand(lengths.tolist(), seqlen, width, *(t.tolist() if t is not None else None for t in (slots, free, past)))
    assert got._fields == ("cu_seqlens", "seq_idx", "positions", "tail_rows", "slots", "n_taken")
    for name, a, e in zip(got._fields, got, want):
        if e is None:
            assert a is None
        else:
            assert a.dtype == torch.int32
            assert a.tolist() == e, name


def test_slot_maps_lengths_that_pass_32_bits():
    from causal_conv1d_b200 import slot_maps_from_lengths

    lengths = torch.tensor([5, 2**31 - 1, 2**31 - 1, 7], dtype=torch.int32, device=DEV)
    got = slot_maps_from_lengths(lengths, 12, 2)
    assert got.cu_seqlens.tolist() == [0, 5, 12, 12, 12]
    assert got.seq_idx.tolist() == [[0] * 5 + [1] * 7]
    with pytest.raises(AssertionError):
        slot_maps_from_lengths(lengths, 12, slots=torch.zeros(4, dtype=torch.int32))  # not on the device


def c_problem(ops):
    """ops (on the device, contiguous, grouped B and C) as the header's structure."""
    from causal_conv1d_b200 import _native as n

    b, t, d = ops["x"].shape
    q = n.SsmProblem(batch=b, seqlen=t, dim=d, dstate=ops["A"].shape[1], groups=ops["B"].shape[2],
                     x_dtype=n.DTYPE_CODE[ops["x"].dtype], dt_softplus=1)
    for k in ("x", "dt", "z", "B", "C"):
        s = ops[k].stride()
        setattr(q, k, n.Tokens(ops[k].data_ptr(), s[0], s[1], s[2] if k in "BC" else 0))
    for k in ("A", "D", "dt_bias", "initial_states"):
        setattr(q, k, n.Param(ops[k].data_ptr(), 0))
    return q


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [1, 2])
def test_c_abi_outputs_at_any_element(dtype, groups):
    """Outputs and gradients that start at any element of a buffer: rows of 16 bytes' multiples from there on
    have the same values as aligned ones, and their neighbours are left alone."""
    from causal_conv1d_b200 import _native as n

    ops = to_dev(ref.case(101, 2, 40, 48, 16, groups, dtype, init=True))
    q, stream, size = c_problem(ops), torch.cuda.current_stream().cuda_stream, 2 * 40 * 48
    dout = torch.randn(2, 40, 48, device=DEV).to(dtype)
    dout_c = n.Tokens(dout.data_ptr(), dout.stride(0), dout.stride(1), 0)
    work = [n.lib.cc1d_ssm_workspace_bytes(2, 40, 48, 16, groups, q.x_dtype, k) for k in (0, 1)]
    ws = torch.empty(max(16, *work), device=DEV, dtype=torch.uint8)
    kept = torch.empty(n.lib.cc1d_ssm_kept_bytes(2, 40, 48, 16), device=DEV, dtype=torch.uint8)

    def run(offset):
        wide = {k: torch.full((size + 16,), 7.0, device=DEV, dtype=dtype) for k in ("out", "dx", "ddt", "dz")}
        at = {k: v.data_ptr() + offset * v.element_size() for k, v in wide.items()}
        dB, dC, dA = torch.empty_like(ops["B"]), torch.empty_like(ops["C"]), torch.empty_like(ops["A"])
        dD, db, di = torch.empty_like(ops["D"]), torch.empty_like(ops["dt_bias"]), torch.empty_like(ops["initial_states"])
        grads = n.SsmGrads(at["dx"], at["ddt"], at["dz"], *(t.data_ptr() for t in (dB, dC, dA, dD, db, di)))
        n.check(n.lib.cc1d_ssm_fwd(ctypes.byref(q), at["out"], None, kept.data_ptr(), None, 0, 0, None, 0, ws.data_ptr(),
                                   work[0], stream), "cc1d_ssm_fwd")
        n.check(n.lib.cc1d_ssm_bwd(ctypes.byref(q), ctypes.byref(dout_c), kept.data_ptr(), None, ctypes.byref(grads),
                                   ws.data_ptr(), work[1], stream), "cc1d_ssm_bwd")
        for v in wide.values():
            assert (v[:offset] == 7).all() and (v[offset + size:] == 7).all()
        return [v[offset:offset + size] for v in wide.values()] + [dB, dC, dA, dD, db, di]

    plain = run(0)
    for offset in (1, 2, 3):
        for a, e in zip(run(offset), plain):
            assert torch.equal(a, e)


@pytest.mark.parametrize("n, seqlen", [(7, 1030), (4097, 9001)])
def test_c_abi_slot_maps_at_any_element(n, seqlen):
    from causal_conv1d_b200 import _native, slot_maps_from_lengths

    lengths = torch.randint(0, 2 * seqlen // n, (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32).to(DEV)
    want = slot_maps_from_lengths(lengths, seqlen, 4)
    for a, b in ((1, 0), (0, 3), (2, 2)):
        seq, pos = (torch.full((seqlen + 8,), 7, device=DEV, dtype=torch.int32) for _ in range(2))
        cu, tail, taken = (torch.empty(k, device=DEV, dtype=torch.int32) for k in (n + 1, 3 * n, 1))
        _native.check(_native.lib.cc1d_slot_maps(
            lengths.data_ptr(), n, seqlen, 4, None, None, None, 0, cu.data_ptr(), seq.data_ptr() + 4 * a, pos.data_ptr() + 4 * b,
            tail.data_ptr(), None, taken.data_ptr(), torch.cuda.current_stream().cuda_stream), "cc1d_slot_maps")
        assert torch.equal(seq[a:a + seqlen], want.seq_idx[0]) and torch.equal(pos[b:b + seqlen], want.positions[0])
        for buf, k in ((seq, a), (pos, b)):
            assert (buf[:k] == 7).all() and (buf[k + seqlen:] == 7).all()
        assert torch.equal(cu, want.cu_seqlens) and torch.equal(tail.view(n, 3), want.tail_rows)


def test_backward_offsets_past_32_bits():
    """So many groups that the sums of the last ones lie past 2^31: one token, so that dB is delta x dy C and
    dC is dy delta x B."""
    from causal_conv1d_b200 import ssm_scan

    groups, n = 2**24 + 40, 33
    g = torch.Generator(device=DEV).manual_seed(3)
    x, dt, dout = (torch.randn(1, 1, groups, generator=g, device=DEV).to(BF16) for _ in range(3))
    B, C = (torch.randn(1, 1, groups, n, generator=g, device=DEV).to(BF16).requires_grad_(True) for _ in range(2))
    A = torch.full((groups, n), -1.0, device=DEV, dtype=BF16)
    dB, dC = torch.autograd.grad(ssm_scan(x, dt, A, B, C), [B, C], dout)
    for part in (slice(0, 1000), slice(groups - 1000, groups)):
        u = (dt[..., part].double() * x[..., part].double() * dout[..., part].double()).unsqueeze(-1)
        ref.assert_near(dB[:, :, part], u * C[:, :, part].double(), 1, "dB")
        ref.assert_near(dC[:, :, part], u * B[:, :, part].double(), 1, "dC")


def test_scan_of_the_longest_row():
    """The most tokens that the header allows, zero but for the last ones: the last of the pieces would end past
    2^31."""
    from causal_conv1d_b200 import ssm_scan

    T, tail = 2**31 - 64, 100
    end = to_dev(ref.case(103, 1, tail, 1, 1, dtype=BF16, D=False, z=False))
    ops = {k: torch.zeros(1, T, 1, device=DEV, dtype=BF16) if k in ("x", "dt", "B", "C") else v for k, v in end.items()}
    for k in ("x", "dt", "B", "C"):
        ops[k][:, -tail:] = end[k]
    out = ssm_scan(**ops, dt_softplus=True)
    ref.assert_near(out[:, -tail:], ref.scan(**ref.wide(end), dt_softplus=True)[0], tail)
    assert not out[:, :-tail].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("seqlen, dstate", [(40, 16), (700, 16), (40, 40)])
def test_nan_in_a_decay_rate(dtype, seqlen, dstate):
    """It reaches its channel's outputs, its own state and its own gradient, and no other channel or state."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(107, 1, seqlen, 24, dstate, dtype=dtype))
    assert (pieces(ops, False) > 1) == (seqlen > 100)
    bad = dict(ops, A=ops["A"].clone())
    bad["A"][5, 3] = float("nan")
    outs = []
    for o in (ops, bad):
        o["A"].requires_grad_(True)
        out, fin = ssm_scan(**o, dt_softplus=True, return_final_states=True)
        (dA,) = torch.autograd.grad(out, [o["A"]], torch.ones_like(out))
        state = torch.zeros(1, 24, dstate, device=DEV)
        token = {k: v.detach() if v is not None else v for k, v in token_ops(o, 0).items()}
        y = ssm_update(ssm_state=state, dt_softplus=True, **token)
        y3 = ssm_update(ssm_state=state.clone(), dt_softplus=True, **{k: v.detach() if v is not None else v for k, v in
                                                                      token_ops(o, slice(0, 3)).items()})
        outs.append((out.detach(), fin.detach(), dA, state, y, y3))
    for clean, got, axis in zip(*outs, (-1, None, None, None, -1, -1)):
        where = torch.zeros_like(clean, dtype=torch.bool)
        if axis == -1:
            where[..., 5] = True
        else:
            where[..., 5, 3] = True
        assert not clean.isnan().any()
        if clean is outs[0][2]:  # the channel's other gradients pass through its output's sum alone
            assert got[5, 3].isnan() and torch.equal(got[~where], clean[~where])
        else:
            assert torch.equal(got.isnan(), where) and torch.equal(got[~where], clean[~where])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("seqlen", [40, 300, 700])  # one piece; pieces chained by themselves, and by a kernel
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("rate", [-20.0, -60.0])
def test_states_stay_non_finite_across_pieces(dtype, seqlen, bad, rate):
    """A state or gradient that is infinite or NaN stays so where a piece's decay underflows, and ends where a
    sequence starts; the others have their usual bits. At a rate of -60 single steps underflow too, where an
    infinity times 0 becomes a NaN."""
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(109, 1, seqlen, 24, 16, dtype=dtype, init=True))
    ops["A"][5, 3] = rate
    ops["dt_bias"][:] = 0.0  # steps of about 0.7: 32 of them times 20 pass what 32 bits hold
    n = pieces(ops, False)
    assert n == 1 if seqlen == 40 else 2 < n <= 16 if seqlen == 300 else n > 16
    dfin = torch.randn(1, 24, 16, device=DEV)
    res = []
    for first, last in ((ops["initial_states"], dfin), [t.index_put((torch.tensor(0), torch.tensor(5), torch.tensor(3)),
                                                                    torch.tensor(bad, device=DEV)) for t in (ops["initial_states"], dfin)]):
        h0 = first.clone().requires_grad_(True)
        out, fin = ssm_scan(**dict(ops, initial_states=h0), dt_softplus=True, return_final_states=True)
        (dh0,) = torch.autograd.grad(fin, h0, last)
        res.append((fin.detach(), dh0))
    for clean, got in zip(*res):
        assert not got[0, 5, 3].isfinite()
        if rate == -20.0:
            assert torch.equal(got[0, 5, 3].nan_to_num(nan=5.0), torch.tensor(bad, device=DEV).nan_to_num(nan=5.0))
        got[0, 5, 3] = clean[0, 5, 3]
        assert clean.isfinite().all() and torch.equal(got, clean)
    # Packed rows: the next sequence does not receive it.
    seq = torch.zeros(1, seqlen, device=DEV, dtype=torch.int32)
    seq[:, seqlen // 2:] = 1
    packed = []
    for first in (0.0, bad):
        h0 = torch.zeros(1, 24, 16, device=DEV)
        h0[0, 5, 3] = first
        packed.append(ssm_scan(**dict(ops, initial_states=h0, seq_idx=seq), dt_softplus=True))
    assert torch.equal(packed[1][:, seqlen // 2:], packed[0][:, seqlen // 2:]) and packed[0].isfinite().all()
    assert not packed[1][0, :seqlen // 2, 5].isfinite().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("seqlen", [300, 700])
def test_nothing_grows_out_of_zero_across_pieces(dtype, seqlen):
    """Growing states (A > 0) whose growth over a piece passes what 32 bits hold: no state before the last tokens,
    no gradient behind the first ones."""
    from causal_conv1d_b200 import ssm_scan

    ops = to_dev(ref.case(113, 1, seqlen, 24, 16, dtype=dtype, z=False))
    # Steps of about 0.7: 32 of them times 5 pass what 32 bits hold, three do not.
    ops["A"], ops["dt_bias"] = 5.0 + ops["A"].abs() / 16, torch.zeros(24, device=DEV)
    ops["x"][:, :-3] = 0.0
    assert pieces(ops, False) > 1 and pieces(ops, True) > 1
    mine = {k: v.clone().requires_grad_(True) if k in ("x", "dt", "B", "C") else v for k, v in ops.items()}
    want = ref.wide(ops)
    out = ssm_scan(**mine, dt_softplus=True)
    wout, _ = ref.scan(**want, dt_softplus=True)
    ref.assert_near(out, wout, seqlen, "out")
    # Only the first three outputs count: the gradient ends there.
    dout = torch.zeros_like(ops["x"])
    dout[:, :3] = torch.randn(1, 3, 24, device=DEV).to(dtype)
    for k in ("x", "dt", "B", "C"):
        want[k] = want[k][:, :3].requires_grad_(True)
    wout, _ = ref.scan(**want, dt_softplus=True)
    got = torch.autograd.grad(out, [mine[k] for k in ("x", "dt", "B", "C")], dout)
    exp = torch.autograd.grad(wout, [want[k] for k in ("x", "dt", "B", "C")], dout[:, :3].double())
    for k, a, e in zip(("x", "dt", "B", "C"), got, exp):
        ref.assert_near(a[:, :3], e, seqlen, "d" + k)
        assert not a[:, 3:].any(), k


def test_autograd_sees_states_written_in_place():
    """A graph that saved a state before an operator wrote to it refuses its backward, as after any in-place
    operation; a state made under inference mode, which has no version, can still be written."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(127, 1, 20, 24, 16, lengths=[[8, 12]]))
    slots = torch.tensor([0, 1], device=DEV)
    token = {k: v.expand(2, *v.shape[1:]) if k in ("x", "dt", "B", "C", "z") else v for k, v in token_ops(ops, 0).items()}
    writes = (lambda s: ssm_update(ssm_state=s, ssm_state_indices=slots, **token),
              lambda s: ssm_scan(**ops, ssm_state=s, ssm_state_indices=slots[None]))
    for write in writes:
        state, w = torch.ones(2, 24, 16, device=DEV), torch.ones(16, device=DEV, requires_grad=True)
        y = (state * w).sum()
        with torch.no_grad():
            write(state)
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
        with torch.inference_mode():
            made = torch.ones(2, 24, 16, device=DEV)
            write(made)
        with torch.no_grad():
            write(made)


@pytest.mark.parametrize("dtype", [F32, F16, torch.float64, torch.complex64])
def test_ids_and_slots_are_integers(dtype):
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(131, 2, 6, 8, 4, lengths=[[2, 4], [6]]))
    state, slots = torch.zeros(4, 8, 4, device=DEV), torch.tensor([[0, 1], [2, -1]], device=DEV)
    with pytest.raises(TypeError, match="seq_idx must be integer"):
        ssm_scan(**dict(ops, seq_idx=ops["seq_idx"].to(dtype)))
    with pytest.raises(TypeError, match="ssm_state_indices must be integer"):
        ssm_scan(**ops, ssm_state=state, ssm_state_indices=slots.to(dtype))
    with pytest.raises(TypeError, match="ssm_state_indices must be integer"):
        ssm_update(ssm_state=state, ssm_state_indices=slots[:, 0].to(dtype), **token_ops(ops, 0))
    assert not state.any()
    for kind in (torch.int64, torch.int32, torch.int16):
        ssm_update(ssm_state=state, ssm_state_indices=slots[:, 0].to(kind), **token_ops(ops, 0))


@pytest.mark.parametrize("dtype, mean", [(F32, 5e-9), (BF16, 1.5e-8), (F16, 1.5e-8)])
def test_decays_have_no_side(dtype, mean):
    """A state left alone for 2000 tokens is the product of 2000 decays: a mean error m of a decay leaves it 2000 m
    off. Arguments of 2^-14 to 2^-5 (in powers of two), the long memories, where that counts.

    16-bit operands: the exponential with its addend, measured per octave over generic arguments, is 1.2e-8 off on
    average at most. 32 bits: rounding to nearest, 5e-8 a step without a side, so five deviations of a state are 5
    sqrt(2000) 5e-8 = 1.1e-5 or 5.6e-9 a token, and the mean over many states lies far inside."""
    from causal_conv1d_b200 import ssm_scan

    T, batch, dim = 2000, 300, 64
    g = torch.Generator(device=DEV).manual_seed(137)
    octave = torch.arange(-14, -6, device=DEV).repeat_interleave(2).float()
    A = -(0.6931471805599453 * 2.0**octave * (1 + 0.5 * torch.rand(dim, 16, generator=g, device=DEV)))
    dt = (1 + torch.rand(batch, T, dim, generator=g, device=DEV) * 0.99).to(dtype)
    x, zero = torch.zeros_like(dt), torch.zeros(batch, T, 16, device=DEV, dtype=dtype)
    ops = dict(x=x, dt=dt, A=A, B=zero, C=zero, seq_idx=None)
    assert pieces(ops, False) == 1
    ones = torch.ones(batch, dim, 16, device=DEV)
    _, fin = ssm_scan(x, dt, A, zero, zero, initial_states=ones, return_final_states=True)
    want = torch.exp(A.double() * dt.double().sum(1)[..., None])
    off = (fin.double() / want - 1).mean((0, 1)) / T
    assert (off.abs() <= mean).all(), off.tolist()


def test_packed_rows_hold_new_requests():
    """What a slot held before does not enter a packed scan; the documented ways to continue a request do."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(139, 1, 30, 24, 16, lengths=[[12, 18]]))
    slots = torch.tensor([2, 0], device=DEV)
    states = []
    for held in (0.0, 3.0):
        states.append(torch.full((4, 24, 16), held, device=DEV))
        with torch.no_grad():
            ssm_scan(**ops, dt_softplus=True, ssm_state=states[-1], ssm_state_indices=slots)
    assert torch.equal(states[0][slots], states[1][slots]) and (states[1][[1, 3]] == 3).all()
    # The first request once more, as the continuation of what its slot holds now.
    first = {k: v[:, :12] if k in ("x", "dt", "B", "C", "z") else v for k, v in ops.items() if k != "seq_idx"}
    whole = dict(ref.wide(ops), seq_idx=None)
    for k in ("x", "dt", "B", "C", "z"):
        whole[k] = torch.cat([whole[k][:, :12]] * 2, 1)
    wout, wh = ref.scan(**whole, dt_softplus=True)
    out, fin = ssm_scan(**dict(first, initial_states=states[0][2:3]), dt_softplus=True, return_final_states=True)
    ref.assert_near(out, wout[:, 12:], 24)
    ref.assert_near(fin, wh[:, -1], 24)
    first.pop("initial_states")
    assert torch.equal(ssm_update(ssm_state=states[0], dt_softplus=True, ssm_state_indices=slots[:1], **first), out)
    assert torch.equal(states[0][2:3], fin)


def test_requests_cut_off_take_their_slots():
    """By their length: the row ends before the last two, whose slots no scan writes."""
    from causal_conv1d_b200 import slot_maps_from_lengths, ssm_scan

    maps = slot_maps_from_lengths(torch.tensor([6, 9, 4, 0, 2], device=DEV), 10, slots=torch.full((5,), -1, device=DEV),
                                  free_slots=torch.arange(7, device=DEV))
    assert maps.slots.tolist() == [0, 1, 2, -1, 3] and maps.n_taken.tolist() == [4]
    assert maps.cu_seqlens.tolist() == [0, 6, 10, 10, 10, 10]
    ops = to_dev(ref.case(149, 1, 10, 8, 4))
    state = torch.full((7, 8, 4), 3.0, device=DEV)
    ssm_scan(**dict(ops, seq_idx=maps.seq_idx), dt_softplus=True, ssm_state=state, ssm_state_indices=maps.slots)
    assert (state[2:] == 3).all() and not (state[:2] == 3).any()


def check_norms(ops, slots=None):
    """Like check_scan, and what comes out in 32 bits also as a whole: within 1e-5 of the 64-bit form in norm.

    A state is carried by decays that are off by 2e-7 each way (exponential, argument, step size), or, over a piece
    of L tokens, by one decay of a sum of L steps, whose argument of size 16 or less (beyond, nothing is left of
    the state) is off by 16 x 2^-24 for its own rounding and as much again for the sum's: 2e-6. A state remembers about
    1/|log a| tokens, and in steps of 0.05 the slowest of them forgets within 20: 20 x 2e-7 + 2e-6 = 6e-6, and the
    gradients, sums of such products without a common sign, stay below that too."""
    from causal_conv1d_b200 import ssm_scan

    g = torch.Generator().manual_seed(11)
    dout = torch.randn(ops["x"].shape, generator=g).to(ops["x"].dtype).to(DEV)
    mine, want = to_dev(ops), ref.wide(to_dev(ops))
    names = [k for k in GRADS if ops[k] is not None]
    final = ops["seq_idx"] is None
    for d in (mine, want):
        for k in names:
            d[k] = d[k].detach().clone().requires_grad_(True)
    res = ssm_scan(**mine, dt_softplus=True, return_final_states=final)
    wout, wh = ref.scan(**want, dt_softplus=True)
    got, exp = {}, {}
    got["out"], exp["out"] = (res[0] if final else res), wout
    if final:
        got["final"], exp["final"] = res[1], wh[:, -1]
    for d, o, w in ((got, mine, dout), (exp, want, dout.double())):
        d.update(zip(names, torch.autograd.grad(d["out"], [o[k] for k in names], w)))
    for k, a in got.items():
        ref.assert_near(a, exp[k], ops["x"].shape[1], k)
        if a.dtype == F32:
            off = ((a.double() - exp[k]).norm() / exp[k].norm()).item()
            assert off <= 1e-5, f"{k}: {off:.3g} off in norm"
    return wh


@pytest.mark.parametrize("batch, seqlen, dim, dstate, groups, dtype, kw, forward, backward", [
    # Pieces chained by themselves, of 2 tiles and of 4 to 16, through which the buffers come round again.
    (1, 300, 200, 16, 0, BF16, {}, 10, 10),
    (2, 1024, 512, 16, 0, F16, dict(init=True), 16, 16),
    (2, 1024, 512, 16, 0, F32, {}, 16, 8),
    (1, 1000, 510, 40, 2, F32, dict(init=True), 8, 4),
    (2, 1000, 1024, 24, 0, BF16, {}, 4, 16),
    # By themselves forward and by the join kernel backward; by the join kernel, 6 tiles each.
    (2, 700, 512, 24, 0, BF16, dict(init=True), 8, 22),
    (1, 3000, 512, 16, 0, BF16, {}, 32, 32),
    # Packed rows: sequences inside a piece, over several, from one's last token to the next one's first.
    (2, 1024, 512, 16, 0, BF16, dict(init=True, lengths=[[10, 500, -2, 1, 319, 64, 128], [1024]]), 16, 16),
    (3, 1021, 516, 12, 3, F32, dict(init=True, lengths=[[1021], [63, 1, 64, 700, -193], [-64, 957]]), 16, 16),
    (1, 3000, 512, 16, 0, F16, dict(lengths=[[96, 95, 1, 1000, 1, 7, -100, 1700]]), 32, 32),
])
def test_pieces_of_every_plan(batch, seqlen, dim, dstate, groups, dtype, kw, forward, backward):
    ops = ref.case(seqlen + dim, batch, seqlen, dim, dstate, groups, dtype, **kw)
    assert (pieces(ops, False), pieces(ops, True)) == (forward, backward)
    check_norms(ops)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch, seqlen, dim, dstate, forward", [(2, 1024, 512, 16, 16), (1, 3000, 200, 16, 32), (2, 700, 512, 24, 8)])
def test_slots_of_a_row_in_pieces(dtype, batch, seqlen, dim, dstate, forward):
    """Sequences that end inside a piece, at its last token and at the row's, each state from its own pieces."""
    from causal_conv1d_b200 import ssm_scan

    rows = [[96, 64, 1, 200, 31, -8, seqlen - 400], [seqlen]][:batch]
    ops = to_dev(ref.case(151, batch, seqlen, dim, dstate, dtype=dtype, lengths=rows))
    assert pieces(ops, False) == forward
    _, h = ref.scan(**ref.wide(ops), dt_softplus=True)
    cache = torch.full((9, dim, dstate), 7.0, device=DEV)
    slots = torch.tensor([[4, 0, 8, 1, -1, 2], [3, 5, 5, 5, 5, 5]], device=DEV)[:batch]
    ssm_scan(**ops, dt_softplus=True, ssm_state=cache, ssm_state_indices=slots)
    ends = {4: (0, 95), 0: (0, 159), 8: (0, 160), 1: (0, 360), 2: (0, seqlen - 1), 3: (1, seqlen - 1)}
    for slot, (b, t) in ends.items():
        if b < batch:
            ref.assert_near(cache[slot], h[b, t], seqlen, f"slot {slot}")
            assert ((cache[slot].double() - h[b, t]).norm() / h[b, t].norm()) <= 1e-5  # check_norms
    for slot in (5, 6, 7, *([3] if batch == 1 else [])):
        assert (cache[slot] == 7).all()


@pytest.mark.parametrize("dtype, state_dtype", [(BF16, F32), (F16, F16), (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("batch, dim, dstate, groups", [
    (77, 2030, 16, 2),   # two groups of rows a CTA, the last one of 5 rows, 14 channels in the last CTA of a row
    (45, 1604, 32, 1),
    (29, 1210, 64, 0),
    (9, 100, 16, 0),     # one group a CTA
    (9, 52, 32, 2),
    (5, 20, 64, 1),
])
def test_decode_batches(dtype, state_dtype, batch, dim, dstate, groups):
    """The one-token kernel with both counts of rows a CTA, rows and channels that fill no CTA, slots in any order."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(157 + batch, batch, 1, dim, dstate, groups, dtype))
    g = torch.Generator(device=DEV).manual_seed(batch)
    state0 = torch.randn(batch + 3, dim, dstate, generator=g, device=DEV).to(state_dtype)
    slots = torch.randperm(batch + 3, generator=g, device=DEV)[:batch]
    skipped = torch.arange(batch, device=DEV) % 11 == 3
    state = state0.clone()
    out = ssm_update(ssm_state=state, dt_softplus=True, ssm_state_indices=torch.where(skipped, -1, slots), **token_ops(ops, 0))
    full = dict(ops, initial_states=state0[slots].float())
    wout, wh = ref.scan(**ref.wide(full), dt_softplus=True)
    live = ~skipped
    ref.assert_near(out[live], wout[live, 0], 1, "out")
    ref.assert_near(state[slots[live]], wh[live, 0], 1, "state")
    untouched = torch.ones(batch + 3, device=DEV, dtype=torch.bool)
    untouched[slots[live]] = False
    assert torch.equal(state[untouched], state0[untouched])
    same, fin = ssm_scan(**full, dt_softplus=True, return_final_states=True)
    assert torch.equal(out[live], same[live, 0])
    if state_dtype == F32:
        assert torch.equal(state[slots[live]], fin[live])


def test_decode_after_a_prompt_in_pieces():
    """A prompt cut in pieces, whose states come through the decay of a summed step, continued token by token:
    within the tolerance of the 64-bit form over the whole sequence, which a scan of it keeps too."""
    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = to_dev(ref.case(163, 1, 520, 512, 16, dtype=BF16))
    prompt = {k: v[:, :512] if k in ("x", "dt", "B", "C", "z") else v for k, v in ops.items()}
    assert pieces(prompt, False) > 1
    wout, wh = ref.scan(**ref.wide(ops), dt_softplus=True)
    out, state = ssm_scan(**prompt, dt_softplus=True, return_final_states=True)
    steps = [ssm_update(ssm_state=state, dt_softplus=True, **token_ops(ops, t)) for t in range(512, 520)]
    ref.assert_near(torch.cat([out, torch.stack(steps, 1)], 1), wout, 520, "out")
    ref.assert_near(state, wh[:, -1], 520, "state")
    assert ((state.double() - wh[:, -1]).norm() / wh[:, -1].norm()) <= 1e-5  # check_norms
