"""State-space operators without a GPU: the 64-bit restatement against differences, the package's
refusals, and the C entry points' checks of their arguments, which come before any CUDA call."""

import ctypes

import pytest
import torch

import _ssm_ref as ref


def test_restatement_gradients_match_differences():
    ops = ref.wide(ref.case(0, 2, 7, 4, 3, groups=2, init=True, lengths=[[3, 2, -2], [-1, 4, 2]]))
    names = [k for k, v in ops.items() if torch.is_tensor(v) and v.is_floating_point()]

    def f(*vals):
        return ref.scan(**{**ops, **dict(zip(names, vals))}, dt_softplus=True)[0]

    assert torch.autograd.gradcheck(f, [ops[k].requires_grad_(True) for k in names])


def operands(**kw):
    ops = ref.case(1, 2, 5, 6, 4, groups=0, init=False)
    ops.update(kw)
    return ops


@pytest.mark.parametrize("kw, error", [
    (dict(x=torch.randn(5, 6)), AssertionError),
    (dict(dt=torch.randn(2, 5, 7)), AssertionError),
    (dict(z=torch.randn(2, 4, 6)), AssertionError),
    (dict(A=torch.randn(5, 4)), AssertionError),
    (dict(A=torch.randn(6, 65), B=torch.randn(2, 5, 65), C=torch.randn(2, 5, 65)), AssertionError),
    (dict(A=torch.randn(6, 0), B=torch.randn(2, 5, 0), C=torch.randn(2, 5, 0)), AssertionError),
    (dict(B=torch.randn(2, 5, 3)), AssertionError),
    (dict(B=torch.randn(2, 5, 4, 4), C=torch.randn(2, 5, 4, 4)), AssertionError),  # 6 channels, 4 groups
    (dict(D=torch.randn(7)), AssertionError),
    (dict(dt_bias=torch.randn(6, 1)), AssertionError),
    (dict(x=torch.randn(2, 5, 6).double()), TypeError),
    (dict(B=torch.randn(2, 5, 4).half()), TypeError),
    (dict(A=torch.ones(6, 4, dtype=torch.int32)), TypeError),
    (dict(), AssertionError),  # not on a CUDA device
])
def test_scan_refuses(kw, error):
    from causal_conv1d_b200 import ssm_scan

    with pytest.raises(error):
        ssm_scan(**operands(**kw))


@pytest.mark.parametrize("kw, error", [
    (dict(x=torch.randn(2, 1, 1, 6)), AssertionError),
    (dict(A=torch.randn(5, 4)), AssertionError),
    (dict(B=torch.randn(2, 5, 4), C=torch.randn(2, 5, 4)), AssertionError),  # 6 channels, 5 groups
    (dict(dt=torch.randn(2, 6).half()), TypeError),
    (dict(), AssertionError),
])
def test_update_refuses(kw, error):
    from causal_conv1d_b200 import ssm_update

    ops = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in operands().items()
           if k not in ("seq_idx", "initial_states")}
    ops.update(kw)
    with pytest.raises(error):
        ssm_update(ssm_state=torch.zeros(2, 6, 4), **ops)


@pytest.mark.parametrize("args, kw, error", [
    ((torch.ones(2, 2, dtype=torch.int32), 8), {}, AssertionError),
    ((torch.ones(2), 8), {}, TypeError),
    ((torch.ones(2, dtype=torch.int32), -1), {}, AssertionError),
    ((torch.ones(2, dtype=torch.int32), 8), dict(width=0), AssertionError),
    ((torch.ones(2, dtype=torch.int32), 8), dict(free_slots=torch.arange(3)), AssertionError),
    ((torch.ones(2, dtype=torch.int32), 8), dict(slots=torch.zeros(3, dtype=torch.int32)), AssertionError),
    ((torch.ones(2, dtype=torch.int32), 8), {}, AssertionError),  # not on a CUDA device
])
def test_slot_maps_refuses(args, kw, error):
    from causal_conv1d_b200 import slot_maps_from_lengths

    with pytest.raises(error):
        slot_maps_from_lengths(*args, **kw)


def test_c_entry_points_refuse_before_any_device_work():
    from causal_conv1d_b200 import _native as n

    lib = n.lib

    def problem(**kw):
        q = n.SsmProblem(batch=1, seqlen=8, dim=6, dstate=4, groups=1, x_dtype=2)
        for k, v in kw.items():
            setattr(q, k, v)
        return ctypes.byref(q)

    def fwd(q, out=None, packed=None):
        return lib.cc1d_ssm_fwd(q, out, None, None, packed, 0, 1, None, 0, None, 0, None)

    bad = n.CC1D_ERR_INVALID
    assert lib.cc1d_ssm_fwd(None, None, None, None, None, 0, 0, None, 0, None, 0, None) == bad
    assert fwd(problem(x_dtype=9)) == bad
    assert fwd(problem(batch=-1)) == bad
    assert fwd(problem(dim=7, groups=2)) == bad
    assert fwd(problem(dstate=0)) == bad
    assert fwd(problem(dstate=65)) == n.CC1D_ERR_UNSUPPORTED
    assert fwd(problem()) == bad  # operands missing
    assert fwd(problem(), packed=8) == bad  # a packed state without seq_idx
    assert fwd(problem(seqlen=0)) == n.CC1D_OK
    assert lib.cc1d_ssm_bwd(problem(), None, None, None, None, None, 0, None) == bad
    assert lib.cc1d_ssm_update(problem(), None, 5, 1, None, None, None) == bad
    assert lib.cc1d_ssm_update(problem(batch=3), None, 0, 2, None, None, None) == bad  # fewer slots than rows
    assert lib.cc1d_ssm_kept_bytes(1, 17, 8, 16) == 2 * 8 * 16 * 4
    assert lib.cc1d_ssm_kept_bytes(1, 17, 8, 65) == -1
    assert lib.cc1d_ssm_workspace_bytes(1, 8, 7, 4, 2, 0, 0) == -1
    assert lib.cc1d_ssm_workspace_bytes(1, 8, 8, 4, 2, 7, 0) == -1
    assert lib.cc1d_ssm_workspace_bytes(0, 8, 8, 4, 2, 2, 1) == 0
    assert lib.cc1d_slot_maps(None, 2, 8, 1, None, None, None, 0, None, None, None, None, None, None, None) == bad
    assert lib.cc1d_slot_maps(None, -1, 8, 1, None, None, None, 0, None, None, None, None, None, None, None) == bad


def test_c_entry_points_refuse_unaligned_scratch():
    """Kept states and workspaces move in 16-byte vectors. The addresses are never read: the refusal comes
    before any device work."""
    from causal_conv1d_b200 import _native as n

    q = n.SsmProblem(batch=1, seqlen=8, dim=8, dstate=4, groups=1, x_dtype=2)
    for k in ("x", "dt", "B", "C"):
        setattr(q, k, n.Tokens(4096, 64, 8, 8))
    q.A = n.Param(4096, 0)
    grads = n.SsmGrads(*([4096] * 6))
    dout = n.Tokens(4096, 64, 8, 0)
    for kept, workspace in ((4100, 4096), (4096, 4104)):
        assert n.lib.cc1d_ssm_fwd(ctypes.byref(q), 4096, None, kept, None, 0, 0, None, 0, workspace, 1 << 30, None) == n.CC1D_ERR_INVALID
        assert n.lib.cc1d_ssm_bwd(ctypes.byref(q), ctypes.byref(dout), kept, None, ctypes.byref(grads), workspace, 1 << 30,
                                  None) == n.CC1D_ERR_INVALID


@pytest.mark.parametrize("name", ["x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_states", "ssm_state"])
def test_forward_mode_is_refused(name):
    """A tangent would be lost without a word (nothing requires grad in forward mode)."""
    import torch.autograd.forward_ad as fwad

    from causal_conv1d_b200 import ssm_scan, ssm_update

    ops = operands(initial_states=torch.zeros(2, 6, 4))
    token = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in ops.items() if k not in ("seq_idx", "initial_states")}
    token["ssm_state"] = torch.zeros(2, 6, 4)
    with fwad.dual_level():
        for fn, args in ((ssm_scan, ops), (ssm_update, token)):
            if name in args:
                dual = fwad.make_dual(args[name], torch.ones_like(args[name]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(**{**args, name: dual})


def test_error_texts_name_no_other_entry_point():
    from causal_conv1d_b200 import _native as n

    text = n.lib.cc1d_error_string(n.CC1D_ERR_WORKSPACE).decode()
    assert "workspace" in text and "cc1d_bwd" not in text
