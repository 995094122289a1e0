"""Policy rows and optimizer, host side: what the C-ABI and the Python wrappers refuse without a GPU."""
import ctypes as C

import pytest
import torch

from muzero_amd import _lib, optim, policy


def args(**kw):
    a = _lib.PolicyArgs()
    a.rows, a.n_actions, a.inverse_temperature, a.logits_stride = 2, 5, 1.0, 5
    for name in ("logits", "entropy", "row_stats", "log_prob", "log_z"):
        setattr(a, name, 4096)      # never followed: every case is refused before a launch
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=3), b"fp32"), (dict(dtype=-1), b"fp32"), (dict(rows=-1), b"rows"), (dict(n_actions=0), b"n_actions"),
    (dict(n_actions=2 ** 31), b"n_actions"), (dict(top=33), b"top"), (dict(top=-1), b"top"),
    (dict(inverse_temperature=0.0), b"temperature"), (dict(inverse_temperature=-1.0), b"temperature"),
    (dict(inverse_temperature=float("inf")), b"temperature"), (dict(inverse_temperature=float("nan")), b"temperature"),
    (dict(logits_stride=-5), b"stride"), (dict(mask_stride=-1), b"stride"), (dict(action=4096, action_bytes=2), b"int32"),
    (dict(logits=None), b"null"), (dict(entropy=None), b"null"), (dict(row_stats=None), b"null"),
    (dict(log_prob=None), b"null"), (dict(log_z=None), b"null"), (dict(top=1), b"null")])
def test_forward_refusals(kw, word):
    lib = _lib.load()
    assert lib.mzs_policy_log_probs(C.byref(args(**kw)), None) == -1
    assert word in lib.mzs_last_error()


@pytest.mark.parametrize("kw, word", [
    (dict(), b"null gradient"), (dict(grad_logits=8192, grad_stride=4), b"overlap"), (dict(grad_logits=8192), b"overlap"),
    (dict(grad_logits=4096, grad_stride=6), b"in place"), (dict(grad_logits=8192, grad_stride=5, entropy=None), b"null")])
def test_gradient_refusals(kw, word):
    lib = _lib.load()
    for call in (lib.mzs_policy_log_probs_grad, lib.mzs_policy_log_probs_train):
        assert call(C.byref(args(**kw)), None) == -1
        assert word in lib.mzs_last_error()


def test_null_arguments():
    lib, size = _lib.load(), C.c_size_t()
    assert lib.mzs_policy_log_probs(None, None) == -1
    assert lib.mzs_policy_workspace(None, C.byref(size)) == -1
    assert lib.mzs_policy_workspace(C.byref(args()), None) == -1
    assert lib.mzs_adamw_step(None, None) == -1
    assert lib.mzs_optim_table(0, 1, None, None, None, None, None) == -1


def test_no_rows_is_nothing_to_do():
    assert _lib.load().mzs_policy_log_probs(C.byref(args(rows=0, logits=None)), None) == 0


def step_args(**kw):
    a = _lib.AdamWArgs()
    a.n, a.n_tiles, a.state_bits, a.lr, a.beta1, a.beta2, a.eps, a.grad_scale = 1, 1, 32, 1e-3, 0.9, 0.999, 1e-8, 1.0
    for name in ("params_table", "grads_table", "exp_avg", "exp_avg_sq", "control_dev", "norm_dev", "workspace"):
        setattr(a, name, 4096)
    a.workspace_bytes = 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, word", [
    (dict(n=-1), b"null"), (dict(params_table=None), b"null"), (dict(grads_table=None), b"null"), (dict(control_dev=None), b"null"),
    (dict(param_dtype=9), b"fp32"), (dict(grad_dtype=-1), b"fp32"), (dict(state_bits=16), b"state_bits"),
    (dict(exp_avg=None), b"null state"), (dict(state_bits=8), b"null state"), (dict(beta1=1.0), b"betas"),
    (dict(beta2=-0.1), b"betas"), (dict(beta1=float("nan")), b"betas"), (dict(eps=-1.0), b"eps"),
    (dict(weight_decay=float("nan")), b"weight_decay"), (dict(max_norm=-1.0), b"max_norm"), (dict(lr=-1.0), b"lr"),
    (dict(grad_scale=float("inf")), b"grad_scale"), (dict(max_norm=1.0, norm_given=1, norm_dev=None), b"norm_given"),
    (dict(max_norm=1.0, workspace=None), b"workspace"), (dict(max_norm=1.0, workspace_bytes=4), b"workspace")])
def test_step_refusals(kw, word):
    lib = _lib.load()
    assert lib.mzs_adamw_step(C.byref(step_args(**kw)), None) == -1
    assert word in lib.mzs_last_error()


def test_norm_refusals():
    lib = _lib.load()
    assert lib.mzs_grad_norm(0, 1, 4096, 1, 7, 1.0, 4096, 4096, 8, None) == -1 and b"fp32" in lib.mzs_last_error()
    assert lib.mzs_grad_norm(0, 1, None, 1, 0, 1.0, 4096, 4096, 8, None) == -1 and b"null" in lib.mzs_last_error()
    assert lib.mzs_grad_norm(0, 1, 4096, 9, 0, 1.0, 4096, 4096, 8, None) == -1 and b"workspace" in lib.mzs_last_error()
    assert lib.mzs_grad_norm(0, 1, 4096, 1, 0, float("nan"), 4096, 4096, 8, None) == -1 and b"scale" in lib.mzs_last_error()
    counts = (C.c_int64 * 1)(-3)
    tiles = C.c_int64()
    assert lib.mzs_optim_table(0, 1, (C.c_void_p * 1)(4096), counts, 4096, C.byref(tiles), None) == -1
    assert b"size" in lib.mzs_last_error()


def test_wrappers_refuse_host_tensors_and_bad_types():
    x = torch.zeros(3, 4)
    with pytest.raises(_lib.MzsError, match="GPU"):
        policy.policy_log_probs(x)
    with pytest.raises(_lib.MzsError, match="GPU"):
        policy.policy_log_probs_grad(x)
    with pytest.raises(ValueError, match="logits"):
        policy.policy_log_probs([1.0, 2.0])
    with pytest.raises(_lib.MzsError, match="GPU"):
        optim.grad_norm([x])
    with pytest.raises(_lib.MzsError, match="GPU"):
        optim.AdamW([x])
    with pytest.raises(ValueError, match="empty"):
        optim.AdamW([])
    with pytest.raises(ValueError, match="empty"):
        optim.grad_norm([None])
    with pytest.raises(ValueError, match="one type"):
        optim.grad_norm([x, x.double()])
    with pytest.raises(ValueError, match="contiguous"):
        optim.grad_norm([torch.zeros(4, 4).t()[1:]])
