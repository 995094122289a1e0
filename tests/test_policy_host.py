"""Policy rows and optimizer, host side: what the C-ABI and the Python wrappers refuse without a GPU."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from muzero_amd import _lib, optim, policy

HERE = os.path.dirname(os.path.abspath(__file__))


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


def plan_check(tmp_path, calls):
    """(launches, workspace bytes, chunks a row) of each call [rows, logits, logits per vector, top]; the program fails on a plan whose launches
    need more workspace than the call was told."""
    exe = tmp_path / "policy_plan_check"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-o", str(exe), os.path.join(HERE, "csrc", "policy_plan_check.cpp")])
    out = subprocess.run([str(exe), *(str(v) for c in calls for v in c)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
    return [tuple(int(v) for v in line.split()) for line in out.stdout.splitlines()[:-1]]


def test_every_launch_of_a_call_follows_the_call_s_plan(tmp_path):
    """Rows around 128 (fewer are cut) and around whole launches, whose rest must not be cut by itself."""
    rows = [k * 2 ** 20 + r for k in (0, 1, 2, 16, 17) for r in (0, 1, 2, 5, 40, 127, 128, 129, 2 ** 20 - 1) if k or r]
    calls = [(r, n, per, top) for r in rows for n in (1, 8, 9, 2048, 2049, 4096, 4097, 8192, 8193, 49151, 49152, 50000, 2 ** 20, 2 ** 28)
             for per in (4, 8) for top in (0, 5)]
    plans = plan_check(tmp_path, calls)
    assert max(p[0] for p in plans) > 16 and max(p[2] for p in plans) == 256
    lib, size = _lib.load(), C.c_size_t()
    for (r, n, per, top), (_, workspace, _) in zip(calls, plans):
        a = args(rows=r, n_actions=n, dtype=_lib.DTYPE_FLOAT if per == 4 else _lib.DTYPE_HALF, top=top)
        assert lib.mzs_policy_workspace(C.byref(a), C.byref(size)) == 0 and size.value == workspace
        if n <= _lib.POLICY_NARROW or r >= _lib.POLICY_MANY:
            assert workspace == 0


def test_a_cut_call_without_its_workspace_is_refused():
    lib = _lib.load()
    a = args(rows=5, n_actions=50000, logits_stride=0, dtype=_lib.DTYPE_BFLOAT)
    size = C.c_size_t()
    assert lib.mzs_policy_workspace(C.byref(a), C.byref(size)) == 0 and size.value > 0
    for given, at in ((0, None), (size.value - 1, 4096), (size.value, None)):
        a.workspace, a.workspace_bytes = at, given
        assert lib.mzs_policy_log_probs(C.byref(a), None) == -1 and b"workspace" in lib.mzs_last_error()


def test_what_a_capture_would_leave_unwritten_is_not_made_there(monkeypatch):
    """Refused before anything is allocated."""
    monkeypatch.setattr(optim, "_check_tensors", lambda tensors, what: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for make in (optim.AdamW, optim.TensorList):
        with pytest.raises(ValueError, match="before the capture"):
            make([torch.zeros(3)])


def test_forward_mode_derivatives_are_refused():
    """A dual tensor has no requires_grad: without a look for its tangent the call would drop it."""
    from torch.autograd import forward_ad
    x, one = torch.zeros(3, 4), torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3, 4))
        for call in (lambda: policy.policy_log_probs(dual), lambda: policy.policy_log_probs_grad(dual),
                     lambda: policy.policy_log_probs_grad(x, None, forward_ad.make_dual(one, one)),
                     lambda: policy.policy_log_probs_grad(x, None, None, forward_ad.make_dual(one, one)),
                     lambda: policy.policy_log_probs_grad(x, None, None, None, forward_ad.make_dual(one, one))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        with pytest.raises(_lib.MzsError, match="GPU"):     # a tensor without a tangent is none of its business
            policy.policy_log_probs(x)


@pytest.mark.parametrize("optimizer", ["adam", "sgd"])
def test_the_trainer_refuses_options_of_another_optimizer(optimizer):
    from muzero_amd.train import Trainer
    for kw, word in ((dict(weight_decay=0.1), "weight_decay"), (dict(weight_decay=0.0), "weight_decay"), (dict(max_grad_norm=1.0), "max_grad_norm")):
        with pytest.raises(ValueError, match=word):
            Trainer(None, 5, 8, optimizer, **kw)        # before it looks at the engine
