"""Policy rows of any width on the MI355X: log-probabilities of given actions, entropy, log partition, the top
alternatives, and the gradient (muzero_amd/csrc/mzs_policy.hip through the C-ABI; formulas and conventions:
include/mzsearch.h, mzs_policy_args).

The reference computes these inside its policy loss (muzero_model.py:690-700) and action selection (game.py:176-225)
for the few actions of one environment; the actions of a Box space are the cartesian product of
`bin_decomposition_number` samples per dimension (muzero_model.py:994-1051), 10 ** 5 for five dimensions.

There is no CPU path: tensors that are not on a GPU are refused.
"""
import ctypes as C
from typing import NamedTuple

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_FLOAT, torch.bfloat16: _lib.DTYPE_BFLOAT, torch.float16: _lib.DTYPE_HALF}


class PolicyLogProbs(NamedTuple):
    """fp32 tensors of the logits' leading shape (top_*: one more dimension, `top` long; None for top = 0)."""
    log_prob: torch.Tensor      # of the given actions; 0 where the action is negative or none were given
    entropy: torch.Tensor
    log_z: torch.Tensor         # log of the sum of exponentials of the tempered logits
    top_log_prob: torch.Tensor  # descending; -inf behind the last allowed action
    top_action: torch.Tensor    # int32; equal logits: the lower index first; -1 behind the last allowed action


def _check(logits, actions, mask, temperature, top):
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise ValueError("logits: a tensor [..., n_actions]")
    if not logits.is_cuda:
        raise _lib.MzsError("policy_log_probs: logits must be on a GPU (there is no CPU path)")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits are {logits.dtype}: float32, bfloat16 or float16")
    n = logits.shape[-1]
    if not 1 <= n <= 2 ** 28:
        raise ValueError(f"{n} actions: 1 .. 2^28")
    if not 1e-30 <= temperature < float("inf"):
        raise ValueError(f"temperature={temperature!r}: positive and finite (at least 1e-30)")
    if not 0 <= top <= _lib.POLICY_MAX_TOP:
        raise ValueError(f"top={top!r}: 0 .. {_lib.POLICY_MAX_TOP}")
    lead = logits.shape[:-1]
    if actions is not None:
        if actions.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"actions are {actions.dtype}: int64 or int32")
        if actions.shape != lead or actions.device != logits.device:
            raise ValueError(f"actions {tuple(actions.shape)} on {actions.device}: expected {tuple(lead)} on {logits.device}")
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"mask is {mask.dtype}: bool (or uint8, 0 / 1)")
        if mask.device != logits.device or mask.shape not in (logits.shape, logits.shape[-1:]):
            raise ValueError(f"mask {tuple(mask.shape)} on {mask.device}: expected {tuple(logits.shape)} or ({n},) on {logits.device}")


def _rows(t, n):
    """`t` as rows of n values, and the elements between two rows (0: every row is the same one); a copy only where the layout
    has no such form."""
    if t.dim() != 2:
        t = t.reshape(-1, n)
    if (n > 1 and t.stride(1) != 1) or t.stride(0) < 0:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else n)


def _coefficient(g, name, lead, device):
    if g is None:
        return None
    if g.shape != lead or g.device != device:
        raise ValueError(f"{name} {tuple(g.shape)} on {g.device}: expected {tuple(lead)} on {device}")
    return g.to(torch.float32).contiguous()


class _Call:
    """The tensors of one library call and its argument block."""

    def __init__(self, logits, actions, mask, temperature, top):
        self.lead, self.device = logits.shape[:-1], logits.device
        n = logits.shape[-1]
        self.logits, stride = _rows(logits, n)
        self.rows = self.logits.shape[0]
        a = self.args = _lib.PolicyArgs()
        a.device, a.dtype, a.rows, a.n_actions = self.device.index, _DTYPES[logits.dtype], self.rows, n
        a.logits, a.logits_stride = self.logits.data_ptr(), stride
        a.inverse_temperature, a.top = 1.0 / temperature, top
        self.actions = self.mask = None
        if actions is not None:
            self.actions = actions.contiguous()
            a.action, a.action_bytes = self.actions.data_ptr(), self.actions.element_size()
        if mask is not None:
            if mask.dim() == 1 and len(self.lead) != 0:
                self.mask, a.mask_stride = mask.contiguous(), 0
            else:
                self.mask, a.mask_stride = _rows(mask, n)
            a.mask = self.mask.data_ptr()

    def outputs(self):
        a, top = self.args, self.args.top
        flat = torch.empty(5 * self.rows, dtype=torch.float32, device=self.device)
        at = flat.data_ptr()
        a.log_prob, a.entropy, a.log_z, a.row_stats = at, at + 4 * self.rows, at + 8 * self.rows, at + 12 * self.rows
        lp, h, z, self.stats = flat.split((self.rows, self.rows, self.rows, 2 * self.rows))
        self.entropy = h
        tl = ta = None
        if top:
            tl = torch.empty(self.lead + (top,), dtype=torch.float32, device=self.device)
            ta = torch.empty(self.lead + (top,), dtype=torch.int32, device=self.device)
            a.top_log_prob, a.top_action = tl.data_ptr(), ta.data_ptr()
        if len(self.lead) != 1:
            lp, h, z = (t.view(self.lead) for t in (lp, h, z))
        return PolicyLogProbs(lp, h, z, tl, ta)

    def gradient(self, grad_log_prob, grad_entropy, grad_log_z, out=None):
        a = self.args
        self.upstream = (grad_log_prob, grad_entropy, grad_log_z)
        a.grad_log_prob, a.grad_entropy, a.grad_log_z = (None if g is None else g.data_ptr() for g in self.upstream)
        if out is None:
            out = torch.empty(self.lead + (a.n_actions,), dtype=self.logits.dtype, device=self.device)
        rows = out if out.dim() == 2 else out.view(-1, a.n_actions)
        a.grad_logits, a.grad_stride = out.data_ptr(), rows.stride(0)
        return out

    def run(self, name):
        lib = _lib.load()
        if self.rows == 0:
            return
        size = C.c_size_t()
        _lib.check(lib.mzs_policy_workspace(C.byref(self.args), C.byref(size)), "mzs_policy_workspace")
        if size.value:
            self.workspace = torch.empty(size.value, dtype=torch.uint8, device=self.device)
            self.args.workspace, self.args.workspace_bytes = self.workspace.data_ptr(), size.value
        stream = torch.cuda.current_stream(self.device).cuda_stream
        _lib.check(getattr(lib, name)(C.byref(self.args), C.c_void_p(stream)), name)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, mask, temperature, top):
        call = _Call(logits, actions, mask, temperature, top)
        out = call.outputs()
        call.run("mzs_policy_log_probs")
        ctx.save_for_backward(logits, actions, mask, out.entropy, call.stats)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(*(t for t in out[3:] if t is not None))
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_log_prob, g_entropy, g_log_z, *_):
        logits, actions, mask, entropy, stats = ctx.saved_tensors
        call = _Call(logits, actions, mask, ctx.temperature, 0)
        if g_log_prob is None and g_entropy is None and g_log_z is None:
            return None, None, None, None, None
        grads = (_coefficient(g, "gradient", call.lead, call.device) for g in (g_log_prob, g_entropy, g_log_z))
        call.args.entropy, call.args.row_stats = entropy.data_ptr(), stats.data_ptr()
        grad = call.gradient(*grads)
        call.run("mzs_policy_log_probs_grad")
        return grad, None, None, None, None


def policy_log_probs(logits, actions=None, mask=None, temperature=1.0, top=0):
    """PolicyLogProbs of logits [..., n_actions] (float32, bfloat16 or float16, any row stride): the log-probability of actions [...]
    (int64 / int32; negative: none), the entropy, the log partition and the `top` (<= 32) most likely alternatives of
    softmax(logits / temperature) over the actions that mask ([..., n_actions] or [n_actions], bool) allows.

    Differentiable by the logits through log_prob, entropy and log_z (once).  Inside a graph capture a differentiable
    call is refused: there policy_log_probs_grad takes the coefficients directly.  Rows that allow nothing: log_prob and log_z -inf, entropy 0,
    gradient 0.  An action >= n_actions gives NaN.  Runs on the current stream of the logits' device."""
    _check(logits, actions, mask, temperature, top)
    if torch.is_grad_enabled() and logits.requires_grad:
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("policy_log_probs: a differentiable call is not captured into a graph (its backward pass would meet the "
                             "leaves' eager streams there, which ends the process); capture policy_log_probs_grad, or detach the logits")
        return PolicyLogProbs(*_LogProbs.apply(logits, actions, mask, float(temperature), int(top)))
    call = _Call(logits, actions, mask, float(temperature), int(top))
    out = call.outputs()
    call.run("mzs_policy_log_probs")
    return out


@torch.no_grad()
def policy_log_probs_grad(logits, actions=None, grad_log_prob=None, grad_entropy=None, grad_log_z=None, mask=None,
                          temperature=1.0, top=0, out=None):
    """(PolicyLogProbs, gradient of sum(grad_log_prob * log_prob + grad_entropy * entropy + grad_log_z * log_z) by the logits) in
    one call, for coefficients that are known beforehand (advantages over the batch, an entropy bonus): without
    autograd, so it can be captured into a graph.  The coefficients are tensors [...] or None (0).  out: where the
    gradient goes, of the logits' shape and type with dense rows — `logits` itself is allowed and is then overwritten."""
    _check(logits, actions, mask, temperature, top)
    lead, dev = logits.shape[:-1], logits.device
    coefficients = [_coefficient(g, name, lead, dev) for g, name in
                    ((grad_log_prob, "grad_log_prob"), (grad_entropy, "grad_entropy"), (grad_log_z, "grad_log_z"))]
    if out is not None:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
            raise ValueError(f"out: expected {logits.dtype} {tuple(logits.shape)} on {dev}")
        if not (out.is_contiguous() or (out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= out.shape[1])):
            raise ValueError("out: rows must be dense and apart")
        if out.data_ptr() == logits.data_ptr() and out.stride() != logits.stride():
            raise ValueError("out: in place of the logits it must be the logits' own view")
    call = _Call(logits, actions, mask, float(temperature), int(top))
    values = call.outputs()
    grad = call.gradient(*coefficients, out=out)
    call.run("mzs_policy_log_probs_train")
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return values, grad
