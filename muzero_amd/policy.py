"""Policy rows of any width on the MI355X: log-probabilities of given actions, entropy, log partition, the top
alternatives, and the gradient (muzero_amd/csrc/mzs_policy.hip through the C-ABI; formulas and conventions:
include/mzsearch.h, mzs_policy_args).

The reference computes these inside its policy loss (muzero_model.py:690-700) and action selection (game.py:176-225)
for the few actions of one environment; the actions of a Box space are the cartesian product of
`bin_decomposition_number` samples per dimension (muzero_model.py:994-1051), 10 ** 5 for five dimensions.

There is no CPU path: tensors that are not on a GPU are refused.
"""
import ctypes as C
import struct
from typing import NamedTuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_FLOAT, torch.bfloat16: _lib.DTYPE_BFLOAT, torch.float16: _lib.DTYPE_HALF}


class PolicyLogProbs(NamedTuple):
    """fp32 tensors of the logits' leading shape (top_*: one more dimension, `top` long; None for top = 0)."""
    log_prob: torch.Tensor      # of the given actions; 0 where the action is negative or none were given
    entropy: torch.Tensor
    log_z: torch.Tensor         # log of the sum of exponentials of the tempered logits
    top_log_prob: torch.Tensor  # descending; -inf behind the last allowed action
    top_action: torch.Tensor    # int32; equal logits: the lower index first; -1 behind the last allowed action


# mzs_policy_args as one packed block: filling it field by field through ctypes costs more than the launch
_ARGS = struct.Struct("@iiqqPqPqPiifxxxxPPPPPPPPPPqPN")
assert _ARGS.size == C.sizeof(_lib.PolicyArgs)
_calls = {}


def _call(name):
    f = _calls.get(name)
    if f is None:
        f = _lib.load()[name]       # a function object of its own: the binding in _lib takes the structure
        f.restype, f.argtypes = C.c_int, [C.c_char_p, C.c_void_p]
        _calls[name] = f
    return f


def _no_tangent(*tensors):
    for t in tensors:
        if t is not None and unpack_dual(t).tangent is not None:
            raise ValueError("policy_log_probs: no forward-mode derivatives (a dual tensor); backward ones through the logits")


def _check(logits, actions, mask, temperature, top):
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise ValueError("logits: a tensor [..., n_actions]")
    _no_tangent(logits)
    if not logits.is_cuda:
        raise _lib.MzsError("policy_log_probs: logits must be on a GPU (there is no CPU path)")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits are {logits.dtype}: float32, bfloat16 or float16")
    shape = logits.shape
    n = shape[-1]
    if not 1 <= n <= 2 ** 28:
        raise ValueError(f"{n} actions: 1 .. 2^28")
    if not 1e-30 <= temperature < float("inf"):
        raise ValueError(f"temperature={temperature!r}: positive and finite (at least 1e-30)")
    if not 0 <= top <= _lib.POLICY_MAX_TOP:
        raise ValueError(f"top={top!r}: 0 .. {_lib.POLICY_MAX_TOP}")
    if actions is not None:
        if actions.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"actions are {actions.dtype}: int64 or int32")
        if actions.shape != shape[:-1] or actions.device != logits.device:
            raise ValueError(f"actions {tuple(actions.shape)} on {actions.device}: expected {tuple(shape[:-1])} on {logits.device}")
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"mask is {mask.dtype}: bool (or uint8, 0 / 1)")
        if mask.device != logits.device or mask.shape not in (shape, shape[-1:]):
            raise ValueError(f"mask {tuple(mask.shape)} on {mask.device}: expected {tuple(shape)} or ({n},) on {logits.device}")


def _rows(t, n):
    """`t` as rows of n values, and the elements between two rows (0: every row is the same one); a copy only where the layout
    has no such form."""
    if t.dim() != 2:
        t = t.reshape(-1, n)
    pitch, step = t.stride()
    if (n > 1 and step != 1) or pitch < 0:
        t = t.contiguous()
        pitch = n
    return t, (pitch if t.shape[0] > 1 else n)


def _coefficient(g, name, lead, device):
    if g is None:
        return None
    if g.shape != lead or g.device != device:
        raise ValueError(f"{name} {tuple(g.shape)} on {g.device}: expected {tuple(lead)} on {device}")
    return g if g.dtype is torch.float32 and g.is_contiguous() else g.to(torch.float32).contiguous()


def _overlap(out, logits):
    """Whether the two share elements without being the same view (columns of one wide buffer are apart)."""
    if out.untyped_storage().data_ptr() != logits.untyped_storage().data_ptr() or not out.numel():
        return False
    if out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride():
        return False
    reach = lambda t: 1 + sum((d - 1) * s for d, s in zip(t.shape, t.stride()))  # noqa: E731
    ahead = (out.data_ptr() - logits.data_ptr()) // out.element_size()
    if ahead >= reach(logits) or -ahead >= reach(out):
        return False
    if out.dim() == 2 and out.stride() == logits.stride() and out.shape[0] > 1:
        n, pitch = out.shape[1], out.stride(0)
        return not n <= ahead % pitch <= pitch - n
    return True


def _run(name, logits, actions, mask, temperature, top, saved=None, upstream=None, out=None):
    """One library call.  saved: (entropy, row statistics) of an earlier forward pass, or None: forward values are made here.  upstream:
    the gradient's coefficients, or None: no gradient.  Returns (PolicyLogProbs or None, row statistics, gradient or None)."""
    shape, device = logits.shape, logits.device
    n, dim = shape[-1], logits.dim()
    rows_of, pitch = _rows(logits, n)
    rows = rows_of.shape[0]
    mask_ptr = mask_pitch = action_ptr = action_bytes = 0
    if actions is not None:
        if not actions.is_contiguous():
            actions = actions.contiguous()
        action_ptr, action_bytes = actions.data_ptr(), actions.element_size()
    if mask is not None:
        if mask.dim() == 1 and dim != 1:
            mask = mask.contiguous()
        else:
            mask, mask_pitch = _rows(mask, n)
        mask_ptr = mask.data_ptr()
    values = stats = None
    top_lp = top_at = grad = None
    lp = h = z = st = tl = ta = 0
    if saved is None:
        # tensors of their own: views of one would not take operations in place that autograd records (1.9 us a call more;
        # new_empty for each would be 3.3)
        log_prob = logits.new_empty(shape[:-1], dtype=torch.float32)
        entropy, log_z = torch.empty_like(log_prob), torch.empty_like(log_prob)
        stats = torch.empty_strided((2 * rows,), (1,), dtype=torch.float32, device=device)
        lp, h, z, st = log_prob.data_ptr(), entropy.data_ptr(), log_z.data_ptr(), stats.data_ptr()
        if top:
            top_lp = logits.new_empty((*shape[:-1], top), dtype=torch.float32)
            top_at = torch.empty_like(top_lp, dtype=torch.int32)
            tl, ta = top_lp.data_ptr(), top_at.data_ptr()
        values = PolicyLogProbs(log_prob, entropy, log_z, top_lp, top_at)
    else:
        h, st = saved[0].data_ptr(), saved[1].data_ptr()
    g_lp = g_h = g_z = g = g_pitch = 0
    if upstream is not None:
        g_lp, g_h, g_z = (0 if u is None else u.data_ptr() for u in upstream)
        grad = logits.new_empty(shape) if out is None else out
        g, g_pitch = grad.data_ptr(), (grad.stride(0) if dim == 2 else n)
    if rows:
        args = [device.index, _DTYPES[logits.dtype], rows, n, rows_of.data_ptr(), pitch, mask_ptr, mask_pitch, action_ptr, action_bytes,
                top, 1.0 / temperature, lp, h, z, st, tl, ta, g_lp, g_h, g_z, g, g_pitch, 0, 0]
        if n > _lib.POLICY_NARROW and rows < _lib.POLICY_MANY and saved is None:
            size = C.c_size_t()
            _lib.check(_lib.load().mzs_policy_workspace(_lib.PolicyArgs.from_buffer_copy(_ARGS.pack(*args)), C.byref(size)),
                       "mzs_policy_workspace")
            if size.value:
                workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
                args[-2:] = workspace.data_ptr(), size.value
        rc = _call(name)(_ARGS.pack(*args), _lib.raw_stream(device.index))
        if rc:
            _lib.check(rc, name)
    return values, stats, grad


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, mask, temperature, top):
        out, stats, _ = _run("mzs_policy_log_probs", logits, actions, mask, temperature, top)
        ctx.save_for_backward(logits, actions, mask, out.entropy, stats)
        ctx.temperature = temperature
        if top:
            ctx.mark_non_differentiable(out.top_log_prob, out.top_action)
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    def backward(ctx, *grads):
        # once_differentiable's bookkeeping costs as much as the launch: only where a graph of the gradient is asked for
        return (_slope_once if torch.is_grad_enabled() else _slope)(ctx, *grads)


def _slope(ctx, g_log_prob, g_entropy, g_log_z, *_):
    if g_log_prob is None and g_entropy is None and g_log_z is None:
        return None, None, None, None, None
    logits, actions, mask, entropy, stats = ctx.saved_tensors
    lead, device = logits.shape[:-1], logits.device
    upstream = [g if g is None else _coefficient(g, "gradient", lead, device) for g in (g_log_prob, g_entropy, g_log_z)]
    _, _, grad = _run("mzs_policy_log_probs_grad", logits, actions, mask, ctx.temperature, 0, (entropy, stats), upstream)
    return grad, None, None, None, None


_slope_once = torch.autograd.function.once_differentiable(_slope)


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
    return _run("mzs_policy_log_probs", logits, actions, mask, float(temperature), int(top))[0]


def policy_log_probs_grad(logits, actions=None, grad_log_prob=None, grad_entropy=None, grad_log_z=None, mask=None,
                          temperature=1.0, top=0, out=None):
    """(PolicyLogProbs, gradient of sum(grad_log_prob * log_prob + grad_entropy * entropy + grad_log_z * log_z) by the logits) in
    one call, for coefficients that are known beforehand (advantages over the batch, an entropy bonus): without
    autograd, so it can be captured into a graph.  The coefficients are tensors [...] or None (0).  out: where the
    gradient goes, of the logits' shape and type with dense rows — `logits` itself is allowed and is then overwritten."""
    _no_tangent(grad_log_prob, grad_entropy, grad_log_z)
    _check(logits, actions, mask, temperature, top)
    lead, dev = logits.shape[:-1], logits.device
    coefficients = [_coefficient(g, name, lead, dev) for g, name in
                    ((grad_log_prob, "grad_log_prob"), (grad_entropy, "grad_entropy"), (grad_log_z, "grad_log_z"))]
    if out is not None:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
            raise ValueError(f"out: expected {logits.dtype} {tuple(logits.shape)} on {dev}")
        if not (out.is_contiguous() or (out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= out.shape[1])):
            raise ValueError("out: rows must be dense and apart")
        if _overlap(out, logits):
            raise ValueError("out overlaps the logits: it may be the logits' own view, or apart from them")
    values, _, grad = _run("mzs_policy_log_probs_train", logits, actions, mask, float(temperature), int(top), None,
                           coefficients, out)
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return values, grad
