"""Optimizer over many tensors on the MI355X: the global gradient norm and the AdamW step, each one walk over all tensors
(muzero_amd/csrc/mzs_optim.hip through the C-ABI; formulas: include/mzsearch.h, mzs_adamw_args).

The reference's optimizers are torch.optim.Adam / SGD (muzero_model.py:418-421), which Trainer runs on the built-in models'
weight blob; AdamW here takes any list of parameters in fp32, bf16 or fp16, with fp32 or 8-bit states.
"""
import ctypes as C

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_FLOAT, torch.bfloat16: _lib.DTYPE_BFLOAT, torch.float16: _lib.DTYPE_HALF}


def _check_tensors(tensors, what):
    if not tensors:
        raise ValueError(f"{what}: an empty list")
    first = tensors[0]
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what}[{i}]: not a tensor")
        if t.dtype is not first.dtype or t.device != first.device:
            raise ValueError(f"{what}[{i}] is {t.dtype} on {t.device}, {what}[0] {first.dtype} on {first.device}: one list, one type and device")
        if not t.is_contiguous():
            raise ValueError(f"{what}[{i}]: not contiguous")
    if not first.is_cuda:
        raise _lib.MzsError(f"{what}: tensors must be on a GPU (there is no CPU path)")
    if first.dtype not in _DTYPES:
        raise ValueError(f"{what} are {first.dtype}: float32, bfloat16 or float16")


class _Table:
    """Device table of tensors (mzs_optim_table), written on the current stream."""

    def __init__(self, device, pointers, counts):
        n = len(counts)
        self.counts, self.device = counts, device
        self.memory = torch.empty((n + 1) * _lib.OPTIM_ENTRY_BYTES, dtype=torch.uint8, device=device)
        tiles = C.c_int64()
        _lib.check(_lib.load().mzs_optim_table(device.index, n, (C.c_void_p * n)(*pointers), (C.c_int64 * n)(*counts),
                                               self.memory.data_ptr(), C.byref(tiles), _lib.raw_stream(device.index)),
                   "mzs_optim_table")
        self.n, self.tiles, self.ptr = n, tiles.value, self.memory.data_ptr()


class _Written:
    """Memory that the current stream has written last, for users on other streams: use() before each."""

    def __init__(self, device, tensors):
        stream = torch.cuda.current_stream(device)
        self.device, self.tensors, self._seen = device, tensors, {stream.cuda_stream}
        self._event = torch.cuda.Event()
        self._event.record(stream)

    def use(self, raw_stream):
        if raw_stream not in self._seen:
            self._event.synchronize()       # once per stream; on the host, so that a capture records nothing of it
            stream = torch.cuda.current_stream(self.device)
            for t in self.tensors:          # freed, it is not given out again before that stream's work so far is done
                t.record_stream(stream)
            self._seen.add(raw_stream)


class TensorList:
    """A list of tensors laid out once for grad_norm and AdamW.step: for gradients that stay in the same buffers from step
    to step.  The list refers to (and keeps alive) the memory the tensors have now: gradients that zero_grad() drops and
    backward() makes anew are not in it.  Not made inside a graph capture; used inside one (grad_norm) it has to live as
    long as the graph, AdamW.step keeps it itself."""

    def __init__(self, tensors):
        tensors = list(tensors)
        _check_tensors(tensors, "tensors")
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("TensorList: its table would hold nothing before the graph's first replay; make it before the capture")
        self.tensors = [t.detach() for t in tensors]
        self.dtype, self.device = tensors[0].dtype, tensors[0].device
        self.counts = tuple(t.numel() for t in tensors)
        self.table = _Table(self.device, [t.data_ptr() for t in tensors], self.counts)
        self._written = _Written(self.device, [self.table.memory])

    def __len__(self):
        return len(self.counts)


def grad_norm(grads, scale=1.0):
    """sqrt of the sum of squares over all gradients, times |scale|: a 0-d float32 tensor, summed in fp64 in a fixed order.
    grads: a tensor, a list of tensors of one type (None: left out), or a TensorList.  No gradient flows through it."""
    if isinstance(grads, TensorList):
        dev, dtype, table = grads.device, grads.dtype, grads.table
        stream = _lib.raw_stream(dev.index)
        grads._written.use(stream)
    else:
        grads = [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]
        _check_tensors(grads, "grads")
        dev, dtype = grads[0].device, grads[0].dtype
        table = _Table(dev, [g.data_ptr() for g in grads], [g.numel() for g in grads])
        stream = _lib.raw_stream(dev.index)
    lib = _lib.load()
    size = lib.mzs_grad_norm_workspace(table.tiles)
    memory = torch.empty(size // 4 + 1, dtype=torch.float32, device=dev)
    _lib.check(lib.mzs_grad_norm(dev.index, table.n, table.ptr, table.tiles, _DTYPES[dtype], float(scale),
                                 memory.data_ptr() + size, memory.data_ptr(), size, stream), "mzs_grad_norm")
    return memory[size // 4]


class AdamW:
    """AdamW (decoupled weight decay, bias correction) over a list of contiguous parameters of one type and device.

    state_bits 32: fp32 moments.  8: the first moment and the root of the second as e4m3 codes, one power-of-two exponent per 32 elements,
    rounded up or down by a counter-based dither from `seed` (2.06 bytes per parameter instead of 8).
    master_weights: fp32 copies of bf16 / fp16 parameters are what the step updates; the parameters are their roundings, so
    values written into the parameters afterwards last until the next step unless they go into state_tensors()["master"] too.
    max_grad_norm: gradients are scaled so that their global norm is at most that; a norm that is not finite skips the step.

    The step counter is on the device: a captured step() replays as the steps that follow.  lr may be a float or a 0-d
    float32 tensor on the GPU (which a captured step reads at every replay).  lr, betas, eps, weight_decay, max_grad_norm and
    seed are read by every step() and may be changed between steps (a replayed step keeps those of its capture).
    Parameters whose gradient is None are left as they are.  Not made inside a graph capture."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 master_weights=False, max_grad_norm=None, seed=0):
        params = list(params)
        _check_tensors(params, "params")
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("AdamW: its states and table would hold nothing before the graph's first replay; make it before the capture")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits={state_bits!r}: 32 or 8")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas={betas!r}: each in [0, 1)")
        if not (eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError("eps and weight_decay must not be negative")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm={max_grad_norm!r}: positive, or None")
        if master_weights and params[0].dtype is torch.float32:
            raise ValueError("master_weights: the parameters are float32 already")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("params overlap in memory: a tensor may appear once")
        self.params, self.lr, self.betas, self.eps, self.weight_decay = params, lr, tuple(betas), eps, weight_decay
        self.state_bits, self.max_grad_norm, self.seed = state_bits, max_grad_norm, int(seed)
        self.device = dev = params[0].device
        self.counts = tuple(p.numel() for p in params)
        self.starts, end = [], 0
        for c in self.counts:
            self.starts.append(end)
            end += -(-c // _lib.OPTIM_ALIGN) * _lib.OPTIM_ALIGN
        self.control = torch.zeros(_lib.OPTIM_CONTROL_BYTES // 4, dtype=torch.int32, device=dev)
        self.grad_norm = torch.zeros((), dtype=torch.float32, device=dev)
        zeros = lambda n, t: torch.zeros(n, dtype=torch.uint8, device=dev).view(t)  # noqa: E731
        self._state = {"exp_avg": torch.zeros(end, device=dev) if state_bits == 32 else zeros(end, torch.float8_e4m3fn)}
        if state_bits == 32:
            self._state["exp_avg_sq"] = torch.zeros(end, device=dev)
        else:
            self._state["exp_avg_exponent"] = zeros(end // _lib.OPTIM_BLOCK, torch.float8_e8m0fnu)
            self._state["exp_avg_root"] = zeros(end, torch.float8_e4m3fn)
            self._state["exp_avg_root_exponent"] = zeros(end // _lib.OPTIM_BLOCK, torch.float8_e8m0fnu)
        if master_weights:
            self._state["master"] = master = torch.zeros(end, device=dev)
            with torch.no_grad():
                for p, at in zip(params, self.starts):
                    master[at:at + p.numel()].copy_(p.detach().reshape(-1))
        self._pointers = [p.data_ptr() for p in params]
        self._params_table = _Table(dev, self._pointers, self.counts)
        a = self._args = _lib.AdamWArgs()
        size = _lib.load().mzs_grad_norm_workspace(self._params_table.tiles)
        self._workspace = torch.empty(size, dtype=torch.uint8, device=dev)      # as the states, for one step at a time
        a.workspace, a.workspace_bytes = self._workspace.data_ptr(), size
        a.device, a.n, a.param_dtype, a.state_bits = dev.index, len(params), _DTYPES[params[0].dtype], state_bits
        a.exp_avg = self._state["exp_avg"].data_ptr()
        a.exp_avg_sq = self._state["exp_avg_sq" if state_bits == 32 else "exp_avg_root"].data_ptr()
        if state_bits == 8:
            a.exp_avg_exponent = self._state["exp_avg_exponent"].data_ptr()
            a.exp_avg_sq_exponent = self._state["exp_avg_root_exponent"].data_ptr()
        if master_weights:
            a.master = self._state["master"].data_ptr()
        a.control_dev = self.control.data_ptr()
        self._written = _Written(dev, [self.control, self.grad_norm, self._workspace, *self._state.values()])
        self._params_written = _Written(dev, [self._params_table.memory])
        self._captured = []     # what graphs read of tables, for as long as this optimizer lives

    # ------------------------------------------------------------------ state
    def state_tensors(self):
        """The flat state buffers (tensor i: counts[i] elements from starts[i] on; zeros between)."""
        return dict(self._state)

    @property
    def step_count(self):
        """Steps taken so far (reads the device)."""
        return int(self.control[0].item())

    @property
    def skipped_count(self):
        """Steps skipped for a norm that was not finite (reads the device)."""
        return int(self.control[1].item())

    def state_dict(self):
        return {"step": self.step_count, "seed": self.seed, **{k: v.clone() for k, v in self._state.items()}}

    def load_state_dict(self, state):
        """Copies the values in (keys of state_dict(); "seed" may be left out)."""
        missing = {"step", *self._state} - set(state)
        unknown = set(state) - {"step", "seed", *self._state}
        if missing or unknown:
            raise ValueError(f"optimizer state: missing {sorted(missing)}, unknown {sorted(unknown)}")
        for k, v in self._state.items():
            if state[k].shape != v.shape or state[k].dtype is not v.dtype:
                raise ValueError(f"optimizer state {k!r}: {state[k].dtype} {tuple(state[k].shape)}, expected {v.dtype} {tuple(v.shape)}")
        if int(state["step"]) < 0:
            raise ValueError("optimizer state: negative step")
        for k, v in self._state.items():
            v.view(torch.uint8).copy_(state[k].view(torch.uint8))
        self.control[0] = int(state["step"])
        if "seed" in state:
            self.seed = int(state["seed"])

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    # ------------------------------------------------------------------- step
    def _grad_table(self, grads):
        if isinstance(grads, TensorList):
            if grads.counts != self.counts or grads.device != self.device:
                raise ValueError("gradients do not match the parameters (sizes and device)")
            return grads.table, grads.dtype
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        there = [g for g in grads if g is not None]
        if not there:
            raise ValueError("no parameter has a gradient")
        _check_tensors(there, "grads")
        if there[0].device != self.device:
            raise ValueError(f"gradients on {there[0].device}, parameters on {self.device}")
        for i, (g, c) in enumerate(zip(grads, self.counts)):
            if g is not None and g.numel() != c:
                raise ValueError(f"grads[{i}]: {g.numel()} elements, the parameter has {c}")
        return _Table(self.device, [None if g is None else g.data_ptr() for g in grads], self.counts), there[0].dtype

    def step(self, grads=None, norm=None, grad_scale=1.0):
        """One step on the current stream.  grads: a list (None entries: no gradient), a TensorList, or None: the parameters'
        .grad.  norm: the norm to clip by (a 0-d float32 tensor) where it covers more than these parameters; None: computed
        here when max_grad_norm is set.  grad_scale multiplies the gradients (1 / loss scale).  grad_norm holds the norm."""
        stream = _lib.raw_stream(self.device.index)
        self._written.use(stream)
        if isinstance(grads, TensorList):
            grads._written.use(stream)
        capturing = torch.cuda.is_current_stream_capturing()
        table, dtype = self._grad_table(grads)
        pointers = [p.data_ptr() for p in self.params]
        params_table = self._params_table
        if pointers != self._pointers:      # a parameter's storage was replaced
            _check_tensors(self.params, "params")
            if (tuple(p.numel() for p in self.params) != self.counts or self.params[0].device != self.device or
                    _DTYPES[self.params[0].dtype] != self._args.param_dtype):
                raise ValueError("the parameters' sizes, type or device changed")
            params_table = _Table(self.device, pointers, self.counts)
            if not capturing:       # a table written inside a graph is that graph's alone
                self._params_table, self._pointers = params_table, pointers
                self._params_written = _Written(self.device, [params_table.memory])
        else:
            self._params_written.use(stream)
        if capturing:
            read = [t for t in (params_table, grads) if t is self._params_table or isinstance(t, TensorList)]
            self._captured += [t for t in read if all(t is not c for c in self._captured)]
        a = self._args
        a.n_tiles, a.params_table, a.grads_table = params_table.tiles, params_table.ptr, table.ptr
        a.grad_dtype, a.grad_scale = _DTYPES[dtype], float(grad_scale)
        a.beta1, a.beta2 = self.betas
        a.eps, a.weight_decay, a.seed = self.eps, self.weight_decay, self.seed & (2 ** 64 - 1)
        lr = self.lr
        if isinstance(lr, torch.Tensor):
            if lr.dtype is not torch.float32 or lr.device != self.device or lr.numel() != 1:
                raise ValueError("lr: a float, or one float32 value on the parameters' device")
            a.lr_dev, a.lr = lr.data_ptr(), 0.0
        else:
            a.lr_dev, a.lr = None, float(lr)
        a.max_norm, a.norm_given, a.norm_dev = float(self.max_grad_norm or 0.0), 0, self.grad_norm.data_ptr()
        if norm is not None:
            if self.max_grad_norm is None:
                raise ValueError("norm: this optimizer has no max_grad_norm")
            if norm.dtype is not torch.float32 or norm.device != self.device or norm.numel() != 1:
                raise ValueError("norm: one float32 value on the parameters' device")
            self.grad_norm.copy_(norm.reshape(()))
            a.norm_given = 1
        _lib.check(_lib.load().mzs_adamw_step(C.byref(a), stream), "mzs_adamw_step")
        torch.autograd.graph.increment_version(self.params)
