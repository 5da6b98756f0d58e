"""AdamW over many tensors at once (C ABI: dp_adamw_step), moments in 32 bits or in 8 bits.

Beside the signed update of the patch (``ops.project_update``): for what is trained by its gradient's moments — the patterns
and masks of many images (``DorPatch.generate(update="adamw")``), or a classifier's own weights.  One step is one launch for
up to 98 tensors, plus two small ones where the gradients are clipped by their global norm; it never synchronises.
"""
import ctypes

import numpy as np
import torch

from . import _lib, ops

BLOCK = _lib.DP_ADAMW_BLOCK
# for map() over a hundred tensors a step
_DTYPE, _SHAPE, _NUMEL = torch.Tensor.dtype.__get__, torch.Tensor.shape.__get__, torch.Tensor.numel
_DENSE, _DEVICE, _POINTER = torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.data_ptr


def _per_tensor(value, count, name):
    values = [float(value)] * count if not isinstance(value, (list, tuple)) else [float(v) for v in value]
    if len(values) != count:
        raise ValueError("`%s` must be a number or one for each of the %d tensors, got %d" % (name, count, len(values)))
    if not all(0.0 <= v < float("inf") for v in values):
        raise ValueError("`%s` must be finite and >= 0" % name)
    return values


class AdamW(object):
    """AdamW with decoupled weight decay over ``params``, a list of dense GPU tensors (float32 / bfloat16 / float16, any mix).

    ``lr`` and ``weight_decay``: a number, or one for each tensor.  ``state_bits``: 32 (float32 moments) or 8 (e4m3 codes with a
    power-of-two scale for each 128 elements, rounded stochastically from ``seed`` and the step, so that runs repeat bit for bit).
    ``max_norm``: the gradients are scaled down to this global norm; a step whose norm is not finite changes nothing and does not
    count.  ``box`` (low, high): parameters are clamped to it after the update (pixels: (0, 1)).  ``capturable``: the step counter
    lives on the device (it does wherever ``max_norm`` is set), so that a captured step counts on every replay.

    ``exp_avg``, ``exp_avg_sq`` (float32 or float8_e4m3fn) hold the moments of all tensors one after the other, each tensor's part
    padded to a multiple of 128 with zeroes (``offsets``); with 8 bits ``exp_avg_scale``, ``exp_avg_sq_scale`` hold a float32 for
    each 128 of them: a moment is code * scale."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=None, box=None,
                 capturable=False, seed=0):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one tensor")
        spans = []
        for k, p in enumerate(self.params):
            self._check(p, "params[%d]" % k)
            if p.device != self.params[0].device:
                raise ValueError("`params` must be on one device, got %s and %s" % (self.params[0].device, p.device))
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        spans.sort()
        if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
            raise ValueError("`params` must not overlap (the same tensor twice?)")
        if state_bits not in (8, 32):
            raise ValueError("`state_bits` must be 8 or 32, got %r" % (state_bits,))
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
            raise ValueError("need 0 <= betas < 1 and eps >= 0, got %r, %r" % (betas, eps))
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError("`max_norm` must be > 0 or None, got %r" % (max_norm,))
        if box is not None and not box[0] <= box[1]:
            raise ValueError("`box` must be (low, high) or None, got %r" % (box,))
        count = len(self.params)
        self.lr = lr
        self._versioned = [p for p in self.params if not p.is_inference()]
        self.offsets, at = [], 0
        for p in self.params:
            self.offsets.append(at)
            at += -(-p.numel() // BLOCK) * BLOCK
        at = max(at, BLOCK)                                # (of empty tensors alone too: the kernels take no null states)
        dev = self.params[0].device
        self.state_bits, self.max_norm = state_bits, max_norm
        dtype = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.exp_avg = torch.zeros(at, dtype=torch.uint8 if state_bits == 8 else dtype, device=dev).view(dtype)
        self.exp_avg_sq = torch.zeros(at, dtype=torch.uint8 if state_bits == 8 else dtype, device=dev).view(dtype)
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg_scale = torch.zeros(at // BLOCK, dtype=torch.float32, device=dev)
            self.exp_avg_sq_scale = torch.zeros(at // BLOCK, dtype=torch.float32, device=dev)
        self._steps = 0
        self._counter = torch.zeros((), dtype=torch.int64, device=dev) if capturable or max_norm is not None else None
        low, high = (0.0, 0.0) if box is None else (float(box[0]), float(box[1]))
        self._cfg = _lib.DpAdamwCfg(float(betas[0]), float(betas[1]), float(eps), 0.0 if max_norm is None else float(max_norm),
                                    low, high, 0 if box is None else 1, state_bits, 0, int(seed) & 0xFFFFFFFF)
        self._table = (_lib.DpAdamwTensor * count)()
        self._rows = np.frombuffer(self._table, dtype=np.dtype(_lib.DpAdamwTensor))     # the same memory, a column at a time
        self._numel = np.array([p.numel() for p in self.params], dtype=np.int64)
        self._shapes, self._devices = [p.shape for p in self.params], {self.params[0].get_device()}
        self._types, self._sizes = [p.dtype for p in self.params], [p.numel() for p in self.params]
        self._rows["at"] = self.offsets
        self._rows["lr"] = _per_tensor(lr, count, "lr")
        self._rows["weight_decay"] = _per_tensor(weight_decay, count, "weight_decay")
        self._rows["param_dtype"] = [ops.ELEMENT_TYPES[p.dtype] for p in self.params]

    @staticmethod
    def _check(t, name):
        if not isinstance(t, torch.Tensor) or t.dtype not in ops.ELEMENT_TYPES:
            raise TypeError("`%s` must be a float32, bfloat16 or float16 tensor" % name)
        ops._chk(t, t.dtype, name)

    @property
    def steps(self):
        """Steps taken (reads the device where the counter lives there)."""
        return self._steps if self._counter is None else int(self._counter)

    def _same(self):
        """The launch writes where the parameters lie now: one given other data since (``p.data = ...``) must fit the states."""
        ps = self.params
        if (list(map(_DTYPE, ps)) != self._types or list(map(_NUMEL, ps)) != self._sizes
                or not all(map(_DENSE, ps)) or set(map(_DEVICE, ps)) != self._devices):
            raise ValueError("`params` have other sizes, types or strides, or another device, than the optimiser was made for")

    def _grads(self, grads):
        """Columns of the table: (pointers, element types, element counts)."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError("`grads` must have one entry for each of the %d tensors, got %d" % (len(self.params), len(grads)))
        numel = self._numel
        missing = [k for k, g in enumerate(grads) if g is None]
        if missing:                                        # no gradient: the tensor and its moments stay
            numel = numel.copy()
            numel[missing] = 0
            grads = [self.params[k] if g is None else g for k, g in enumerate(grads)]
        try:
            good = (list(map(_SHAPE, grads)) == self._shapes and all(map(_DENSE, grads))
                    and set(map(_DEVICE, grads)) == self._devices)
            types = set(map(_DTYPE, grads))
            kinds = [ops.ELEMENT_TYPES[g.dtype] for g in grads] if len(types) > 1 else ops.ELEMENT_TYPES[types.pop()]
        except (TypeError, KeyError):
            good = False
        if not good:                                       # which one, and why
            for k, (g, p) in enumerate(zip(grads, self.params)):
                self._check(g, "grads[%d]" % k)
                if g.shape != p.shape:
                    raise ValueError("`grads[%d]` has the shape %s, its parameter %s" % (k, tuple(g.shape), tuple(p.shape)))
                if g.device != p.device:
                    raise ValueError("`grads[%d]` is on %s, its parameter on %s" % (k, g.device, p.device))
        return list(map(_POINTER, grads)), kinds, numel

    def step(self, grads=None, lr=None):
        """One step from ``grads`` (a list; None: every parameter's ``.grad``; an entry None: that tensor stays), in place.
        A gradient may not lie on a parameter that the step writes, but for its own as a whole.
        ``lr``: a number or one for each tensor, for this and the next steps.  Returns the global gradient norm before clipping
        (a 0-dim float32 tensor) where ``max_norm`` is set, else None."""
        lib = _lib.load()
        rows = self._rows
        self._same()
        pointers, kinds, numel = self._grads(grads)
        ops._here(self.exp_avg, "params")
        if self._counter is None and self.params[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step is being captured: the step count would stay what it is (use capturable=True)")
        if lr is not None:
            rows["lr"] = _per_tensor(lr, len(self.params), "lr")
            self.lr = lr
        rows["param"], rows["grad"] = list(map(_POINTER, self.params)), pointers
        rows["grad_dtype"], rows["n"] = kinds, numel
        cfg, count = self._cfg, len(self.params)
        norm = work = None
        dev = self.params[0].device
        if self._counter is not None:
            n = lib.dp_adamw_workspace(ctypes.byref(cfg), self._table, count)
            work = torch.empty((n,), dtype=torch.uint8, device=dev)
            if self.max_norm is not None:
                norm = torch.empty((), dtype=torch.float32, device=dev)
        cfg.step = self._steps + 1
        ptr = ops._ptr
        _lib.check(lib.dp_adamw_step(ctypes.byref(cfg), self._table, count, ptr(self.exp_avg), ptr(self.exp_avg_scale),
                                     ptr(self.exp_avg_sq), ptr(self.exp_avg_sq_scale), ptr(self._counter), ptr(norm), ptr(work),
                                     ops._stream()), "dp_adamw_step")
        self._steps += 1
        torch.autograd.graph.increment_version(self._versioned)     # written in place, as autograd has to know
        return norm

    def moments(self, k):
        """(exp_avg, exp_avg_sq) of tensor ``k`` as new float32 tensors of its shape."""
        p, at = self.params[k], self.offsets[k]
        out = []
        for m, scale in ((self.exp_avg, self.exp_avg_scale), (self.exp_avg_sq, self.exp_avg_sq_scale)):
            n = p.numel()
            part = m[at:at + -(-n // BLOCK) * BLOCK].float()
            if scale is not None:
                part = (part.view(-1, BLOCK) * scale[at // BLOCK:(at + part.numel()) // BLOCK, None]).view(-1)
            out.append(part[:n].reshape(p.shape))
        return tuple(out)

    def state_dict(self):
        """The moments' buffers (not copied) and the steps taken."""
        state = {"exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "steps": self.steps}
        if self.state_bits == 8:
            state.update(exp_avg_scale=self.exp_avg_scale, exp_avg_sq_scale=self.exp_avg_sq_scale)
        return state

    def load_state_dict(self, state):
        self.load_state(state["exp_avg"], state["exp_avg_sq"], state["steps"], state.get("exp_avg_scale"), state.get("exp_avg_sq_scale"))

    def load_state(self, exp_avg, exp_avg_sq, steps, exp_avg_scale=None, exp_avg_sq_scale=None):
        """Copies moments in the layout of ``exp_avg`` / ``exp_avg_sq`` (and their scales) in, and sets the steps taken."""
        mine = [self.exp_avg, self.exp_avg_sq, self.exp_avg_scale, self.exp_avg_sq_scale]
        given = [exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale]
        for a, b in zip(mine, given):
            if (a is None) != (b is None) or (a is not None and (a.shape != b.shape or a.dtype != b.dtype)):
                raise ValueError("the state does not fit: it is for other tensors or another `state_bits`")
        if int(steps) < 0:
            raise ValueError("`steps` must be >= 0")
        for a, b in zip(mine, given):
            if a is not None:
                a.copy_(b)
        self._steps = int(steps)
        if self._counter is not None:
            self._counter.fill_(int(steps))
