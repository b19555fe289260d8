"""AdamW over many tensors at once, as HIP kernels (csrc/plmpm_adamw.hip; C ABI include/plmpm_policy.h).

``AdamW`` stands beside ``Adam`` and ``Momentum`` (optim.py: the same constructor, config keys and ``step``) for a policy that lives on the
GPU: its parameters are a list of tensors, updated where they are, with moments in 32 or in 8 bits.  ``adamw_step`` is the update itself, on
tensors that the caller keeps; ``adamw_values`` reads 8-bit moments back.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from .. import policy as P
from .optim import Optimizer

BLOCK = 256                             # elements that share a scale where moments are held in 8 bits


def _split(moments, what):
    """-> the lists of codes and of scales of a list of (codes, scales) pairs."""
    for k, entry in enumerate(moments):
        if not isinstance(entry, (tuple, list)) or len(entry) != 2:
            P._refuse(f"{what} {k}: all moments have 32 bits, or all have 8 and are pairs of codes and scales")
    return [entry[0] for entry in moments], [entry[1] for entry in moments]


def _not_tensors(optional=(), **lists):
    """Called for a TypeError of the binding: a ValueError that names the first entry which is no tensor, if that was it."""
    for name, entries in lists.items():
        for k, t in enumerate(entries):
            if isinstance(t, (tuple, list)):
                raise ValueError(f"{name} {k}: all moments have 32 bits, or all have 8") from None
            P._not_tensors((f"{name} {k}",) if name in optional else (), **{f"{name} {k}": t})


def adamw_step(params, grads, first, second, step, *, lr=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-8, weight_decay=0.01, max_norm=0.0,
               bounds=(-math.inf, math.inf), masters=None):
    """One AdamW update of all ``params`` in place: -> the gradients' global norm before clipping (a float32 scalar on the GPU), or None
    without ``max_norm``.

        k = min(1, max_norm / |g|) if max_norm > 0 else 1                 |g| over all tensors, summed in float64
        m = beta_1 m + (1 - beta_1) k g;   v = beta_2 v + (1 - beta_2) (k g)^2;   t = updates + 1
        w = clip(w - lr weight_decay w - lr / (1 - beta_1^t) m / (sqrt(v / (1 - beta_2^t)) + epsilon), *bounds)

    params, grads: float32, bfloat16 or float16 (each gradient of its parameter's type; types may differ between tensors).  A gradient of
    None leaves its parameter and moments as they are.  first, second: float32 tensors of the parameters' sizes, or (codes, scales) pairs for 8
    bits: int8 codes (first) and uint8 codes (second) of the parameter's size, one float32 scale for each 256 of them; all of one kind, zeros at
    the start.  masters: for each parameter a float32 copy that is updated in its place, the parameter being its rounding, or None; without one
    a 16-bit parameter is itself updated in float32 and rounded, and loses updates below its last bit.  step: int64 (2,) on the GPU, zeros at the
    start: the updates done, and those begun.  lr and the other numbers are fixed in a captured graph; the count is not.
    No tensor that the update writes may be in the call twice or share memory with another one of it (but for a gradient that is its parameter itself).  A call without any gradient does nothing.
    A gradient that is not finite makes its element's moments and weight not finite (moments of 8 bits: its 256's).  With max_norm a NaN does so to all of
    them; an infinity makes k zero, so all other elements move as with a gradient of zero.
    """
    bits, first_scales, second_scales = 32, [], []
    if len(first) and isinstance(first[0], (tuple, list)):
        bits = 8
        (first, first_scales), (second, second_scales) = _split(first, "first moment"), _split(second, "second moment")
    if masters is None:
        masters = []
    elif len(masters) != len(params):
        P._refuse("params, grads, first, second and masters have to be of one length")
    try:
        return P._binding().adamw_step(params, grads, first, second, first_scales, second_scales, masters, step, bits, lr, beta_1, beta_2, epsilon, weight_decay, max_norm,
                                       bounds[0], bounds[1])
    except TypeError:
        _not_tensors(("gradient", "master"), **{"parameter": params, "gradient": grads, "first moment": first, "second moment": second, "scales of first moment": first_scales,
                                                "scales of second moment": second_scales, "master": masters})
        P._not_tensors(step=step)
        raise


def adamw_values(moments, out=None):
    """The float32 values that 8-bit moments stand for: ``moments`` a list of (codes, scales) pairs, int8 codes for first moments and uint8 for
    second; -> ``out``, a list of float32 tensors of the codes' sizes (made if None)."""
    codes, scales = _split(list(moments), "moment")
    if out is None:
        out = [torch.empty(t.shape, dtype=torch.float32, device=t.device) for t in codes]
    try:
        P._binding().adamw_values(codes, scales, out)
    except TypeError:
        _not_tensors(codes=codes, scales=scales, out=out)
        raise
    return out


class AdamW(Optimizer):
    """``AdamW(parameters, cfg, **kw)``: parameters a list of tensors on one GPU; ``step(grads)`` (default: their ``.grad``) updates them in place
    and returns them.  Config keys beside Adam's: ``weight_decay``, ``state_bits`` (32 or 8), ``max_norm`` (of all gradients together, before the
    update; 0: no clipping).  16-bit parameters get a float32 master copy, which is made anew from a parameter that was written to between two
    updates (torch's version counter says so; writes through ``.data`` go unnoticed; before a capture ``renew_masters`` has to do it, since the copy would
    be part of the graph and each replay would lose what the master holds beyond the parameter).  ``grad_norm`` is the last norm (on the GPU)."""
    extra_keys = {"lr": 1e-3, "bounds": (-np.inf, np.inf), "beta_1": 0.9, "beta_2": 0.999, "epsilon": 1e-8, "weight_decay": 0.01, "state_bits": 32, "max_norm": 0.0}

    def __init__(self, parameters, cfg=None, **kwargs):
        if isinstance(parameters, (torch.Tensor, np.ndarray)):
            raise TypeError("AdamW takes a list of tensors (policy.parameters()); Adam and Momentum take a numpy array")
        super().__init__(list(parameters), cfg, **kwargs)
        if not self.parameters or not all(isinstance(p, torch.Tensor) for p in self.parameters):
            P._refuse("AdamW needs a list of at least one tensor")
        if self.cfg.state_bits not in (8, 32):
            P._refuse(f"state_bits has to be 32 or 8, got {self.cfg.state_bits}")
        device = self.parameters[0].device
        P._binding().require_device(self.parameters[0])  # a GPU's, or refused
        for k, p in enumerate(self.parameters):
            if p.dtype not in P.DTYPES or not p.is_contiguous() or p.device != device:
                P._refuse(f"parameter {k} has to be a contiguous float32, bfloat16 or float16 tensor on {device}")
        self._count = torch.zeros(2, dtype=torch.int64, device=device)
        self.grad_norm = None
        self.masters = [None if p.dtype == torch.float32 else p.detach().float() for p in self.parameters]
        self._seen = [p._version for p in self.parameters]
        self.state = {"first": [self._moment(p, torch.int8) for p in self.parameters], "second": [self._moment(p, torch.uint8) for p in self.parameters]}

    def _moment(self, p, codes):
        if self.cfg.state_bits == 32:
            return torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return torch.zeros(p.shape, dtype=codes, device=p.device), torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)

    # the update count lives on the GPU (a replayed graph counts too): reading it waits for the device
    @property
    def updates(self):
        return int(self._count[0])

    @updates.setter
    def updates(self, value):
        if hasattr(self, "_count"):                      # (the base class sets it before there is one)
            self._count[0] = int(value)

    def _values(self, name):
        return [t.clone() for t in self.state[name]] if self.cfg.state_bits == 32 else adamw_values(self.state[name])

    @property
    def momentum_buffer(self):
        return self._values("first")

    @property
    def v_buffer(self):
        return self._values("second")

    def _capturing(self):
        with torch.cuda.device_of(self._count):              # (the stream asked about is the current one of the parameters' device)
            return self._count.is_cuda and torch.cuda.is_current_stream_capturing()

    @torch.no_grad()
    def renew_masters(self):
        """Make the masters of parameters that were written to since the last update anew (``step`` does it by itself, outside a capture)."""
        stale = [k for k, (p, w, seen) in enumerate(zip(self.parameters, self.masters, self._seen)) if w is not None and p._version != seen]
        if stale and self._capturing():
            raise P.L.EngineError(f"parameter {stale[0]} was written to since the last update: call renew_masters() before the capture")
        for k in stale:
            self.masters[k].copy_(self.parameters[k])
            self._seen[k] = self.parameters[k]._version

    @torch.no_grad()
    def step(self, grads=None):
        c = self.cfg
        grads = [p.grad for p in self.parameters] if grads is None else list(grads)
        self.renew_masters()
        self.grad_norm = adamw_step(self.parameters, grads, self.state["first"], self.state["second"], self._count, lr=self.lr, beta_1=c.beta_1, beta_2=c.beta_2,
                                    epsilon=c.epsilon, weight_decay=c.weight_decay, max_norm=c.max_norm, bounds=self.bounds, masters=self.masters)
        self._seen = [p._version for p in self.parameters]
        return self.parameters

    # ---- checkpoints: the state is handed out and taken back as copies
    def state_dict(self):
        copy = lambda x: None if x is None else tuple(t.clone() for t in x) if isinstance(x, tuple) else x.clone()      # noqa: E731
        return {"iter": self.updates, "state_bits": self.cfg.state_bits, "first": [copy(x) for x in self.state["first"]],
                "second": [copy(x) for x in self.state["second"]], "masters": [copy(x) for x in self.masters]}

    def load_state_dict(self, saved):
        """Take a ``state_dict`` back.  The parameters are the caller's to restore, before this call (a later write makes their masters anew)."""
        if saved["state_bits"] != self.cfg.state_bits:
            P._refuse(f"the saved moments have {saved['state_bits']} bits, this optimizer's {self.cfg.state_bits}")
        pairs = []
        for mine, theirs in ((self.state["first"], saved["first"]), (self.state["second"], saved["second"]), (self.masters, saved["masters"])):
            if len(mine) != len(theirs):
                P._refuse("the saved state is of another list of parameters")
            for a, b in zip(mine, theirs):
                for t, s in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, (tuple, list)) else (b,)):
                    if (t is None) != (s is None) or (t is not None and (t.shape != s.shape or t.dtype != s.dtype)):
                        P._refuse("the saved state is of other parameters")
                    if t is not None:
                        pairs.append((t, s))
        for t, s in pairs:
            t.copy_(s)
        self._seen = [p._version for p in self.parameters]
        self.updates = saved["iter"]
