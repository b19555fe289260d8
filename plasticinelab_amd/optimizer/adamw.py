"""AdamW over many tensors at once, as HIP kernels (csrc/plmpm_adamw.hip; C ABI include/plmpm_policy.h).

``AdamW`` stands beside ``Adam`` and ``Momentum`` (optim.py: the same constructor, config keys and ``step``) for a policy that lives on the
GPU: its parameters are a list of tensors, updated where they are, with moments in 32 or in 8 bits.  ``adamw_step`` is the update itself, on
tensors that the caller keeps; ``adamw_values`` reads 8-bit moments back.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from .. import _lib as L
from .. import policy as P
from .optim import Optimizer

BLOCK = 256                             # elements that share a scale where moments are held in 8 bits


def _pair(entry, n, device, codes_dtype, name):
    codes, scales = entry
    P._need(codes.dtype == codes_dtype and codes.numel() == n and codes.is_contiguous() and codes.device == device,
            f"{name}: codes have to be {n} contiguous {codes_dtype} values on {device}")
    P._need(scales.dtype == torch.float32 and scales.numel() == -(-n // BLOCK) and scales.is_contiguous() and scales.device == device,
            f"{name}: scales have to be {-(-n // BLOCK)} contiguous float32 values on {device}")
    return codes.data_ptr(), scales.data_ptr()


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
    start: the updates done, and a word that the kernels use.  lr and the other numbers are fixed in a captured graph; the count is not.
    A gradient that is not finite makes its element's moments and weight not finite (with max_norm: all of them).
    """
    params, grads, first, second = list(params), list(grads), list(first), list(second)
    masters = [None] * len(params) if masters is None else list(masters)
    P._need(len(params) == len(grads) == len(first) == len(second) == len(masters), "params, grads, first, second and masters have to be of one length")
    P._need(isinstance(step, torch.Tensor) and step.shape == (2,) and step.dtype == torch.int64 and step.is_contiguous(), "step has to be an int64 tensor of two values")
    device = step.device
    bits = 8 if first and isinstance(first[0], (tuple, list)) else 32
    rows, keep, touched = [], [], []
    for k, (p, g, m, v, w) in enumerate(zip(params, grads, first, second, masters)):
        if g is None:
            continue
        n = p.numel()
        P._need(p.dtype in P.DTYPES and p.is_contiguous() and p.device == device, f"parameter {k} has to be a contiguous float32, bfloat16 or float16 tensor on {device}")
        P._need(g.shape == p.shape and g.dtype == p.dtype and g.device == device, f"gradient {k} has to match its parameter: {tuple(p.shape)} {p.dtype} on {device}")
        if not g.is_contiguous():
            g = g.contiguous()
            keep.append(g)
        P._need(isinstance(m, (tuple, list)) == (bits == 8) and isinstance(v, (tuple, list)) == (bits == 8), f"moments of parameter {k}: all moments have 32 bits, or all have 8")
        if bits == 8:
            (m, ms), (v, vs) = _pair(m, n, device, torch.int8, f"first moment {k}"), _pair(v, n, device, torch.uint8, f"second moment {k}")
        else:
            for t in (m, v):
                P._need(t.dtype == torch.float32 and t.numel() == n and t.is_contiguous() and t.device == device, f"moments of parameter {k} have to be {n} contiguous float32 values on {device}")
            m, v, ms, vs = m.data_ptr(), v.data_ptr(), None, None
        if w is not None:
            P._need(p.dtype != torch.float32, f"parameter {k} is float32: a master copy goes with 16 bits")
            P._need(w.dtype == torch.float32 and w.numel() == n and w.is_contiguous() and w.device == device, f"master {k} has to be {n} contiguous float32 values on {device}")
            w = w.data_ptr()
        rows.append((p.data_ptr(), g.data_ptr(), m, v, ms, vs, w, n, P.DTYPES[p.dtype], 0))
        touched.append(p)
    lo, hi = bounds
    norm = torch.empty((), dtype=torch.float32, device=device) if max_norm > 0 else None
    a = L.AdamWStep(state_bits=bits, lr=lr, beta_1=beta_1, beta_2=beta_2, epsilon=epsilon, weight_decay=weight_decay, max_norm=max_norm, lo=lo, hi=hi,
                    step=step.data_ptr(), grad_norm=P._ptr(norm))
    if not sum(r[7] for r in rows):
        return None if norm is None else norm.zero_()
    table = (L.AdamWTensor * len(rows))(*rows)
    lib, need = P._library(), C.c_size_t()
    L.check(lib.plmpm_adamw_workspace(C.byref(a), table, len(rows), C.byref(need)), lib)
    work = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    a.workspace, a.workspace_bytes = P._ptr(work), need.value
    P._call("plmpm_adamw_step", step, C.byref(a), table, len(rows))
    torch.autograd.graph.increment_version(touched)         # (a graph that saved a parameter notices that it changed)
    return norm


def adamw_values(moments, out=None):
    """The float32 values that 8-bit moments stand for: ``moments`` a list of (codes, scales) pairs, int8 codes for first moments and uint8 for
    second; -> ``out``, a list of float32 tensors of the codes' sizes (made if None)."""
    moments = list(moments)
    if out is None:
        out = [torch.empty(codes.shape, dtype=torch.float32, device=codes.device) for codes, _ in moments]
    P._need(len(out) == len(moments), "out has to have a tensor for each moment")
    n = len(moments)
    if not n:
        return out
    device = moments[0][0].device
    for k, ((codes, scales), o) in enumerate(zip(moments, out)):
        P._need(codes.dtype in (torch.int8, torch.uint8), f"moment {k}: codes have to be int8 or uint8")
        _pair((codes, scales), codes.numel(), device, codes.dtype, f"moment {k}")
        P._need(o.dtype == torch.float32 and o.numel() == codes.numel() and o.is_contiguous() and o.device == device, f"out {k} has to be {codes.numel()} contiguous float32 values on {device}")
    pointers = [(C.c_void_p * n)(*(t.data_ptr() for t in ts)) for ts in ([c for c, _ in moments], [s for _, s in moments], out)]
    sizes, which = (C.c_int64 * n)(*(c.numel() for c, _ in moments)), (C.c_int32 * n)(*(int(c.dtype == torch.uint8) for c, _ in moments))
    P._call("plmpm_adamw_values", moments[0][0], *pointers, sizes, which, n)
    return out


class AdamW(Optimizer):
    """``AdamW(parameters, cfg, **kw)``: parameters a list of tensors on one GPU; ``step(grads)`` (default: their ``.grad``) updates them in place
    and returns them.  Config keys beside Adam's: ``weight_decay``, ``state_bits`` (32 or 8), ``max_norm`` (of all gradients together, before the
    update; 0: no clipping).  16-bit parameters get a float32 master copy.  ``grad_norm`` is the last norm (on the GPU)."""
    extra_keys = {"lr": 1e-3, "bounds": (-np.inf, np.inf), "beta_1": 0.9, "beta_2": 0.999, "epsilon": 1e-8, "weight_decay": 0.01, "state_bits": 32, "max_norm": 0.0}

    def __init__(self, parameters, cfg=None, **kwargs):
        if isinstance(parameters, (torch.Tensor, np.ndarray)):
            raise TypeError("AdamW takes a list of tensors (policy.parameters()); Adam and Momentum take a numpy array")
        super().__init__(list(parameters), cfg, **kwargs)
        P._need(self.parameters and all(isinstance(p, torch.Tensor) for p in self.parameters), "AdamW needs at least one tensor")
        P._need(self.cfg.state_bits in (8, 32), f"state_bits has to be 32 or 8, got {self.cfg.state_bits}")
        device = self.parameters[0].device
        P._site(self.parameters[0])
        for k, p in enumerate(self.parameters):
            P._need(p.dtype in P.DTYPES and p.is_contiguous() and p.device == device, f"parameter {k} has to be a contiguous float32, bfloat16 or float16 tensor on {device}")
        self._count = torch.zeros(2, dtype=torch.int64, device=device)
        self.grad_norm = None
        self.masters = [None if p.dtype == torch.float32 else p.detach().float() for p in self.parameters]
        self.state = {"first": [self._moment(p, torch.int8) for p in self.parameters], "second": [self._moment(p, torch.uint8) for p in self.parameters]}

    def _moment(self, p, codes):
        if self.cfg.state_bits == 32:
            return torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return torch.zeros(p.shape, dtype=codes, device=p.device), torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)

    @property
    def iter(self):
        return int(self._count[0])

    @iter.setter
    def iter(self, value):
        self._count[0] = int(value)

    updates = property(lambda self: self.iter, lambda self, value: None if not hasattr(self, "_count") else AdamW.iter.fset(self, value))

    def _values(self, name):
        return [t.clone() for t in self.state[name]] if self.cfg.state_bits == 32 else adamw_values(self.state[name])

    @property
    def momentum_buffer(self):
        return self._values("first")

    @property
    def v_buffer(self):
        return self._values("second")

    @torch.no_grad()
    def step(self, grads=None):
        c = self.cfg
        grads = [p.grad for p in self.parameters] if grads is None else list(grads)
        self.grad_norm = adamw_step(self.parameters, grads, self.state["first"], self.state["second"], self._count, lr=self.lr, beta_1=c.beta_1, beta_2=c.beta_2,
                                    epsilon=c.epsilon, weight_decay=c.weight_decay, max_norm=c.max_norm, bounds=self.bounds, masters=self.masters)
        return self.parameters

    # ---- checkpoints: the state is handed out and taken back as copies
    def state_dict(self):
        copy = lambda x: None if x is None else tuple(t.clone() for t in x) if isinstance(x, tuple) else x.clone()      # noqa: E731
        return {"iter": self.iter, "state_bits": self.cfg.state_bits, "first": [copy(x) for x in self.state["first"]],
                "second": [copy(x) for x in self.state["second"]], "masters": [copy(x) for x in self.masters]}

    def load_state_dict(self, saved):
        P._need(saved["state_bits"] == self.cfg.state_bits, f"the saved moments have {saved['state_bits']} bits, this optimizer's {self.cfg.state_bits}")
        pairs = []
        for mine, theirs in ((self.state["first"], saved["first"]), (self.state["second"], saved["second"]), (self.masters, saved["masters"])):
            P._need(len(mine) == len(theirs), "the saved state is of another list of parameters")
            for a, b in zip(mine, theirs):
                for t, s in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, (tuple, list)) else (b,)):
                    P._need((t is None) == (s is None) and (t is None or (t.shape == s.shape and t.dtype == s.dtype)), "the saved state is of other parameters")
                    if t is not None:
                        pairs.append((t, s))
        for t, s in pairs:
            t.copy_(s)
        self.iter = saved["iter"]
