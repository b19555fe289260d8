"""Operators of a policy that is a sequence model, as HIP kernels (csrc/plmpm_scan.hip, csrc/plmpm_norm.hip; C ABI include/plmpm_policy.h), and
the policy built from them.

    h, last = gated_scan(x, r, i, decay, h0, reset)         # a gated linear recurrence over whole sequences, differentiable
    h = gated_scan_step(x, r, i, decay, state)              # one observation: ``state`` moves on in place
    y, z = block_norm(x, u, gate, scale, post, pre)         # norms before and after a block, its gate and residual scale
    policy = RecurrentPolicy(obs_dim, action_dim)           # what SolverNN drives (optimizer/solver_nn.py)

Tensors live on one GPU; kernels go to the current stream of that GPU and nothing synchronises, so calls can be captured into a graph.
There is no CPU path.  The reference's counterpart is a per-step MLP (plb/engine/nn/mlp.py:11-183) without a memory.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

import torch

from . import _lib as L

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
GATES = {"identity": 0, "sigmoid": 1, "silu": 2}
MAX_WIDTH = 8192                        # of block_norm (a row stays in one workgroup's registers)
CHECKPOINT = 64                         # steps between the states that gated_scan keeps for its backward pass


# ---- plumbing: the library, the device and the stream of a call (one place)
def _library():
    return L.load_policy()


def _site(t: torch.Tensor):
    """-> (stream handle, device guard) of a call on ``t``'s GPU."""
    if t.device.type != "cuda":
        raise L.EngineError(f"policy operators run on a ROCm device, got a tensor on {t.device}: there is no CPU path")
    guard = contextlib.nullcontext() if torch.cuda.current_device() == t.device.index else torch.cuda.device(t.device)
    return torch.cuda.current_stream(t.device).cuda_stream, guard


def _call(name, t, *args):
    stream, guard = _site(t)
    lib = _library()
    with guard:
        L.check(getattr(lib, name)(*args, C.c_void_p(stream)), lib)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(cond, message):
    if not cond:
        raise ValueError(message)


def _same_device(first, **others):
    for name, t in others.items():
        if t is not None:
            _need(isinstance(t, torch.Tensor), f"{name} has to be a tensor")
            _need(t.device == first.device, f"{name} is on {t.device}, not on {first.device}")


def _rows(t):
    """Unit stride over the last dimension (a copy if need be)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


# ---------------------------------------------------------------------------------------------- gated linear recurrence
def _scan_args(x, r, i, decay, h0, reset, c):
    B, T, D = x.shape
    s = L.Scan(dtype=DTYPES[x.dtype], batch=B, steps=T, width=D, c=c, x=_ptr(x), r=_ptr(r), i=_ptr(i), decay=_ptr(decay), h0=_ptr(h0), reset=_ptr(reset))
    for k, t in enumerate((x, r, i)):
        s.stride_b[k], s.stride_t[k] = t.stride(0), t.stride(1)
    return s


def _scan_run(name, s, x, backward):
    lib, need = _library(), C.c_size_t()
    L.check(lib.plmpm_scan_workspace(C.byref(s), int(backward), C.byref(need)), lib)
    work = torch.empty(need.value, dtype=torch.uint8, device=x.device) if need.value else None
    s.workspace, s.workspace_bytes = _ptr(work), need.value
    _call(name, x, C.byref(s))


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, decay, h0, reset, c):
        x, r, i = _rows(x), _rows(r), _rows(i)
        B, T, D = x.shape
        h = torch.empty(B, T, D, dtype=x.dtype, device=x.device)
        last = torch.empty(B, D, dtype=torch.float32, device=x.device)
        keep = any(ctx.needs_input_grad[:5])
        checkpoint = torch.empty((T + CHECKPOINT - 1) // CHECKPOINT, B, D, dtype=torch.float32, device=x.device) if keep else None
        if h.numel():
            s = _scan_args(x, r, i, decay, h0, reset, c)
            s.h, s.h_last, s.checkpoint = _ptr(h), _ptr(last), _ptr(checkpoint)
            _scan_run("plmpm_scan_forward", s, x, False)
        elif h0 is not None:
            last.copy_(h0)
        else:
            last.zero_()
        ctx.save_for_backward(x, r, i, decay, reset, checkpoint)
        ctx.c, ctx.has_h0 = c, h0 is not None
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        x, r, i, decay, reset, checkpoint = ctx.saved_tensors
        B, T, D = x.shape
        dx, dr, di = (torch.empty(B, T, D, dtype=x.dtype, device=x.device) for _ in range(3))
        ddecay = torch.empty_like(decay)
        dh0 = torch.empty(B, D, dtype=torch.float32, device=x.device) if ctx.has_h0 else None
        dh = None if dh is None else dh.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        if dx.numel():
            s = _scan_args(x, r, i, decay, None, reset, ctx.c)
            s.checkpoint, s.dh, s.dlast = _ptr(checkpoint), _ptr(dh), _ptr(dlast)
            s.dx, s.dr, s.di, s.ddecay, s.dh0 = _ptr(dx), _ptr(dr), _ptr(di), _ptr(ddecay), _ptr(dh0)
            _scan_run("plmpm_scan_backward", s, x, True)
        else:
            ddecay.zero_()
            if dh0 is not None:
                dh0.zero_() if dlast is None else dh0.copy_(dlast)
        return dx, dr, di, ddecay, dh0, None, None


def _scan_checks(x, r, i, decay, c, dims):
    _need(isinstance(x, torch.Tensor) and x.dim() == dims, f"x has to be a tensor of {dims} dimensions")
    _same_device(x, r=r, i=i, decay=decay)
    _need(x.dtype in DTYPES, f"x has to be float32, bfloat16 or float16, got {x.dtype}")
    for name, t in (("r", r), ("i", i)):
        _need(t.shape == x.shape and t.dtype == x.dtype, f"{name} has to match x: {tuple(x.shape)} {x.dtype}, got {tuple(t.shape)} {t.dtype}")
    _need(decay.shape == x.shape[-1:] and decay.dtype == torch.float32 and decay.is_contiguous(),
          f"decay has to be a contiguous float32 tensor of {x.shape[-1]} values")
    _need(0.0 < c < 1e30, f"c has to be positive and finite, got {c}")


def gated_scan(x, r, i, decay, h0=None, reset=None, *, c: float = 8.0):
    """Gated linear recurrence over sequences: ``-> (h, last)``.

        a_t = exp(-c softplus(decay) sigmoid(r_t));   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t

    x, r, i: (B, T, D), float32, bfloat16 or float16; batch and time strides are free (slices of one projection are read in place).
    decay: (D,) float32.  h0: (B, D) float32, the state before the first step (zeros if None).  reset: (B, T) bool; where it is set, a_t is 0:
    the sequence starts anew and nothing of what came before, a NaN either, reaches it.  h has x's type, ``last`` (B, D) is the float32
    state behind step T-1 (all rows of a batch have T steps: pack shorter episodes with ``reset``).  The state is carried in float32; gradients
    reach x, r, i, decay and h0 (its backward pass makes the states again from one float32 state in 64 steps).
    """
    _scan_checks(x, r, i, decay, c, 3)
    B, T, D = x.shape
    _same_device(x, h0=h0, reset=reset)
    if h0 is not None:
        _need(h0.shape == (B, D) and h0.dtype == torch.float32, f"h0 has to be float32 ({B}, {D}), got {tuple(h0.shape)} {h0.dtype}")
        h0 = h0.contiguous()
    if reset is not None:
        _need(reset.shape == (B, T) and reset.dtype == torch.bool, f"reset has to be bool ({B}, {T}), got {tuple(reset.shape)} {reset.dtype}")
        reset = reset.contiguous()
    return _GatedScan.apply(x, r, i, decay, h0, reset, float(c))


def gated_scan_step(x, r, i, decay, state, *, c: float = 8.0):
    """One step of ``gated_scan`` for (B, D) inputs: -> h (B, D); ``state`` (B, D) float32 moves on in place.  No gradients (serving and
    evaluation; a differentiable step is ``gated_scan`` with T = 1)."""
    _scan_checks(x, r, i, decay, c, 2)
    _same_device(x, state=state)
    _need(state is not None and state.shape == x.shape and state.dtype == torch.float32 and state.is_contiguous(),
          f"state has to be a contiguous float32 tensor of {tuple(x.shape)}")
    _need(not (torch.is_grad_enabled() and any(t.requires_grad for t in (x, r, i, decay, state))),
          "gated_scan_step has no gradients: call it under torch.no_grad(), or gated_scan with one step")
    x, r, i = _rows(x), _rows(r), _rows(i)
    B, D = x.shape
    h = torch.empty(B, D, dtype=x.dtype, device=x.device)
    if h.numel():
        s = L.Scan(dtype=DTYPES[x.dtype], batch=B, steps=1, width=D, c=c, x=_ptr(x), r=_ptr(r), i=_ptr(i), decay=_ptr(decay), h0=_ptr(state), h=_ptr(h), h_last=_ptr(state))
        for k, t in enumerate((x, r, i)):
            s.stride_b[k] = t.stride(0)
        _scan_run("plmpm_scan_forward", s, x, False)
        torch.autograd.graph.increment_version(state)
    return h


# ---------------------------------------------------------------------------------------------- norms around a block
def _as_rows(t, D):
    t = _rows(t.reshape(-1, D))
    return t, (t.stride(0) if t.shape[0] > 1 else D)


def _norm_args(x, u, gate, scale, post, pre, u_dtype, eps, fn, keep):
    D = x.shape[-1]
    n = L.Norm(x_dtype=DTYPES[x.dtype], u_dtype=DTYPES[u_dtype], gate_fn=fn, width=D, eps=eps, scale=_ptr(scale), post=_ptr(post), pre=_ptr(pre))
    n.w_dtype = next((DTYPES[w.dtype] for w in (pre, post, scale) if w is not None), 0)
    for name, t in (("x", x), ("u", u), ("gate", gate)):
        if t is not None:
            t, stride = _as_rows(t, D)
            keep.append(t)
            setattr(n, name, _ptr(t))
            setattr(n, "stride_" + name, stride)
    n.rows = keep[0].shape[0]
    return n


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, u, gate, scale, post, pre, u_dtype, eps, fn):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if u is not None else None
        z = torch.empty(x.shape, dtype=u_dtype, device=x.device) if pre is not None else None
        if x.numel():
            keep = []
            n = _norm_args(x, u, gate, scale, post, pre, u_dtype, eps, fn, keep)
            n.y, n.z = _ptr(y), _ptr(z)
            _call("plmpm_norm_forward", x, C.byref(n))
        ctx.save_for_backward(x, u, gate, scale, post, pre)
        ctx.how = (u_dtype, eps, fn)
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz):
        x, u, gate, scale, post, pre = ctx.saved_tensors
        u_dtype, eps, fn = ctx.how
        if dy is None and dz is None:
            return (None,) * 9
        D = x.shape[-1]
        keep, out = [], {}
        for name, t in (("dx", x), ("du", u), ("dgate", gate), ("dscale", scale), ("dpost", post), ("dpre", pre)):
            out[name] = None if t is None else torch.empty(t.shape, dtype=t.dtype, device=x.device)
        if x.numel():
            n = _norm_args(x, u, gate, scale, post, pre, u_dtype, eps, fn, keep)
            for name, t in (("dy", dy), ("dz", dz)):
                if t is not None:
                    t, stride = _as_rows(t, D)
                    keep.append(t)
                    setattr(n, name, _ptr(t))
                    setattr(n, "stride_" + name, stride)
            for name, t in out.items():
                setattr(n, name, _ptr(t))
            lib, need = _library(), C.c_size_t()
            L.check(lib.plmpm_norm_workspace(C.byref(n), C.byref(need)), lib)
            work = torch.empty(need.value, dtype=torch.uint8, device=x.device)
            n.workspace, n.workspace_bytes = _ptr(work), need.value
            _call("plmpm_norm_backward", x, C.byref(n))
        else:
            for name in ("dscale", "dpost", "dpre"):
                if out[name] is not None:
                    out[name].zero_()
        return out["dx"], out["du"], out["dgate"], out["dscale"], out["dpost"], out["dpre"], None, None, None


def block_norm(x, u=None, gate=None, scale=None, post=None, pre=None, *, eps: float = 1e-6, gate_fn: str = "sigmoid", dtype=None):
    """The norms before and after a block with its gate and residual scale: ``-> (y, z)``.

        y = x + scale * f(gate) * post * u / rms(u)         the residual stream behind a block that answered u
        z = pre * y / rms(y)                                what the next block reads;  rms(v) = sqrt(mean(v^2) + eps)

    x: (..., D), the residual stream, float32, bfloat16 or float16.  u, gate: x's shape; u's type is x's, or a 16-bit one next to a float32 x.
    f: ``gate_fn``, "identity", "sigmoid" or "silu"; no gate counts as ones (a gate that many rows share is expanded to x's shape; its gradient is
    then summed by torch).  scale, post, pre: (D,), of one type; scale and post may be None (ones).  Without u, y is x itself (the norm before
    the first block); without pre there is no z (None: behind the last).  z has u's type (without u: ``dtype``, x's by default) and comes
    from the unrounded y.  D is at most 8192.  Sums in float32; gradients reach every tensor given.
    """
    _need(isinstance(x, torch.Tensor) and x.dim() >= 1, "x has to be a tensor with at least one dimension")
    _same_device(x, u=u, gate=gate, scale=scale, post=post, pre=pre)
    _need(x.dtype in DTYPES, f"x has to be float32, bfloat16 or float16, got {x.dtype}")
    D = x.shape[-1]
    _need(D <= MAX_WIDTH, f"rows of {D} values, at most {MAX_WIDTH}")
    _need(u is not None or pre is not None, "u, pre or both are needed")
    _need(gate_fn in GATES, f"gate_fn has to be one of {sorted(GATES)}, got {gate_fn!r}")
    _need(0.0 <= eps < 1e30, f"eps has to be zero or above, and finite, got {eps}")
    if u is None:
        _need(gate is None and scale is None and post is None, "gate, scale and post go with u")
        u_dtype = x.dtype if dtype is None else dtype
    else:
        u_dtype = u.dtype
        _need(dtype is None or dtype == u_dtype, f"z has u's type {u_dtype}: dtype is for calls without u")
    _need(u_dtype in DTYPES and (u_dtype == x.dtype or x.dtype == torch.float32), f"u (or dtype) has to be x's type, or 16 bits next to a float32 x: got {u_dtype} with {x.dtype}")
    for name, t in (("u", u), ("gate", gate)):
        _need(t is None or (t.shape == x.shape and t.dtype == u_dtype), f"{name} has to have x's shape {tuple(x.shape)} and the type {u_dtype}")
    weights = [(n, w) for n, w in (("scale", scale), ("post", post), ("pre", pre)) if w is not None]
    for name, w in weights:
        _need(w.shape == (D,) and w.is_contiguous() and w.dtype in DTYPES and w.dtype == weights[0][1].dtype,
              f"{name} has to be a contiguous tensor of {D} values, of one floating type with the other weights")
    y, z = _BlockNorm.apply(x, u, gate, scale, post, pre, u_dtype, float(eps), GATES[gate_fn])
    return (x if u is None else y), z
