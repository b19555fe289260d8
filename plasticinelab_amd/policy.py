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

import ctypes as C

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
    """-> (stream handle, device guard or None) of a call on ``t``'s GPU."""
    index = t.get_device()
    if index < 0:
        raise L.EngineError(f"policy operators run on a ROCm device, got a tensor on {t.device}: there is no CPU path")
    return torch._C._cuda_getCurrentRawStream(index), None if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def _call(name, t, *args):
    stream, guard = _site(t)
    lib = _library()
    if guard is None:
        L.check(getattr(lib, name)(*args, stream), lib)
    else:
        with guard:
            L.check(getattr(lib, name)(*args, stream), lib)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _refuse(message):
    raise ValueError(message)


def _together(first, *others):
    """Whether the others (None left out) are tensors on the device of the first."""
    where = first.get_device()
    try:
        for t in others:
            if t is not None and t.get_device() != where:
                return False
    except AttributeError:
        return False
    return True


def _same_device(first, **others):
    where = first.get_device()
    for name, t in others.items():
        if t is not None:
            if not isinstance(t, torch.Tensor):
                _refuse(f"{name} has to be a tensor")
            if t.get_device() != where:
                _refuse(f"{name} is on {t.device}, not on {first.device}")


def _tracked(*ts):
    """Whether autograd has to know of a call (without it the kernels are called directly: Function.apply costs more than they do)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _written(t):
    """A tensor was changed in place: a graph that saved it has to notice (tensors of inference mode are in none)."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _rows(t):
    """Unit stride over the last dimension (a copy if need be)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# ---------------------------------------------------------------------------------------------- gated linear recurrence
def _scan_args(x, r, i, decay, h0, reset, c):
    B, T, D = x.shape
    (xb, xt, _), (rb, rt, _), (ib, it, _) = x.stride(), r.stride(), i.stride()
    return L.Scan(DTYPES[x.dtype], 0, B, T, D, (xb, rb, ib), (xt, rt, it), c, x.data_ptr(), r.data_ptr(), i.data_ptr(), decay.data_ptr(), _ptr(h0), _ptr(reset))


def _scan_run(name, s, x, backward):
    lib, need = _library(), C.c_size_t()
    L.check(lib.plmpm_scan_workspace(s, backward, need), lib)
    if need.value:
        work = x.new_empty(need.value, dtype=torch.uint8)
        s.workspace, s.workspace_bytes = work.data_ptr(), need.value
    _call(name, x, s)


def _scan_forward(x, r, i, decay, h0, reset, c, keep):
    """-> h, last, checkpoint (what the backward pass starts from; None unless ``keep``)."""
    B, T, D = x.shape
    h, last = x.new_empty((B, T, D)), decay.new_empty((B, D))
    checkpoint = decay.new_empty(((T + CHECKPOINT - 1) // CHECKPOINT, B, D)) if keep else None
    if B and T and D:
        s = _scan_args(x, r, i, decay, h0, reset, c)
        s.h, s.h_last, s.checkpoint = h.data_ptr(), last.data_ptr(), _ptr(checkpoint)
        _scan_run("plmpm_scan_forward", s, x, 0)
    elif h0 is not None:
        last.copy_(h0)
    else:
        last.zero_()
    return h, last, checkpoint


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, decay, h0, reset, c):
        h, last, checkpoint = _scan_forward(x, r, i, decay, h0, reset, c, True)
        ctx.save_for_backward(x, r, i, decay, reset, checkpoint)
        ctx.c, ctx.has_h0 = c, h0 is not None
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dlast):
        x, r, i, decay, reset, checkpoint = ctx.saved_tensors
        B, T, D = x.shape
        dx, dr, di, ddecay = x.new_empty((B, T, D)), x.new_empty((B, T, D)), x.new_empty((B, T, D)), decay.new_empty(D)
        dh0 = decay.new_empty((B, D)) if ctx.has_h0 else None
        dh = None if dh is None else dh.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        if B and T and D:
            s = _scan_args(x, r, i, decay, None, reset, ctx.c)
            s.checkpoint, s.dh, s.dlast = checkpoint.data_ptr(), _ptr(dh), _ptr(dlast)
            s.dx, s.dr, s.di, s.ddecay, s.dh0 = dx.data_ptr(), dr.data_ptr(), di.data_ptr(), ddecay.data_ptr(), _ptr(dh0)
            _scan_run("plmpm_scan_backward", s, x, 1)
        else:
            ddecay.zero_()
            if dh0 is not None:
                dh0.zero_() if dlast is None else dh0.copy_(dlast)
        return dx, dr, di, ddecay, dh0, None, None


def _scan_checks(x, r, i, decay, c, dims):
    if not isinstance(x, torch.Tensor) or x.dim() != dims:
        _refuse(f"x has to be a tensor of {dims} dimensions")
    if r is None or i is None or decay is None or not _together(x, r, i, decay):
        _same_device(x, r=r, i=i, decay=decay)
        _refuse("r, i and decay are needed")
    shape, dtype = x.shape, x.dtype
    if dtype not in DTYPES:
        _refuse(f"x has to be float32, bfloat16 or float16, got {dtype}")
    if r.shape != shape or i.shape != shape or r.dtype != dtype or i.dtype != dtype:
        _refuse(f"r and i have to match x: {tuple(shape)} {dtype}, got {tuple(r.shape)} {r.dtype} and {tuple(i.shape)} {i.dtype}")
    if decay.shape != shape[-1:] or decay.dtype != torch.float32 or not decay.is_contiguous():
        _refuse(f"decay has to be a contiguous float32 tensor of {shape[-1]} values")
    if not 0.0 < c < 1e30:
        _refuse(f"c has to be positive and finite, got {c}")


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
    if h0 is not None:
        if not _together(x, h0):
            _same_device(x, h0=h0)
        if h0.shape != (B, D) or h0.dtype != torch.float32:
            _refuse(f"h0 has to be float32 ({B}, {D}), got {tuple(h0.shape)} {h0.dtype}")
        h0 = h0.contiguous()
    if reset is not None:
        if not _together(x, reset):
            _same_device(x, reset=reset)
        if reset.shape != (B, T) or reset.dtype != torch.bool:
            _refuse(f"reset has to be bool ({B}, {T}), got {tuple(reset.shape)} {reset.dtype}")
        reset = reset.contiguous()
    x, r, i = _rows(x), _rows(r), _rows(i)
    if _tracked(x, r, i, decay, h0):
        return _GatedScan.apply(x, r, i, decay, h0, reset, float(c))
    return _scan_forward(x, r, i, decay, h0, reset, float(c), False)[:2]


def gated_scan_step(x, r, i, decay, state, *, c: float = 8.0):
    """One step of ``gated_scan`` for (B, D) inputs: -> h (B, D); ``state`` (B, D) float32 moves on in place.  No gradients (serving and
    evaluation; a differentiable step is ``gated_scan`` with T = 1)."""
    _scan_checks(x, r, i, decay, c, 2)
    if not _together(x, state):
        _same_device(x, state=state)
    if state is None or state.shape != x.shape or state.dtype != torch.float32 or not state.is_contiguous():
        _refuse(f"state has to be a contiguous float32 tensor of {tuple(x.shape)}")
    if _tracked(x, r, i, decay, state):
        _refuse("gated_scan_step has no gradients: call it under torch.no_grad(), or gated_scan with one step")
    x, r, i = _rows(x), _rows(r), _rows(i)
    B, D = x.shape
    h = x.new_empty((B, D))
    if B and D:
        p = state.data_ptr()
        s = L.Scan(DTYPES[x.dtype], 0, B, 1, D, (x.stride(0), r.stride(0), i.stride(0)), (0, 0, 0), c, x.data_ptr(), r.data_ptr(), i.data_ptr(), decay.data_ptr(), p, None,
                   h.data_ptr(), p)
        _call("plmpm_scan_forward", x, s)           # (a single step needs no workspace)
        _written(state)
    return h


# ---------------------------------------------------------------------------------------------- norms around a block
def _as_rows(t, D):
    t = _rows(t) if t.dim() == 2 else _rows(t.reshape(-1, D))
    return t, (t.stride(0) if t.shape[0] > 1 else D)


def _norm_args(x, u, gate, scale, post, pre, u_dtype, eps, fn, keep):
    D = x.shape[-1]
    w = pre if pre is not None else post if post is not None else scale
    at = [0, 0, 0]
    strides = [0, 0, 0]
    for k, t in enumerate((x, u, gate)):
        if t is not None:
            t, strides[k] = _as_rows(t, D)
            keep.append(t)
            at[k] = t.data_ptr()
    return L.Norm(DTYPES[x.dtype], DTYPES[u_dtype], 0 if w is None else DTYPES[w.dtype], fn, keep[0].shape[0], D, strides[0], strides[1], strides[2], 0, 0, eps,
                  at[0], at[1], at[2], _ptr(scale), _ptr(post), _ptr(pre))


def _norm_forward(x, u, gate, scale, post, pre, u_dtype, eps, fn):
    y = x.new_empty(x.shape) if u is not None else None
    z = x.new_empty(x.shape, dtype=u_dtype) if pre is not None else None
    if x.numel():
        keep = []
        n = _norm_args(x, u, gate, scale, post, pre, u_dtype, eps, fn, keep)
        n.y, n.z = _ptr(y), _ptr(z)
        _call("plmpm_norm_forward", x, n)
    return y, z


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, u, gate, scale, post, pre, u_dtype, eps, fn):
        ctx.save_for_backward(x, u, gate, scale, post, pre)
        ctx.how = (u_dtype, eps, fn)
        ctx.set_materialize_grads(False)
        return _norm_forward(x, u, gate, scale, post, pre, u_dtype, eps, fn)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz):
        x, u, gate, scale, post, pre = saved = ctx.saved_tensors
        u_dtype, eps, fn = ctx.how
        if dy is None and dz is None:
            return (None,) * 9
        D = x.shape[-1]
        out = [None if t is None else t.new_empty(t.shape) for t in saved]
        if x.numel():
            keep = []
            n = _norm_args(x, u, gate, scale, post, pre, u_dtype, eps, fn, keep)
            if dy is not None:
                dy, n.stride_dy = _as_rows(dy, D)
                n.dy = dy.data_ptr()
            if dz is not None:
                dz, n.stride_dz = _as_rows(dz, D)
                n.dz = dz.data_ptr()
            n.dx, n.du, n.dgate, n.dscale, n.dpost, n.dpre = (_ptr(t) for t in out)
            lib, need = _library(), C.c_size_t()
            L.check(lib.plmpm_norm_workspace(n, need), lib)
            work = x.new_empty(need.value, dtype=torch.uint8)
            n.workspace, n.workspace_bytes = work.data_ptr(), need.value
            _call("plmpm_norm_backward", x, n)
        else:
            for t in out[3:]:
                if t is not None:
                    t.zero_()
        return (*out, None, None, None)


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
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        _refuse("x has to be a tensor with at least one dimension")
    if not _together(x, u, gate, scale, post, pre):
        _same_device(x, u=u, gate=gate, scale=scale, post=post, pre=pre)
    if x.dtype not in DTYPES:
        _refuse(f"x has to be float32, bfloat16 or float16, got {x.dtype}")
    D = x.shape[-1]
    if D > MAX_WIDTH:
        _refuse(f"rows of {D} values, at most {MAX_WIDTH}")
    if u is None and pre is None:
        _refuse("u, pre or both are needed")
    if gate_fn not in GATES:
        _refuse(f"gate_fn has to be one of {sorted(GATES)}, got {gate_fn!r}")
    if not 0.0 <= eps < 1e30:
        _refuse(f"eps has to be zero or above, and finite, got {eps}")
    if u is None:
        if gate is not None or scale is not None or post is not None:
            _refuse("gate, scale and post go with u")
        u_dtype = x.dtype if dtype is None else dtype
    else:
        u_dtype = u.dtype
        if dtype is not None and dtype != u_dtype:
            _refuse(f"z has u's type {u_dtype}: dtype is for calls without u")
        if u.shape != x.shape:
            _refuse(f"u has to have x's shape {tuple(x.shape)}, got {tuple(u.shape)}")
    if u_dtype not in DTYPES or (u_dtype != x.dtype and x.dtype != torch.float32):
        _refuse(f"u (or dtype) has to be x's type, or 16 bits next to a float32 x: got {u_dtype} with {x.dtype}")
    if gate is not None and (gate.shape != x.shape or gate.dtype != u_dtype):
        _refuse(f"gate has to have x's shape {tuple(x.shape)} and the type {u_dtype}, got {tuple(gate.shape)} {gate.dtype}")
    w_dtype = None
    for name, w in (("scale", scale), ("post", post), ("pre", pre)):
        if w is not None:
            w_dtype = w.dtype if w_dtype is None else w_dtype
            if w.dim() != 1 or w.shape[0] != D or not w.is_contiguous() or w.dtype != w_dtype or w_dtype not in DTYPES:
                _refuse(f"{name} has to be a contiguous tensor of {D} values, of one floating type with the other weights")
    run = _BlockNorm.apply if _tracked(x, u, gate, scale, post, pre) else _norm_forward
    y, z = run(x, u, gate, scale, post, pre, u_dtype, float(eps), GATES[gate_fn])
    return (x if u is None else y), z


# ---------------------------------------------------------------------------------------------- the policy
class RecurrentPolicy(torch.nn.Module):
    """Observations to actions with a memory: a linear embedding, ``depth`` blocks around a gated linear recurrence, and a linear head.

        z = pre * y / rms(y);   x, r, i, g = z W_in;   u = gated_scan(x, r, i) W_out;   y += scale * f(g) * post * u / rms(u)

    ``forward`` takes whole sequences, ``step`` one observation of each row (both differentiable, the same numbers), ``act`` the same without
    gradients, with the state moved on in place.  ``dtype`` is the type of the matrices and of what passes through them; the residual stream, the norms'
    weights, the decays and the state are float32.  Actions are not bounded here (SolverNN clamps them, as plb/engine/nn/mlp.py:98 does).
    """

    def __init__(self, obs_dim, action_dim, width=128, depth=2, *, gate_fn="sigmoid", c=8.0, eps=1e-6, device="cuda", dtype=torch.float32):
        super().__init__()
        if dtype not in DTYPES:
            _refuse(f"dtype has to be float32, bfloat16 or float16, got {dtype}")
        if not 1 <= width <= MAX_WIDTH or depth < 1:
            _refuse(f"width has to lie in 1..{MAX_WIDTH} and depth has to be at least 1, got {width} and {depth}")
        if gate_fn not in GATES:
            _refuse(f"gate_fn has to be one of {sorted(GATES)}, got {gate_fn!r}")
        self.width, self.depth, self.gate_fn, self.c, self.eps = int(width), int(depth), gate_fn, float(c), float(eps)
        how = {"device": device, "dtype": dtype}
        vectors = lambda n, value: torch.nn.ParameterList([torch.nn.Parameter(torch.full((width,), value, device=device)) for _ in range(n)])    # noqa: E731
        self.embed = torch.nn.Linear(obs_dim, width, **how)
        self.into = torch.nn.ModuleList([torch.nn.Linear(width, 4 * width, **how) for _ in range(depth)])
        self.out = torch.nn.ModuleList([torch.nn.Linear(width, width, **how) for _ in range(depth)])
        self.head = torch.nn.Linear(width, action_dim, **how)
        self.pre, self.post, self.scale = vectors(depth + 1, 1.0), vectors(depth, 1.0), vectors(depth, 0.5)
        # decays of 0.9 .. 0.999 a step at a fully open gate
        at = torch.linspace(0.9, 0.999, width, dtype=torch.float64)
        start = torch.log(torch.expm1(-torch.log(at) / c)).float().to(device)
        self.decay = torch.nn.ParameterList([torch.nn.Parameter(start.clone()) for _ in range(depth)])

    def initial_state(self, batch=1):
        """The state before the first observation: float32 (depth, batch, width), zeros."""
        return torch.zeros(self.depth, batch, self.width, device=self.decay[0].device)

    def _run(self, obs, memory):
        """obs (..., obs_dim) -> actions; ``memory(k, x, r, i)`` is block k's recurrence."""
        dtype = self.embed.weight.dtype
        y = self.embed(obs.to(dtype)).float()
        _, z = block_norm(y, pre=self.pre[0], eps=self.eps, dtype=dtype)
        for k in range(self.depth):
            x, r, i, g = self.into[k](z).split(self.width, dim=-1)
            u = self.out[k](memory(k, x, r, i))
            y, z = block_norm(y, u, g, self.scale[k], self.post[k], self.pre[k + 1], eps=self.eps, gate_fn=self.gate_fn)
        return self.head(z)

    def forward(self, obs, state=None, reset=None):
        """obs (batch, steps, obs_dim) -> (actions (batch, steps, action_dim), state behind the last step).  ``reset``: (batch, steps) bool, where a new
        episode begins."""
        if obs.dim() != 3:
            _refuse(f"obs has to be (batch, steps, obs_dim), got {tuple(obs.shape)}")
        states = []

        def memory(k, x, r, i):
            h, last = gated_scan(x, r, i, self.decay[k], None if state is None else state[k], reset, c=self.c)
            states.append(last)
            return h

        actions = self._run(obs, memory)
        return actions, torch.stack(states)

    def step(self, obs, state):
        """obs (batch, obs_dim), state -> (actions (batch, action_dim), next state)."""
        if obs.dim() != 2:
            _refuse(f"obs has to be (batch, obs_dim), got {tuple(obs.shape)}")
        actions, state = self.forward(obs[:, None], state)
        return actions[:, 0], state

    @torch.no_grad()
    def act(self, obs, state):
        """``step`` without gradients: -> actions; ``state`` moves on in place."""
        if obs.dim() != 2:
            _refuse(f"obs has to be (batch, obs_dim), got {tuple(obs.shape)}")
        return self._run(obs, lambda k, x, r, i: gated_scan_step(x, r, i, self.decay[k], state[k], c=self.c))
