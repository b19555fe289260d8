"""Operators of a policy that is a sequence model, as HIP kernels (csrc/plmpm_scan.hip, csrc/plmpm_norm.hip; C ABI include/plmpm_policy.h), and
the policy built from them.

    h, last = gated_scan(x, r, i, decay, h0, reset)         # a gated linear recurrence over whole sequences, differentiable
    h = gated_scan_step(x, r, i, decay, state)              # one observation: ``state`` moves on in place
    y, z = block_norm(x, u, gate, scale, post, pre)         # norms before and after a block, its gate and residual scale
    policy = RecurrentPolicy(obs_dim, action_dim)           # what SolverNN drives (optimizer/solver_nn.py)

Tensors live on one GPU; kernels go to the current stream of that GPU and nothing synchronises, so calls can be captured into a graph (a
backward pass too, as long as no eager graph of the same leaves is alive: torch would join the two streams, which a capture forbids).
There is no CPU path.  Derivatives are first ones in reverse mode; forward-mode tangents, second derivatives and tracing (torch.jit.trace, make_fx) are refused.
The reference's counterpart is a per-step MLP (plb/engine/nn/mlp.py:11-183) without a memory.
"""
from __future__ import annotations

import ctypes as C
import os

import torch

from . import _lib as L

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
GATES = {"identity": 0, "sigmoid": 1, "silu": 2}
MAX_WIDTH = 8192                        # of block_norm (a row stays in one workgroup's registers)

# ---- plumbing: what torch has to be told of these operators is C++ (csrc/policy_binding.cpp: checks, allocations, autograd, the calls)
BINDING_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_policy_binding.so")
_bound = None


def _binding():
    global _bound
    if _bound is None:
        if not os.path.exists(BINDING_PATH):
            raise L.EngineError(f"{BINDING_PATH} not found: it is built with the library.  Run `python -c 'import __graft_entry__ as g; g.build()'` at the repo root.")
        from . import _policy_binding
        _attach(_policy_binding, L.load_policy())
        _bound = _policy_binding
    return _bound


def _attach(binding, lib, host=False):
    """Hand the library's entry points over.  ``host``: they take host memory (the tests' interpreter of the device source)."""
    binding.attach({name: C.cast(getattr(lib, name), C.c_void_p).value for name in (*L.POLICY_SYMBOLS, "plmpm_last_error")}, L.EngineError, host)


def _refuse(message):
    raise ValueError(message)


def _not_tensors(optional=(), **named):
    """Called for a TypeError of the binding: a ValueError that names the argument which is no tensor, if that was it."""
    for name, t in named.items():
        if not isinstance(t, torch.Tensor) and (t is not None or name not in optional):
            raise ValueError(f"{name} has to be a tensor, got {type(t).__name__}") from None


# ---------------------------------------------------------------------------------------------- gated linear recurrence
def gated_scan(x, r, i, decay, h0=None, reset=None, *, c: float = 8.0):
    """Gated linear recurrence over sequences: ``-> (h, last)``.

        a_t = exp(-c softplus(decay) sigmoid(r_t));   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t

    x, r, i: (B, T, D), float32, bfloat16 or float16; batch and time strides are free (slices of one projection are read in place).
    decay: (D,) float32.  h0: (B, D) float32, the state before the first step (zeros if None).  reset: (B, T) bool; where it is set, a_t is 0:
    the sequence starts anew and nothing of what came before, a NaN either, reaches it.  h has x's type, ``last`` (B, D) is the float32
    state behind step T-1 (all rows of a batch have T steps: pack shorter episodes with ``reset``).  The state is carried in float32; gradients
    reach x, r, i, decay and h0 (its backward pass makes the states again from one float32 state in 64 steps).
    """
    try:
        return _binding().gated_scan(x, r, i, decay, h0, reset, c)
    except TypeError:
        _not_tensors(("h0", "reset"), x=x, r=r, i=i, decay=decay, h0=h0, reset=reset)
        raise


def gated_scan_step(x, r, i, decay, state, *, c: float = 8.0):
    """One step of ``gated_scan`` for (B, D) inputs: -> h (B, D); ``state`` (B, D) float32 moves on in place.  No gradients (serving and
    evaluation; a differentiable step is ``gated_scan`` with T = 1).  Inputs may lie in the state: they are read as they were before it moves."""
    try:
        return _binding().gated_scan_step(x, r, i, decay, state, c)
    except TypeError:
        _not_tensors(x=x, r=r, i=i, decay=decay, state=state)
        raise


# ---------------------------------------------------------------------------------------------- norms around a block
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
    if gate_fn not in GATES:
        _refuse(f"gate_fn has to be one of {sorted(GATES)}, got {gate_fn!r}")
    try:
        return _binding().block_norm(x, u, gate, scale, post, pre, eps, GATES[gate_fn], dtype)
    except TypeError:
        _not_tensors(("u", "gate", "scale", "post", "pre"), x=x, u=u, gate=gate, scale=scale, post=post, pre=pre)
        raise


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

    def _check_state(self, state):
        if len(state) != self.depth:
            _refuse(f"state has to be of {self.depth} blocks, got {len(state)}")

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
        episode begins (its first input then enters with a gain of 1, as ``gated_scan``'s reset has it; behind a state of zeros it is sqrt(1 - a^2))."""
        if obs.dim() != 3:
            _refuse(f"obs has to be (batch, steps, obs_dim), got {tuple(obs.shape)}")
        if state is not None:
            self._check_state(state)
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
        self._check_state(state)
        return self._run(obs, lambda k, x, r, i: gated_scan_step(x, r, i, self.decay[k], state[k], c=self.c))
