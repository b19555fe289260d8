"""Policy-in-the-loop differentiation: mirror of /root/reference/plb/optimizer/solver_nn.py:3-76 with the
hand-rolled Taichi MLP (plb/engine/nn/mlp.py) replaced by any ``torch.nn.Module``.

At every env step the policy sees the observation the reference's MLP builds (mlp.py:63-84): position and
``velocity_weight`` x velocity of every ``obs_step``-th particle at the step's first frame, then the 7-number pose of
every manipulator; its output, clamped to [-1, 1] (mlp.py:98), is the step's action.  The gradient of the rollout
loss w.r.t. the policy parameters flows

    loss -> (HIP adjoint of the step) -> d loss / d action[t] -> torch autograd through the policy
         -> d loss / d obs[t] -> back into the HIP adjoint of frame t*substeps (particle x, v and manipulator poses)

the last arrow through ``Tape(after_step_grad=...)`` / ``Engine.add_frame_grad`` / ``add_primitive_grad``.

A policy on the CPU runs in float64.  A policy on a GPU keeps its own type and place, may have a memory (``initial_state`` and ``step``, as
``policy.RecurrentPolicy`` has them: its gradient then also flows from each step's state to the one before), and is what ``optim.type =
"AdamW"`` and ``imitate`` are for.
"""
from __future__ import annotations

import inspect

import numpy as np
import torch

from ..config import CfgNode
from ..engine.taichi_env import TaichiEnv, Tape
from .adamw import AdamW
from .optim import Adam, Momentum

OPTIMS = {"Adam": Adam, "Momentum": Momentum, "AdamW": AdamW}


class Observation:
    """mlp.py:31-38,63-84: which particles are observed and how an observation vector is laid out."""

    def __init__(self, env: TaichiEnv, n_observed_particles=200, velocity_weight=1.0):
        self.env = env
        n = env.simulator.n_particles
        self.obs_step = n // n_observed_particles
        self.obs_num = n // self.obs_step
        self.index = np.arange(self.obs_num) * self.obs_step
        self.velocity_weight = float(velocity_weight)
        self.dim = self.obs_num * 6 + 7 * len(env.primitives)

    def read(self, f) -> np.ndarray:
        sim = self.env.simulator
        fr = sim.engine.get_frame(f, want=("x", "v"))
        part = np.concatenate([fr["x"][self.index], fr["v"][self.index] * self.velocity_weight], axis=1).reshape(-1)
        prim = [p.get_state(f)[:7] for p in self.env.primitives]
        return np.concatenate([part] + prim) if prim else part

    def push_grad(self, f, g: np.ndarray):
        """d loss / d obs -> adjoint of frame ``f`` (which must be the resident adjoint frame)."""
        sim = self.env.simulator
        n = sim.n_particles
        gp = g[:self.obs_num * 6].reshape(self.obs_num, 6)
        xa, va = np.zeros((n, 3)), np.zeros((n, 3))
        xa[self.index] = gp[:, :3]
        va[self.index] = gp[:, 3:] * self.velocity_weight
        sim.engine.add_frame_grad(f, xa=xa, va=va)
        base = self.obs_num * 6
        for i in range(len(self.env.primitives)):
            sim.engine.add_primitive_grad(i, f, g[base + 7 * i: base + 7 * i + 7])


class SolverNN:
    def __init__(self, env: TaichiEnv, policy: torch.nn.Module, logger=None, cfg=None, n_observed_particles=200,
                 velocity_weight=1.0, **kwargs):
        self.cfg = self.default_config()
        if cfg is not None:
            self.cfg.merge(dict(cfg), strict=False)
        for k, v in kwargs.items():
            node = self.cfg
            parts = k.split(".")
            for p in parts[:-1]:
                node = node[p]
            node[parts[-1]] = v
        self.cfg.optim.lr *= 0.001                         # solver_nn.py:6-7
        self.cfg.optim.bounds = (-np.inf, np.inf)
        self.env = env
        first = next(policy.parameters(), None)
        self.policy = policy if first is not None and first.is_cuda else policy.double()
        first = next(self.policy.parameters(), None)
        self.place = {"dtype": torch.float64, "device": "cpu"} if first is None else {"dtype": first.dtype, "device": first.device}
        self.logger = logger
        self.obs = Observation(env, n_observed_particles, velocity_weight)
        self.total_steps = 0

    @classmethod
    def default_config(cls):                               # solver_nn.py:65-76
        return CfgNode({"optim": {"lr": 0.1, "bounds": (-1.0, 1.0), "type": "Adam"}, "n_iters": 100, "softness": 666.0,
                        "horizon": 50, "init_range": 0.0, "init_sampler": "uniform"})

    # ---- flat parameter vector, as nn.get_params / set_params / get_grad (mlp.py:154-183)
    def get_params(self):
        return np.concatenate([p.detach().double().cpu().numpy().reshape(-1) for p in self.policy.parameters()])

    def set_params(self, flat):
        flat = np.asarray(flat, np.float64)
        o = 0
        with torch.no_grad():
            for p in self.policy.parameters():
                n = p.numel()
                p.copy_(torch.as_tensor(flat[o:o + n].reshape(p.shape), dtype=p.dtype))
                o += n

    def forward(self, sim_state, params=None):             # solver_nn.py:28-43
        env, sim = self.env, self.env.simulator
        if params is not None:
            self.set_params(params)
        env.set_state(sim_state, self.cfg.softness, False)
        if self.logger is not None:
            self.logger.reset()
        for p in self.policy.parameters():
            p.grad = None
        graph = {}                                         # step -> (obs tensor, action tensor[, state in, state out])
        A = env.primitives.action_dim
        memory = hasattr(self.policy, "initial_state")
        state = self.policy.initial_state(1) if memory else None
        from_later = []                                    # d loss / d state handed to the next step, from the reverse sweep

        def after_step_grad(step, first_frame):
            obs_t, act_t, *states = graph.pop(step)
            g = torch.as_tensor(sim.engine.get_action_grad(step + 1)[step].reshape(-1)[:A].copy()).to(**self.place)
            ends, grads = [act_t], [g]
            later = from_later.pop() if from_later else None
            if later is not None and states[1].requires_grad:      # (a policy may leave its memory out of the graph)
                ends.append(states[1])
                grads.append(later)
            torch.autograd.backward(ends, grads)           # accumulates into policy.parameters().grad, fills obs_t.grad
            if states:
                from_later[:] = [states[0].grad]
            self.obs.push_grad(first_frame, obs_t.grad.double().cpu().numpy())

        with Tape(env, after_step_grad=after_step_grad):
            for i in range(self.cfg.horizon):
                obs_t = torch.tensor(self.obs.read(sim.cur), requires_grad=True, **self.place)
                if memory:
                    before = state.detach().requires_grad_()
                    act_t, state = self.policy.step(obs_t[None], before)
                    act_t = torch.clamp(act_t[0], -1.0, 1.0)
                    graph[i] = (obs_t, act_t, before, state)
                else:
                    act_t = torch.clamp(self.policy(obs_t), -1.0, 1.0)          # mlp.py:98
                    graph[i] = (obs_t, act_t)
                env.step(act_t.detach().double().cpu().numpy())
                self.total_steps += 1
                info = env.compute_loss()
                if self.logger is not None:
                    self.logger.step(None, None, info["reward"], None, i == self.cfg.horizon - 1, info)
        grad = np.concatenate([(p.grad if p.grad is not None else torch.zeros_like(p)).double().cpu().numpy().reshape(-1)
                               for p in self.policy.parameters()])
        return env.loss.loss, grad

    def solve(self, callbacks=()):                         # solver_nn.py:14-63
        env = self.env
        params = self.get_params()
        on_device = self.cfg.optim.type == "AdamW"         # updates the policy's tensors where they are; the others a flat vector
        optim = OPTIMS[self.cfg.optim.type](list(self.policy.parameters()) if on_device else params, self.cfg.optim)
        env_state = env.get_state()
        self.total_steps = 0
        best, best_loss = None, 1e10
        for _ in range(self.cfg.n_iters):
            self.params = params
            loss, grad = self.forward(env_state["state"], None if on_device else params)
            if loss < best_loss:
                best_loss, best = loss, params.copy()
            if on_device:
                optim.step()
                params = self.get_params()
            else:
                params = optim.step(grad)
            for cb in callbacks:
                cb(self, optim, loss, grad)
        env.set_state(**env_state)
        self.set_params(best)
        return best

    # ---- a warm start from action sequences that another solver found
    def record(self, sim_state, actions):
        """Run ``actions`` (H, action_dim) from ``sim_state``: -> the observations (H, obs.dim) a policy would have seen before each of them.  No
        frames are kept, so H is not bound by ``max_steps``; the environment is left at ``sim_state``."""
        env, seen = self.env, []
        softness, is_copy = env.primitives.get_softness(), env._is_copy
        env.set_state(sim_state, self.cfg.softness, True)
        try:
            for a in actions:
                seen.append(self.obs.read(env.simulator.cur))
                env.step(a)
        finally:
            env.set_state(sim_state, softness, is_copy)
        return np.stack(seen)

    def _whole_sequences(self, obs, reset):
        """The policy's actions over sequences (B, H, obs.dim).  A policy with a memory whose ``forward`` takes ``reset`` gets them at once and answers
        (actions, state); any other one goes through ``initial_state`` and ``step``, row by row where there are resets (which part of a state is a
        row's is the policy's business).  A policy without a memory has nothing to reset."""
        if not hasattr(self.policy, "initial_state"):
            return self.policy(obs)
        try:
            at_once = "reset" in inspect.signature(self.policy.forward).parameters
        except (TypeError, ValueError):                    # (a compiled forward has no signature to ask)
            at_once = False
        if at_once:
            out = self.policy(obs, reset=reset)
            if not isinstance(out, (tuple, list)) or len(out) != 2:
                raise ValueError(f"a policy whose forward takes reset has to answer (actions, state), got {type(out).__name__}")
            return out[0]

        def walk(rows, begins):
            state, answers = self.policy.initial_state(rows.shape[0]), []
            for t in range(rows.shape[1]):
                if begins[t]:
                    state = self.policy.initial_state(rows.shape[0])
                answer, state = self.policy.step(rows[:, t], state)
                answers.append(answer)
            return torch.stack(answers, 1)

        if reset is None:
            return walk(obs, [False] * obs.shape[1])
        return torch.cat([walk(row[None], begins) for row, begins in zip(obs, reset.tolist())])

    def imitate(self, observations, actions, n_iters=100, reset=None):
        """Fit the policy to recorded sequences by least squares: observations (B, H, obs.dim), actions (B, H, action_dim); ``reset`` (B, H) marks steps
        that begin an episode (sequences of several).  Whole sequences go through the policy at once (one with a memory whose ``forward`` takes no
        ``reset`` goes through its ``step``); AdamW with this solver's optimiser settings updates it.  -> the mean squared errors, one an iteration."""
        obs, target = (torch.as_tensor(np.asarray(a)).to(**self.place) for a in (observations, actions))
        if hasattr(self.policy, "initial_state") and obs.dim() != 3:
            raise ValueError(f"observations of a policy with a memory have to be (B, H, obs.dim), got {tuple(obs.shape)}")
        if reset is not None:
            reset = torch.as_tensor(np.asarray(reset, bool)).to(self.place["device"])
            if reset.shape != obs.shape[:-1]:
                raise ValueError(f"reset has to be {tuple(obs.shape[:-1])}, got {tuple(reset.shape)}")
        optim = AdamW(list(self.policy.parameters()), self.cfg.optim)
        losses = []
        for _ in range(int(n_iters)):
            for p in self.policy.parameters():
                p.grad = None
            out = self._whole_sequences(obs, reset)
            if out.shape != target.shape:
                raise ValueError(f"the policy answers {tuple(out.shape)} to these observations, actions are {tuple(target.shape)}")
            loss = torch.nn.functional.mse_loss(out.float(), target.float())
            loss.backward()
            optim.step()
            losses.append(loss.detach())
        return [float(x) for x in losses]
