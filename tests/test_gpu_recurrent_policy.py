"""-m gpu: the policy built from the operators (policy.RecurrentPolicy), alone and in the simulator's loop (SolverNN), and what trains it there."""
import numpy as np
import pytest
import torch

from plasticinelab_amd.policy import RecurrentPolicy
from tests.util import O, oracle_prims, sparse_target
from tests.gpu_util import relerr
from tests.test_gpu_loss import c_sdf

pytestmark = pytest.mark.gpu
DEV = "cuda"

# float32 against float64, largest difference over largest value: a layer's product of K <= 320 terms is off by at most (K + 1) 2^-24 of its
# terms' absolute sum, the operators around it by some 60 2^-24, three layers a block and two blocks: 8 * 380 * 2^-24 = 1.8e-4 at the worst
TOL = 2e-4


def plain(policy, obs, state=None, reset=None):
    """The policy's formulas in float64 on the CPU, one step after the other; differentiable w.r.t. the copies it returns."""
    w = {k: v.detach().double().cpu().requires_grad_() for k, v in policy.named_parameters()}
    lin = lambda n, v: v @ w[n + ".weight"].T + w[n + ".bias"]                                               # noqa: E731
    rms = lambda v: v / torch.sqrt((v * v).mean(-1, keepdim=True) + policy.eps)                               # noqa: E731
    f = {"identity": lambda g: g, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[policy.gate_fn]

    def step(o, hs, cut):
        y, new = lin("embed", o), []
        for k in range(policy.depth):
            x, r, i, g = lin(f"into.{k}", rms(y) * w[f"pre.{k}"]).split(policy.width, dim=-1)
            la = -policy.c * torch.nn.functional.softplus(w[f"decay.{k}"]) * torch.sigmoid(r)
            a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
            a, m = torch.where(cut, 0.0, a), torch.where(cut, 1.0, m)
            h = a * hs[k] + m * torch.sigmoid(i) * x
            new.append(h)
            y = y + w[f"scale.{k}"] * f(g) * w[f"post.{k}"] * rms(lin(f"out.{k}", h))
        return lin("head", rms(y) * w[f"pre.{policy.depth}"]), new

    B, T = obs.shape[:2]
    hs = [torch.zeros(B, policy.width, dtype=torch.float64) if state is None else state[k].double().cpu() for k in range(policy.depth)]
    out = []
    for t in range(T):
        cut = torch.zeros(B, 1, dtype=torch.bool) if reset is None else reset[:, t:t + 1].cpu()
        a, hs = step(obs[:, t].double().cpu() if not obs.requires_grad else obs[:, t], hs, cut)
        out.append(a)
    return torch.stack(out, 1), torch.stack(hs), w, step


def off(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).abs().max() / b.abs().max().clamp(min=1e-30))


@pytest.mark.parametrize("gate_fn,resets", [("sigmoid", False), ("silu", True)])
def test_sequence_steps_and_gradients(gate_fn, resets):
    torch.manual_seed(0)
    policy = RecurrentPolicy(33, 6, width=72, depth=2, gate_fn=gate_fn)
    B, T = 3, 90
    obs, state = torch.randn(B, T, 33, device=DEV), torch.randn(2, B, 72, device=DEV)
    reset = torch.rand(B, T, device=DEV) < 0.05 if resets else None
    weight = torch.randn(B, T, 6, device=DEV)
    out, last = policy(obs, state, reset)
    ref, ref_last, w, _ = plain(policy, obs, state, reset)
    assert off(out, ref) < TOL and off(last, ref_last) < TOL
    (out * weight).sum().backward()
    (ref * weight.double().cpu()).sum().backward()
    for k, p in policy.named_parameters():
        assert off(p.grad, w[k].grad) < 4 * TOL, k            # (forward and backward, and sums over the steps)
    if reset is None:                                         # the same, an observation at a time
        s1, s2 = state, state.clone()
        for t in range(T):
            a1, s1 = policy.step(obs[:, t], s1)
            a2 = policy.act(obs[:, t], s2)
            assert off(a1, ref[:, t]) < TOL and off(a2, ref[:, t]) < TOL
        assert off(s1, ref_last) < TOL and off(s2, ref_last) < TOL


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_policy_of_16_bits(dtype):
    """Matrices and what passes through them in 16 bits: some 20 roundings of half a step each on the way from an observation to an action."""
    torch.manual_seed(1)
    policy = RecurrentPolicy(40, 6, width=128, depth=2, dtype=dtype)
    obs = torch.randn(2, 50, 40, device=DEV).to(dtype)
    out, last = policy(obs)
    ref, ref_last, w, _ = plain(policy, obs)
    tol = 20 * torch.finfo(dtype).eps / 2
    assert out.dtype == dtype and last.dtype == torch.float32 and off(out, ref) < tol and off(last, ref_last) < tol
    out.float().square().sum().backward()
    assert all(torch.isfinite(p.grad).all() and float(p.grad.float().abs().max()) > 0 for p in policy.parameters())


def make_env(n, n_obs):
    from plasticinelab_amd.engine import taichi_env as te
    from plasticinelab_amd.envs.scenes import load_scene

    class Sub(te.Shapes):
        def get(self):
            x, c = super().get()
            k = len(x) // n
            return np.ascontiguousarray(x[::k][:n]), c[::k][:n]

    cfg = load_scene("Move", 1)
    cfg.ENV.loss.target_path = ""
    orig, te.Shapes = te.Shapes, Sub
    try:
        env = te.TaichiEnv(cfg, compute_dtype="float64")
    finally:
        te.Shapes = orig
    env.initialize()
    env.loss.load_target_density(grids=sparse_target("Move3D-v1"))
    env.loss.set_weights(10, 10, 1, True)
    return cfg, env, (n // (n // n_obs)) * 6 + 7 * len(env.primitives)


def test_recurrent_policy_in_the_loop_matches_oracle(oracle_c):
    """Gradient of a rollout's loss w.r.t. the parameters, through the simulator, the observations AND the policy's memory, against the same closed loop
    on one autograd graph (float64 engine; the policy's float32 sets the difference)."""
    from plasticinelab_amd.optimizer.solver_nn import SolverNN
    n, H, n_obs, vw = 1500, 3, 50, 0.5
    cfg, env, obs_dim = make_env(n, n_obs)
    torch.manual_seed(2)
    policy = RecurrentPolicy(obs_dim, env.primitives.action_dim, width=32, depth=2)
    solver = SolverNN(env, policy, horizon=H, n_observed_particles=n_obs, velocity_weight=vw)
    assert solver.policy.embed.weight.dtype == torch.float32 and solver.obs.dim == obs_dim
    loss, grad = solver.forward(env.get_state()["state"])

    prims, s = oracle_prims(cfg), cfg.SIMULATOR
    sim = O.SimCfg(n_particles=n, yield_stress=s.yield_stress, E=s.E, nu=s.nu, ground_friction=s.ground_friction)
    tgt = sparse_target("Move3D-v1")
    sdf, td = torch.as_tensor(c_sdf(oracle_c, tgt, sim.dx).reshape(-1)), torch.as_tensor(tgt.reshape(-1))
    state, mats, poses = O.init_state(env.init_particles), O.materials(sim), O.init_poses(prims)
    idx = torch.as_tensor(solver.obs.index)
    _, _, w, step = plain(policy, torch.zeros(1, 1, obs_dim))
    memory, total, no = [torch.zeros(1, 32, dtype=torch.float64) for _ in range(2)], 0.0, torch.zeros(1, 1, dtype=torch.bool)
    for _ in range(H):
        obs = torch.cat([torch.cat([state[0][idx], state[1][idx] * vw], 1).reshape(-1)] + [torch.cat(po[:2]) for po in poses])
        act, memory = step(obs[None], memory, no)
        state, poses = O.env_step(sim, prims, 666.0, state, mats, poses, torch.clamp(act[0], -1.0, 1.0))
        l, _ = O.compute_loss(sim, O.LossCfg(soft_contact=True), prims, state[0], poses, td, sdf)
        total = total + l
    total.backward()
    ref = np.concatenate([w[k].grad.numpy().reshape(-1) for k, _ in policy.named_parameters()])
    print(f"\n[recurrent policy] loss rel {abs(loss - float(total.detach())) / abs(float(total.detach())):.2e}  gradient max-norm rel {relerr(grad, ref):.2e}")
    assert abs(loss - float(total.detach())) / abs(float(total.detach())) < 1e-5 and np.abs(ref).max() > 0 and relerr(grad, ref) < 4 * TOL


class Counting(torch.nn.Module):
    """A policy whose memory is outside the graph (``how``: a count kept without gradients, or handed on untouched) and does not reach its actions."""

    def __init__(self, obs_dim, action_dim, how):
        super().__init__()
        self.lin, self.how = torch.nn.Linear(obs_dim, action_dim, device=DEV), how

    def forward(self, obs):
        return self.lin(obs)

    def initial_state(self, batch):
        return torch.zeros(batch, 1, device=DEV)

    def step(self, obs, state):
        return self.lin(obs), state.detach() + 1 if self.how == "count" else state


@pytest.mark.parametrize("how", ["count", "untouched"])
def test_a_memory_outside_the_graph(how):
    from plasticinelab_amd.optimizer.solver_nn import SolverNN
    _, env, obs_dim = make_env(1000, 40)
    torch.manual_seed(4)
    policy = Counting(obs_dim, env.primitives.action_dim, how)
    state = env.get_state()["state"]
    _, grad = SolverNN(env, policy, horizon=3, n_observed_particles=40).forward(state)
    _, want = SolverNN(env, policy.lin, horizon=3, n_observed_particles=40).forward(state)
    assert np.abs(want).max() > 0 and relerr(grad, want) < TOL


@pytest.mark.parametrize("bits", [32, 8])
def test_solver_updates_a_policy_on_the_gpu(bits):
    """SolverNN.solve with AdamW, after a warm start from a recorded action sequence: the parameters it hands back are those of its best rollout."""
    from plasticinelab_amd.optimizer.solver_nn import SolverNN
    _, env, obs_dim = make_env(1000, 40)
    torch.manual_seed(3)
    policy = RecurrentPolicy(obs_dim, env.primitives.action_dim, width=32, depth=1)
    solver = SolverNN(env, policy, horizon=3, n_observed_particles=40, n_iters=3,
                      **{"optim.type": "AdamW", "optim.lr": 1.0, "optim.state_bits": bits, "optim.max_norm": 1.0})
    state = env.get_state()["state"]
    actions = np.random.RandomState(0).uniform(-0.5, 0.5, (3, env.primitives.action_dim))
    seen = solver.record(state, actions)
    assert seen.shape == (3, obs_dim)
    errors = solver.imitate(seen[None], actions[None], n_iters=4, reset=np.array([[True, False, False]]))
    assert len(errors) == 4 and all(np.isfinite(errors))
    env.set_state(state, 666.0, False)
    losses = []
    best = solver.solve(callbacks=[lambda s, optim, loss, grad: losses.append((loss, optim.iter, float(optim.grad_norm), np.linalg.norm(grad)))])
    assert len(losses) == 3 and [i for _, i, _, _ in losses] == [1, 2, 3]
    for _, _, norm, whole in losses:                      # the norm that the update saw is that of the gradient the solver reports
        assert abs(norm - whole) <= 1e-6 * whole
    assert np.array_equal(best, solver.get_params())
    again, _ = solver.forward(state, best)
    assert abs(again - min(l for l, _, _, _ in losses)) <= 1e-5 * abs(again)


def test_policy_refusals():
    with pytest.raises(ValueError, match="dtype"):
        RecurrentPolicy(4, 2, dtype=torch.float64)
    with pytest.raises(ValueError, match="width"):
        RecurrentPolicy(4, 2, width=9000)
    with pytest.raises(ValueError, match="gate_fn"):
        RecurrentPolicy(4, 2, gate_fn="tanh")
    policy = RecurrentPolicy(4, 2, width=8)
    with pytest.raises(ValueError, match="batch, steps"):
        policy(torch.zeros(3, 4, device=DEV))
    with pytest.raises(ValueError, match="batch, obs_dim"):
        policy.step(torch.zeros(4, device=DEV), policy.initial_state(1))
    with pytest.raises(ValueError, match="float32"):
        RecurrentPolicy(4, 2, width=8).double()(torch.zeros(1, 2, 4, device=DEV))


def test_act_in_inference_mode():
    policy = RecurrentPolicy(9, 4, width=24, depth=2)
    obs = torch.randn(5, 3, 9, device=DEV)
    with torch.no_grad():
        want, end = policy(obs)
    with torch.inference_mode():
        state = policy.initial_state(5)
        got = torch.stack([policy.act(obs[:, t], state) for t in range(3)], 1)
        again, last = policy(obs)
    assert off(got, want) < TOL and off(state, end) < TOL and torch.equal(again, want) and torch.equal(last, end)


def test_act_captured_and_replayed():
    """A rollout's step as a graph: the state moves on from replay to replay, with eager work and synchronisation in between."""
    policy = RecurrentPolicy(9, 4, width=64, depth=2)
    obs = torch.randn(8, 5, 9, device=DEV)
    state, slot = policy.initial_state(5), torch.zeros(5, 9, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        policy.act(slot, state.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = policy.act(slot, state)
    state.zero_()
    eager = policy.initial_state(5)
    for t in range(8):
        slot.copy_(obs[t])
        graph.replay()
        want = policy.act(obs[t], eager)
        torch.cuda.synchronize()
        assert off(out, want) < TOL and off(state, eager) < TOL, t


def test_recording_longer_than_the_frames_and_what_it_leaves():
    """A recording keeps no frames: more steps than max_steps holds, the same observations as with frames kept, and the environment where it began."""
    from plasticinelab_amd.optimizer.solver_nn import SolverNN
    _, env, obs_dim = make_env(1000, 40)
    torch.manual_seed(6)
    policy = RecurrentPolicy(obs_dim, env.primitives.action_dim, width=16, depth=1)
    solver = SolverNN(env, policy, horizon=2, n_observed_particles=40, n_iters=1, **{"optim.type": "AdamW"})
    state = env.get_state()["state"]
    steps = env.simulator.max_steps // env.simulator.substeps + 4
    actions = np.random.RandomState(1).uniform(-0.3, 0.3, (steps, env.primitives.action_dim))
    softness, copying = env.primitives.get_softness(), env._is_copy
    seen = solver.record(state, actions)
    assert seen.shape == (steps, obs_dim) and np.isfinite(seen).all()
    assert env.primitives.get_softness() == softness and env._is_copy == copying
    after = env.get_state()["state"]
    assert all(np.array_equal(np.asarray(a), np.asarray(b)) for a, b in zip(after, state))
    env.set_state(state, solver.cfg.softness, False)
    kept = []
    for a in actions[:5]:
        kept.append(solver.obs.read(env.simulator.cur))
        env.step(a)
    assert np.abs(np.stack(kept) - seen[:5]).max() < 1e-9         # (a float64 engine whose scatters add in any order)
    env.set_state(state, softness, copying)
    losses = []
    solver.record(state, actions[:2])
    solver.solve(callbacks=[lambda s, optim, loss, grad: losses.append(loss)])        # straight on, as imitation's warm start ends
    assert len(losses) == 1 and np.isfinite(losses[0])


def test_a_recording_that_fails_leaves_the_environment_where_it_began(monkeypatch):
    from plasticinelab_amd.optimizer.solver_nn import SolverNN
    _, env, obs_dim = make_env(1000, 40)
    solver = SolverNN(env, torch.nn.Linear(obs_dim, env.primitives.action_dim), horizon=2, n_observed_particles=40)
    state, softness, copying = env.get_state()["state"], env.primitives.get_softness(), env._is_copy
    step, steps = env.step, []

    def failing(action):
        if len(steps) == 2:
            raise RuntimeError("stopped")
        steps.append(action)
        step(action)

    monkeypatch.setattr(env, "step", failing)
    with pytest.raises(RuntimeError, match="stopped"):
        solver.record(state, np.full((4, env.primitives.action_dim), 0.3))
    assert len(steps) == 2 and env.primitives.get_softness() == softness and env._is_copy == copying
    assert all(np.array_equal(np.asarray(a), np.asarray(b)) for a, b in zip(env.get_state()["state"], state))
