"""CPU tier: the policy-training operators' device source on the CPU interpreter (tests/host_emul/hipemu), against their 64-bit forms.
tests/test_gpu_policy_ops.py runs the same checks, and larger ones, on a GPU."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from plasticinelab_amd import _lib
from plasticinelab_amd import policy as P
from plasticinelab_amd.optimizer import AdamW, adamw_step, adamw_values
from tests import policy_cases as cases
from tests.util import ROOT

HERE = os.path.join(ROOT, "tests", "host_emul")
SOURCES = "plmpm_capi.hip plmpm_kinematics.hip plmpm_loss.hip plmpm_migrate.hip plmpm_peer.hip plmpm_scan.hip plmpm_norm.hip plmpm_adamw.hip"


@pytest.fixture(scope="module")
def interpreter():
    """The operators' library compiled by g++ for the interpreter; tensors on the CPU stand for device memory.  (PLMPM_EMUL_VARIANT=asan: under
    AddressSanitizer; LD_PRELOAD then holds libasan.so and, for the C++ exceptions of the binding, libstdc++.so.6.)"""
    tag = "_asan" if os.environ.get("PLMPM_EMUL_VARIANT") == "asan" else ""
    out = f"libplmpm_policy_emul{tag}.so"
    subprocess.check_call(["make", "-s", "-j", "6", "-C", HERE, f"OBJDIR=build_emul_policy{tag}", f"OUT={out}", f"SAN={1 if tag else 0}",
                           "HDRS=" + " ".join(os.path.join("../../plasticinelab_amd/csrc", h) for h in ("plmpm_nn.h", "plmpm_kernels.h")) + " ../../include/plmpm_policy.h",
                           "SRCS=" + SOURCES, out])
    lib = _lib.bind(C.CDLL(os.path.join(HERE, out)), {**_lib.POLICY_SYMBOLS, "plmpm_last_error": _lib.SYMBOLS["plmpm_last_error"]})
    binding = P._binding()
    P._attach(binding, lib, host=True)
    yield "cpu"
    P._attach(binding, _lib.load_policy())


def test_policy_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "plmpm_policy.h")).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(plmpm_[a-z_0-9]+)\s*\(", text))) == sorted(_lib.POLICY_SYMBOLS)
    lib = _lib.load_policy()
    for name in _lib.POLICY_SYMBOLS:
        assert hasattr(lib, name)
    assert C.sizeof(_lib.Scan) == 4 * 8 + 6 * 8 + 8 + 18 * 8 and C.sizeof(_lib.Norm) == 16 + 7 * 8 + 8 + 18 * 8
    assert C.sizeof(_lib.AdamWTensor) == 72 and C.sizeof(_lib.AdamWStep) == 8 + 8 * 8 + 4 * 8


@pytest.mark.parametrize("B,T,D,dtype,layout,resets", [
    (1, 1, 1, "f32", "plain", 0.0), (2, 7, 64, "bf16", "plain", 0.3), (1, 64, 65, "f32", "packed", 0.0), (2, 65, 130, "f16", "packed", 0.1),
    (1, 129, 128, "f32", "time_major", 0.05), (3, 20, 33, "bf16", "odd", 0.0), (1, 200, 6, "f32", "plain", 0.0)])
def test_scan(interpreter, B, T, D, dtype, layout, resets):
    cases.run_scan(interpreter, 11, B, T, D, dtype, layout, resets=resets, with_h0=T != 20)


@pytest.mark.parametrize("B,T,D,dtype,layout,resets", [
    (2, 70, 65, "bf16", "plain", 0.1), (1, 200, 193, "f16", "odd", 0.05), (2, 130, 129, "bf16", "packed", 0.0), (2, 20, 128, "f16", "odd", 0.0), (1, 65, 127, "bf16", "time_major", 0.2),
    (1, 2, 255, "bf16", "plain", 0.0)])
def test_scan_of_16_bits_between_words(interpreter, B, T, D, dtype, layout, resets):
    cases.run_scan(interpreter, 12, B, T, D, dtype, layout, resets=resets, with_h0=T != 20)


@pytest.mark.parametrize("use", [("h",), ("last",)])
def test_scan_with_one_gradient(interpreter, use):
    cases.run_scan(interpreter, 5, 2, 70, 16, "f32", use=use)


def test_scan_step(interpreter):
    cases.run_step(interpreter, 3, 5, 66, "bf16")


@pytest.mark.parametrize("T,cut,at", [(16, 9, 12), (40, 16, 17), (200, 65, 130), (300, 129, 130)])
def test_nothing_behind_a_reset_reaches_gradients_before_it(interpreter, T, cut, at):
    cases.run_reset_and_what_is_not_finite_behind_it(interpreter, T, cut, at)


@pytest.mark.parametrize("T", [3, 17, 130])
def test_a_last_step_that_begins_anew_at_infinity(interpreter, T):
    cases.run_last_step_reset_to_infinity(interpreter, T)


@pytest.mark.parametrize("shape,tx,tu,fn,strided", [
    ((3, 8), "f32", "f32", "sigmoid", False), ((2, 5, 33), "bf16", "bf16", "silu", False), ((9, 130), "f32", "f16", "identity", True),
    ((5, 520), "f16", "f16", "sigmoid", True), ((2, 2050), "f32", "bf16", "silu", False), ((70, 1), "f32", "f32", "sigmoid", False),
    ((5, 9), "f16", "f16", "silu", True), ((3, 71), "f32", "bf16", "identity", False), ((2, 7), "bf16", "bf16", "sigmoid", False)])
def test_norm(interpreter, shape, tx, tu, fn, strided):
    cases.run_norm(interpreter, 21, shape, tx, tu, fn, strided=strided)


@pytest.mark.parametrize("use,grads", [(("pre",), ("dz",)), (("u",), ("dy",)), (("u", "pre"), ("dz",)), (("u", "gate", "post"), ("dy",)), (("u", "gate", "pre"), ("dy",))])
def test_norm_parts(interpreter, use, grads):
    cases.run_norm(interpreter, 22, (6, 72), "f32", "f32", use=use, grads=grads)
    cases.run_norm(interpreter, 23, (3, 600), "bf16", "bf16", use=use, grads=grads, weights=torch.bfloat16)


def test_norm_first_of_a_16_bit_block_next_to_a_float_stream(interpreter):
    cases.run_norm(interpreter, 24, (4, 40), "f32", "bf16", use=("pre",), grads=("dz",), dtype=torch.bfloat16)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes,dtypes,offset", [((1, 5, 300, 4096), ("f32",), 0), ((4097, 255), ("bf16", "f32", "f16"), 0), ((700, 4100), ("f32", "bf16"), 1)])
def test_adamw(interpreter, bits, sizes, dtypes, offset):
    cases.run_adamw(interpreter, 31, sizes, dtypes, bits, lr=1e-2, offset=offset, max_norm=0.05)


def test_adamw_without_masters_or_a_gradient_and_with_bounds(interpreter):
    cases.run_adamw(interpreter, 32, (40, 33), ("bf16",), 32, lr=0.1, masters=False)
    cases.run_adamw(interpreter, 33, (40, 33, 7), ("f32",), 8, lr=0.5, missing=(1,), bounds=(-0.3, 0.2), max_norm=1e3)


def test_adamw_more_tensors_than_one_launch_takes(interpreter):
    cases.run_adamw(interpreter, 34, tuple(range(1, 102)), ("f32",), 32, steps=2, max_norm=0.1)


def test_numbers_out_of_range_are_refused_at_the_c_entry(interpreter):
    p, step = torch.zeros(10), torch.zeros(2, dtype=torch.int64)
    z = lambda: [torch.zeros(10)]                                                                        # noqa: E731
    for kw, text in (({"beta_1": 1.0}, "betas"), ({"beta_2": -0.1}, "betas"), ({"epsilon": -1.0}, "epsilon"), ({"max_norm": -1.0}, "max_norm"), ({"bounds": (1.0, -1.0)}, "bounds"),
                     ({"max_norm": float("nan")}, "max_norm")):
        with pytest.raises(_lib.EngineError, match=text):
            adamw_step([p], [p], z(), z(), step, **kw)
    assert float(p.abs().sum()) == 0 and step.tolist() == [0, 0]


def leaves(*shapes):
    gen = torch.Generator().manual_seed(3)
    return [torch.randn(shape, generator=gen).requires_grad_() for shape in shapes]


def test_second_derivatives_are_refused(interpreter):
    x, r, i, decay = leaves((2, 7, 8), (2, 7, 8), (2, 7, 8), (8,))
    for value, name in ((P.gated_scan(x, r, i, decay)[0], "gated_scan"), (P.block_norm(x, pre=decay)[1], "block_norm")):
        grad, = torch.autograd.grad(value.square().sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match=f"{name} has no second derivative"):
            grad.sum().backward()


def test_a_saved_tensor_that_was_changed_is_noticed(interpreter):
    x, r, i, decay = leaves((2, 7, 8), (2, 7, 8), (2, 7, 8), (8,))
    for value in (P.gated_scan(x, r, i, decay)[0], P.block_norm(x, r, post=decay)[0]):
        with torch.no_grad():
            decay.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            value.sum().backward()


@pytest.mark.parametrize("reentrant", [False, True])
def test_under_activation_checkpointing(interpreter, reentrant):
    from torch.utils.checkpoint import checkpoint
    args = leaves((2, 70, 8), (2, 70, 8), (2, 70, 8), (8,), (2, 8))

    def run(x, r, i, decay, h0):
        return P.block_norm(P.gated_scan(x, r, i, decay, h0)[0], r, i, decay, decay, decay, gate_fn="silu")[1]

    run(*args).square().sum().backward()
    want = [t.grad.clone() for t in args]
    for t in args:
        t.grad = None
    checkpoint(run, *args, use_reentrant=reentrant).square().sum().backward()
    assert all(torch.equal(t.grad, w) for t, w in zip(args, want))


def test_only_the_gradients_that_are_asked_for(interpreter):
    x, r, i, decay = leaves((2, 7, 8), (2, 7, 8), (2, 7, 8), (8,))
    full = torch.autograd.grad(P.gated_scan(x, r, i, decay)[1].sum(), [x, r, i, decay])
    h, last = P.gated_scan(x.detach(), r.detach(), i.detach(), decay)
    assert torch.equal(torch.autograd.grad(last.sum(), [decay])[0], full[3])
    y, z = P.block_norm(x, r, pre=decay)
    assert [t is None for t in torch.autograd.grad(y.sum(), [x, r, decay], allow_unused=True, retain_graph=True)] == [False] * 3
    assert torch.equal(torch.autograd.grad(y.sum(), [x], retain_graph=True)[0], torch.ones_like(x))
    assert P.block_norm(x, pre=decay)[0] is x


def test_norm_of_rows_far_apart(interpreter):
    cases.run_norm_of_rows_far_apart(interpreter)


# ---- what torch carries beside a tensor's values, or records of a call, and a kernel does not see
def test_forward_mode_tangents_are_refused(interpreter):
    import torch.autograd.forward_ad as forward_ad
    x, r, i, decay, h0 = (t.detach() for t in leaves((2, 7, 8), (2, 7, 8), (2, 7, 8), (8,), (2, 8)))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))                                     # noqa: E731
        for call in (lambda: P.gated_scan(dual(x), r, i, decay), lambda: P.gated_scan(x, r, i, dual(decay)), lambda: P.gated_scan(x, r, i, decay, dual(h0)),
                     lambda: P.gated_scan_step(dual(x[:, 0]), r[:, 0], i[:, 0], decay, h0), lambda: P.gated_scan_step(x[:, 0], r[:, 0], i[:, 0], decay, dual(h0)),
                     lambda: P.block_norm(dual(x), pre=decay), lambda: P.block_norm(x, dual(r)), lambda: P.block_norm(x, r, pre=dual(decay)),
                     lambda: adamw_step([dual(decay)], [decay.clone()], [torch.zeros(8)], [torch.zeros(8)], torch.zeros(2, dtype=torch.int64)),
                     lambda: adamw_step([decay], [dual(decay.clone())], [torch.zeros(8)], [torch.zeros(8)], torch.zeros(2, dtype=torch.int64))):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode derivative"):      # (tangents are carried there too)
                call()
        leaf = x.clone().requires_grad_()                    # a tangent that only the gradient has: through a weight behind the operator
        for out in (P.gated_scan(leaf, r, i, decay)[0], P.gated_scan(leaf, r, i, decay)[1], P.block_norm(leaf, r)[0], P.block_norm(leaf, r, pre=decay)[1]):
            with pytest.raises((ValueError, RuntimeError), match="no forward-mode derivative"):
                torch.autograd.grad((out * dual(torch.ones_like(out))).sum(), leaf)
        with forward_ad._set_fwd_grad_enabled(False):        # where torch itself leaves tangents out
            assert torch.equal(P.gated_scan(dual(x), r, i, decay)[0], P.gated_scan(x, r, i, decay)[0])


def test_recorders_of_programs_are_refused(interpreter):
    """A traced program would hold the calls' allocations without their kernels and hand out what happens to lie in that memory."""
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, r, i, decay = leaves((2, 7, 8), (2, 7, 8), (2, 7, 8), (8,))
    plain = [t.detach() for t in (x, r, i, decay)]
    first, second, step = [torch.zeros(8)], [torch.zeros(8)], torch.zeros(2, dtype=torch.int64)
    h = P.gated_scan(x, r, i, decay)[0]
    calls = (lambda t: P.gated_scan(t, *plain[1:])[0], lambda t: P.gated_scan_step(t[:, 0], plain[1][:, 0], plain[2][:, 0], plain[3], torch.zeros(2, 8)), lambda t: P.block_norm(t, plain[1])[0],
             lambda t: P.block_norm(t, pre=plain[3])[1], lambda t: P.gated_scan(t.detach().requires_grad_(), *plain[1:])[0], lambda t: torch.autograd.grad(h, x, t, retain_graph=True)[0],
             lambda t: adamw_step([t[0, 0]], [plain[3]], first, second, step) or t + 1)
    for call in calls:
        for record in (lambda f, t: torch.jit.trace(f, (t,), check_trace=False), lambda f, t: make_fx(f)(t), lambda f, t: make_fx(f, pre_dispatch=True)(t)):
            with pytest.raises(RuntimeError, match="cannot be traced|Cannot insert a Tensor that requires grad"):      # (the second: torch's own, of a backward pass)
                record(call, plain[0].clone())
    with FakeTensorMode() as mode, pytest.raises(_lib.EngineError, match="cannot be traced"):
        P.block_norm(mode.from_tensor(plain[0]), mode.from_tensor(plain[1]))
    from torch.utils.flop_counter import FlopCounterMode           # a mode that only looks on
    with FlopCounterMode(display=False):
        assert torch.equal(P.gated_scan(*plain)[0], h)


@pytest.mark.parametrize("how", ["imag", "view"])
def test_negative_views_and_zeros_without_memory(interpreter, how):
    """x.conj().imag and the gradients of complex products are views with a sign that torch only notes: the operators see the values."""
    B, T, D = 2, 7, 8
    noted = lambda t: torch.complex(torch.zeros_like(t), t).conj().imag if how == "imag" and t.dim() > 1 else torch._neg_view(t)                  # noqa: E731
    args = leaves((B, T, D), (B, T, D), (B, T, D), (D,), (B, D))
    minus = [noted(t) for t in args]
    assert all(t.is_neg() for t in minus)
    for one, other in ((P.gated_scan(*minus), P.gated_scan(*[-t for t in args])), (P.gated_scan(*[t.detach() for t in minus]), P.gated_scan(*[-t for t in args]))):
        assert all(torch.equal(a, b) for a, b in zip(one, other))
    x, r, i, decay, h0 = args
    weights = [noted(t) for t in leaves((D,), (D,), (D,))]
    for a, b in zip(P.block_norm(minus[0], minus[1], minus[2], *weights), P.block_norm(-x, -r, -i, *[w.clone() for w in weights])):
        assert torch.equal(a, b)
    y, z = P.block_norm(minus[0], pre=weights[0])
    assert y is minus[0] and torch.equal(z, P.block_norm(-x, pre=weights[0].clone())[1])
    out = P.gated_scan_step(*[t.detach()[:, 0] for t in minus[:3]], minus[3].detach(), h0.detach().clone())
    assert torch.equal(out, P.gated_scan_step(*[-t.detach()[:, 0] for t in args[:3]], -decay.detach(), h0.detach().clone()))
    # gradients of the inputs, and incoming ones.  block_norm has decay three times here, and torch adds its three gradients in the order in which they come: two
    # orders of a + b + c differ by at most 2 roundings each, 4 x 2^-24 (|a| + |b| + |c|)
    three = [(-decay).detach().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(P.block_norm(-x, -r, -i, *three)[1].square().sum(), three)
    orders = 4 * 2.0 ** -24 * sum(t.abs() for t in parts)
    same = lambda a, b: (a is None and b is None) or torch.equal(a, b) or (a.shape == decay.shape and bool(((a - b).abs() <= orders).all()))          # noqa: E731
    for call in (lambda s: P.gated_scan(s[0], s[1], s[2], s[3], s[4])[0], lambda s: P.gated_scan(s[0], s[1], s[2], s[3], s[4])[1], lambda s: P.block_norm(s[0], s[1], s[2], s[3], s[3], s[3])[0],
                 lambda s: P.block_norm(s[0], s[1], s[2], s[3], s[3], s[3])[1]):
        got = torch.autograd.grad(call([noted(t) for t in args]).square().sum(), args, allow_unused=True)
        want = torch.autograd.grad(call([-t for t in args]).square().sum(), args, allow_unused=True)
        assert all(same(a, b) for a, b in zip(got, want))
        value = call(args)
        got = torch.autograd.grad(value, args, torch._neg_view(torch.ones_like(value)), allow_unused=True, retain_graph=True)
        want = torch.autograd.grad(value, args, -torch.ones_like(value), allow_unused=True, retain_graph=True)
        assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(got, want))
        got = torch.autograd.grad(value, args, torch._efficientzerotensor(value.shape), allow_unused=True)
        assert all(a is None or float(a.abs().sum()) == 0 for a in got)
    zeros = torch._efficientzerotensor((B, T, D))
    assert torch.equal(P.block_norm(x, zeros, pre=weights[0])[0], x) and torch.equal(P.gated_scan(zeros, r, i, decay)[1], torch.zeros(B, D))
    # an update: the gradient's values; nothing that it writes to
    p, one, two = (torch.ones(D) for _ in range(3))
    new = lambda: [torch.zeros(D)]                                                                       # noqa: E731
    count = lambda: torch.zeros(2, dtype=torch.int64)                                                    # noqa: E731
    adamw_step([one], [noted(decay).detach()], new(), new(), count())
    adamw_step([two], [-decay.detach()], new(), new(), count())
    assert torch.equal(one, two)
    for args in (([torch._neg_view(p)], [p.clone()], new(), new(), count()), ([p], [p.clone()], [torch._neg_view(p.clone())], new(), count()),
                 ([p], [p.clone()], new(), new(), torch._neg_view(count())), ([p.half()], [p.half()], new(), new(), count(), [torch._neg_view(p.clone())])):
        masters = {"masters": args[5]} if len(args) > 5 else {}
        with pytest.raises(ValueError, match="written in place"):
            adamw_step(*args[:5], **masters)
    with pytest.raises(ValueError, match="written in place"):
        P.gated_scan_step(*[t.detach()[:, 0] for t in (x, r, i)], decay.detach(), torch._neg_view(h0.detach()))


def test_wrappers_without_memory_are_refused(interpreter):
    x, r = (t.detach() for t in leaves((4, 8), (4, 8)))
    with pytest.raises(_lib.EngineError, match="holds no memory"):
        torch.func.functionalize(lambda u: P.block_norm(x, u)[0])(r)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_notices_whatever_an_update_changed(interpreter, bits):
    """Moments, their scales, masters and the count are written in place like the parameters: a graph that saved one of them has to say so."""
    n = 300
    z = lambda dt=torch.float32, size=n: torch.zeros(size, dtype=dt)                                     # noqa: E731
    p, master, step = z(torch.bfloat16), z(), z(torch.int64, 2)
    first, second = ([z()], [z()]) if bits == 32 else ([(z(torch.int8), z(size=2))], [(z(torch.uint8), z(size=2))])
    changed = [p, master, step] + [t for m in (first[0], second[0]) for t in (m if bits == 8 else [m])]
    leaf = torch.ones((), requires_grad=True)
    graphs = [(leaf * t).sum() for t in changed]
    versions = [t._version for t in changed]
    g = torch.ones(n, dtype=torch.bfloat16)
    kept = (leaf * g).sum()
    adamw_step([p], [g], first, second, step, masters=[master])
    assert all(t._version > v for t, v in zip(changed, versions))
    for loss in graphs:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    kept.backward()                                          # the gradient was only read
    idle = z()
    before = idle._version
    adamw_step([idle], [None], [z()], [z()], step)
    assert idle._version == before


def test_a_step_whose_inputs_lie_in_its_state(interpreter):
    """A row of the state for every row's input, the state itself, a part of it as the decays: as with copies of them."""
    B, D = 9, 130
    x, r, i, decay, state = (t.detach() for t in leaves((B, D), (B, D), (B, D), (D,), (B, D)))
    halves = torch.empty(2 * B * D - D)                      # the state, and an input that begins in its last row
    for pick in (lambda s: (s[:1].expand(B, D), r, i, decay), lambda s: (x, s[2:3].expand(B, D), i, decay), lambda s: (x, r, s[-1:].expand(B, D), decay), lambda s: (s, s, s, decay),
                 lambda s: (x, r, i, s[0]), lambda s: (x, r, i, s[B - 1]), lambda s: (s[0].view(D)[:1].expand(B, D), r, i, decay), lambda s: (halves[(B - 1) * D:].view(B, D), r, i, decay)):
        halves.copy_(torch.linspace(-1, 1, halves.numel()))
        mine = halves[:B * D].view(B, D)
        mine.copy_(state)
        args = pick(mine)
        other = mine.clone()
        want = P.gated_scan_step(*[t.clone().contiguous() for t in args], other)
        got = P.gated_scan_step(*args, mine)
        assert torch.equal(got, want) and torch.equal(mine, other)


def test_a_master_is_not_made_anew_inside_a_capture(interpreter, monkeypatch):
    p, g = torch.zeros(40, dtype=torch.bfloat16), torch.ones(40, dtype=torch.bfloat16)
    opt = AdamW([p], lr=1e-3)
    p.fill_(1.0)
    with monkeypatch.context() as m:
        m.setattr(AdamW, "_capturing", lambda self: True)
        with pytest.raises(_lib.EngineError, match="renew_masters"):
            opt.step([g])
        assert float(p[0]) == 1.0 and opt.iter == 0
    opt.renew_masters()
    assert float(opt.masters[0][0]) == 1.0
    with monkeypatch.context() as m:
        m.setattr(AdamW, "_capturing", lambda self: True)
        opt.step([g])
    assert opt.iter == 1 and float(opt.masters[0][0]) != float(p[0])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_adamw_gradients_that_are_not_finite(interpreter, bits, value):
    """What becomes of an element, of its block of 256 and of the rest, with and without clipping."""
    n = 1000
    z = lambda dt=torch.float32, size=n: torch.zeros(size, dtype=dt)                                     # noqa: E731
    g = torch.linspace(-1, 1, n)
    g[700] = value
    for max_norm in (0.0, 1.0):
        results = []
        for grad in (g, torch.where(torch.isfinite(g), g, torch.zeros(()))):
            p = torch.ones(n)
            first, second = ([z()], [z()]) if bits == 32 else ([(z(torch.int8), z(size=4))], [(z(torch.uint8), z(size=4))])
            norm = adamw_step([p], [grad * 0 if max_norm and grad is not g else grad], first, second, z(torch.int64, 2), max_norm=max_norm)
            m, v = ((first[0], second[0]) if bits == 32 else adamw_values([first[0], second[0]]))
            results.append((p, m, v, norm))
        (p, m, v, norm), (rest_p, rest_m, rest_v, _) = results
        touched = torch.zeros(n, dtype=torch.bool)
        touched[700] = True
        if max_norm and value != value:
            assert not torch.isfinite(p).any() and not torch.isfinite(m).any() and not torch.isfinite(norm)
            continue
        assert not torch.isfinite(p[700])
        moments = touched if bits == 32 else (torch.arange(n) // 256 == 700 // 256)
        assert not torch.isfinite(m[moments]).any() and not torch.isfinite(v[moments]).any()
        assert torch.equal(p[~touched], rest_p[~touched]) and torch.equal(m[~moments], rest_m[~moments]) and torch.equal(v[~moments], rest_v[~moments])
        if max_norm:
            assert float(norm) == float("inf")


def test_a_state_of_another_policy_is_refused(interpreter):
    """Before anything moves: too few blocks ended in an IndexError with the first ones moved on, too many went unnoticed."""
    policy, obs = P.RecurrentPolicy(5, 2, width=8, depth=2, device="cpu"), torch.randn(3, 5)
    for blocks in (1, 3):
        state = torch.zeros(blocks, 3, 8)
        for call in (lambda: policy.act(obs, state), lambda: policy.step(obs, state), lambda: policy(obs[:, None], state)):
            with pytest.raises(ValueError, match="of 2 blocks"):
                call()
        assert float(state.abs().sum()) == 0
    state = policy.initial_state(3)
    action, after = policy.step(obs, state)
    assert torch.allclose(policy.act(obs, state), action.detach()) and torch.allclose(state, after)


class Sums(torch.nn.Module):
    """A policy with a memory of the documented kind: ``initial_state`` and ``step``, its ``forward`` for one observation."""

    def __init__(self):
        super().__init__()
        self.lin = torch.nn.Linear(4, 2)

    def initial_state(self, batch):
        return [torch.zeros(batch, 4)]

    def step(self, obs, state):
        state = [0.5 * state[0] + obs]
        return self.lin(state[0]), state

    def forward(self, obs):
        return self.lin(obs)


def imitation(policy):
    from plasticinelab_amd.config import CfgNode
    from plasticinelab_amd.optimizer.solver_nn import SolverNN
    solver = SolverNN.__new__(SolverNN)                      # (a simulator needs a GPU; imitation does without one)
    solver.policy, solver.place = policy, {"dtype": torch.float32, "device": "cpu"}
    solver.cfg = CfgNode({"optim": {"lr": 1e-3, "bounds": (-float("inf"), float("inf")), "type": "Adam"}})
    return solver


def test_imitation_by_policies_of_every_kind(interpreter):
    B, H = 3, 6
    gen = torch.Generator().manual_seed(8)
    obs, target = torch.randn(B, H, 4, generator=gen), torch.randn(B, H, 2, generator=gen)
    reset = torch.rand(B, H, generator=gen) < 0.3
    assert reset.any()

    def expected(policy, reset):
        if reset is not None and isinstance(policy, P.RecurrentPolicy):          # (there a reset is a = 0 with a gain of 1, not a state of zeros)
            return float(((policy(obs, reset=reset)[0] - target).detach() ** 2).mean())
        out = []
        for b in range(B):
            state = policy.initial_state(1)
            for t in range(H):
                if reset is not None and reset[b, t]:
                    state = policy.initial_state(1)
                a, state = policy.step(obs[b:b + 1, t], state)
                out.append(a)
        return float(((torch.cat(out).view(B, H, 2) - target).detach() ** 2).mean())

    for make in (Sums, lambda: P.RecurrentPolicy(4, 2, width=8, depth=2, device="cpu")):
        for cuts in (None, reset):
            torch.manual_seed(9)
            policy = make()
            want = expected(policy, cuts)
            before = [p.detach().clone() for p in policy.parameters()]
            losses = imitation(policy).imitate(obs, target, n_iters=3, reset=cuts)
            assert len(losses) == 3 and abs(losses[0] - want) <= 1e-5 * want
            assert not any(torch.equal(a, b) for a, b in zip(policy.parameters(), before))
            want = expected(policy, cuts)                    # (of the policy as the updates left it)
            assert abs(imitation(policy).imitate(obs, target, n_iters=1, reset=cuts)[0] - want) <= 1e-5 * want

    linear = torch.nn.Linear(4, 2)                           # without a memory: nothing to reset
    want = float(((linear(obs) - target).detach() ** 2).mean())
    for cuts in (None, reset):
        fresh = torch.nn.Linear(4, 2)
        fresh.load_state_dict(linear.state_dict())
        assert abs(imitation(fresh).imitate(obs, target, n_iters=1, reset=cuts)[0] - want) <= 1e-5 * want


def test_imitation_refuses_what_does_not_fit(interpreter):
    class Odd(Sums):
        def forward(self, obs, reset=None):
            return self.lin(obs)

    obs, target = torch.zeros(3, 6, 4), torch.zeros(3, 6, 2)
    for policy, args, kw, text in ((Odd(), (obs, target), {}, "answer \\(actions, state\\)"), (Sums(), (obs, target[:, :, :1]), {}, "actions are"), (Sums(), (obs, target[0]), {}, "actions are"),
                                   (torch.nn.Linear(4, 2), (obs, target[0]), {}, "actions are"), (Sums(), (obs[0], target[0]), {}, "B, H, obs.dim"),
                                   (Sums(), (obs, target), {"reset": torch.zeros(3, 5)}, "reset has to be"), (P.RecurrentPolicy(4, 2, width=8, device="cpu"), (obs, target[0]), {}, "actions are")):
        before = [p.detach().clone() for p in policy.parameters()]
        with pytest.raises(ValueError, match=text):
            imitation(policy).imitate(*args, n_iters=1, **kw)
        assert all(torch.equal(a, b) for a, b in zip(policy.parameters(), before))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scan_gradients_of_gates_far_out(interpreter, dtype):
    cases.run_gates_far_out(interpreter, dtype)


@pytest.mark.parametrize("tx,tu", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
def test_norm_gradients_of_gates_far_out(interpreter, tx, tu):
    cases.run_norm_gates_far_out(interpreter, tx, tu)


def test_decay_gradient_of_many_rows(interpreter):
    cases.run_decay_gradient_of_many_rows(interpreter, 4099)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gate_of_a_reset_that_is_no_number(interpreter, dtype):
    cases.run_gate_of_a_reset_that_is_no_number(interpreter, dtype)


def test_imitation_by_a_policy_whose_forward_has_no_signature(interpreter):
    class Compiled:
        __signature__ = "none"

        def __call__(self, obs):
            raise AssertionError("not reached")

    torch.manual_seed(10)
    policy = Sums()
    policy.forward = Compiled()
    obs, target = torch.randn(2, 3, 4), torch.randn(2, 3, 2)
    assert len(imitation(policy).imitate(obs, target, n_iters=1)) == 1
