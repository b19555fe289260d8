"""CPU tier: what the policy-training operators refuse -- in Python before anything is touched, and at the C entries of the library itself."""
import ctypes as C

import pytest
import torch

from plasticinelab_amd import _lib
from plasticinelab_amd import policy as P
from plasticinelab_amd.optimizer import AdamW, adamw_step, adamw_values


def tensors(B=2, T=3, D=8, dtype=torch.float32):
    return [torch.zeros(B, T, D, dtype=dtype) for _ in range(3)] + [torch.zeros(D)]


def test_scan_refusals():
    x, r, i, decay = tensors()
    for args, kw, text in (
            ((x[0], r[0], i[0], decay), {}, "3 dimensions"), ((x.double(), r.double(), i.double(), decay), {}, "float32, bfloat16 or float16"),
            ((x, r[:, :2], i, decay), {}, "have to match x"), ((x, r.half(), i, decay), {}, "have to match x"), ((x, r, i, decay[:4]), {}, "8 values"),
            ((x, r, i, decay.half()), {}, "float32"), ((x, r, i, torch.zeros(16)[::2]), {}, "contiguous"), ((x, r, i, decay, torch.zeros(2, 7)), {}, "h0"),
            ((x, r, i, decay, torch.zeros(2, 8).double()), {}, "h0"), ((x, r, i, decay, None, torch.zeros(2, 3)), {}, "bool"),
            ((x, r, i, decay, None, torch.zeros(3, 2, dtype=torch.bool)), {}, "bool"), ((x, r, i, decay), {"c": 0.0}, "c has to be positive"),
            ((x, r, i, decay), {"c": float("nan")}, "c has to be positive"), ((x, 1.0, i, decay), {}, "r has to be a tensor")):
        with pytest.raises(ValueError, match=text):
            P.gated_scan(*args, **kw)
    s = torch.zeros(2, 8)
    for args, text in (((x, r, i, decay, s), "2 dimensions"), ((x[:, 0], r[:, 0], i[:, 0], decay, s.half()), "state"), ((x[:, 0], r[:, 0], i[:, 0], decay, torch.zeros(8, 2).T), "contiguous"),
                       ((x[:, 0], r[:, 0], i[:, 0], decay.requires_grad_(), s), "no gradients")):
        with pytest.raises(ValueError, match=text):
            P.gated_scan_step(*args)
    decay = decay.detach()
    with pytest.raises(_lib.EngineError, match="no CPU path"):
        P.gated_scan(x, r, i, decay)


def test_norm_refusals():
    x, u, w = torch.zeros(4, 8), torch.zeros(4, 8), torch.ones(8)
    for kw, text in (({"x": x}, "u, pre or both"), ({"x": x, "gate": u, "pre": w}, "go with u"), ({"x": x, "u": u[:, :4]}, "shape"), ({"x": x, "u": u.double()}, "16 bits"),
                     ({"x": x.half(), "u": u}, "16 bits"), ({"x": x, "u": u, "gate": u.half()}, "gate"), ({"x": x, "u": u, "pre": w[:4]}, "8 values"),
                     ({"x": x, "u": u, "pre": w, "post": w.half()}, "one floating type"), ({"x": x, "pre": torch.ones(16)[::2]}, "contiguous"), ({"x": x, "u": u, "gate_fn": "tanh"}, "gate_fn"),
                     ({"x": x, "u": u, "eps": -1.0}, "eps"), ({"x": x, "u": u, "dtype": torch.float16}, "calls without u"), ({"x": torch.zeros(1, 8193), "pre": torch.ones(8193)}, "at most 8192"),
                     ({"x": torch.zeros(4, 8, dtype=torch.int32), "pre": w}, "float32, bfloat16 or float16"), ({"x": torch.zeros(()), "pre": w}, "one dimension")):
        with pytest.raises(ValueError, match=text):
            P.block_norm(**kw)
    with pytest.raises(_lib.EngineError, match="no CPU path"):
        P.block_norm(x, u)


def test_adamw_refusals():
    p, step = torch.zeros(300), torch.zeros(2, dtype=torch.int64)
    z = lambda n=300, dt=torch.float32: torch.zeros(n, dtype=dt)                                         # noqa: E731
    eight = lambda: ((z(300, torch.int8), z(2)), (z(300, torch.uint8), z(2)))                            # noqa: E731
    m8, v8 = eight()
    for args, kw, text in (
            (([p], [p], [z()], [], step), {}, "one length"), (([p], [p], [z()], [z()], step[:1]), {}, "two values"), (([p.double()], [p.double()], [z()], [z()], step), {}, "parameter 0"),
            (([torch.zeros(600)[::2]], [p], [z()], [z()], step), {}, "contiguous"), (([p], [z(299)], [z()], [z()], step), {}, "gradient 0"), (([p], [p.half()], [z()], [z()], step), {}, "gradient 0"),
            (([p], [p], [z(299)], [z()], step), {}, "first moment"), (([p], [p], [z()], [z().half()], step), {}, "second moment"), (([p], [p], [m8], [z()], step), {}, "all have 8"),
            (([p], [p], [v8], [v8], step), {}, "int8"), (([p], [p], [m8], [(v8[0], z(1))], step), {}, "2 contiguous float32"), (([p], [p], [z()], [z()], step), {"masters": [z()]}, "goes with 16 bits"),
            (([p.half()], [p.half()], [z()], [z()], step), {"masters": [z(5)]}, "master")):
        with pytest.raises(ValueError, match=text):
            adamw_step(*args, **kw)
    for args in (([p, p], [p, p], [z(), z()], [z(), z()], step), ([p, z()], [p, p], [m8[0].float()] * 2, [z(), z()], step), ([p, z()], [p, p], [m8, eight()[0]], [v8, (v8[0].clone(), v8[1])], step)):
        with pytest.raises(ValueError, match="twice"):
            adamw_step(*args)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([p.half(), z().half()], [p.half()] * 2, [z(), z()], [z(), z()], step, masters=[p, p])
    for entry, text in (((z(), z(2)), "int8 or uint8"), ((z(300, torch.int8), z(3)), "scales")):
        with pytest.raises(ValueError, match=text):
            adamw_values([entry])
    with pytest.raises(ValueError, match="for each moment"):
        adamw_values([m8], out=[])
    with pytest.raises(_lib.EngineError, match="no CPU path"):
        AdamW([p])
    with pytest.raises(TypeError, match="list of tensors"):
        AdamW(p)
    with pytest.raises(ValueError, match="at least one"):
        AdamW([])


def test_what_is_no_tensor_is_named():
    x, r, i, decay = tensors()
    p, step = torch.zeros(300), torch.zeros(2, dtype=torch.int64)
    for call, text in ((lambda: P.gated_scan(x, r, i, decay, 3), "h0 has to be a tensor"), (lambda: P.gated_scan(None, r, i, decay), "x has to be a tensor, got NoneType"),
                       (lambda: P.gated_scan_step(x[:, 0], r[:, 0], i[:, 0], decay, None), "state has to be a tensor"), (lambda: P.block_norm(x, 1.0), "u has to be a tensor"),
                       (lambda: adamw_step([p], [0.0], [p], [p], step), "gradient 0 has to be a tensor"), (lambda: adamw_step([p], [p], [p], [p], None), "step has to be a tensor"),
                       (lambda: adamw_step([p], [p], [p], [(p, p)], step), "all have 8"), (lambda: adamw_values([p]), "pairs of codes and scales")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError):
        P.gated_scan(x, r, i, decay, c="8")


def test_c_entries_check_before_they_launch():
    """Null pointers, sizes and alignments at the C entries of the library itself: a message and non-zero, nothing launched."""
    lib = _lib.load_policy()
    error = lambda: lib.plmpm_last_error().decode()                                                      # noqa: E731
    some = 1 << 20
    ok = dict(dtype=0, batch=1, steps=300, width=8, c=8.0, x=some, r=some, i=some, decay=some, h=some)
    need = C.c_size_t()
    for change, text in (({"dtype": 3}, "dtype"), ({"batch": -1}, "negative"), ({"width": 1 << 31}, "too large"), ({"steps": 1 << 40}, "too many"), ({"c": -1.0}, "c has to be"),
                         ({"x": None}, "needed"), ({"h": None}, "needed"), ({"r": some + 2}, "aligned"), ({"batch": 1 << 29, "width": 1 << 20}, "too large"), ({}, "workspace")):
        assert lib.plmpm_scan_forward(_lib.Scan(**{**ok, **change}), None) != 0 and text in error(), (change, error())
    assert lib.plmpm_scan_forward(None, None) != 0 and lib.plmpm_scan_workspace(_lib.Scan(**ok), 0, None) != 0
    assert lib.plmpm_scan_workspace(_lib.Scan(**ok), 0, need) == 0 and need.value > 0
    assert lib.plmpm_scan_backward(_lib.Scan(**ok), None) != 0 and "needed" in error()
    assert lib.plmpm_scan_forward(_lib.Scan(**{**ok, "workspace": some + 4, "workspace_bytes": 1 << 20}), None) != 0 and "aligned" in error()
    room = dict(workspace=some, workspace_bytes=1 << 60)
    assert lib.plmpm_scan_forward(_lib.Scan(**{**ok, **room, "width": 1 << 27}), None) != 0 and "too large" in error()
    assert lib.plmpm_scan_forward(_lib.Scan(**{**ok, **room, "batch": 1 << 23, "width": 1}), None) != 0 and "one launch" in error()
    assert lib.plmpm_scan_forward(_lib.Scan(**{**ok, **room, "h0": some + 2}), None) != 0 and "aligned" in error()
    assert lib.plmpm_scan_forward(_lib.Scan(**{**ok, "steps": 0}), None) == 0                           # nothing to do
    ok = dict(rows=4, width=8, eps=1e-6, x=some, u=some, y=some, z=some, pre=some, stride_x=8, stride_u=8)
    for change, text in (({"x_dtype": 5}, "dtype"), ({"x_dtype": 1}, "u has x's type"), ({"rows": -1}, "negative"), ({"width": 9000}, "at most"), ({"gate_fn": 7}, "gate function"),
                         ({"eps": -1.0}, "eps"), ({"x": None}, "x is needed"), ({"u": None, "gate": some}, "go with u"), ({"y": None}, "y goes with u"), ({"pre": None}, "z with pre"),
                         ({"x": some + 1}, "aligned"), ({"stride_x": -8}, "stride"), ({"stride_u": 1 << 28}, "stride")):
        assert lib.plmpm_norm_forward(_lib.Norm(**{**ok, **change}), None) != 0 and text in error(), (change, error())
    assert lib.plmpm_norm_backward(_lib.Norm(**ok), None) != 0 and "dx" in error()
    assert lib.plmpm_norm_backward(_lib.Norm(**{**ok, "dx": some, "du": some}), None) != 0 and "workspace" in error()
    assert lib.plmpm_norm_forward(_lib.Norm(**{**ok, "rows": 0}), None) == 0
    ok = dict(state_bits=32, lr=0.1, beta_1=0.9, beta_2=0.99, step=some)
    t = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(p=some, g=some, m=some, v=some, n=5))
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**{**ok, "state_bits": 16}), t, 1, None) != 0 and "32 or 8" in error()
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**{**ok, "state_bits": 8}), t, 1, None) != 0 and "null" in error()
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**{**ok, "step": None}), t, 1, None) != 0 and "step" in error()
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**{**ok, "max_norm": 1.0}), t, 1, None) != 0 and "workspace" in error()
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**ok), None, 1, None) != 0 and lib.plmpm_adamw_step(_lib.AdamWStep(**ok), t, -1, None) != 0
    t[0].master = some
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**ok), t, 1, None) != 0 and "16-bit" in error()
    t[0].n = 0
    assert lib.plmpm_adamw_step(_lib.AdamWStep(**ok), t, 1, None) == 0
    assert lib.plmpm_adamw_values(None, None, None, None, None, 1, None) != 0 and "null" in error()


def test_adamw_refuses_tensors_that_share_memory():
    """Whatever an update writes: the other tensor begins before it, behind its start, or is what another parameter reads."""
    n, step = 300, torch.zeros(2, dtype=torch.int64)
    z = lambda dt=torch.float32: torch.zeros(n, dtype=dt)                                                # noqa: E731
    wide = torch.zeros(2 * n)
    halves, shifted = [wide[:n], wide[n:]], [wide[:n], wide[n - 1:2 * n - 1]]
    eight = lambda: ((z(torch.int8), torch.zeros(2)), (z(torch.uint8), torch.zeros(2)))                  # noqa: E731
    a, b = eight(), eight()
    scales = torch.zeros(3)
    two = lambda: [z(), z()]                                                                             # noqa: E731
    words = torch.zeros(n, dtype=torch.int64)
    for args, kw in (((shifted, two(), two(), two(), step), {}), ((shifted[::-1], two(), two(), two(), step), {}), ((two(), two(), shifted, two(), step), {}), ((two(), two(), two(), shifted, step), {}),
                     (([z()], [wide[:n]], [wide[n - 1:2 * n - 1]], [z()], step), {}), ((halves, [wide[1:n + 1], z()], two(), two(), step), {}), ((halves, [z(), wide[:n]], two(), two(), step), {}),
                     (([z(torch.float16)], [z(torch.float16)], [wide[:n]], [z()], step), {"masters": [wide[1:n + 1]]}),
                     (([words.view(torch.float32)[:n]], [z()], [z()], [z()], words[1:3]), {}),
                     ((two(), two(), [(a[0][0], scales[:2]), (b[0][0], scales[1:])], [a[1], b[1]], step), {}), ((two(), two(), [a[0], b[0]], [(a[1][0], scales[:2]), (b[1][0], scales[1:])], step), {})):
        with pytest.raises(ValueError, match="overlaps"):
            adamw_step(*args, **kw)
    g = z()                                                  # side by side, a gradient for two, a gradient that is its parameter: on to the check of the device
    for args in ((halves, [g, g], two(), two(), step), ([g], [g], [z()], [z()], step)):
        with pytest.raises(_lib.EngineError, match="no CPU path"):
            adamw_step(*args)
    codes = lambda: (z(torch.int8), torch.zeros(2))                                                      # noqa: E731
    for moments, out in (([codes(), codes()], shifted), ([(wide.view(torch.int8)[4:4 + n], torch.zeros(2))], [wide[:n]]), ([(z(torch.int8), wide[n - 1:n + 1])], [wide[:n]])):
        with pytest.raises(ValueError, match="overlaps"):
            adamw_values(moments, out=out)
    one = codes()
    with pytest.raises(_lib.EngineError, match="no CPU path"):
        adamw_values([one, one], out=halves)


def test_a_forward_call_is_refused_where_its_backward_call_would_be():
    """10^7 rows of 50 steps of one channel: the forward launch takes them, the backward one, whose waves hold half the steps, does not."""
    lib = _lib.load_policy()
    some = 1 << 20
    for steps, batch in ((50, 10 ** 7), (1, 1 << 27)):
        s = _lib.Scan(dtype=0, batch=batch, steps=steps, width=1, c=8.0, x=some, r=some, i=some, decay=some, h=some, checkpoint=some, workspace=some, workspace_bytes=1 << 60)
        assert lib.plmpm_scan_forward(s, None) != 0 and "one launch" in lib.plmpm_last_error().decode()
