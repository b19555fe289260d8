"""Plain 64-bit forms of the policy-training operators, step by step, and how far float32 arithmetic may be from them.

The bounds are running error bounds: beside each quantity its majorant (the same sum with absolute values) and its error are walked through
the definition, every operation adding its own rounding.  u = 2^-24 is half a step of float32; a hardware exp2 / rcp / rsq / sqrt is within one
step (2 u).  From that, for arguments |r| <= 6:
    sigmoid: scaling 6 u, exp2 2 u, sum 1 u, rcp 2 u                                                        -> 11 u
    la = -c softplus(decay) sigmoid(r): softplus and its products 8 u more                                  -> 20 u, so a: (20 |la| + 2) u
    m = sqrt(1 - a^2): half of the cubic's 4.5 u and la's 20 u, or of 2 (20 |la| + 2) u a^2 / (1 - a^2)
    at a^2 = 0.78, and the root                                                                             -> 16 u
    m sigmoid(i) x                                                                                          -> 30 u
Outputs of 16 bits add half a step of their own type (torch.finfo(t).eps / 2 relative)."""
import numpy as np
import torch

U = 2.0 ** -24
F64 = torch.float64
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def rounding(ref, dtype):
    """Half a step of ``dtype`` at each value (float32 results are rounded within the counted operations, which U covers)."""
    return ref.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype]


def far(got, ref, bound):
    """Largest |got - ref| / bound; infinities and NaN have to be where the reference has them."""
    got, ref, bound = got.detach().cpu().to(F64), ref.detach().cpu().to(F64), bound.detach().cpu().to(F64)
    assert got.shape == ref.shape, (got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(got)), "not finite in different places"
    if not got.numel() or not fine.any():
        return 0.0
    return float(((got - ref).abs() / bound.clamp(min=1e-300))[fine].max())


def scan(x, r, i, decay, h0=None, reset=None, c=8.0, dh=None, dlast=None):
    """-> ({name: value}, {name: error bound of float32 arithmetic}) of gated_scan and, with dh / dlast, of its gradients."""
    B, T, D = x.shape
    dtype = x.dtype
    x, r, i, decay = (t.detach().cpu().to(F64) for t in (x, r, i, decay))
    cut = torch.zeros(B, T, 1, dtype=torch.bool) if reset is None else reset.cpu()[..., None]
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    la = -c * torch.nn.functional.softplus(decay) * sr
    a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    a, m = torch.where(cut, 0.0, a), torch.where(cut, 1.0, m)
    push = m * si * x
    now = torch.zeros(B, D, dtype=F64) if h0 is None else h0.detach().cpu().to(F64)
    start, big, err = now, now.abs(), torch.zeros(B, D, dtype=F64)
    h, before, bigs, errs = [], [], [], []
    for t in range(T):
        before.append((now, big, err))
        keep = ~cut[:, t]
        zero = torch.zeros_like(now)
        old, old_big, old_err = (torch.where(keep, v, zero) for v in (now, big, err))
        now = a[:, t] * old + push[:, t]
        err = a[:, t] * old_err + U * ((20 * la[:, t].abs() + 4) * a[:, t] * old_big + 32 * push[:, t].abs())
        big = a[:, t] * old_big + push[:, t].abs()
        h.append(now)
        bigs.append(big)
        errs.append(err)
    out, tol = {}, {}
    out["h"], tol["h"] = torch.stack(h, 1), torch.stack(errs, 1)
    out["last"], tol["last"] = now, err + TINY[torch.float32]
    tol["h"] = tol["h"] + rounding(out["h"], dtype)
    if dh is None and dlast is None:
        return out, tol
    dh = torch.zeros(B, T, D, dtype=F64) if dh is None else dh.detach().cpu().to(F64)
    back = torch.zeros(B, D, dtype=F64) if dlast is None else dlast.detach().cpu().to(F64)
    bback, eback = back.abs(), torch.zeros(B, D, dtype=F64)
    res = {k: torch.zeros(B, T, D, dtype=F64) for k in ("dx", "dr", "di", "dla", "bla", "ela")}
    ers = {k: torch.zeros(B, T, D, dtype=F64) for k in ("dx", "dr", "di")}
    for t in range(T - 1, -1, -1):
        g, G, E = dh[:, t] + back, dh[:, t].abs() + bback, eback + 2 * U * (dh[:, t].abs() + bback)
        hp, hb, he = (torch.where(cut[:, t], torch.zeros_like(g), v) for v in before[t])
        at, mt, s, q = a[:, t], m[:, t], si[:, t], sr[:, t]
        pull = torch.where(mt > 0, s * x[:, t] * at * at / mt.clamp(min=1e-300), torch.zeros_like(g))
        # (a where() keeps what is not finite before a reset out of the products)
        dla = torch.where(cut[:, t], torch.zeros_like(g), g * (at * hp - pull))
        bla = torch.where(cut[:, t], torch.zeros_like(g), G * (at * hb + pull.abs()))
        ela = torch.where(cut[:, t], torch.zeros_like(g), E * (at * hb + pull.abs()) + G * at * he + 60 * U * bla + G * (20 * la[:, t].abs()) * U * (at * hb + 2 * pull.abs()))
        res["dx"][:, t], ers["dx"][:, t] = g * mt * s, mt * s * (E + 32 * U * G)
        res["di"][:, t], ers["di"][:, t] = g * mt * x[:, t] * s * (1 - s), (mt * x[:, t].abs()) * s * ((1 - s) * (E + 48 * U * G) + 12 * U * G)
        res["dr"][:, t], ers["dr"][:, t] = dla * la[:, t] * (1 - q), la[:, t].abs() * ((1 - q) * (ela + 24 * U * bla) + 12 * U * bla)
        res["dla"][:, t], res["bla"][:, t], res["ela"][:, t] = dla, bla, ela
        keep = ~cut[:, t]
        zero = torch.zeros_like(g)
        back, bback, eback = torch.where(keep, at * g, zero), torch.where(keep, at * G, zero), torch.where(keep, at * E + U * (20 * la[:, t].abs() + 4) * at * G, zero)
    for k in ("dx", "dr", "di"):
        out[k], tol[k] = res[k], ers[k] + rounding(res[k], dtype)
    pull = c * torch.sigmoid(decay)
    rows = B * ((T + 63) // 64)
    out["ddecay"] = -pull * (res["dla"] * sr).sum((0, 1))
    tol["ddecay"] = pull * (((res["ela"] + 24 * U * res["bla"]) * sr).sum((0, 1)) + (48 + rows / 16) * U * (res["bla"] * sr).sum((0, 1))) + TINY[torch.float32]
    out["dh0"], tol["dh0"] = back, eback + TINY[torch.float32]
    return out, tol


def norm(x, u=None, gate=None, scale=None, post=None, pre=None, eps=1e-6, fn="sigmoid", dy=None, dz=None, u_dtype=None):
    """-> ({name: value}, {name: error bound}) of block_norm and, with dy / dz, of its gradients.  A sum of squares over a row: at most 8 + 10 + 4
    additions on a path, 24 u; its root half of that, and rsq 2 u -> 14 u for 1 / rms."""
    D = x.shape[-1]
    tx, tu = x.dtype, (u_dtype or (u.dtype if u is not None else x.dtype))
    wt = next((w.dtype for w in (pre, post, scale) if w is not None), torch.float32)
    f64 = lambda t: None if t is None else t.detach().cpu().to(F64)                                                 # noqa: E731
    X, Uu, G = (None if t is None else f64(t).reshape(-1, D) for t in (x, u, gate))
    one = torch.ones(D, dtype=F64)
    S, P = (one if f64(t) is None else f64(t) for t in (scale, post))
    out, tol = {}, {}
    y, Ey = X, torch.zeros_like(X)
    if u is not None:
        ru = 1 / torch.sqrt((Uu * Uu).mean(1, keepdim=True) + eps)
        uh = Uu * ru
        if gate is None:
            f, df, ef = torch.ones_like(uh), torch.zeros_like(uh), 0.0 * uh
        else:
            sg = torch.sigmoid(G)
            f, df = {"identity": (G, torch.ones_like(G)), "sigmoid": (sg, sg * (1 - sg)), "silu": (G * sg, sg * (1 + G * (1 - sg)))}[fn]
            ef = 12 * U * (1 + G.abs())
        v = S * f * P * uh
        y = X + v
        Ey = 24 * U * v.abs() + 12 * U * (S * P * uh).abs() * (0 if gate is None else 1 + (G.abs() if fn == "silu" else 0)) + U * y.abs()
        out["y"], tol["y"] = y, Ey + rounding(y, tx)
    if pre is not None:
        Q = f64(pre)
        ry = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
        er = 14 * U + Ey.norm(dim=1, keepdim=True) / y.norm(dim=1, keepdim=True).clamp(min=1e-300)
        yh = y * ry
        out["z"] = yh * Q
        tol["z"] = Q.abs() * (Ey * ry + yh.abs() * (er + 4 * U)) + rounding(out["z"], tu)
    if dy is None and dz is None:
        return _shaped(out, tol, x)
    g = torch.zeros_like(X) if dy is None else f64(dy).reshape(-1, D)
    Eg = U * g.abs()
    rows = X.shape[0]
    add = (rows / 512 + 2 + rows / 256 / 16 + 48) * U
    if dz is not None:
        Z = f64(dz).reshape(-1, D)
        q = Z * Q
        mean = (q * yh).mean(1, keepdim=True)
        Em = (q * yh).abs().mean(1, keepdim=True) * (er + 30 * U) + (q.abs() * Ey * ry).mean(1, keepdim=True)
        g = g + ry * (q - yh * mean)
        Eg = Eg + U * g.abs() + ry * (3 * U * q.abs() + yh.abs() * Em + mean.abs() * (Ey * ry + yh.abs() * (er + 4 * U)) + (er + 2 * U) * (q.abs() + (yh * mean).abs()))
        out["dpre"] = (Z * yh).sum(0)
        tol["dpre"] = (Z.abs() * (Ey * ry + yh.abs() * (er + 4 * U))).sum(0) + add * (Z * yh).abs().sum(0) + rounding(out["dpre"], wt)
    elif pre is not None:
        out["dpre"], tol["dpre"] = torch.zeros(D, dtype=F64), torch.full((D,), 1e-300, dtype=F64)
    out["dx"], tol["dx"] = g, Eg + rounding(g, tx)
    if u is not None:
        Euh = uh.abs() * 15 * U
        dv = g * S * f
        Ev = (S * f).abs() * Eg + (g * S).abs() * (ef + 3 * U * f.abs())
        out["dscale"], out["dpost"] = (g * f * P * uh).sum(0), (dv * uh).sum(0)
        tol["dscale"] = ((f * P * uh).abs() * Eg + (g * P * uh).abs() * ef + 20 * U * (g * f * P * uh).abs()).sum(0) + add * (g * f * P * uh).abs().sum(0) + rounding(out["dscale"], wt)
        tol["dpost"] = (Ev * uh.abs() + dv.abs() * Euh).sum(0) + add * (dv * uh).abs().sum(0) + rounding(out["dpost"], wt)
        w, Ew = dv * P, Ev * P.abs() + 2 * U * (dv * P).abs()
        mean = (w * uh).mean(1, keepdim=True)
        Em = (Ew * uh.abs() + w.abs() * Euh).mean(1, keepdim=True) + 26 * U * (w * uh).abs().mean(1, keepdim=True)
        out["du"] = ru * (w - uh * mean)
        tol["du"] = ru * (Ew + uh.abs() * Em + Euh * mean.abs() + 18 * U * (w.abs() + (uh * mean).abs())) + rounding(out["du"], tu)
        if gate is not None:
            edf = 0.0 if fn == "identity" else 26 * U * (1 + G.abs())
            k = S * P * uh
            out["dgate"] = g * k * df
            tol["dgate"] = (k * df).abs() * Eg + (g * k).abs() * edf + 22 * U * (g * k * df).abs() + rounding(out["dgate"], tu)
    return _shaped(out, tol, x)


def _shaped(out, tol, x):
    for k in out:
        if out[k].dim() == 2:
            out[k], tol[k] = out[k].reshape(x.shape), tol[k].reshape(x.shape)
    return out, tol


# ---- AdamW: float32 arithmetic has one answer when every operation rounds by itself, and numpy's does
F = np.float32


def moment_values(codes, scales, second):
    n = codes.size
    s = np.repeat(scales, 256)[:n].astype(F)
    q = codes.astype(F) * F(1.0 / (255.0 if second else 127.0))
    if second:
        q = q * q
        return (q * q) * s
    return (q * np.abs(q)) * s


def moment_codes(v, second):
    n = v.size
    pad = np.zeros(-(-n // 256) * 256, F)
    pad[:n] = np.abs(v)
    scales = pad.reshape(-1, 256).max(1) if n else np.zeros(0, F)
    s = np.repeat(np.where(scales > 0, scales, F(1)), 256)[:n].astype(F)
    q = np.sqrt(np.abs(v) / s)
    if second:
        q = np.rint(np.sqrt(q) * F(255))
        return np.where(v > 0, np.maximum(q, 1), q).astype(np.uint8), scales
    return (np.rint(q * F(127)) * np.sign(v)).astype(np.int8), scales


def adamw(w, g, m, v, t, norm=None, lr=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-8, weight_decay=0.01, max_norm=0.0, bounds=(-np.inf, np.inf)):
    """One update of one tensor in float32, each operation rounded by itself -> (w, m, v).  norm: of all tensors' gradients, in float64."""
    g = g.astype(F)
    if max_norm > 0:
        g = g * F(min(1.0, max_norm / norm if norm else 1.0))
    m = F(beta_1) * m + F(1 - beta_1) * g
    v = F(beta_2) * v + F(1 - beta_2) * (g * g)
    den = np.sqrt(v) * F(1.0 / np.sqrt(1 - beta_2 ** t)) + F(epsilon)
    w = w - F(lr * weight_decay) * w - (F(lr / (1 - beta_1 ** t)) * m) / den
    return np.clip(w, F(bounds[0]), F(bounds[1])), m, v
