"""Plain 64-bit forms of the sequence operators (gan_amd/sequence.py) on the CPU, each with its gradients and, beside every value, a MAJORANT:
the same formula with every term's absolute value.  A float32 evaluation that takes at most k successive roundings from the inputs to a value is
off by at most k * 2^-24 * majorant (first order: each rounding is relative to a partial result, and every partial result is at most its
majorant), whatever the order of the sums.  That is the tests' tolerance; bfloat16 outputs add their own rounding, 2^-8 of the value."""
import torch
import torch.nn.functional as F

U = 2.0 ** -24


def close(got, ref, major, k, what):
    """|got - ref| <= k 2^-24 majorant + half a step of got's type (+ its smallest normal number: kernels may flush below it)."""
    got, dtype = got.detach().cpu().double(), got.dtype
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), what
    tol = k * U * major + (2.0 ** -8 * ref.abs() * (1 + 1e-3) if dtype == torch.bfloat16 else 0.0) + 1.2e-38
    err = (got - ref).abs()
    worst = float((err / tol.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the tolerance (largest error {float(err.max()):.3g})"


def silu(v):
    s = torch.sigmoid(v)
    return v * s, s * (1 + v * (1 - s))


def d(t):
    return None if t is None else t.detach().cpu().double()


def keep_rows(lengths, B, T):
    n = torch.full((B,), T) if lengths is None else lengths.detach().cpu().long().clamp(0, T)
    return torch.arange(T)[None, :] < n[:, None], n


def conv(x, w, bias, act, state, lengths, dy=None, dlast=None):
    """{name: (value, majorant)}"""
    x, w, bias, state, dy, dlast = d(x), d(w), d(bias), d(state), d(dy), d(dlast)
    B, T, C = x.shape
    K = w.shape[1]
    keep, n = keep_rows(lengths, B, T)
    keep = keep[..., None]
    x = torch.where(keep, x, 0.0)
    rows = torch.cat([torch.zeros(B, K - 1, C, dtype=x.dtype) if state is None else state, x], 1)
    pre = sum(rows[:, k:k + T] * w[:, k] for k in range(K)) + (0.0 if bias is None else bias)
    mpre = sum((rows[:, k:k + T] * w[:, k]).abs() for k in range(K)) + (0.0 if bias is None else bias.abs())
    y, slope = silu(pre) if act else (pre, torch.ones_like(pre))
    # |silu'| <= 1.1 and |silu''| <= 0.5: an error e of pre moves y by 1.1 e and the slope by 0.5 e
    out = {"y": (torch.where(keep, y, 0.0), torch.where(keep, 1.1 * mpre if act else mpre, 0.0))}
    at = (n[:, None] + torch.arange(K - 1))[..., None].expand(B, K - 1, C)
    last = rows.gather(1, at)
    out["last"] = (last, 0 * last)
    if dy is None:
        return out
    g = torch.where(keep, dy * slope, 0.0)
    mg = torch.where(keep, dy.abs() * (slope.abs() + 0.5 * mpre if act else 1.0), 0.0)
    drows, mrows = torch.zeros_like(rows), torch.zeros_like(rows)
    if dlast is not None:
        drows.scatter_add_(1, at, dlast)
        mrows.scatter_add_(1, at, dlast.abs())
    dw, mw = torch.zeros_like(w), torch.zeros_like(w)
    for k in range(K):
        drows[:, k:k + T] += g * w[:, k]
        mrows[:, k:k + T] += mg * w[:, k].abs()
        dw[:, k] = (g * rows[:, k:k + T]).sum((0, 1))
        mw[:, k] = (mg * rows[:, k:k + T].abs()).sum((0, 1))
    out["x"] = (torch.where(keep, drows[:, K - 1:], 0.0), torch.where(keep, mrows[:, K - 1:], 0.0))
    out["state"] = (drows[:, :K - 1], mrows[:, :K - 1])
    out["weight"], out["bias"] = (dw, mw), (g.sum((0, 1)), mg.sum((0, 1)))
    return out


def scan(u, delta, A, Bm, Cm, D, z, delta_bias, softplus, state, lengths, dy=None, dlast=None):
    """{name: (value, majorant)}; Bm, Cm [B, T, G, N].  The decay's own error is relative: exp(step A) carries (3 + 2 |step A|) roundings of its
    argument, which the caller counts in k."""
    u, delta, A, Bm, Cm, D, z, delta_bias, state, dy, dlast = (d(t) for t in (u, delta, A, Bm, Cm, D, z, delta_bias, state, dy, dlast))
    B, T, C = u.shape
    G, N = Bm.shape[2:]
    keep, n = keep_rows(lengths, B, T)
    keep = keep[..., None]
    raw = delta + (0.0 if delta_bias is None else delta_bias)
    step = torch.where(keep, F.softplus(raw, threshold=1e9) if softplus else raw, 0.0)
    u = torch.where(keep, u, 0.0)
    z = None if z is None else torch.where(keep, z, 0.0)
    Bc, Cc = (torch.where(keep[..., None], m, 0.0).repeat_interleave(C // G, 2) for m in (Bm, Cm))
    Dv = torch.zeros(C, dtype=u.dtype) if D is None else D
    gate, slope = (torch.ones_like(u), None) if z is None else silu(z)

    def whole(absolute):
        f = (lambda t: t.abs()) if absolute else (lambda t: t)
        h = f(state) if state is not None else torch.zeros(B, C, N, dtype=u.dtype)
        hs, ys, decay = [h], [], []
        for t in range(T):
            a = torch.exp(step[:, t, :, None] * A)
            h = a * h + f((step[:, t] * u[:, t])[..., None] * Bc[:, t])
            hs.append(h)
            decay.append(a)
            ys.append((f(Cc[:, t]) * h).sum(-1) + f(Dv * u[:, t]))
        y0 = torch.stack(ys, 1)
        out = {"y": torch.where(keep, y0 * f(gate), 0.0), "last": h}
        if dy is None:
            return out
        gy = torch.where(keep, dy, 0.0)
        d0 = f(gy * gate)
        c = f(dlast) if dlast is not None else torch.zeros(B, C, N, dtype=u.dtype)
        dA = torch.zeros(C, N, dtype=u.dtype)
        du, ds, dB, dC = torch.zeros_like(u), torch.zeros_like(u), torch.zeros(B, T, C, N, dtype=u.dtype), torch.zeros(B, T, C, N, dtype=u.dtype)
        for t in range(T - 1, -1, -1):
            g = c + d0[:, t, :, None] * f(Cc[:, t])
            dC[:, t] = d0[:, t, :, None] * hs[t + 1]
            dB[:, t] = g * f(step[:, t] * u[:, t])[..., None]
            gb = (g * f(Bc[:, t])).sum(-1)
            c = decay[t] * g
            q = c * hs[t]
            du[:, t] = f(step[:, t]) * gb + f(Dv) * d0[:, t]
            ds[:, t] = (q * f(A)).sum(-1) + f(u[:, t]) * gb
            dA += (q * f(step[:, t])[..., None]).sum(0)
        if softplus:
            ds = ds * torch.sigmoid(raw)
        ds = torch.where(keep, ds, 0.0)
        out.update(u=torch.where(keep, du, 0.0), delta=ds, A=dA, D=(d0 * f(u)).sum((0, 1)), delta_bias=ds.sum((0, 1)), state=c,
                   Bm=dB.view(B, T, G, C // G, N).sum(3), Cm=dC.view(B, T, G, C // G, N).sum(3))
        if z is not None:
            out["z"] = f(gy) * y0 * f(slope)
        return out

    val, maj = whole(False), whole(True)
    return {k: (val[k], maj[k]) for k in val}


def norm(x, branch, gate, w, b, wp, bp, scale, ab, post, layer, eps, dr=None, dy=None):
    """{name: (value, majorant)}.  A norm's row is divided by its own deviation, so the majorants take the row's values at |v| + |mean|."""
    x, branch, gate, w, b, wp, bp, scale, ab, dr, dy = (d(t) for t in (x, branch, gate, w, b, wp, bp, scale, ab, dr, dy))
    B, T, C = x.shape
    one, zero = torch.ones(C, dtype=x.dtype), torch.zeros(C, dtype=x.dtype)

    def hat(v, mv):
        c = v - v.mean(-1, keepdim=True) if layer else v
        mc = mv + mv.mean(-1, keepdim=True) if layer else mv
        rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + eps)
        # error of c / rms(c): c's own, and c times the relative error of the mean square (Cauchy-Schwarz over the row)
        return c * rstd, mc * rstd + (c * rstd).abs() * (mc.square().mean(-1, keepdim=True).sqrt() * rstd), rstd

    def back(g, mg, vh, mvh, rstd):
        dv = g - vh * (g * vh).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if layer else 0.0)
        m = mg + mvh * (mg * mvh).mean(-1, keepdim=True) + (mg.mean(-1, keepdim=True) if layer else 0.0)
        return rstd * dv, rstd * m * (1 + mvh.square().mean(-1, keepdim=True).sqrt())

    sc = one if scale is None else scale
    gt = one if gate is None else gate[:, None] if gate.dim() == 2 else gate
    vw, vb = one if w is None else w, zero if b is None else b
    pw, pb = one if wp is None else wp, zero if bp is None else bp
    if branch is None:
        r, mr = x, x.abs()
    else:
        oh, moh, orstd = hat(branch, branch.abs()) if post else (branch, branch.abs(), None)
        n, mn = (oh * pw + pb, moh * pw.abs() + pb.abs()) if post else (branch, branch.abs())
        r, mr = x + sc * gt * n, x.abs() + (sc * gt).abs() * mn
    rh, mrh, rrstd = hat(r, mr)
    a, s = (zero, zero) if ab is None else ab[:, None].chunk(2, -1)
    m, mm = rh * vw + vb, mrh * vw.abs() + vb.abs()
    out = {"r": (r, mr), "y": (m * (1 + a) + s, mm * (1 + a).abs() + s.abs() + mm * a.abs())}
    if dr is None and dy is None:
        return out
    q, mq = (torch.zeros_like(x), torch.zeros_like(x)) if dr is None else (dr, dr.abs())
    dy0 = torch.zeros_like(x) if dy is None else dy
    dm, mdm = dy0 * (1 + a), dy0.abs() * (1 + a.abs())
    out["ab"] = (torch.cat([(dy0 * m).sum(1), dy0.sum(1)], -1), torch.cat([(dy0.abs() * mm).sum(1), dy0.abs().sum(1)], -1))
    out["weight"], out["bias"] = ((dm * rh).sum((0, 1)), (mdm * mrh).sum((0, 1))), (dm.sum((0, 1)), mdm.sum((0, 1)))
    if dy is not None:
        v, mv = back(dm * vw, mdm * vw.abs(), rh, mrh, rrstd)
        q, mq = q + v, mq + mv
    out["x"] = (q, mq)
    if branch is None:
        return out
    full = torch.ones(B, T, C, dtype=x.dtype)
    dn, mdn = q * sc * gt, mq * (sc * gt).abs()
    dg, mdg = q * sc * n, mq * sc.abs() * mn
    out["gate"] = (dg.sum(1), mdg.sum(1)) if gate is not None and gate.dim() == 2 else (dg, mdg)
    out["scale"] = ((q * gt * n * full).sum((0, 1)), (mq * gt.abs() * mn * full).sum((0, 1)))
    if post:
        out["post_weight"], out["post_bias"] = ((dn * oh).sum((0, 1)), (mdn * moh).sum((0, 1))), (dn.sum((0, 1)), mdn.sum((0, 1)))
        out["branch"] = back(dn * pw, mdn * pw.abs(), oh, moh, orstd)
    else:
        out["branch"] = (dn, mdn)
    return out
