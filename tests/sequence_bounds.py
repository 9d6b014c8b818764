"""The selective scan in 64 bits on the CPU with its gradients and, beside every value, how far a float32 evaluation may be off: first-order errors
carried along the recurrence, so that they decay as the states do (a bound that grows with the length alone lets states of too few bits pass).

Roundings are counted in U = 2^-24 of the value rounded, or of a majorant of it (the same formula with every term's absolute value) where the
order of a sum is the kernel's own.  What is counted:
    step        raw = delta + delta_bias: 1;  softplus: 16 (exp2, log2, reciprocal and their arguments), and raw's error times its slope
    decay       exp(step A): A log2(e) and its product with the step 3 of the argument, exp2 4; where chunks of `tiles` tiles are joined, the sum
                of their steps takes tiles + 64 additions: as many more of every row's argument
    state       decay * h + (step u) B: 2 of the input, 2 of the sum; what float32 flushes below its normal numbers (1.2e-38, of a decay: times
                the state), carried along as well
    sums        over N states N + 8, over the channels of a group 12 + their blocks of 64 + the products, over a chunk's rows 16 tiles + 40 (and in
                double from there on)
    gates       z sigmoid(z): 2 |z| + 8;  its slope (1 + |z|) sigmoid(z) (2 |z| + 12)
The adjoint is the same recurrence run backwards.  Second-order terms: 2 % on top."""
import torch
import torch.nn.functional as F

from tests.sequence_ref import U, d, keep_rows, silu

FLUSH = 1.2e-38


def close(got, ref, err, what):
    """|got - ref| <= err + half a step of got's type"""
    got, dtype = got.detach().cpu().double(), got.dtype
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), what
    tol = 1.02 * err + (2.0 ** -8 * ref.abs() * (1 + 1e-3) if dtype == torch.bfloat16 else 0.0) + FLUSH
    off = (got - ref).abs()
    worst = float((off / tol).max())
    assert worst <= 1.0, f"{what}: {worst:.2f} times the tolerance (largest error {float(off.max()):.3g})"


def scan(u, delta, A, Bm, Cm, D, z, delta_bias, softplus, state, lengths, tiles, dy=None, dlast=None):
    """{name: (value, error)}; Bm, Cm [B, T, G, N]"""
    u, delta, A, Bm, Cm, D, z, delta_bias, state, dy, dlast = (d(t) for t in (u, delta, A, Bm, Cm, D, z, delta_bias, state, dy, dlast))
    B, T, C = u.shape
    G, N = Bm.shape[2:]
    Cg = C // G
    keep, _ = keep_rows(lengths, B, T)
    keep = keep[..., None]
    zero = torch.zeros((), dtype=u.dtype)
    bias = zero if delta_bias is None else delta_bias
    raw = torch.where(keep, delta + bias, zero)
    eraw = U * raw.abs()
    step = F.softplus(raw, threshold=1e9) if softplus else raw
    estep = 16 * U * step.abs() + eraw * torch.sigmoid(raw) if softplus else eraw
    step, estep = torch.where(keep, step, zero), torch.where(keep, estep, zero)
    u = torch.where(keep, u, zero)
    z = None if z is None else torch.where(keep, z, zero)
    Bm, Cm = (torch.where(keep[..., None], m, zero) for m in (Bm, Cm))
    Dv = torch.zeros(C, dtype=u.dtype) if D is None else D
    su, esu = step * u, u.abs() * estep + U * (step * u).abs()
    gate, egate = torch.ones_like(u), torch.zeros_like(u)
    if z is not None:
        gate, slope = silu(z)
        egate = gate.abs() * (2 * z.abs() + 8) * U
        eslope = (1 + z.abs()) * torch.sigmoid(z) * (2 * z.abs() + 12) * U

    def per_channel(m, t):  # [B, G, N] -> [B, C, N]
        return m[:, t].repeat_interleave(Cg, 1)

    def decay(t):
        x = step[:, t, :, None] * A
        a = torch.exp(x)
        return a, a * (A.abs() * estep[:, t, :, None] + ((3 + tiles + 64) * x.abs() + 4) * U)

    h = torch.zeros(B, C, N, dtype=u.dtype) if state is None else state
    m, e = h.abs(), torch.zeros(B, C, N, dtype=u.dtype)
    hs, y0, my0, ey0 = [(h, m, e)], torch.empty_like(u), torch.empty_like(u), torch.empty_like(u)
    for t in range(T):
        a, ea = decay(t)
        b, c = per_channel(Bm, t), per_channel(Cm, t)
        x = su[:, t, :, None] * b
        e = a * e + ea * m + esu[:, t, :, None] * b.abs() + FLUSH * (1 + m)
        h, m = a * h + x, a * m + x.abs()
        e = e + 2 * U * (x.abs() + m)
        y0[:, t] = (c * h).sum(-1) + Dv * u[:, t]
        my0[:, t] = (c.abs() * m).sum(-1) + (Dv * u[:, t]).abs()
        ey0[:, t] = (c.abs() * e).sum(-1) + (N + 8) * U * my0[:, t]
        hs.append((h, m, e) if dy is not None else None)
    out = {"y": (torch.where(keep, y0 * gate, zero), torch.where(keep, gate.abs() * ey0 + egate * my0 + U * (gate * my0).abs(), zero)), "last": (h, e)}
    if dy is None:
        return out
    gy = torch.where(keep, dy, zero)
    d0, ed0 = gy * gate, gy.abs() * egate + U * (gy * gate).abs()
    if z is not None:
        out["z"] = (gy * y0 * slope, gy.abs() * (slope.abs() * ey0 + my0 * eslope + 4 * U * my0 * slope.abs()))
    c = torch.zeros(B, C, N, dtype=u.dtype) if dlast is None else dlast
    mc, ec = c.abs(), torch.zeros(B, C, N, dtype=u.dtype)
    new = lambda *s: torch.zeros(*s, dtype=u.dtype)  # noqa: E731
    dB, eB, dC, eC = (new(B, T, G, N) for _ in range(4))
    du, eu, ds, es, ms = (new(B, T, C) for _ in range(5))
    dA, eA = new(C, N), new(C, N)
    kc, rows = 12 + (Cg + 63) // 64, 16 * tiles + 40
    group = lambda v: v.view(B, G, Cg, N).sum(2)  # noqa: E731
    for t in range(T - 1, -1, -1):
        a, ea = decay(t)
        b, cm = per_channel(Bm, t), per_channel(Cm, t)
        g0, eg0 = d0[:, t, :, None], ed0[:, t, :, None]
        s, esu_t = su[:, t, :, None], esu[:, t, :, None]
        (h, m, e), (hp, mp, ep) = hs[t + 1], hs[t]
        g, mg = c + g0 * cm, mc + (g0 * cm).abs()
        eg = ec + eg0 * cm.abs() + 2 * U * mg
        dC[:, t], eC[:, t] = group(g0 * h), group(g0.abs() * e + eg0 * m + kc * U * g0.abs() * m)
        dB[:, t], eB[:, t] = group(g * s), group(s.abs() * eg + esu_t * mg + kc * U * s.abs() * mg)
        gb, mgb = (g * b).sum(-1), (mg * b.abs()).sum(-1)
        egb = (eg * b.abs()).sum(-1) + (N + 8) * U * mgb
        c, mc = a * g, a * mg
        ec = a * eg + ea * mg + U * mc + FLUSH * (1 + mg)
        q, mq = c * hp, mc * mp
        eq = mc * ep + mp * ec + U * mq
        st, est = step[:, t], estep[:, t]
        du[:, t] = st * gb + Dv * d0[:, t]
        eu[:, t] = est * mgb + st.abs() * egb + Dv.abs() * ed0[:, t] + 3 * U * (st.abs() * mgb + (Dv * d0[:, t]).abs())
        ds[:, t] = (q * A).sum(-1) + u[:, t] * gb
        ms[:, t] = (mq * A.abs()).sum(-1) + u[:, t].abs() * mgb
        es[:, t] = (eq * A.abs()).sum(-1) + u[:, t].abs() * egb + (N + 12) * U * ms[:, t]
        dA += (q * st[..., None]).sum(0)
        eA += (eq * st.abs()[..., None] + mq * est[..., None] + rows * U * mq * st.abs()[..., None]).sum(0)
    if softplus:
        sig = torch.sigmoid(raw)
        es = sig * (es + (16 + raw.abs()) * U * ms)
        ds, ms = ds * sig, ms * sig
    ds, ms, es = (torch.where(keep, v, zero) for v in (ds, ms, es))
    out.update(u=(torch.where(keep, du, zero), torch.where(keep, eu, zero)), delta=(ds, es), A=(dA, eA), Bm=(dB, eB), Cm=(dC, eC), state=(c, ec),
               D=((d0 * u).sum((0, 1)), (u.abs() * ed0 + rows * U * (d0 * u).abs()).sum((0, 1))),
               delta_bias=(ds.sum((0, 1)), (es + rows * U * ms).sum((0, 1))))
    return out


def scan_rounded(u, delta, A, Bm, Cm, D, z, delta_bias, softplus, state, lengths, round_state=lambda h: h, round_step=lambda s: s):
    """The forward recurrence row by row in float32, the state (and the steps) rounded as told: (y, last).  What the bounds above have to tell from
    an honest float32 evaluation."""
    B, T, C = u.shape
    Cg = C // Bm.shape[2]
    keep, _ = keep_rows(lengths, B, T)
    f = lambda t: torch.where(keep.view(B, T, *[1] * (t.dim() - 2)), t.float(), torch.zeros(()))  # noqa: E731
    raw = f(delta) + (0.0 if delta_bias is None else delta_bias)
    step = round_step(f(F.softplus(raw, threshold=1e9) if softplus else raw))
    u, Bm, Cm = f(u), f(Bm), f(Cm)
    h = torch.zeros(B, C, A.shape[1]) if state is None else state.float()
    y = torch.empty(B, T, C)
    for t in range(T):
        h = round_state(torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * u[:, t])[..., None] * Bm[:, t].repeat_interleave(Cg, 1))
        y[:, t] = (Cm[:, t].repeat_interleave(Cg, 1) * h).sum(-1) + (0.0 if D is None else D * u[:, t])
    if z is not None:
        zz = f(z)
        y = y * (zz * torch.sigmoid(zz))
    return torch.where(keep[..., None], y, torch.zeros(())), h
