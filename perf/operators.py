"""The sequence operators' workloads: a short causal convolution, a selective state space scan (both for whole sequences and for single
tokens) and the norms at a block's two edges with its gate and residual scale, forward and backward.

Every case is one call as a program makes it (`run`), in two forms on the same inputs: the plain one, elementary torch operations in
32 bits, and this package's kernels (`own`).  `exact` gives the same outputs from the definitions in 64 bits.  Activations are
channels-last [B, T, C]; parameters, recurrent states and per-item conditions are float32.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one stream generating frame by frame: the smallest call there is, pure latency
        dict(name="scan_step_one", op="scan_step", dtype="bf16", B=1, C=512, N=16, G=1, z=True),
        # 256 streams served together, one frame each: the state's read and write
        dict(name="scan_step_batch", op="scan_step", dtype="bf16", B=256, C=1024, N=16, G=1, z=True),
        # a 30 s clip (2250 codec frames) taken in before generation starts: one sequence, outputs and the state behind it
        dict(name="scan_prompt_clip", op="scan", train=False, dtype="bf16", B=1, T=2250, C=512, N=16, G=1, z=True, ragged=False, state=False),
        # the reference's default batch of 12 clips of 5 s (375 frames), a training step's forward and backward
        dict(name="scan_train", op="scan", train=True, dtype="bf16", B=12, T=375, C=512, N=16, G=1, z=True, ragged=False, state=False),
        # 16 clips of 30 s at 1024 channels, forward and backward: the largest
        dict(name="scan_train_long", op="scan", train=True, dtype="bf16", B=16, T=2250, C=1024, N=16, G=1, z=True, ragged=False, state=False),
        # float32 mode, odd sizes, two groups, clips of different lengths in one padded batch, carried state and its gradient
        dict(name="scan_train_ragged", op="scan", train=True, dtype="fp32", B=5, T=411, C=202, N=11, G=2, z=False, ragged=True, state=True),
        # 64 streams, one frame each, through the convolution's window
        dict(name="conv_step", op="conv_step", dtype="bf16", B=64, C=1024, K=4),
        # the benchmark's batch of 64 clips of 5 s at 512 channels, forward and backward
        dict(name="conv_train", op="conv", train=True, dtype="bf16", B=64, T=375, C=512, K=4, silu=True, ragged=False, state=False),
        # float32 mode, an odd channel count and length, a padded batch that goes on from a carried window
        dict(name="conv_train_ragged", op="conv", train=True, dtype="fp32", B=7, T=1003, C=131, K=3, silu=False, ragged=True, state=True),
        # one frame of 64 streams between two blocks: latency
        dict(name="norm_token", op="norm", train=False, dtype="bf16", residual="bf16", B=64, T=1, C=512, kind="rms", post=True, gate="none",
             scale=True, ab=False),
        # the translator's width (256) at the benchmark's batch, layer norm with a gate and a scale / shift from each item's condition
        dict(name="norm_train_film", op="norm", train=True, dtype="bf16", residual="bf16", B=64, T=375, C=256, kind="layer", post=False,
             gate="item", scale=False, ab=True),
        # 16 clips of 30 s, float32 residual stream, a gate per frame and a learned residual scale, forward and backward
        dict(name="norm_train_long", op="norm", train=True, dtype="bf16", residual="fp32", B=16, T=2250, C=1024, kind="rms", post=True,
             gate="token", scale=True, ab=False),
    ]


def draw(rng):
    """A case of the same ranges: batches of 1 to 256, 1 to 4096 frames, odd widths, both types, every option."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["scan", "scan", "scan", "conv", "norm", "scan_step", "conv_step"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if op in ("scan", "scan_step"):
        G = rng.choice([1, 1, 1, 2, 4])
        C = G * max(1, log(16, 2048) // G)
        N = rng.choice([4, 8, 16, 16, 16, 32, 64, rng.randint(1, 64)])
        if op == "scan_step":
            return dict(op=op, dtype=dtype, B=log(1, 256), C=C, N=N, G=G, z=flag())
        T = log(1, 4096)
        B = max(1, min(log(1, 64), 300_000_000 // (T * C * N)))
        T = max(1, min(T, 300_000_000 // (B * C * N)))
        return dict(op=op, train=flag(), dtype=dtype, B=B, T=T, C=C, N=N, G=G, z=flag(), ragged=flag(), state=flag())
    if op == "conv_step":
        return dict(op=op, dtype=dtype, B=log(1, 256), C=log(1, 4096), K=rng.randint(2, 8))
    if op == "conv":
        T, C, K = log(1, 4096), log(1, 2048), rng.randint(1, 8)
        return dict(op=op, train=flag(), dtype=dtype, B=max(1, min(log(1, 64), 20_000_000 // (T * C))), T=T, C=C, K=K, silu=flag(),
                    ragged=flag(), state=K > 1 and flag())
    T, C = log(1, 4096), log(16, 4096)
    return dict(op=op, train=flag(), dtype=dtype, residual=rng.choice([dtype, "fp32"]), B=max(1, min(log(1, 64), 20_000_000 // (T * C))), T=T,
                C=C, kind=rng.choice(["rms", "layer"]), post=flag(), gate=rng.choice(["none", "item", "token"]), scale=flag(), ab=flag())


def work(case):
    """What one pass reads, writes and computes at the least."""
    op, B, C = case["op"], case["B"], case["C"]
    T = case.get("T", 1)
    e = 2 if case["dtype"] == "bf16" else 4
    el = B * T * C
    train = case.get("train", False)
    if op in ("scan", "scan_step"):
        N, G = case["N"], case["G"]
        maps, params, state = 2 * B * T * G * N * e, 4 * C * (N + 2), 4 * B * C * N
        if op == "scan_step":
            return {"bytes": (3 + case["z"]) * el * e + maps + params + 2 * state, "flops": el * (7 * N + 20)}
        acts = 3 + case["z"]  # u, delta, z in; y out
        if not train:
            return {"bytes": acts * el * e + maps + params + (1 + case["state"]) * state, "flops": el * (7 * N + 20)}
        # the inputs once, y, dy, and a gradient for each input
        return {"bytes": (2 * acts) * el * e + 2 * maps + 2 * params + (4 * state if case["state"] else 0), "flops": el * (24 * N + 60)}
    if op in ("conv", "conv_step"):
        K = case["K"]
        if op == "conv_step":
            return {"bytes": (2 * el + 2 * B * (K - 1) * C) * e + 4 * C * (K + 1), "flops": el * (2 * K + 6)}
        state = B * (K - 1) * C * e
        return {"bytes": (4 if train else 2) * el * e + (2 if train else 1) * 4 * C * (K + 1) + (1 + train) * (1 + case["state"]) * state,
                "flops": el * (2 * K + 6) * (4 if train else 1)}
    er = 2 if case["residual"] == "bf16" else 4
    gate = {"none": 0, "item": 4 * B * C, "token": el * e}[case["gate"]]
    cond = 8 * B * C if case["ab"] else 0
    fwd = el * (2 * er + 2 * e) + gate + cond + 4 * C * 3
    return {"bytes": fwd + (el * (2 * er + 2 * e) + gate + cond + 4 * C * 3 if train else 0), "flops": el * (40 if train else 12)}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    def rand(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    op, B, C = case["op"], case["B"], case["C"]
    T, train = case.get("T", 1), case.get("train", False)
    s, grads = {}, {}
    if case.get("ragged"):  # clips of T // 3 to T frames in one padded batch
        s["lengths"] = (T // 3 + (rand(B) * (T - T // 3 + 1)).long()).clamp(max=T).to(torch.int32)
    if op in ("scan", "scan_step"):
        N, G = case["N"], case["G"]
        # decays spread over the states and step sizes of 1e-3 to 1e-1, as such layers are initialised, and moved a little by training
        s["A"] = -(torch.arange(1, N + 1, device="cuda").float() * (1 + 0.1 * randn(C, N).clamp(-3, 3)))
        s["D"] = 1 + 0.1 * randn(C)
        step = torch.exp(math.log(1e-3) + math.log(100.0) * rand(C))
        s["delta_bias"] = step + torch.log(-torch.expm1(-step))  # softplus^-1
        lead = (B,) if op == "scan_step" else (B, T)
        s["u"] = randn(*lead, C, dtype=dt)
        s["delta"] = randn(*lead, C, dtype=dt, scale=0.5)
        s["Bm"], s["Cm"] = randn(*lead, G, N, dtype=dt), randn(*lead, G, N, dtype=dt)
        if case["z"]:
            s["z"] = randn(*lead, C, dtype=dt)
        if op == "scan_step" or case["state"]:
            s["state"] = randn(B, C, N, scale=0.3)
        if train:
            grads["y"] = randn(B, T, C, dtype=dt)
            if case["state"]:
                grads["last"] = randn(B, C, N)
    elif op in ("conv", "conv_step"):
        K = case["K"]
        s["weight"], s["bias"] = randn(C, K, scale=1 / math.sqrt(K)), randn(C, scale=0.1)
        s["x"] = randn(*((B,) if op == "conv_step" else (B, T)), C, dtype=dt)
        if op == "conv_step" or case["state"]:
            s["state"] = randn(B, K - 1, C, dtype=dt)
        if train:
            grads["y"] = randn(B, T, C, dtype=dt)
            if case["state"]:
                grads["last"] = randn(B, K - 1, C, dtype=dt)
    else:
        rt = DTYPES[case["residual"]]
        s["x"], s["branch"] = randn(B, T, C, dtype=rt, scale=2.0), randn(B, T, C, dtype=dt)
        s["weight"] = 1 + 0.2 * randn(C)
        if case["kind"] == "layer":
            s["bias"] = 0.1 * randn(C)
        if case["post"]:
            s["post_weight"] = 1 + 0.2 * randn(C)
            if case["kind"] == "layer":
                s["post_bias"] = 0.1 * randn(C)
        if case["gate"] != "none":
            s["gate"] = randn(B, C) if case["gate"] == "item" else randn(B, T, C, dtype=dt)
        if case["scale"]:
            s["scale"] = 0.5 + 0.1 * randn(C)
        if case["ab"]:
            s["ab"] = 0.3 * randn(B, 2 * C)
        if train:
            grads["r"], grads["y"] = randn(B, T, C, dtype=rt), randn(B, T, C, dtype=dt)
    if train:
        for t in s.values():
            if t.is_floating_point():
                t.requires_grad_(True)
    return {"case": dict(case), "in": s, "grads": grads}


def run(state):
    case, s, grads = state["case"], state["in"], state["grads"]
    return (_own if own else _plain)(case, s, grads)


# ------------------------------------------------------------------------------------------------ this package's kernels
def _own(case, s, grads):
    from gan_amd import _lib as L
    from gan_amd import sequence as S

    op = case["op"]
    if op == "scan_step":
        y = S.selective_scan_step(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], s["state"], D=s["D"], z=s.get("z"), delta_bias=s["delta_bias"])
        return {"y": y, "state": s["state"]}
    if op == "conv_step":
        return {"y": S.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], act=L.ACT_SILU), "state": s["state"]}
    if op == "scan":
        y, last = S.selective_scan(s["u"], s["delta"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s.get("z"), delta_bias=s["delta_bias"],
                                   state=s.get("state"), lengths=s.get("lengths"), return_state=True)
        out = {"y": y, "last": last}
    elif op == "conv":
        y, last = S.causal_conv(s["x"], s["weight"], s["bias"], act=L.ACT_SILU if case["silu"] else L.ACT_NONE, state=s.get("state"),
                                lengths=s.get("lengths"), return_state=True)
        out = {"y": y, "last": last}
    else:
        r, y = S.block_norm(s["x"], s["branch"], weight=s["weight"], bias=s.get("bias"), post_norm=case["post"], post_weight=s.get("post_weight"),
                            post_bias=s.get("post_bias"), gate=s.get("gate"), scale=s.get("scale"), ab=s.get("ab"), kind=case["kind"], eps=1e-5)
        out = {"r": r, "y": y}
    if not case["train"]:
        return out
    wrt = [k for k in s if s[k].requires_grad]
    got = torch.autograd.grad([out[k] for k in grads], [s[k] for k in wrt], list(grads.values()))
    return {**{k: v.detach() for k, v in out.items()}, **{"d_" + k: g for k, g in zip(wrt, got)}}


# ------------------------------------------------------------------------------------------------ plain forms, in 32 bits
def _plain(case, s, grads):
    op = case["op"]
    if op == "scan_step":
        return _plain_scan_step(s)
    if op == "conv_step":
        return _plain_conv_step(s)
    if op == "scan":
        return _plain_scan(case, s, grads)
    f = {k: v.detach().float().requires_grad_(case["train"]) if v.is_floating_point() else v for k, v in s.items()}
    with torch.enable_grad():
        out = _plain_conv(case, f) if op == "conv" else _plain_norm(case, f)
    kinds = {"r": s["x"].dtype, "y": s["branch"].dtype if "branch" in s else s["x"].dtype, "last": s["x"].dtype}
    res = {k: v.detach().to(kinds[k]) for k, v in out.items()}
    if case["train"]:
        wrt = [k for k in f if f[k].is_floating_point()]
        got = torch.autograd.grad([out[k] for k in grads], [f[k] for k in wrt], [g.float() for g in grads.values()])
        res.update({"d_" + k: g.to(s[k].dtype) for k, g in zip(wrt, got)})
    return res


def _plain_conv(case, f):
    x, w = f["x"], f["weight"]
    B, T, C = x.shape
    K = w.shape[1]
    past = f["state"] if "state" in f else x.new_zeros(B, K - 1, C)
    if "lengths" in f:
        keep = (torch.arange(T, device=x.device) < f["lengths"][:, None])[..., None]
        x = torch.where(keep, x, 0.0)
    full = torch.cat([past, x], 1)
    pre = (full.unfold(1, K, 1) * w).sum(-1) + f["bias"]
    y = pre * torch.sigmoid(pre) if case["silu"] else pre
    if "lengths" in f:
        y = torch.where(keep, y, 0.0)
        rows = f["lengths"].long()[:, None] + torch.arange(K - 1, device=x.device)
        last = full.gather(1, rows[..., None].expand(B, K - 1, C))
    else:
        last = full[:, T:]
    return {"y": y, "last": last}


def _plain_conv_step(s):
    full = torch.cat([s["state"], s["x"][:, None]], 1)
    pre = (full.float().transpose(1, 2) * s["weight"]).sum(-1) + s["bias"]
    s["state"].copy_(full[:, 1:])
    return {"y": (pre * torch.sigmoid(pre)).to(s["x"].dtype), "state": s["state"]}


def _plain_norm(case, f):
    def norm(v, w, b):
        if case["kind"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5)
        v = v * w if w is not None else v
        return v + b if b is not None else v

    n = f["branch"]
    if case["post"]:
        n = norm(n, f.get("post_weight"), f.get("post_bias"))
    if "gate" in f:
        n = n * (f["gate"][:, None] if case["gate"] == "item" else f["gate"])
    if "scale" in f:
        n = n * f["scale"]
    r = f["x"] + n
    y = norm(r, f.get("weight"), f.get("bias"))
    if "ab" in f:
        a, b = f["ab"][:, None].chunk(2, -1)
        y = y * (1 + a) + b
    return {"r": r, "y": y}


def _per_channel(m, C):
    """[..., G, N] -> [..., C, N] in 32 bits: each group's row for every one of its channels."""
    return m.float().repeat_interleave(C // m.shape[-2], -2)


def _plain_scan_step(s):
    u, C = s["u"].float(), s["u"].shape[-1]
    step = F.softplus(s["delta"].float() + s["delta_bias"])
    h = torch.exp(step[..., None] * s["A"]) * s["state"] + (step * u)[..., None] * _per_channel(s["Bm"], C)
    y = (h * _per_channel(s["Cm"], C)).sum(-1) + s["D"] * u
    if "z" in s:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    s["state"].copy_(h)
    return {"y": y.to(s["u"].dtype), "state": s["state"]}


def _recur(a, x):
    """h_t = a_t h_{t-1} + x_t along axis 1 (h before the first row 0), in blocks of sqrt(T) rows: inside all blocks at once, then the
    carries from block to block, then the carries' share of every row."""
    B, T = x.shape[:2]
    S = max(1, math.isqrt(T))
    n = -(-T // S)
    if n * S > T:
        a = torch.cat([a, a.new_ones(B, n * S - T, *a.shape[2:])], 1)
        x = torch.cat([x, x.new_zeros(B, n * S - T, *x.shape[2:])], 1)
    a, x = a.reshape(B, n, S, *a.shape[2:]).clone(), x.reshape(B, n, S, *x.shape[2:]).clone()
    for i in range(1, S):
        x[:, :, i].addcmul_(a[:, :, i], x[:, :, i - 1])
        a[:, :, i].mul_(a[:, :, i - 1])
    carry = torch.zeros_like(x[:, :, 0])
    for j in range(1, n):
        carry[:, j] = x[:, j - 1, -1] + a[:, j - 1, -1] * carry[:, j - 1]
    return x.addcmul_(a, carry[:, :, None]).flatten(1, 2)[:, :T]


def _plain_scan(case, s, grads):
    s = {k: v.detach() for k, v in s.items()}
    dt, C, T = s["u"].dtype, case["C"], case["T"]
    u, raw = s["u"].float(), s["delta"].float() + s["delta_bias"]
    step = F.softplus(raw)
    z = s["z"].float() if "z" in s else None
    if "lengths" in s:
        keep = (torch.arange(T, device=u.device) < s["lengths"][:, None])[..., None]
        step, u = torch.where(keep, step, 0.0), torch.where(keep, u, 0.0)
    Bc, Cc = _per_channel(s["Bm"], C), _per_channel(s["Cm"], C)
    a = torch.exp(step[..., None] * s["A"])
    x = (step * u)[..., None] * Bc
    first = s["state"] if "state" in s else torch.zeros_like(x[:, 0])
    x[:, 0] += a[:, 0] * first
    h = _recur(a, x)
    y0 = (h * Cc).sum(-1) + s["D"] * u
    gate = z * torch.sigmoid(z) if z is not None else 1.0
    y = y0 * gate
    if "lengths" in s:
        y = torch.where(keep, y, 0.0)
    out = {"y": y.to(dt), "last": h[:, -1].clone()}
    if not case["train"]:
        return out
    dy = grads["y"].float()
    if "lengths" in s:
        dy = torch.where(keep, dy, 0.0)
    d0 = dy * gate
    G = d0[..., None] * Cc
    if "last" in grads:
        G[:, -1] += grads["last"]
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _recur(after.flip(1), G.flip(1)).flip(1)
    out["d_state"] = a[:, 0] * g[:, 0]
    before = torch.cat([first[:, None], h[:, :-1]], 1)
    q = g * a * before
    gB = (g * Bc).sum(-1)
    d_step = (q * s["A"]).sum(-1) + u * gB
    d_raw = d_step * torch.sigmoid(raw)
    d_u = step * gB + s["D"] * d0
    if "lengths" in s:
        d_raw, d_u = torch.where(keep, d_raw, 0.0), torch.where(keep, d_u, 0.0)
    groups = (*d0.shape[:2], case["G"], C // case["G"], case["N"])
    out["d_u"], out["d_delta"] = d_u.to(dt), d_raw.to(dt)
    out["d_A"] = (q * step[..., None]).sum((0, 1))
    out["d_Bm"] = (g * (step * u)[..., None]).view(groups).sum(3).to(dt)
    out["d_Cm"] = (h * d0[..., None]).view(groups).sum(3).to(dt)
    out["d_D"], out["d_delta_bias"] = (d0 * u).sum((0, 1)), d_raw.sum((0, 1))
    if z is not None:
        sig = torch.sigmoid(z)
        dz = dy * y0 * sig * (1 + z * (1 - sig))
        out["d_z"] = (torch.where(keep, dz, 0.0) if "lengths" in s else dz).to(dt)
    if "state" not in s:
        del out["d_state"]
    return out


# ------------------------------------------------------------------------------------------------ definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    s = {k: v.detach().double() if v.is_floating_point() else v.long() for k, v in st["in"].items()}
    grads = {k: v.double() for k, v in st["grads"].items()}
    if case["op"] in ("scan", "scan_step"):
        return _exact_scan(case, s, grads)
    if case["op"] in ("conv", "conv_step"):
        return _exact_conv(case, s, grads)
    return _exact_norm(case, s, grads)


def _silu_and_slope(v):
    e = torch.exp(-v.abs())
    sig = torch.where(v >= 0, 1 / (1 + e), e / (1 + e))
    return v * sig, sig + v * sig * (1 - sig)


def _exact_scan(case, s, grads):
    """Time step by time step, then the adjoint recurrence backwards; the reductions gathered as the steps go."""
    single = case["op"] == "scan_step"
    seq = (lambda t: t[:, None]) if single else (lambda t: t)
    u, raw = seq(s["u"]), seq(s["delta"]) + s["delta_bias"]
    Bm, Cm = seq(s["Bm"]), seq(s["Cm"])
    z = seq(s["z"]) if "z" in s else None
    nb, T, C = u.shape
    G, N = case["G"], case["N"]
    Cg = C // G
    length = s["lengths"] if "lengths" in s else torch.full((nb,), T, device=u.device)
    live = torch.arange(T, device=u.device) < length[:, None]
    step = raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs()))
    step = torch.where(live[..., None], step, torch.zeros_like(step))
    u = torch.where(live[..., None], u, torch.zeros_like(u))
    h = s["state"].reshape(nb, G, Cg, N) if "state" in s else u.new_zeros(nb, G, Cg, N)
    A = s["A"].view(G, Cg, N)
    sv, uv = step.view(nb, T, G, Cg), u.view(nb, T, G, Cg)
    hist = u.new_empty((T + 1 if grads else 1, nb, G, Cg, N))
    hist[0] = h
    y0 = u.new_empty(nb, T, G, Cg)
    for t in range(T):
        h = torch.exp(sv[:, t, ..., None] * A) * h + (sv[:, t] * uv[:, t])[..., None] * Bm[:, t, :, None]
        y0[:, t] = (h @ Cm[:, t, ..., None])[..., 0]
        if grads:
            hist[t + 1] = h
    y0 = y0.view(nb, T, C) + s["D"] * u
    gate, slope = _silu_and_slope(z) if z is not None else (torch.ones_like(y0), None)
    y = torch.where(live[..., None], y0 * gate, torch.zeros_like(y0))
    if single:
        return {"y": y[:, 0], "state": h.reshape(nb, C, N)}
    out = {"y": y, "last": h.reshape(nb, C, N)}
    if not grads:
        return out
    dy = torch.where(live[..., None], grads["y"], torch.zeros_like(y0))
    d0 = (dy * gate).view(nb, T, G, Cg)
    carry = grads["last"].reshape(nb, G, Cg, N) if "last" in grads else torch.zeros_like(h)
    dA = torch.zeros_like(A)
    dB, dC = torch.zeros_like(Bm), torch.zeros_like(Cm)
    d_step, d_u = torch.zeros_like(sv), torch.zeros_like(uv)
    for t in range(T - 1, -1, -1):
        st, ut, dt0 = sv[:, t], uv[:, t], d0[:, t]
        a = torch.exp(st[..., None] * A)
        g = carry + dt0[..., None] * Cm[:, t, :, None]
        dC[:, t] = (dt0[:, :, None] @ hist[t + 1])[:, :, 0]
        dB[:, t] = ((st * ut)[:, :, None] @ g)[:, :, 0]
        gb = (g @ Bm[:, t, ..., None])[..., 0]
        carry = g * a
        q = carry * hist[t]
        d_u[:, t] = st * gb
        d_step[:, t] = (q * A).sum(-1) + ut * gb
        dA += (q * st[..., None]).sum(0)
    d0, zero = d0.reshape(nb, T, C), torch.zeros_like(u)
    d_raw = torch.where(live[..., None], d_step.view(nb, T, C) / (1 + torch.exp(-raw)), zero)
    out["d_u"] = torch.where(live[..., None], d_u.view(nb, T, C) + s["D"] * d0, zero)
    out["d_delta"], out["d_delta_bias"] = d_raw, d_raw.sum((0, 1))
    out["d_A"], out["d_Bm"], out["d_Cm"], out["d_D"] = dA.view(C, N), dB, dC, (d0 * u).sum((0, 1))
    if z is not None:
        out["d_z"] = torch.where(live[..., None], dy * y0 * slope, zero)
    if "state" in s:
        out["d_state"] = carry.reshape(nb, C, N)
    return out


def _exact_conv(case, s, grads):
    """Tap by tap on the joined rows (window, then sequence)."""
    single = case["op"] == "conv_step"
    x = s["x"][:, None] if single else s["x"]
    nb, T, C = x.shape
    w = s["weight"]
    K = w.shape[1]
    length = s["lengths"] if "lengths" in s else torch.full((nb,), T, device=x.device)
    live = (torch.arange(T, device=x.device) < length[:, None])[..., None]
    x = torch.where(live, x, torch.zeros_like(x))
    rows = torch.zeros(nb, T + K - 1, C, dtype=x.dtype, device=x.device)
    rows[:, K - 1:] = x
    if "state" in s:
        rows[:, :K - 1] = s["state"]
    pre = s["bias"].expand(nb, T, C).clone()
    for k in range(K):
        pre += rows[:, k:k + T] * w[:, k]
    y, slope = _silu_and_slope(pre) if single or case["silu"] else (pre, torch.ones_like(pre))
    y = torch.where(live, y, torch.zeros_like(y))
    at = (length[:, None] + torch.arange(K - 1, device=x.device))[..., None].expand(nb, K - 1, C)
    last = rows.gather(1, at)
    if single:
        return {"y": y[:, 0], "state": last}
    out = {"y": y, "last": last}
    if not grads:
        return out
    g = torch.where(live, grads["y"] * slope, torch.zeros_like(y))
    d_rows = torch.zeros_like(rows)
    if "last" in grads:
        d_rows.scatter_add_(1, at, grads["last"])
    d_w = torch.zeros_like(w)
    for k in range(K):
        d_rows[:, k:k + T] += g * w[:, k]
        d_w[:, k] = (g * rows[:, k:k + T]).sum((0, 1))
    out["d_weight"], out["d_bias"] = d_w, g.sum((0, 1))
    out["d_x"] = torch.where(live, d_rows[:, K - 1:], torch.zeros_like(x))
    if "state" in s:
        out["d_state"] = d_rows[:, :K - 1]
    return out


def _exact_norm(case, s, grads):
    """The two norms' closed forms: d v = rstd (g - mean(g) - vhat mean(g vhat)), without mean(g) for the root mean square."""
    layer = case["kind"] == "layer"
    one = torch.ones(case["C"], dtype=torch.float64, device=s["x"].device)

    def hat(v):
        v = v - v.mean(-1, keepdim=True) if layer else v
        rstd = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)
        return v * rstd, rstd

    def hat_back(g, vh, rstd):
        d = g - vh * (g * vh).mean(-1, keepdim=True)
        return rstd * (d - g.mean(-1, keepdim=True) if layer else d)

    w, wp = s.get("weight", one), s.get("post_weight", one)
    b, bp = s.get("bias", 0 * one), s.get("post_bias", 0 * one)
    if case["post"]:
        oh, orstd = hat(s["branch"])
        n = oh * wp + bp
    else:
        n = s["branch"]
    gate = s["gate"][:, None] if case["gate"] == "item" else s["gate"] if case["gate"] == "token" else one
    scale = s.get("scale", one)
    r = s["x"] + scale * gate * n
    rh, rrstd = hat(r)
    m = rh * w + b
    a, shift = (s["ab"][:, None].chunk(2, -1)) if case["ab"] else (0 * one, 0 * one)
    out = {"r": r, "y": m * (1 + a) + shift}
    if not grads:
        return out
    dy = grads["y"]
    if case["ab"]:
        out["d_ab"] = torch.cat([(dy * m).sum(1), dy.sum(1)], -1)
    dm = dy * (1 + a)
    out["d_weight"] = (dm * rh).sum((0, 1))
    if "bias" in s:
        out["d_bias"] = dm.sum((0, 1))
    dr = grads["r"] + hat_back(dm * w, rh, rrstd)
    out["d_x"] = dr
    if case["scale"]:
        out["d_scale"] = (dr * gate * n).sum((0, 1))
    if case["gate"] != "none":
        dg = dr * scale * n
        out["d_gate"] = dg.sum(1) if case["gate"] == "item" else dg
    dn = dr * scale * gate
    if case["post"]:
        out["d_post_weight"] = (dn * oh).sum((0, 1))
        if "post_bias" in s:
            out["d_post_bias"] = dn.sum((0, 1))
        out["d_branch"] = hat_back(dn * wp, oh, orstd)
    else:
        out["d_branch"] = dn
    return out
