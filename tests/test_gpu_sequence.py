"""GPU: the sequence operators (gan_amd/sequence.py: causal convolution, selective scan, block norms; forward, gradients, single-token steps)
against their plain 64-bit forms (tests/sequence_ref.py), at the sizes, strides, lengths and masks where they can go wrong, on other
streams, in captured graphs, together as one block, and bit for bit from run to run.

Tolerance: k roundings of 2^-24 times the majorant of the value (see sequence_ref), plus half a bf16 step for bf16 results.  k counts the longest
path: K_CONV = taps + activation; K_SCAN per row walked, forward and backward, with exp's argument (12 roundings of step * A, |step * A| <= 2 in
these tests) and the sums over rows, channels and states; K_NORM = the row sums (a tree over 64 lanes of C / 64 values) and the chain through two
norms and their gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from gan_amd import _lib as L
from gan_amd import sequence as S
from tests import sequence_ref as R

DEV = torch.device("cuda")
BF, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def lens(B, T):
    """Items of every kind: none, one row, all, some, more than there are (counts as all), less than none (none)."""
    return torch.tensor([[0, 1, T, T // 2 + 1, T + 9, -3][i % 6] for i in range(B)], dtype=torch.int32, device=DEV)


def poison(t, lengths, value=NAN):
    """Garbage in the rows behind each item's end."""
    t = t.clone()
    for b, n in enumerate(lengths.clamp(0, t.shape[1]).tolist()):
        t[b, n:] = value
    return t


def grads(outs, wrt, cot):
    pairs = [(o, c) for o, c in zip(outs, cot) if c is not None]
    return torch.autograd.grad([o for o, _ in pairs], wrt, [c for _, c in pairs])


# ------------------------------------------------------------------------------------------------ causal convolution
CONV = [  # B, T, C, K, dtype, silu, bias, state, ragged
    (1, 1, 1, 1, F32, False, True, False, False),
    (1, 1, 8, 4, BF, True, True, True, False),
    (2, 2, 6, 8, F32, True, True, True, False),      # fewer rows than taps
    (3, 16, 64, 4, BF, True, True, False, False),    # exactly one run
    (2, 17, 260, 3, F32, False, False, True, False),  # one row past a run; several piece blocks
    (6, 37, 33, 4, F32, True, True, True, True),
    (6, 40, 72, 5, BF, True, False, True, True),
    (7, 65, 20, 2, BF, False, True, False, True),
    (2, 300, 12, 7, F32, True, True, False, False),
    (40, 33, 512, 4, BF, True, True, True, False),   # more runs than blocks along time
    (3, 5, 9, 6, BF, True, True, True, True),
]


def make_conv(case, seed=0):
    B, T, C, K, dt, silu, bias, state, ragged = case
    g = gen(seed + T * 7 + C)
    ln = lens(B, T) if ragged else None
    x = rnd(g, B, T, C, dtype=dt)
    a = dict(x=poison(x, ln) if ragged else x, weight=rnd(g, C, K, scale=0.5), bias=rnd(g, C, scale=0.3) if bias else None,
             state=rnd(g, B, K - 1, C, dtype=dt) if state else None)
    dy, dl = rnd(g, B, T, C, dtype=dt), rnd(g, B, K - 1, C, dtype=dt)
    return a, ln, (poison(dy, ln) if ragged else dy), dl


def k_conv(case):
    B, T, C, K = case[:4]
    return 2 * K + 24 + B * T  # taps, the gate's exp / reciprocal / products, and the weight gradient's sum over all rows


@pytest.mark.parametrize("case", CONV, ids=str)
def test_causal_conv_and_its_gradients(case):
    B, T, C, K, dt, silu, *_ = case
    a, ln, dy, dl = make_conv(case)
    act = L.ACT_SILU if silu else L.ACT_NONE
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items() if v is not None}
    y, last = S.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), act, leaves.get("state"), ln, return_state=True)
    got = dict(zip(leaves, grads([y, last], list(leaves.values()), [dy, dl if K > 1 else None])))
    ref = R.conv(a["x"], a["weight"], a["bias"], silu, a["state"], ln, dy, dl)
    k = k_conv(case)
    for name, t in (("y", y), ("last", last), *got.items()):
        R.close(t, *ref[name], k, name)
    with torch.no_grad():  # the call without gradients is the same call
        y2 = S.causal_conv(a["x"], a["weight"], a["bias"], act, a["state"], ln)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("K", [1, 2, 4, 8])
def test_causal_conv_step_goes_on_where_the_sequence_ended(dt, K):
    B, T, C = 5, 11, 70
    g = gen(K)
    x, w, b = rnd(g, B, T, C, dtype=dt), rnd(g, C, K, scale=0.5), rnd(g, C)
    whole = S.causal_conv(x, w, b, L.ACT_SILU)
    pool = rnd(g, 2 * B, K - 1, C, dtype=dt)  # the state is every other item of a larger buffer
    y, last = S.causal_conv(x[:, :4], w, b, L.ACT_SILU, return_state=True)
    other = pool[1::2].clone()
    pool[::2] = last
    for t in range(4, T):
        yt = S.causal_conv_step(x[:, t], pool[::2], w, b, L.ACT_SILU)
        assert torch.equal(yt, whole[:, t]) or float((yt.float() - whole[:, t].float()).abs().max()) <= 2 ** -8 * float(whole.float().abs().max())
        R.close(yt, *(v[:, t] for v in R.conv(x, w, b, True, None, None)["y"]), 2 * K + 24, "step")
    if K > 1:
        assert torch.equal(pool[::2], torch.cat([torch.zeros(B, K - 1, C, device=DEV, dtype=dt), x], 1)[:, -(K - 1):])
        assert torch.equal(pool[1::2], other)


def test_causal_conv_in_two_calls_equals_one_with_gradients_through_the_state():
    g = gen(3)
    B, T, C, K = 3, 29, 24, 4
    x, w, b = (rnd(g, *s).requires_grad_() for s in ((B, T, C), (C, 1, K), (C,)))
    dy = rnd(g, B, T, C)
    one = grads([S.causal_conv(x, w, b, L.ACT_SILU)], [x, w, b], [dy])
    y1, s1 = S.causal_conv(x[:, :13], w, b, L.ACT_SILU, return_state=True)
    y2 = S.causal_conv(x[:, 13:], w, b, L.ACT_SILU, state=s1)
    two = grads([torch.cat([y1, y2], 1)], [x, w, b], [dy])
    ref = R.conv(x, w.squeeze(1), b, True, None, None, dy)
    for t1, t2, name in zip(one, two, ("x", "weight", "bias")):
        R.close(t1.reshape(ref[name][0].shape), *ref[name], 2 * K + 24 + B * T, name)
        R.close(t2.reshape(ref[name][0].shape), *ref[name], 2 * K + 26 + B * T, name)


# ------------------------------------------------------------------------------------------------ selective scan
SCAN = [  # B, T, C, N, G, dtype, z, D, bias, softplus, state, ragged
    (1, 1, 1, 1, 1, F32, True, True, True, True, False, False),
    (2, 16, 64, 16, 1, BF, True, True, True, True, False, False),   # one tile, one block
    (2, 17, 65, 16, 1, BF, True, True, True, True, True, False),    # one more of each
    (6, 50, 130, 5, 2, F32, True, True, True, True, True, True),
    (6, 35, 48, 20, 3, F32, False, True, False, True, True, True),
    (1, 40, 70, 64, 1, BF, True, False, True, True, False, False),
    (6, 100, 33, 8, 1, BF, False, False, True, True, False, True),
    (3, 21, 30, 33, 6, F32, True, True, False, False, True, False),
    (1, 1100, 8, 4, 1, F32, True, True, True, True, True, False),   # as many chunks as there can be
    (2, 200, 200, 11, 2, F32, False, True, True, True, True, False),
    (2, 90, 64, 32, 2, BF, True, True, True, True, True, False),
    (4, 3, 2, 3, 2, F32, True, True, True, True, True, True),
]


def make_scan(case, seed=0):
    B, T, C, N, G, dt, z, D, bias, softplus, state, ragged = case
    g = gen(seed + T * 3 + C + N)
    ln = lens(B, T) if ragged else None
    m = (lambda t: poison(t, ln)) if ragged else (lambda t: t)
    delta = rnd(g, B, T, C, dtype=dt, scale=0.5)
    delta = delta - 1.5 if softplus else delta.abs() * 0.5  # steps of 0.05 to 0.8
    a = dict(u=m(rnd(g, B, T, C, dtype=dt)), delta=m(delta), A=-(torch.rand(C, N, generator=g) * 1.4 + 0.1).to(DEV), Bm=m(rnd(g, B, T, G, N, dtype=dt)),
             Cm=m(rnd(g, B, T, G, N, dtype=dt)), D=rnd(g, C) if D else None, z=m(rnd(g, B, T, C, dtype=dt)) if z else None,
             delta_bias=rnd(g, C, scale=0.2) if bias else None, state=rnd(g, B, C, N, scale=0.5) if state else None)
    return a, ln, m(rnd(g, B, T, C, dtype=dt)), rnd(g, B, C, N)


def k_scan(B, T, C, N, G):
    return 2 * 28 * T + N + C // G + B * T + 60


@pytest.mark.parametrize("case", SCAN, ids=str)
def test_selective_scan_and_its_gradients(case):
    B, T, C, N, G = case[:5]
    softplus = case[9]
    a, ln, dy, dl = make_scan(case)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items() if v is not None}
    y, last = S.selective_scan(**leaves, softplus=softplus, lengths=ln, return_state=True)
    got = dict(zip(leaves, grads([y, last], list(leaves.values()), [dy, dl])))
    ref = R.scan(**a, softplus=softplus, lengths=ln, dy=dy, dlast=dl)
    k = k_scan(B, T, C, N, G)
    for name, t in (("y", y), ("last", last), *got.items()):
        R.close(t, *ref[name], k, name)
    with torch.no_grad():
        y2, last2 = S.selective_scan(**a, softplus=softplus, lengths=ln, return_state=True)
    assert torch.equal(y2, y) and torch.equal(last2, last)


@pytest.mark.parametrize("only", ["y", "last"])
def test_selective_scan_gradients_of_one_output_alone(only):
    case = (2, 37, 20, 6, 1, F32, True, True, True, True, True, False)
    a, ln, dy, dl = make_scan(case)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items()}
    y, last = S.selective_scan(**leaves, return_state=True)
    zy, zl = (dy, torch.zeros_like(dl)) if only == "y" else (torch.zeros_like(dy), dl)
    got = torch.autograd.grad([y if only == "y" else last], list(leaves.values()), [dy if only == "y" else dl], allow_unused=True)
    ref = R.scan(**a, softplus=True, lengths=None, dy=zy, dlast=zl)
    for name, t in zip(leaves, got):
        R.close(t, *ref[name], k_scan(*case[:5]), name)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("N, G, C", [(1, 1, 3), (5, 2, 70), (16, 1, 130), (24, 3, 33), (64, 1, 20)])
def test_selective_scan_step_goes_on_where_the_sequence_ended(dt, N, G, C):
    B, T, T0 = 3, 23, 18
    case = (B, T, C, N, G, dt, True, True, True, True, False, False)
    a, _, _, _ = make_scan(case, seed=5)
    ref = R.scan(**a, softplus=True, lengths=None)
    cut = {k: (v[:, :T0] if v is not None and v.dim() > 2 and k != "state" else v) for k, v in a.items()}
    _, last = S.selective_scan(**cut, return_state=True)
    pool = torch.full((2 * B, C, N), 7.0, device=DEV)
    pool[::2] = last
    for t in range(T0, T):
        row = {k: (v[:, t] if v is not None and v.dim() > 2 else v) for k, v in a.items() if k != "state"}
        y = S.selective_scan_step(**row, state=pool[::2])
        R.close(y, *(v[:, t] for v in ref["y"]), k_scan(B, T, C, N, G), f"row {t}")
    R.close(pool[::2], *ref["last"], k_scan(B, T, C, N, G), "state")
    assert bool((pool[1::2] == 7.0).all())


def test_selective_scan_in_two_calls_equals_one_with_gradients_through_the_state():
    case = (2, 70, 40, 16, 1, F32, True, True, True, True, True, False)
    a, _, dy, dl = make_scan(case)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items()}
    seq = ("u", "delta", "Bm", "Cm", "z")

    def part(s, state):
        return S.selective_scan(**{k: (v[:, s] if k in seq else v) for k, v in leaves.items() if k != "state"}, state=state, return_state=True)

    y1, s1 = part(slice(0, 33), leaves["state"])
    y2, s2 = part(slice(33, None), s1)
    got = grads([torch.cat([y1, y2], 1), s2], list(leaves.values()), [dy, dl])
    ref = R.scan(**a, softplus=True, lengths=None, dy=dy, dlast=dl)
    R.close(torch.cat([y1, y2], 1), *ref["y"], k_scan(*case[:5]), "y")
    for name, t in zip(leaves, got):
        R.close(t, *ref[name], k_scan(*case[:5]), name)


def test_no_decay_and_strong_decay():
    """A = 0 keeps every input for good; step * A = -200 forgets at once (exp underflows to zero); a step of zero leaves the state alone."""
    B, T, C, N = 1, 40, 64, 4
    g = gen(1)
    u, Bm, Cm = rnd(g, B, T, C), rnd(g, B, T, N), rnd(g, B, T, N)
    delta = torch.full((B, T, C), 1.0, device=DEV)
    delta[:, 10:20] = 0.0
    A = torch.zeros(C, N, device=DEV)
    A[:, 1] = -200.0
    A[:, 2] = -1e30
    y, last = S.selective_scan(u, delta, A, Bm, Cm, softplus=False, return_state=True)
    ref = R.scan(u, delta, A, Bm[:, :, None], Cm[:, :, None], None, None, None, False, None, None)
    R.close(y, *ref["y"], k_scan(B, T, C, N, 1), "y")
    R.close(last, *ref["last"], k_scan(B, T, C, N, 1), "last")


def test_softplus_over_its_whole_range():
    """One row of steps from exp(-80) to 200: each within 2^-20 of the value in 64 bits (a handful of roundings), read back through u = B = 1, y
    = C h = step."""
    d = torch.cat([torch.linspace(-80, 30, 4001), torch.tensor([0.0, -0.0, 88.0, 100.0, 200.0])]).to(DEV)
    C = d.numel()
    one = torch.ones(1, 1, C, device=DEV)
    y = S.selective_scan(one, d.view(1, 1, C), torch.zeros(C, 1, device=DEV), torch.ones(1, 1, 1, device=DEV), torch.ones(1, 1, 1, device=DEV))
    want = torch.nn.functional.softplus(d.double(), threshold=1e9)
    assert float(((y.view(-1).double() - want) / want).abs().max()) <= 2.0 ** -20


# ------------------------------------------------------------------------------------------------ block norms
NORM = [  # B, T, C, x type, dtype, layer, post, gate, scale, ab, affine
    (1, 1, 1, F32, F32, False, True, None, False, False, True),
    (2, 3, 8, F32, BF, True, True, "item", True, True, True),
    (3, 5, 130, BF, BF, False, True, "row", True, False, True),
    (2, 7, 256, BF, BF, True, False, "item", False, True, True),
    (5, 3, 257, F32, F32, True, True, "row", True, True, True),
    (2, 4, 512, F32, BF, False, True, "row", True, True, True),
    (1, 9, 1000, F32, F32, False, False, None, True, False, False),
    (3, 2, 1024, BF, BF, True, True, "item", True, True, True),
    (2, 3, 1028, F32, BF, False, True, "row", True, False, True),
    (2, 2, 2049, F32, F32, True, True, "item", True, True, True),
    (1, 3, 4096, F32, BF, False, True, None, True, False, True),
    (1, 2, 4093, BF, BF, True, True, "row", True, True, True),
    (300, 1, 64, BF, BF, False, True, "item", True, True, True),
    (2, 700, 36, F32, F32, False, True, "row", True, False, True),
    (4, 6, 48, F32, BF, False, None, None, False, True, True),     # no branch
    (4, 6, 48, BF, BF, True, None, None, False, False, True),
]


def make_norm(case, seed=0):
    B, T, C, xt, dt, layer, post, gate, scale, ab, affine = case
    g = gen(seed + C + T)
    a = dict(x=rnd(g, B, T, C, dtype=xt, scale=2.0), branch=None if post is None else rnd(g, B, T, C, dtype=dt),
             gate=None if gate is None else rnd(g, B, C) if gate == "item" else rnd(g, B, T, C, dtype=dt),
             weight=1 + rnd(g, C, scale=0.3) if affine else None, bias=rnd(g, C, scale=0.2) if affine and layer else None,
             post_weight=1 + rnd(g, C, scale=0.3) if post and affine else None, post_bias=rnd(g, C, scale=0.2) if post and affine and layer else None,
             scale=rnd(g, C, scale=0.5) if scale else None, ab=rnd(g, B, 2 * C, scale=0.3) if ab else None)
    return a, rnd(g, B, T, C, dtype=xt), rnd(g, B, T, C, dtype=dt)


def ref_norm(case, a, dr, dy):
    return R.norm(a["x"], a["branch"], a["gate"], a["weight"], a["bias"], a["post_weight"], a["post_bias"], a["scale"], a["ab"], bool(case[6]), case[5],
                  1e-5, dr, dy)


def k_norm(B, T, C):
    return 6 * (C // 64 + 12) + 60 + B * T


@pytest.mark.parametrize("want", ["both", "y", "r"])
@pytest.mark.parametrize("case", NORM, ids=str)
def test_block_norm_and_its_gradients(case, want):
    B, T, C, xt, dt, layer, post = case[:7]
    if post is None and want != "y":
        pytest.skip("without a branch r is x")
    a, dr, dy = make_norm(case)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items() if v is not None}
    r, y = S.block_norm(**leaves, post_norm=bool(post), kind="layer" if layer else "rms", eps=1e-5, dtype=dt)
    assert r.dtype == xt and y.dtype == dt
    if post is None:
        assert r is leaves["x"]
    cot = [dr if want != "y" else None, dy if want != "r" else None]
    outs = [(o, c) for o, c in zip((r, y), cot) if c is not None]
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [c for _, c in outs], allow_unused=True)
    ref = ref_norm(case, a, *cot)
    k = k_norm(B, T, C)
    R.close(r, *ref["r"], k, "r")
    R.close(y, *ref["y"], k, "y")
    for name, t in zip(leaves, got):
        R.close(t, *ref[name], k, name)
    with torch.no_grad():
        r2, y2 = S.block_norm(**a, post_norm=bool(post), kind="layer" if layer else "rms", eps=1e-5, dtype=dt)
    assert torch.equal(r2, r) and torch.equal(y2, y)


def test_block_norm_of_zero_rows_and_large_means():
    x = torch.zeros(1, 3, 64, device=DEV)
    x[0, 1] = 5.0                                      # no deviation: the norm is zero
    x[0, 2] = 1000.0 + torch.arange(64, device=DEV)    # a mean of 50 deviations
    _, y = S.block_norm(x, kind="layer", eps=1e-6)
    ref = R.norm(x, None, None, None, None, None, None, None, None, False, True, 1e-6)
    assert bool((y[0, :2] == 0).all())
    R.close(y, *ref["y"], k_norm(1, 3, 64), "y")
    _, y = S.block_norm(torch.zeros(1, 2, 65, device=DEV))
    assert bool((y == 0).all())


# ------------------------------------------------------------------------------------------------ strides, orders, streams, graphs
def test_slices_of_one_projection_are_read_in_place_and_other_orders_are_copied():
    B, T, C, N, K = 3, 21, 40, 6, 4
    g = gen(8)
    for dt in (F32, BF):
        wide = rnd(g, B, T, 2 * C + 3, dtype=dt)            # odd row stride, odd offset: no vector access anywhere
        maps = rnd(g, B, T, 1 + 2 * N, dtype=dt)
        w, A, st = rnd(g, C, K), -rnd(g, C, N).abs() - 0.1, rnd(g, B, C, N)
        x, z, delta = wide[..., 1:C + 1], wide[..., C + 1:2 * C + 1], (wide[..., 2:C + 2] * 0.3 - 1.0)
        Bm, Cm = maps[..., 1:N + 1], maps[..., N + 1:]
        assert torch.equal(S.causal_conv(x, w), S.causal_conv(x.contiguous(), w))
        packed = S.selective_scan(x.contiguous(), delta, A, Bm.contiguous(), Cm.contiguous(), z=z.contiguous(), state=st)
        assert torch.equal(S.selective_scan(x, delta, A, Bm, Cm, z=z, state=st), packed)
        turned = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731  channels not innermost
        assert torch.equal(S.selective_scan(turned(x), turned(delta), A, turned(Bm), turned(Cm), z=turned(z), state=st), packed)
        assert torch.equal(S.causal_conv(turned(x), w), S.causal_conv(x.contiguous(), w))
        one = x[:1].expand(B, T, C)                          # a broadcast batch: read in place, its gradient summed by autograd
        assert torch.equal(S.causal_conv(one, w), S.causal_conv(one.contiguous(), w))
        r, y = S.block_norm(turned(x.contiguous()), turned(z.contiguous()), post_norm=True)
        r2, y2 = S.block_norm(x.contiguous(), z.contiguous(), post_norm=True)
        assert torch.equal(r, r2) and torch.equal(y, y2)


def test_gradients_of_broadcast_inputs():
    B, T, C, N = 4, 19, 24, 5
    g = gen(9)
    u1, d1, b1 = rnd(g, 1, T, C).requires_grad_(), (rnd(g, 1, T, C) - 1).requires_grad_(), rnd(g, 1, T, N).requires_grad_()
    A, Cm, dy = -rnd(g, C, N).abs() - 0.1, rnd(g, B, T, N), rnd(g, B, T, C)
    y = S.selective_scan(u1.expand(B, T, C), d1.expand(B, T, C), A, b1.expand(B, T, N), Cm)
    got = torch.autograd.grad(y, [u1, d1, b1], dy)
    ref = R.scan(u1.expand(B, T, C), d1.expand(B, T, C), A, b1.expand(B, T, N)[:, :, None], Cm[:, :, None], None, None, None, True, None, None, dy)
    for t, name in zip(got, ("u", "delta", "Bm")):
        v, m = (x.sum(0, keepdim=True) for x in ref[name])
        R.close(t, v.reshape(t.shape), m.reshape(t.shape), k_scan(B, T, C, N, 1) + B, name)


def _block(p, x, state=None, step=False):
    """A mixer block as a model runs it: in projection, convolution, scan, out projection, and the norms at its edge."""
    N = p["A"].shape[1]
    C = p["A"].shape[0]
    h = x @ p["w_in"]
    xi, z = h[..., :C], h[..., C:]
    conv = (lambda t: S.causal_conv_step(t, state["conv"], p["conv_w"], p["conv_b"], L.ACT_SILU)) if step else None
    if step:
        xc = conv(xi)
    else:
        xc, conv_state = S.causal_conv(xi, p["conv_w"], p["conv_b"], L.ACT_SILU, return_state=True)
    m = xc @ p["w_x"]
    delta, Bm, Cm = m[..., :C], m[..., C:C + N], m[..., C + N:]
    if step:
        y = S.selective_scan_step(xc, delta, p["A"], Bm, Cm, state["scan"], D=p["D"], z=z, delta_bias=p["dt_b"])
        out = S.block_norm(p["res"][:, None], (y @ p["w_out"])[:, None], weight=p["nw"], post_norm=True, post_weight=p["pw"], scale=p["sc"])
        return out[0][:, 0], out[1][:, 0]
    y, scan_state = S.selective_scan(xc, delta, p["A"], Bm, Cm, D=p["D"], z=z, delta_bias=p["dt_b"], return_state=True)
    r, out = S.block_norm(p["res"], y @ p["w_out"], weight=p["nw"], post_norm=True, post_weight=p["pw"], scale=p["sc"])
    return r, out, {"conv": conv_state, "scan": scan_state}


def make_block(B, T, dim, C, N, K, seed=0):
    g = gen(seed)
    p = dict(w_in=rnd(g, dim, 2 * C, scale=dim ** -0.5), conv_w=rnd(g, C, K, scale=0.5), conv_b=rnd(g, C, scale=0.1), w_x=rnd(g, C, C + 2 * N, scale=C ** -0.5),
             A=-(torch.rand(C, N, generator=g) + 0.1).to(DEV), D=rnd(g, C), dt_b=rnd(g, C, scale=0.1) - 1.0, w_out=rnd(g, C, dim, scale=C ** -0.5),
             nw=1 + rnd(g, dim, scale=0.1), pw=1 + rnd(g, dim, scale=0.1), sc=rnd(g, dim, scale=0.5), res=rnd(g, B, T, dim))
    return p, rnd(g, B, T, dim)


def test_operators_together_prompt_then_token_by_token():
    """A block over a whole sequence equals the same block over a prompt and then row by row with its carried states (float32: the two paths
    differ in the order of a few sums only)."""
    p, x = make_block(3, 30, 48, 80, 16, 4)
    with torch.no_grad():
        r, y, _ = _block(p, x)
        cut = dict(p, res=p["res"][:, :19])
        r0, y0, st = _block(cut, x[:, :19])
        assert float((y0 - y[:, :19]).abs().max()) <= 1e-5 * float(y.abs().max())
        for t in range(19, 30):
            rt, yt = _block(dict(p, res=p["res"][:, t]), x[:, t], st, step=True)
            assert float((yt - y[:, t]).abs().max()) <= 1e-5 * float(y.abs().max())
            assert float((rt - r[:, t]).abs().max()) <= 1e-5 * float(r.abs().max())


def test_operators_together_gradients_against_64_bits():
    """The whole block's gradients, through the library's projections: against the same block in 64 bits on the CPU by autograd through plain
    torch operations.  float32 products over up to 160 terms on both sides of every operator: 2^-24 * (a path of about 1500 roundings) = 1e-4
    of each gradient's norm."""
    p, x = make_block(2, 24, 32, 64, 8, 4, seed=4)
    leaves = [t.requires_grad_() for t in (x, *p.values())]
    r, y, _ = _block(p, x)
    g = gen(11)
    dr, dy = rnd(g, *r.shape), rnd(g, *y.shape)
    got = torch.autograd.grad([r, y], leaves, [dr, dy])
    q = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    xd = x.detach().cpu().double().requires_grad_()
    C, N = q["A"].shape
    K = q["conv_w"].shape[1]
    h = xd @ q["w_in"]
    xi, z = h[..., :C], h[..., C:]
    full = torch.cat([torch.zeros(2, K - 1, C, dtype=torch.double), xi], 1)
    xc = torch.nn.functional.silu((full.unfold(1, K, 1) * q["conv_w"]).sum(-1) + q["conv_b"])
    m = xc @ q["w_x"]
    step = torch.nn.functional.softplus(m[..., :C] + q["dt_b"])
    Bm, Cm = m[..., C:C + N], m[..., C + N:]
    hs, out = torch.zeros(2, C, N, dtype=torch.double), []
    for t in range(24):
        hs = torch.exp(step[:, t, :, None] * q["A"]) * hs + (step[:, t] * xc[:, t])[..., None] * Bm[:, t, None]
        out.append((hs * Cm[:, t, None]).sum(-1) + q["D"] * xc[:, t])
    yv = torch.stack(out, 1) * torch.nn.functional.silu(z)
    rms = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    rd = q["res"] + q["sc"] * (rms(yv @ q["w_out"]) * q["pw"])
    yd = rms(rd) * q["nw"]
    want = torch.autograd.grad([rd, yd], [xd, *q.values()], [dr.cpu().double(), dy.cpu().double()])
    for name, a, b in zip(["x", *p], got, want):
        assert float((a.cpu().double() - b).norm() / b.norm()) <= 1e-4, name


def _all_operators(inp):
    """One pass of everything with gradients, as plain tensors."""
    ca, cdy, sa, sdy, na, ndr, ndy = inp
    xs = {k: v.detach().requires_grad_(True) for k, v in ca.items()}
    y, last = S.causal_conv(xs["x"], xs["weight"], xs["bias"], L.ACT_SILU, xs["state"], return_state=True)
    out = [y, last, *torch.autograd.grad(y, list(xs.values()), cdy)]
    xs = {k: v.detach().requires_grad_(True) for k, v in sa.items()}
    y, last = S.selective_scan(**xs, return_state=True)
    out += [y, last, *torch.autograd.grad(y, list(xs.values()), sdy)]
    xs = {k: v.detach().requires_grad_(True) for k, v in na.items()}
    r, y = S.block_norm(**xs, post_norm=True, kind="layer")
    out += [r, y, *torch.autograd.grad([r, y], list(xs.values()), [ndr, ndy])]
    return [t.detach() for t in out]


def _inputs(seed, dt=BF):
    ca, _, cdy, _ = make_conv((4, 150, 72, 4, dt, True, True, True, False), seed)
    sa, _, sdy, _ = make_scan((2, 150, 100, 16, 2, dt, True, True, True, True, True, False), seed)
    na, ndr, ndy = make_norm((4, 60, 320, F32, dt, True, True, "item", True, True, True), seed)
    return ca, cdy, sa, sdy, na, ndr, ndy


@pytest.mark.parametrize("dt", [F32, BF])
def test_results_are_the_same_bits_from_run_to_run(dt):
    inp = _inputs(0, dt)
    first = _all_operators(inp)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, _all_operators(inp)))


def test_on_another_stream_and_on_two_at_once():
    a, b = _inputs(1), _inputs(2)
    want_a, want_b = _all_operators(a), _all_operators(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            got_a = _all_operators(a)
        with torch.cuda.stream(s2):
            got_b = _all_operators(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want_a, got_a)) and all(torch.equal(x, y) for x, y in zip(want_b, got_b))


def test_two_captured_graphs_with_eager_work_between_the_replays():
    """Forward and backward of every operator recorded into two graphs, replayed several times on new inputs in turn, with eager calls of
    other sizes between: every replay equals the eager result on the same inputs."""
    slots = [_inputs(3), _inputs(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in slots:
            _all_operators(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in slots:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all_operators(s))
        graphs.append(g)

    def flat(inp):
        return [t for part in inp for t in (part.values() if isinstance(part, dict) else [part])]

    for round_ in range(3):
        fresh = [_inputs(10 + 2 * round_), _inputs(11 + 2 * round_)]
        want = [_all_operators(f) for f in fresh]
        for slot, f in zip(slots, fresh):
            for dst, src in zip(flat(slot), flat(f)):
                dst.copy_(src)
        graphs[0].replay()
        graphs[1].replay()
        _all_operators(_inputs(77, F32))
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_steps_in_a_captured_graph():
    B, C, N, K = 5, 96, 16, 4
    g = gen(6)
    w, b, A, D = rnd(g, C, K), rnd(g, C), -rnd(g, C, N).abs() - 0.1, rnd(g, C)
    x, delta, Bm, Cm, z = rnd(g, B, C), rnd(g, B, C) - 1, rnd(g, B, N), rnd(g, B, N), rnd(g, B, C)
    conv, scan = rnd(g, B, K - 1, C), rnd(g, B, C, N)

    def token(cs, ss):
        xc = S.causal_conv_step(x, cs, w, b, L.ACT_SILU)
        y = S.selective_scan_step(xc, delta, A, Bm, Cm, ss, D=D, z=z)
        return S.block_norm(x[:, None], y[:, None], post_norm=True)[1]

    e_conv, e_scan, s_conv, s_scan = conv.clone(), scan.clone(), conv.clone(), scan.clone()
    token(conv.clone(), scan.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token(s_conv, s_scan)
    s_conv.copy_(conv)
    s_scan.copy_(scan)
    for t in range(4):
        x.copy_(rnd(g, B, C))
        want = token(e_conv, e_scan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(s_conv, e_conv) and torch.equal(s_scan, e_scan)


def test_refusals_leave_the_tensors_alone():
    g = gen(2)
    x, w, st = rnd(g, 2, 8), rnd(g, 8, 4), rnd(g, 2, 3, 8)
    before = st.clone()
    with pytest.raises(ValueError):
        S.causal_conv_step(x, st, w[:, :2])
    with pytest.raises(RuntimeError, match="GPU only"):
        S.causal_conv_step(x, st, w.cpu())
    assert torch.equal(st, before)


def test_gradients_are_of_first_order():
    x = torch.randn(1, 5, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, 3, device=DEV, requires_grad=True)
    y = S.causal_conv(x, w)
    gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
def test_more_than_two_to_the_31_elements():
    """The last item of a batch whose activations pass 2^31 elements equals the same item alone, bit for bit."""
    C, T = 1024, 4096
    B = 2 ** 31 // (C * T) + 2
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(B, T, C, device=DEV, dtype=BF)
    x[:-1] = 0.5
    x[-1] = torch.randn(T, C, generator=g, device=DEV).to(BF)
    w = torch.randn(C, 4, generator=g, device=DEV)
    one = x[-1:].clone()
    y = S.causal_conv(x, w, act=L.ACT_SILU)
    assert torch.equal(y[-1:], S.causal_conv(one, w, act=L.ACT_SILU))
    del y
    r, y = S.block_norm(x, x, post_norm=True)
    r1, y1 = S.block_norm(one, one, post_norm=True)
    assert torch.equal(r[-1:], r1) and torch.equal(y[-1:], y1)
    del r, y
    A = -torch.rand(C, 2, generator=g, device=DEV) - 0.1
    m = torch.randn(1, T, 2, generator=g, device=DEV).to(BF)
    y = S.selective_scan(x, x, A, m.expand(B, T, 2), m.expand(B, T, 2), z=x)
    y1 = S.selective_scan(one, one, A, m, m, z=one)
    # one item alone is cut into chunks, the large batch is not: the states differ by float32 roundings, the outputs by a bf16 step at most
    assert float((y[-1:].float() - y1.float()).abs().max()) <= 2 ** -7 * float(y1.float().abs().max())
    assert bool((y[0] == y[1]).all())


# ------------------------------------------------------------------------------------------------ calls that the lists above leave out
SCAN_CHUNKS = [  # as SCAN: many chunks in time, items that end chunks before the last row, every number of states a wave can hold
    (6, 700, 40, 16, 1, F32, True, True, True, True, True, True),
    (6, 333, 72, 12, 2, BF, True, True, True, True, True, True),
    (1, 4500, 12, 4, 1, F32, False, True, True, True, True, False),  # more tiles than chunks
    (2, 300, 70, 64, 1, F32, True, True, True, True, True, True),
    (3, 210, 68, 32, 1, BF, True, True, False, True, True, False),
]


@pytest.mark.parametrize("case", SCAN_CHUNKS, ids=str)
def test_selective_scan_in_many_chunks(case):
    test_selective_scan_and_its_gradients(case)


def test_selective_scan_of_rows_far_apart():
    """Rows further apart than the kernels' offsets reach are copied; so is a single row with a stride that nothing uses."""
    B, T, C, N = 2, 3, 40, 5
    g = gen(31)
    A, Bm, Cm = -rnd(g, C, N).abs() - 0.1, rnd(g, B, T, N), rnd(g, B, T, N)
    far = torch.zeros(B * T, L.SCAN_MAX_STRIDE + 9, device=DEV)
    u = far.view(B, T, -1)[..., 3:C + 3]
    u.copy_(rnd(g, B, T, C))
    leaf = u.detach().requires_grad_()
    packed = u.contiguous().requires_grad_()
    dy = rnd(g, B, T, C)
    y, y2 = (S.selective_scan(t, t, A, Bm, Cm, z=t) for t in (leaf, packed))
    assert torch.equal(y, y2)
    got, want = (torch.autograd.grad(o, t, dy)[0] for o, t in ((y, leaf), (y2, packed)))
    # the three gradients of the one leaf (as u, delta and z) are added up in autograd's order, which the copies change: either order makes two
    # roundings of partial sums that are at most |p1| + |p2| + |p3|, so the two differ by at most 4 * 2^-24 of it (and one rounding of the bound)
    apart = [packed.detach().clone().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(S.selective_scan(apart[0], apart[1], A, Bm, Cm, z=apart[2]), apart, dy)
    assert bool(((got - want).abs() <= 4.01 * 2.0 ** -24 * sum(p.abs() for p in parts)).all())
    one = u[:, :1].as_strided((B, 1, C), (u.stride(0), 1 << 40, 1), u.storage_offset())
    want = S.selective_scan(packed[:, :1].detach(), packed[:, :1].detach(), A, Bm[:, :1], Cm[:, :1])
    assert torch.equal(S.selective_scan(one, one, A, Bm[:, :1], Cm[:, :1]), want)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("value", ["-inf", "lowest"])
def test_rows_masked_through_their_step(dt, value):
    """delta = minus infinity, or the type's lowest value, is a step of zero: the row leaves the states alone and gets no gradient through it
    (the reference gets -1e4, whose exp is zero in 64 bits too)."""
    case = (2, 45, 68, 16, 1, dt, True, True, True, True, True, False)
    a, _, dy, dl = make_scan(case)
    cut = float("-inf") if value == "-inf" else torch.finfo(dt).min
    rows = torch.zeros(45, dtype=torch.bool, device=DEV)
    rows[5:9] = rows[16:33] = True
    leaves = {k: v.detach().clone() for k, v in a.items()}
    leaves["delta"][:, rows] = cut
    a["delta"] = a["delta"].clone()
    a["delta"][:, rows] = -1e4
    for v in leaves.values():
        v.requires_grad_(True)
    y, last = S.selective_scan(**leaves, return_state=True)
    got = dict(zip(leaves, grads([y, last], list(leaves.values()), [dy, dl])))
    ref = R.scan(**a, softplus=True, lengths=None, dy=dy, dlast=dl)
    assert float(got["delta"][:, rows].float().abs().max()) <= 1e-37
    for name, t in (("y", y), ("last", last), *got.items()):
        if name != "delta":
            R.close(t, *ref[name], k_scan(*case[:5]), name)
    with torch.no_grad():
        st = leaves["state"].detach().clone()
        row = {k: (v[:, 5].detach() if v.dim() > 2 else v.detach()) for k, v in leaves.items() if k != "state"}
        S.selective_scan_step(**row, state=st)
        assert torch.equal(st, leaves["state"])


@pytest.mark.parametrize("dt", [F32, BF])
def test_selective_scan_step_reads_slices_in_place(dt):
    """Offsets and strides that leave no vector access, and one that leaves it to the state alone: the same bits as packed tensors."""
    B, C, N, G = 5, 70, 12, 2
    g = gen(41)
    wide, maps = rnd(g, B, 3 * C + 1, dtype=dt), rnd(g, B, 1 + 2 * G * N, dtype=dt)
    u, delta, z = wide[:, 1:C + 1], wide[:, C + 1:2 * C + 1], wide[:, 2 * C + 1:]
    Bm, Cm = maps[:, 1:G * N + 1].unflatten(1, (G, N)), maps[:, G * N + 1:].unflatten(1, (G, N))
    A, D, state = -rnd(g, C, N).abs(), rnd(g, C), rnd(g, B, C, N)
    want_state = state.clone()
    want = S.selective_scan_step(u.contiguous(), delta.contiguous(), A, Bm.contiguous(), Cm.contiguous(), want_state, D=D, z=z.contiguous())
    odd = torch.empty(B * C * N + 1, device=DEV)[1:].view(B, C, N)
    apart = torch.empty(B, C * N + 3, device=DEV)[:, :C * N].unflatten(1, (C, N))
    for st in (state.clone(), odd, apart):
        st.copy_(state)
        assert torch.equal(S.selective_scan_step(u, delta, A, Bm, Cm, st, D=D, z=z), want) and torch.equal(st, want_state)


def test_a_graph_that_saved_a_state_refuses_it_after_a_step():
    g = gen(51)
    x, w, st = rnd(g, 2, 6, 8).requires_grad_(), rnd(g, 8, 4), rnd(g, 2, 3, 8)
    y = S.causal_conv(x, w.requires_grad_(), state=st)
    with torch.no_grad():
        S.causal_conv_step(x[:, 0], st, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    h = rnd(g, 2, 8, 3)
    q = rnd(g, 2, 8, 3).requires_grad_()
    prod = q * h
    with torch.no_grad():
        S.selective_scan_step(x[:, 0], x[:, 1], -w[:, :3].abs(), w[:2, :3].contiguous(), w[2:4, :3].contiguous(), h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        prod.sum().backward()
    with torch.inference_mode():
        h2 = torch.zeros(2, 8, 3, device=DEV)
        S.selective_scan_step(x[:, 0], x[:, 1], -w[:, :3].abs(), w[:2, :3].contiguous(), w[2:4, :3].contiguous(), h2)
        assert bool((h2 != 0).any())


@pytest.mark.parametrize("which", ["conv", "scan", "norm"])
def test_backwards_twice_through_one_graph_and_from_a_broadcast_gradient(which):
    """retain_graph: the same bits again (nothing that a backward pass reads is written by it); a gradient without memory of its own (of a sum)
    is that of ones."""
    g = gen(61)
    if which == "conv":
        leaves = [rnd(g, 2, 9, 12), rnd(g, 12, 3), rnd(g, 12)]
        run = lambda x, w, b: S.causal_conv(x, w, b, L.ACT_SILU)  # noqa: E731
    elif which == "scan":
        leaves = [rnd(g, 2, 40, 12), rnd(g, 2, 40, 12) - 1, -rnd(g, 12, 5).abs(), rnd(g, 2, 40, 5), rnd(g, 2, 40, 5)]
        run = S.selective_scan
    else:
        leaves = [rnd(g, 2, 9, 12), rnd(g, 2, 9, 12), rnd(g, 12)]
        run = lambda x, b, w: S.block_norm(x, b, weight=w, post_norm=True)[1]  # noqa: E731
    leaves = [t.requires_grad_() for t in leaves]
    y = run(*leaves)
    first = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
    again = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
    y.sum().backward()
    for a, b, t in zip(first, again, leaves):
        assert torch.equal(a, b) and torch.equal(a, t.grad)
