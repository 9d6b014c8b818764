"""GPU: sizes at which the sequence operators' loops take several turns, as training sizes do: scans with chunks of several tiles or with one chunk,
convolutions with more runs than blocks, norms with more rows than the blocks hold at once; and scans under bounds that do not grow with their
length.  Each case first checks, from the buffer sizes the C entries report, that it takes the turns it is there for."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from gan_amd import _lib as L
from gan_amd import sequence as S
from tests import sequence_bounds as SB
from tests import sequence_ref as R
from tests.sequence_plan import conv_bwd_plan, norm_plan, scan_plan
from tests.test_gpu_sequence import BF, DEV, F32, gen, grads, make_norm, make_scan, poison, ref_norm, rnd

SCAN = [  # ((B, T, C, N, G, dtype, z, D, bias, softplus, state, ragged), (chunks, tiles a chunk at least))
    ((64, 800, 16, 16, 1, BF, True, True, True, True, True, True), (13, 4)),      # quads, the next tile's rows ahead of the backward walk
    ((64, 800, 13, 16, 1, F32, True, True, True, True, True, True), (13, 4)),     # single channels
    ((64, 700, 20, 5, 1, BF, False, True, True, True, False, False), (15, 3)),    # two states a wave
    ((64, 700, 8, 24, 1, F32, True, True, False, True, True, True), (15, 3)),     # eight states a wave: half of them wait
    ((64, 700, 12, 40, 1, BF, True, False, True, True, True, True), (15, 3)),     # sixteen
    ((1030, 70, 4, 16, 1, BF, True, True, True, True, True, True), (1, 5)),       # one chunk
    ((1030, 70, 3, 8, 1, F32, False, True, True, True, True, True), (1, 5)),
    ((520, 60, 8, 33, 2, BF, True, True, True, True, True, True), (1, 4)),
    ((1030, 50, 4, 32, 1, F32, True, True, True, False, True, False), (1, 4)),
    ((1030, 50, 4, 64, 1, BF, True, True, False, True, True, True), (1, 4)),
    ((1, 4096, 8, 4, 1, F32, True, True, True, True, True, False), (256, 1)),     # as many chunks as there can be
    ((1, 9000, 4, 16, 1, F32, True, True, True, True, True, False), (188, 3)),
    ((1, 4500, 12, 4, 1, F32, False, True, True, True, True, False), (141, 2)),
    ((1, 1100, 8, 4, 1, F32, True, True, True, True, True, False), (69, 1)),
]


def inside(T, B, seed):
    """Lengths of every kind, most of them inside a chunk."""
    n = torch.randint(1, T + 1, (B,), generator=gen(seed))
    for i, v in enumerate((0, 1, T, T - 1, T + 9, -3, 17, 33)):
        n[i * 7 % B] = v
    return n.to(torch.int32).to(DEV)


@pytest.mark.parametrize("case, plan", SCAN, ids=str)
def test_selective_scan_over_many_tiles(case, plan):
    B, T, C, N, G, softplus, ragged = *case[:5], case[9], case[11]
    assert scan_plan(B, T, C, N, G) == plan
    a, _, dy, dl = make_scan((*case[:11], False))
    ln = inside(T, B, C) if ragged else None
    if ragged:
        for k in ("u", "delta", "Bm", "Cm", "z"):
            a[k] = None if a[k] is None else poison(a[k], ln)
        dy = poison(dy, ln)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items() if v is not None}
    y, last = S.selective_scan(**leaves, softplus=softplus, lengths=ln, return_state=True)
    got = dict(zip(leaves, grads([y, last], list(leaves.values()), [dy, dl])))
    ref = SB.scan(**a, softplus=softplus, lengths=ln, tiles=plan[1] + 1, dy=dy, dlast=dl)
    for name, t in (("y", y), ("last", last), *got.items()):
        SB.close(t, *ref[name], name)
    with torch.no_grad():
        y2, last2 = S.selective_scan(**a, softplus=softplus, lengths=ln, return_state=True)
    assert torch.equal(y2, y) and torch.equal(last2, last)


CONV = [  # B, T, C, K, dtype, silu, ragged
    (4, 70001, 65, 3, F32, True, False),   # more runs of 128 rows than blocks along time
    (9, 6, 262148, 4, BF, True, True),     # more channel blocks than 1024: one block along time takes all runs
    (14, 5, 65537, 2, F32, False, True),
]


@pytest.mark.parametrize("case", CONV, ids=str)
def test_causal_conv_with_more_runs_than_blocks(case):
    B, T, C, K, dt, silu, ragged = case
    assert conv_bwd_plan(B, T, C, K)[1] >= 2
    g = gen(C)
    ln = inside(T, B, C) if ragged else None
    cut = (lambda t: poison(t, ln)) if ragged else (lambda t: t)
    x, dy = cut(rnd(g, B, T, C, dtype=dt)), cut(rnd(g, B, T, C, dtype=dt))
    w, b, st, dl = rnd(g, C, K, scale=0.5), rnd(g, C, scale=0.3), rnd(g, B, K - 1, C, dtype=dt), rnd(g, B, K - 1, C, dtype=dt)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, st)]
    y, last = S.causal_conv(leaves[0], leaves[1], leaves[2], L.ACT_SILU if silu else L.ACT_NONE, leaves[3], ln, return_state=True)
    got = grads([y, last], leaves, [dy, dl])
    ref = R.conv(x, w, b, silu, st, ln, dy, dl)
    k = 2 * K + 24
    # a thread adds up its runs' rows (of T, 128 at the most, each), a block four threads; the rest is added in double
    runs, parts = B * -(-T // min(T, 128)), max(1, 1024 // -(-C // 64))
    chain = min(T, 128) * -(-runs // (4 * parts)) + 4
    for name, t in zip(("y", "last", "x", "weight", "bias", "state"), (y, last, *got)):
        R.close(t, *ref[name], k + (chain if name in ("weight", "bias") else 0), name)


NORM = [  # B, T, C, x type, dtype, layer, post, gate, scale, ab, affine
    (1, 40000, 8, F32, BF, False, True, "row", True, False, True),
    (3, 20000, 12, F32, F32, True, True, "item", True, True, True),
    (2, 20000, 7, BF, BF, True, True, "row", True, False, True),
    (1, 17000, 260, BF, BF, False, False, None, True, False, True),
    (2, 3000, 516, F32, BF, True, True, "row", True, False, True),
    (2, 2100, 1028, BF, BF, False, True, "item", True, True, True),
    (1, 2500, 2052, F32, F32, True, True, None, True, False, True),
    (1, 5000, 515, F32, F32, False, True, "row", True, False, True),
    (1, 1500, 1030, BF, BF, True, True, "row", True, False, True),
    (2, 20000, 16, F32, BF, False, None, None, False, True, True),
]


@pytest.mark.parametrize("case", NORM, ids=str)
def test_block_norm_with_more_rows_than_the_blocks_hold(case):
    B, T, C, xt, dt, layer, post = case[:7]
    by_item = case[9] or case[7] == "item"
    rows, fwd, bwd = norm_plan(B, T, C, by_item, C % 4 == 0)
    assert fwd >= 2 and bwd >= 2
    a, dr, dy = make_norm(case)
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in a.items() if v is not None}
    r, y = S.block_norm(**leaves, post_norm=bool(post), kind="layer" if layer else "rms", eps=1e-5, dtype=dt)
    cot = [(r, dr), (y, dy)] if post is not None else [(y, dy)]
    got = torch.autograd.grad([o for o, _ in cot], list(leaves.values()), [c for _, c in cot])
    ref = ref_norm(case, a, dr if post is not None else None, dy)
    k = 6 * (C // 64 + 12) + 60
    # a block adds up its rows in float32: at least 256 blocks in all; the rest is added in double
    chain = -(-rows // max(1, 256 // (B if by_item else 1))) + 16
    summed = {"weight", "bias", "post_weight", "post_bias", "scale", "ab"} | ({"gate"} if case[7] == "item" else set())
    for name, t in (("r", r), ("y", y), *zip(leaves, got)):
        if name != "r" or post is not None:
            R.close(t, *ref[name], k + (chain if name in summed else 0), name)
