"""GPU: scans whose states grow as well as decay (A > 0, or negative steps under softplus=False)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from gan_amd import sequence as S
from tests import sequence_bounds as SB
from tests.sequence_plan import scan_plan
from tests.test_gpu_sequence import BF, DEV, F32, gen, rnd


def bands(m, cycles):
    """Rows of a decay of 16 m rows, as many that grow, and a decay again, each by exp(+-96 |A|) in all, `cycles` times: (steps, rows with an input,
    rows with a gradient).  What enters dies down to exp(-72) before it grows, and so does what comes back: every state and adjoint is far
    inside float32, the factor of a growing band alone (exp(96) > 3.4e38) is not."""
    n = 16 * m
    at = torch.arange(3 * n * cycles) % (3 * n)
    grow = (at >= n) & (at < 2 * n)
    step = torch.where(grow, -6.0 / m, 6.0 / m)
    return step, at < n // 4, (at < n // 4) | (at >= 2 * n + 3 * n // 4)


GROW = [  # B, C, N, tiles a band, cycles, dtype, chunks: every form of the kernel that joins chunks, one walk without it, both element paths
    (1, 8, 4, 1, 40, F32, 120),
    (1, 5, 64, 1, 14, F32, 42),
    (64, 16, 16, 2, 5, BF, 15),
    (64, 7, 20, 2, 5, F32, 15),
    (128, 12, 8, 2, 2, F32, 6),
    (1030, 4, 16, 1, 1, F32, 1),
]


@pytest.mark.parametrize("quiet", [False, True], ids=["", "zeros first"])
@pytest.mark.parametrize("case", GROW, ids=str)
def test_scan_of_bands_that_grow(case, quiet):
    """Chunks of a sequence are joined by the factor exp(A * sum of steps): where it passes float32's range, a state that is small, or exactly zero,
    still has to come through."""
    B, C, N, m, cycles, dt, chunks = case
    step, fed, read = (t.to(DEV) for t in bands(m, cycles))
    T = step.numel()
    assert scan_plan(B, T, C, N, 1) == (chunks, m if chunks > 1 else T // 16)
    g = gen(B + N)
    if quiet:
        fed, read = fed & (torch.arange(T, device=DEV) >= T // 2), read & (torch.arange(T, device=DEV) < T // 2)
    u, dy = rnd(g, B, T, C, dtype=dt) * fed[:, None], rnd(g, B, T, C, dtype=dt) * read[:, None]
    delta = step[:, None].expand(B, T, C).contiguous().to(dt)
    A = -(1 + 0.02 * torch.rand(C, N, generator=g)).to(DEV)
    Bm, Cm = rnd(g, B, T, 1, N, dtype=dt), rnd(g, B, T, 1, N, dtype=dt)
    a = dict(u=u, delta=delta, A=A, Bm=Bm, Cm=Cm)
    leaves = {k: v.clone().requires_grad_(True) for k, v in a.items()}
    y, last = S.selective_scan(**leaves, softplus=False, return_state=True)
    got = dict(zip(leaves, torch.autograd.grad([y], list(leaves.values()), [dy])))
    ref = SB.scan(**a, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None, tiles=m, dy=dy)
    for name, t in (("y", y), ("last", last), *got.items()):
        SB.close(t, *ref[name], name)


def test_scan_grows_from_zero_only_where_something_enters():
    """A > 0 and nothing but zeros until ten rows before the end: zero until there, whatever the factors of the chunks before."""
    for B in (1, 64):
        T, C, N = 2000, 8, 4
        g = gen(B)
        u = rnd(g, B, T, C)
        u[:, :-10] = 0
        one, Bm, Cm = torch.ones(B, T, C, device=DEV), rnd(g, B, T, 1, N), rnd(g, B, T, 1, N)
        A = (6 + torch.rand(C, N, generator=g)).to(DEV)
        y, last = S.selective_scan(u, one, A, Bm, Cm, softplus=False, return_state=True)
        ref = SB.scan(u, one, A, Bm, Cm, None, None, None, False, None, None, scan_plan(B, T, C, N, 1)[1])
        assert bool((y[:, :-10] == 0).all())
        SB.close(y, *ref["y"], "y")
        SB.close(last, *ref["last"], "last")
