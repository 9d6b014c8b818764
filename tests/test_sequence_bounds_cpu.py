"""CPU: the scan's error bounds (tests/sequence_bounds.py): the values are the reference's, an honest float32 evaluation is inside, and states or steps
of too few bits are not."""
import pytest
import torch

from tests import sequence_bounds as SB
from tests import sequence_ref as R

BF, F32 = torch.bfloat16, torch.float32


def make(B, T, C, N, G, dt, softplus=True, seed=0):
    g = torch.Generator().manual_seed(seed + T + C + N)
    r = lambda *s, dtype=dt, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype)  # noqa: E731
    delta = r(B, T, C, scale=0.5)
    return dict(u=r(B, T, C), delta=delta - 1.5 if softplus else delta.abs() * 0.5, A=-(torch.rand(C, N, generator=g) * 1.4 + 0.1), Bm=r(B, T, G, N),
                Cm=r(B, T, G, N), D=r(C, dtype=F32), z=r(B, T, C), delta_bias=r(C, dtype=F32, scale=0.2) if softplus else None, state=r(B, C, N, dtype=F32, scale=0.5)), \
        r(B, T, C), r(B, C, N, dtype=F32)


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("ragged", [False, True])
def test_values_are_the_references(softplus, ragged):
    a, dy, dl = make(3, 21, 6, 5, 2, F32, softplus)
    ln = torch.tensor([21, 0, 9], dtype=torch.int32) if ragged else None
    ours = SB.scan(**a, softplus=softplus, lengths=ln, tiles=2, dy=dy, dlast=dl)
    refs = R.scan(**a, softplus=softplus, lengths=ln, dy=dy, dlast=dl)
    assert ours.keys() == refs.keys()
    for k, (v, e) in ours.items():
        assert float((v - refs[k][0]).abs().max()) <= 1e-12 * float(refs[k][1].abs().max()), k
        assert bool((e >= 0).all())


LONG = [(1, 4500, 12, 4, 1), (1, 1100, 8, 4, 1), (2, 700, 16, 16, 1)]


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("size", LONG, ids=str)
def test_float32_is_inside_and_fewer_bits_are_not(size, softplus):
    a, _, _ = make(*size, F32, softplus)
    ref = SB.scan(**a, softplus=softplus, lengths=None, tiles=18)
    y, last = SB.scan_rounded(**a, softplus=softplus, lengths=None)
    SB.close(y, *ref["y"], "y")
    SB.close(last, *ref["last"], "last")
    half = lambda t: t.to(BF).float()  # noqa: E731

    def every(n):
        count = iter(range(10 ** 9))
        return lambda h: half(h) if next(count) % n == n - 1 else h

    for kw in (dict(round_state=half), dict(round_state=every(16)), dict(round_step=half), dict(round_state=lambda t: t.half().float())):
        y, last = SB.scan_rounded(**a, softplus=softplus, lengths=None, **kw)
        with pytest.raises(AssertionError, match="times the tolerance"):
            SB.close(y, *ref["y"], "y")


@pytest.mark.parametrize("size", LONG, ids=str)
def test_bounds_do_not_grow_with_the_length(size):
    a, _, _ = make(*size, F32)
    v, e = SB.scan(**a, softplus=True, lengths=None, tiles=18)["y"]
    rows = e.abs().amax((0, 2)) / v.abs().amax((0, 2))
    assert float(rows.max()) <= 2e-3 and float(rows[-100:].median()) <= 4 * float(rows[100:200].median())


def test_the_long_cases_take_the_turns_they_are_there_for():
    from tests import test_gpu_sequence_turns as turns
    from tests.sequence_plan import conv_bwd_plan, norm_plan, scan_plan
    for case, plan in turns.SCAN:
        assert scan_plan(*case[:5]) == plan, case
    for case in turns.CONV:
        assert conv_bwd_plan(*case[:4])[1] >= 2, case
    for case in turns.NORM:
        assert min(norm_plan(*case[:3], case[9] or case[7] == "item", case[2] % 4 == 0)[1:]) >= 2, case
