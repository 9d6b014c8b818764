"""GPU: block norms at the ends of their documented range of values: rows of 1e18, and rows whose squares are far below the smallest eps."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from gan_amd import sequence as S
from tests import sequence_ref as R
from tests.test_gpu_sequence import BF, F32, gen, rnd


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [64, 340, 341, 1000, 1023, 1024, 2048, 2051, 4096])
def test_block_norm_of_rows_at_the_limit(C, dt, kind):
    """|v| = 1e18 in every column, or 1e18 at the most, forward and backward: the sum of C squares is beyond float32, their mean is not."""
    g = gen(C)
    x = rnd(g, 2, 3, C)
    x[:, 0] = torch.where(x[:, 0] < 0, -1.0, 1.0)
    x = (x / x.abs().amax(-1, keepdim=True) * 0.999e18).to(dt)
    w, b = 1 + rnd(g, C, scale=0.3), rnd(g, C, scale=0.2)
    dy = rnd(g, 2, 3, C, dtype=dt)
    k = 6 * (C // 64 + 12) + 60 + 6  # the row sums (a tree over 64 lanes of C / 64 values), the chain through the norm and its gradients, 6 rows
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    _, y = S.block_norm(leaves[0], weight=leaves[1], bias=leaves[2], kind=kind, eps=1e-5)
    got = torch.autograd.grad(y, leaves, dy)
    ref = R.norm(x, None, None, w, b, None, None, None, None, False, kind == "layer", 1e-5, None, dy)
    R.close(y, *ref["y"], k, "y")
    for t, name in zip(got, ("x", "weight", "bias")):
        R.close(t, *ref[name], k, name)
    # the same rows as a branch, normed before they are added to a small residual stream
    res = rnd(g, 2, 3, C, dtype=dt)
    leaves = [t.clone().requires_grad_(True) for t in (res, x)]
    r, y = S.block_norm(*leaves, post_norm=True, kind=kind, eps=1e-5)
    got = torch.autograd.grad([r, y], leaves, [dy, dy])
    ref = R.norm(res, x, None, None, None, None, None, None, None, True, kind == "layer", 1e-5, dy, dy)
    for t, name in zip((r, y, *got), ("r", "y", "x", "branch")):
        R.close(t, *ref[name], k, name)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("size", [1e-13, 1e-15, 3e-17, 1e-19])
def test_block_norm_of_small_rows_under_the_smallest_eps(size, kind):
    """Squares far above, at, below and far below eps = 1e-30."""
    for C in (8, 67, 1024, 4096):
        x = rnd(gen(C), 2, 3, C, scale=size)
        dy = rnd(gen(C + 1), 2, 3, C)
        leaf = x.clone().requires_grad_(True)
        _, y = S.block_norm(leaf, kind=kind, eps=1e-30)
        got, = torch.autograd.grad(y, leaf, dy)
        ref = R.norm(x, None, None, None, None, None, None, None, None, False, kind == "layer", 1e-30, None, dy)
        k = 6 * (C // 64 + 12) + 60
        R.close(y, *ref["y"], k, "y")
        R.close(got, *ref["x"], k, "x")
