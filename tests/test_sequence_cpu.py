"""CPU: the sequence operators' own 64-bit references (tests/sequence_ref.py) against autograd and against differences, and every refusal of
gan_amd/sequence.py -- arguments are checked before anything touches a GPU, and what passes the checks is refused for being on the CPU."""
import ctypes as C

import pytest
import torch

from gan_amd import _lib as L
from gan_amd import sequence as S
from tests import sequence_ref as R

BF, F32 = torch.bfloat16, torch.float32


def rnd(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype)


# ------------------------------------------------------------------------------------------------ the references themselves
def _against_differences(names, inputs, values, grads_of, cot):
    """The formula's gradients against central differences in 64 bits: f(x + h v) - f(x - h v) over 2 h in a random direction v of each input."""
    ref = grads_of(*inputs)
    for i, name in enumerate(names):
        if inputs[i] is None:
            continue
        v = rnd(*inputs[i].shape, seed=i + 77).double()
        h = 1e-5

        def f(sign):
            got = values(*[t + sign * h * v if j == i else t for j, t in enumerate(inputs)])
            return sum((g * c).sum() for g, c in zip(got, cot))

        num = float(f(1.0) - f(-1.0)) / (2 * h)
        ana = float((ref[name][0] * v).sum())
        # third derivatives enter at h^2 = 1e-10, cancellation at 1e-16 / h of the sums' size
        assert abs(num - ana) <= 1e-6 * max(1.0, abs(ana)), (name, num, ana)


@pytest.mark.parametrize("silu", [False, True])
def test_conv_reference_against_differences(silu):
    ln = torch.tensor([5, 0, 7], dtype=torch.int32)
    ins = [rnd(3, 7, 4).double(), rnd(4, 3).double(), rnd(4).double(), rnd(3, 2, 4).double()]
    dy, dl = rnd(3, 7, 4, seed=5).double(), rnd(3, 2, 4, seed=6).double()

    def vals(x, w, b, st):
        o = R.conv(x, w, b, silu, st, ln)
        return o["y"][0], o["last"][0]

    _against_differences(["x", "weight", "bias", "state"], ins, vals, lambda x, w, b, st: R.conv(x, w, b, silu, st, ln, dy, dl), (dy, dl))


@pytest.mark.parametrize("softplus", [False, True])
def test_scan_reference_against_differences(softplus):
    ln = torch.tensor([6, 0, 3], dtype=torch.int32)
    B, T, Cn, G, N = 3, 6, 4, 2, 3
    ins = [rnd(B, T, Cn).double(), rnd(B, T, Cn, seed=1).double().abs(), -rnd(Cn, N).double().abs(), rnd(B, T, G, N, seed=2).double(),
           rnd(B, T, G, N, seed=3).double(), rnd(Cn).double(), rnd(B, T, Cn, seed=4).double(), rnd(Cn, seed=9).double(), rnd(B, Cn, N).double()]
    dy, dl = rnd(B, T, Cn, seed=5).double(), rnd(B, Cn, N, seed=6).double()
    names = ["u", "delta", "A", "Bm", "Cm", "D", "z", "delta_bias", "state"]

    def go(u, dt, A, Bm, Cm, D, z, db, st, *g):
        return R.scan(u, dt, A, Bm, Cm, D, z, db, softplus, st, ln, *g)

    def vals(*a):
        o = go(*a)
        return o["y"][0], o["last"][0]

    _against_differences(names, ins, vals, lambda *a: go(*a, dy, dl), (dy, dl))


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "item", "row"])
def test_norm_reference_against_differences(layer, post, gate):
    B, T, Cn = 2, 3, 8
    ins = [rnd(B, T, Cn).double(), rnd(B, T, Cn, seed=1).double(), {None: None, "item": rnd(B, Cn), "row": rnd(B, T, Cn, seed=8)}[gate], rnd(Cn).double(),
           rnd(Cn, seed=2).double(), rnd(Cn, seed=3).double() if post else None, rnd(Cn, seed=4).double() if post else None, rnd(Cn, seed=5).double(),
           rnd(B, 2 * Cn).double()]
    ins[2] = None if ins[2] is None else ins[2].double()
    names = ["x", "branch", "gate", "weight", "bias", "post_weight", "post_bias", "scale", "ab"]
    dr, dy = rnd(B, T, Cn, seed=6).double(), rnd(B, T, Cn, seed=7).double()

    def vals(*a):
        o = R.norm(*a, post, layer, 1e-5)
        return o["r"][0], o["y"][0]

    _against_differences(names, ins, vals, lambda *a: R.norm(*a, post, layer, 1e-5, dr, dy), (dr, dy))


# ------------------------------------------------------------------------------------------------ refusals
def conv_args(**kw):
    a = dict(x=rnd(2, 5, 8), weight=rnd(8, 4), bias=rnd(8))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, exc, say", [
    (dict(x=rnd(5, 8)), ValueError, "x:"), (dict(x=rnd(2, 0, 8)), ValueError, "x:"), (dict(x=rnd(2, 5, 8).half()), TypeError, "float32 or bfloat16"),
    (dict(weight=rnd(8, 9)), ValueError, "weight"), (dict(weight=rnd(7, 4)), ValueError, "weight"), (dict(weight=rnd(8, 2, 4)), ValueError, "weight"),
    (dict(weight=rnd(8, 4, dtype=BF)), TypeError, "weight"), (dict(bias=rnd(4)), ValueError, "bias"), (dict(bias=rnd(8).double()), TypeError, "bias"),
    (dict(act=L.ACT_TANH), ValueError, "act"), (dict(state=rnd(2, 4, 8)), ValueError, "state"), (dict(state=rnd(2, 3, 8, dtype=BF)), TypeError, "state"),
    (dict(lengths=torch.tensor([1, 2])), TypeError, "lengths"), (dict(lengths=torch.ones(3, dtype=torch.int32)), ValueError, "lengths"),
    ({}, RuntimeError, "GPU only"), (dict(weight=rnd(8, 1, 4)), RuntimeError, "GPU only"),
])
def test_causal_conv_refuses(kw, exc, say):
    with pytest.raises(exc, match=say):
        S.causal_conv(**conv_args(**kw))


@pytest.mark.parametrize("kw, exc, say", [
    (dict(x=rnd(2, 5, 8)), ValueError, "x:"), (dict(state=rnd(2, 2, 8)), ValueError, "state"), (dict(state=rnd(2, 3, 8, dtype=BF)), TypeError, "state"),
    (dict(state=rnd(1, 3, 8).expand(2, 3, 8)), ValueError, "overlap"), (dict(state=rnd(2, 8, 3).transpose(1, 2)), ValueError, "packed"),
    (dict(weight=rnd(8, 4).requires_grad_()), RuntimeError, "no gradient"), ({}, RuntimeError, "GPU only"),
    (dict(state=rnd(4, 3, 8)[::2]), RuntimeError, "GPU only"),
])
def test_causal_conv_step_refuses(kw, exc, say):
    a = dict(x=rnd(2, 8), state=rnd(2, 3, 8), weight=rnd(8, 4))
    a.update(kw)
    with pytest.raises(exc, match=say):
        S.causal_conv_step(**a)


@pytest.mark.parametrize("kw, exc, say", [
    (dict(u=rnd(5, 8)), ValueError, "u:"), (dict(u=rnd(0, 5, 8)), ValueError, "u:"), (dict(delta=rnd(2, 5, 4)), ValueError, "delta"),
    (dict(delta=rnd(2, 5, 8, dtype=BF)), TypeError, "delta"), (dict(z=rnd(2, 5, 8, dtype=BF)), TypeError, "z"), (dict(z=rnd(2, 4, 8)), ValueError, "z"),
    (dict(Bm=rnd(2, 5, 3, 6), Cm=rnd(2, 5, 3, 6)), ValueError, "groups"), (dict(Bm=rnd(2, 5, 65), Cm=rnd(2, 5, 65)), ValueError, "states"),
    (dict(Bm=rnd(2, 5, 2, 6)), ValueError, "differ"), (dict(Bm=rnd(2, 4, 6)), ValueError, "Bm"), (dict(Cm=rnd(2, 5, 6, dtype=BF)), TypeError, "Cm"),
    (dict(A=rnd(8, 5)), ValueError, "A"), (dict(A=rnd(8, 6).double()), TypeError, "A"), (dict(D=rnd(6)), ValueError, "D"),
    (dict(delta_bias=rnd(1)), ValueError, "delta_bias"), (dict(state=rnd(2, 6, 8)), ValueError, "state"), (dict(state=rnd(2, 8, 6, dtype=BF)), TypeError, "state"),
    (dict(lengths=torch.ones(2)), TypeError, "lengths"), ({}, RuntimeError, "GPU only"),
])
def test_selective_scan_refuses(kw, exc, say):
    a = dict(u=rnd(2, 5, 8), delta=rnd(2, 5, 8), A=-rnd(8, 6).abs(), Bm=rnd(2, 5, 6), Cm=rnd(2, 5, 6))
    a.update(kw)
    with pytest.raises(exc, match=say):
        S.selective_scan(**a)


@pytest.mark.parametrize("kw, exc, say", [
    (dict(u=rnd(2, 5, 8)), ValueError, "u:"), (dict(state=None), ValueError, "state"), (dict(state=rnd(2, 8, 6, dtype=BF)), TypeError, "state"),
    (dict(state=rnd(2, 6, 8).transpose(1, 2)), ValueError, "packed"), (dict(state=rnd(1, 8, 6).expand(2, 8, 6)), ValueError, "overlap"),
    (dict(Bm=rnd(2, 5)), ValueError, "differ"), (dict(A=(-rnd(8, 6).abs()).requires_grad_()), RuntimeError, "no gradient"), ({}, RuntimeError, "GPU only"),
    (dict(state=rnd(6, 8, 6)[::3]), RuntimeError, "GPU only"),
])
def test_selective_scan_step_refuses(kw, exc, say):
    a = dict(u=rnd(2, 8), delta=rnd(2, 8), A=-rnd(8, 6).abs(), Bm=rnd(2, 6), Cm=rnd(2, 6), state=rnd(2, 8, 6))
    a.update(kw)
    with pytest.raises(exc, match=say):
        S.selective_scan_step(**a)


@pytest.mark.parametrize("kw, exc, say", [
    (dict(x=rnd(5, 8)), ValueError, "x:"), (dict(x=rnd(2, 5, 4097), branch=rnd(2, 5, 4097)), ValueError, "channels"), (dict(kind="batch"), ValueError, "kind"),
    (dict(eps=0.0), ValueError, "eps"), (dict(branch=rnd(2, 4, 8)), ValueError, "branch"), (dict(branch=rnd(2, 5, 8).half()), TypeError, "float32 or bfloat16"),
    (dict(x=rnd(2, 5, 8, dtype=BF)), TypeError, "x must be"), (dict(dtype=BF), TypeError, "dtype"), (dict(post_weight=rnd(8)), ValueError, "post_norm"),
    (dict(branch=None, gate=rnd(2, 8)), ValueError, "branch"), (dict(branch=None, post_norm=True), ValueError, "branch"),
    (dict(branch=None, scale=rnd(8)), ValueError, "branch"), (dict(branch=None, dtype=torch.float16), TypeError, "x must be"),
    (dict(gate=rnd(2, 5)), ValueError, "gate"), (dict(gate=rnd(2, 8, dtype=BF)), TypeError, "gate"), (dict(gate=rnd(2, 5, 8, dtype=BF)), TypeError, "gate"),
    (dict(weight=rnd(4)), ValueError, "weight"), (dict(scale=rnd(8, dtype=BF)), TypeError, "scale"), (dict(ab=rnd(2, 8)), ValueError, "ab"),
    ({}, RuntimeError, "GPU only"),
])
def test_block_norm_refuses(kw, exc, say):
    a = dict(x=rnd(2, 5, 8), branch=rnd(2, 5, 8))
    a.update(kw)
    with pytest.raises(exc, match=say):
        S.block_norm(**a)


def test_c_entries_refuse_bad_sizes_without_a_launch():
    """The C ABI's own checks: status codes, no exceptions, before anything is enqueued."""
    if not L.LIB_PATH.exists():
        import __graft_entry__
        __graft_entry__.build()
    lib = L.lib()
    s = L.ScanBuffers()
    for bad in [(0, 1, 1, 1, 1), (1, 0, 1, 1, 1), (1, 1, 6, 65, 1), (1, 1, 6, 4, 4), (1, 1, 6, 0, 1)]:
        assert lib.ga_scan_sizes(*bad, C.byref(s)) == 1
    assert lib.ga_scan_sizes(2, 40, 70, 20, 2, C.byref(s)) == 0
    assert s.maps == 2 * 48 * 2 * 2 * 32 and s.hs == 2 * 3 * 32 * 70 and s.dmaps == s.maps  # 35 channels of a group: one block of 64
    assert lib.ga_scan_sizes(2, 40, 70, 20, 2, None) == 1
    one = 1 << 20  # a non-null address that no refusal reads
    for fn, P in (("ga_scan_fwd", L.ScanParams), ("ga_scan_bwd", L.ScanBwdParams), ("ga_scan_step", L.ScanStepParams), ("ga_causal_conv_fwd", L.CausalConvParams),
                  ("ga_causal_conv_bwd", L.CausalConvBwdParams), ("ga_causal_conv_step", L.CausalConvStepParams)):
        assert getattr(lib, fn)(None, 0, None) == 1
        assert getattr(lib, fn)(C.byref(P()), 0, None) == 1
        p = P()
        for f, v in (("B", 1), ("T", 4), ("C", 8), ("N", 4), ("G", 1), ("K", 2)):
            if hasattr(p, f):
                setattr(p, f, v)
        assert getattr(lib, fn)(C.byref(p), 0, None) == 1        # null pointers
        assert getattr(lib, fn)(C.byref(p), 7, None) == 1        # unknown type
    p = L.BlockNormParams(x=one, y=one, B=1, T=1, C=4097, eps=1e-5)
    assert lib.ga_block_norm_fwd(C.byref(p), 0, 0, None) == 1
    p = L.BlockNormParams(x=one, y=one, B=1, T=1, C=8, eps=0.0)
    assert lib.ga_block_norm_fwd(C.byref(p), 0, 0, None) == 1
    p = L.BlockNormParams(x=one, y=one, gate=one, B=1, T=1, C=8, eps=1e-5)
    assert lib.ga_block_norm_fwd(C.byref(p), 0, 0, None) == 1    # a gate without a branch
    p = L.BlockNormParams(x=one, y=one, stats=one + 4, B=1, T=1, C=8, eps=1e-5)
    assert lib.ga_block_norm_fwd(C.byref(p), 0, 0, None) == 3    # misaligned statistics
    assert lib.ga_block_norm_fwd(C.byref(p), 1, 0, None) == 1    # bf16 residual under float32 activations
    assert lib.ga_block_norm_bwd(C.byref(L.BlockNormBwdParams(B=1, T=1, C=8)), 0, 0, None) == 1
    assert lib.ga_causal_conv_bwd_ws_elems(1, 1, 8, 9) == 0 and lib.ga_causal_conv_bwd_ws_elems(2, 40, 8, 4) > 0
    assert lib.ga_block_norm_bwd_ws_elems(1, 1, 9000, 0) == 0 and lib.ga_block_norm_bwd_ws_elems(3, 5, 8, 1) >= (3 + 3) * 4 * 8


@pytest.mark.parametrize("eps", [float("nan"), float("inf"), -1e-6, 1e-46])
def test_block_norm_refuses_an_eps_that_float32_does_not_hold(eps):
    with pytest.raises(ValueError, match="eps"):
        S.block_norm(rnd(2, 5, 8), eps=eps)


def test_selective_scan_refuses_more_channels_than_its_offsets_reach():
    Cn = L.SCAN_MAX_STRIDE + 1
    u = torch.zeros(1).expand(1, 1, Cn)
    with pytest.raises(ValueError, match="channels"):
        S.selective_scan(u, u, torch.zeros(1, 1).expand(Cn, 1), torch.zeros(1, 1, 1), torch.zeros(1, 1, 1))


def test_c_entries_refuse_lengths_at_the_end_of_the_integers():
    lib, s = L.lib(), L.ScanBuffers()
    for T in (2 ** 31 - 1, 2 ** 31 - 16):
        assert lib.ga_scan_sizes(1, T, 1, 1, 1, C.byref(s)) == 1
        assert lib.ga_causal_conv_bwd_ws_elems(1, T, 1, 1) == 0
    assert lib.ga_scan_sizes(2 ** 20, 2 ** 20, 2 ** 16, 1, 1, C.byref(s)) == 0  # 2^20 items of 1024 blocks: 2^30, a grid has up to 2^31 - 1
    assert lib.ga_scan_sizes(2 ** 21, 2 ** 20, 2 ** 16, 1, 1, C.byref(s)) == 1  # 2^31
