"""CPU: calls of the sequence operators that have to be refused by name, before anything touches a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from gan_amd import sequence as S

ARGS = {
    "causal_conv": lambda: dict(x=torch.randn(2, 5, 8), weight=torch.randn(8, 4), bias=torch.randn(8), state=torch.randn(2, 3, 8)),
    "causal_conv_step": lambda: dict(x=torch.randn(2, 8), state=torch.randn(2, 3, 8), weight=torch.randn(8, 4), bias=torch.randn(8)),
    "selective_scan": lambda: dict(u=torch.randn(2, 5, 8), delta=torch.randn(2, 5, 8), A=-torch.rand(8, 6), Bm=torch.randn(2, 5, 6), Cm=torch.randn(2, 5, 6),
                                   D=torch.randn(8), z=torch.randn(2, 5, 8), delta_bias=torch.randn(8), state=torch.randn(2, 8, 6)),
    "selective_scan_step": lambda: dict(u=torch.randn(2, 8), delta=torch.randn(2, 8), A=-torch.rand(8, 6), Bm=torch.randn(2, 6), Cm=torch.randn(2, 6),
                                        state=torch.randn(2, 8, 6), D=torch.randn(8), z=torch.randn(2, 8), delta_bias=torch.randn(8)),
    "block_norm": lambda: dict(x=torch.randn(2, 5, 8), branch=torch.randn(2, 5, 8), weight=torch.randn(8), bias=torch.randn(8), post_norm=True,
                               post_weight=torch.randn(8), post_bias=torch.randn(8), gate=torch.randn(2, 5, 8), scale=torch.randn(8), ab=torch.randn(2, 16)),
}
TENSORS = [(op, k) for op, make in ARGS.items() for k, v in make().items() if torch.is_tensor(v)]


@pytest.mark.parametrize("grad", [True, False], ids=["", "no_grad"])
@pytest.mark.parametrize("op, which", TENSORS)
def test_forward_mode_derivatives_are_refused(op, which, grad):
    """A dual tensor does not ask for gradients; its tangent would be lost in silence."""
    a = ARGS[op]()
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        a[which] = fwd.make_dual(a[which], torch.randn_like(a[which]))
        with pytest.raises(NotImplementedError, match=f"{op}.*forward-mode"):
            getattr(S, op)(**a)


@pytest.mark.parametrize("op", ARGS)
def test_tensors_without_a_tangent_pass_inside_a_dual_level(op):
    with fwd.dual_level(), pytest.raises(RuntimeError, match="GPU only"):
        getattr(S, op)(**ARGS[op]())


def test_causal_conv_step_without_a_state():
    a = ARGS["causal_conv_step"]()
    with pytest.raises(ValueError, match="state"):
        S.causal_conv_step(**dict(a, state=None))
    with pytest.raises(ValueError, match="state"):
        S.causal_conv_step(a["x"], None, a["weight"][:, :1])


@pytest.mark.parametrize("eps", [1e39, 3.5e38, torch.finfo(torch.float32).max * 1.0000001, 1e300])
def test_block_norm_refuses_an_eps_beyond_float32(eps):
    with pytest.raises(ValueError, match="eps"):
        S.block_norm(torch.randn(2, 5, 8), eps=eps)


def test_block_norm_takes_the_largest_eps():
    assert len(S._pack_norm(*[0] * 18, torch.finfo(torch.float32).max)) > 0
    with pytest.raises(RuntimeError, match="GPU only"):
        S.block_norm(torch.randn(2, 5, 8), eps=torch.finfo(torch.float32).max)


def test_c_entry_refuses_a_misaligned_workspace():
    """The block norms' column sums leave in 16-byte pieces."""
    import ctypes as C

    from gan_amd import _lib as L
    one = 1 << 20  # a non-null address that no refusal reads
    p = L.BlockNormBwdParams(x=one, stats=one, dy=one, dx=one, B=1, T=1, C=8)
    for off in (4, 8, 12):
        p.ws = one + off
        assert L.lib().ga_block_norm_bwd(C.byref(p), 0, 0, None) == 3


@pytest.mark.parametrize("entry, cls, sizes, absent", [
    ("ga_causal_conv_fwd", "CausalConvParams", dict(B=1 << 30, T=1, C=64, K=2), ()),
    ("ga_causal_conv_bwd", "CausalConvBwdParams", dict(B=1, T=1, C=1 << 30, K=2), ()),
    ("ga_causal_conv_step", "CausalConvStepParams", dict(B=1 << 16, C=1 << 16, K=2), ()),
    ("ga_scan_fwd", "ScanParams", dict(B=1 << 24, T=1, C=1, N=1, G=1), ()),
    ("ga_scan_bwd", "ScanBwdParams", dict(B=1 << 24, T=1, C=1, N=1, G=1), ()),
    ("ga_scan_bwd", "ScanBwdParams", dict(B=1, T=1, C=(1 << 22) - 1, N=64, G=1), ()),
    ("ga_scan_step", "ScanStepParams", dict(B=1 << 24, C=1, N=1, G=1), ()),
    ("ga_block_norm_fwd", "BlockNormParams", dict(B=1 << 24, T=1, C=8, eps=1e-5), ("branch", "gate")),
    ("ga_block_norm_bwd", "BlockNormBwdParams", dict(B=1 << 24, T=1, C=8), ("branch", "gate")),
    ("ga_block_norm_bwd", "BlockNormBwdParams", dict(B=1 << 24, T=1, C=8), ("ab",)),
])
def test_c_entries_refuse_more_work_items_than_a_launch_holds(entry, cls, sizes, absent):
    """A launch has at most 2^32 - 1 work-items along an axis: 2^24 - 1 blocks of 256.  Every buffer is there, nothing but the sizes is wrong."""
    import ctypes as C

    from gan_amd import _lib as L
    p = getattr(L, cls)()
    for name, kind in p._fields_:
        if kind is C.c_void_p and name not in absent:
            setattr(p, name, 1 << 20)  # a non-null address that no refusal reads
    for k, v in sizes.items():
        setattr(p, k, v)
    args = (0, 0, None) if "norm" in entry else (0, None)
    assert getattr(L.lib(), entry)(C.byref(p), *args) == 1
