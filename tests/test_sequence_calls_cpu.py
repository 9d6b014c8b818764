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
