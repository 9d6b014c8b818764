"""Linear-time sequence operators on channels-last activations [B, T, C]: a short causal convolution, a selective state space scan (each for
whole sequences, with gradients, and for single tokens, with its state carried in place) and the norms at a residual block's two edges.

    y, window = causal_conv(x, weight, bias, act=ACT_SILU, return_state=True)          ga_causal_conv_fwd / _bwd
    y = causal_conv_step(x_t, window, weight, bias, act=ACT_SILU)                      ga_causal_conv_step
    y, state = selective_scan(u, delta, A, Bm, Cm, D=D, z=z, return_state=True)        ga_scan_fwd / _bwd
    y = selective_scan_step(u_t, delta_t, A, Bm_t, Cm_t, state, D=D, z=z_t)            ga_scan_step
    r, y = block_norm(x, branch, weight=w, post_norm=True, gate=gate, scale=scale)     ga_block_norm_fwd / _bwd

They take what a model around this package's convolutions, LSTM and GroupNorm layers has in hand: activations in float32 or bfloat16 (all of one
call in the same type), parameters, recurrent states and per-item conditions in float32.  All arithmetic, every sum and the states are float32;
what is returned in bfloat16 is rounded once.  An activation may be a channel slice of a wider projection (unit stride along the channels);
anything else that is not packed is copied.  Calls enqueue on the current stream of the tensors' device and keep nothing between calls, so they
may be captured into graphs and run on several streams at once; results do not depend on timing (no atomics).  Gradients are of first order and in
reverse mode (a tensor with a forward-mode tangent is refused, NotImplementedError); a backward pass is captured with torch.autograd.grad, or
with leaves of which no eager graph is alive (a leaf's accumulation belongs to the stream that first used it).  Under softplus delta = -inf
(or the type's lowest value) is a step of zero: the row leaves the states as they are.
Sizes and types are checked here (ValueError / TypeError); like every operator of this package these run on the GPU only.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

Tensor = torch.Tensor
FLOAT_MAX = torch.finfo(torch.float32).max
_pack_conv, _pack_conv_bwd, _pack_conv_step = (L.packer(c) for c in (L.CausalConvParams, L.CausalConvBwdParams, L.CausalConvStepParams))
_pack_scan, _pack_scan_bwd, _pack_scan_step = (L.packer(c) for c in (L.ScanParams, L.ScanBwdParams, L.ScanStepParams))
_pack_norm, _pack_norm_bwd = L.packer(L.BlockNormParams), L.packer(L.BlockNormBwdParams)


# ------------------------------------------------------------------------------------------------ checks and launching
def _act(name: str, t: Optional[Tensor], shape, dtype=None) -> None:
    if t is None:
        return
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")


def _vec(name: str, t: Optional[Tensor], *shape) -> None:
    _act(name, t, shape, torch.float32)


def _lengths(t: Optional[Tensor], B: int) -> None:
    if t is not None:
        _act("lengths", t, (B,), torch.int32)


def _one_device(first: Tensor, *ts) -> None:
    index = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            L.require_cuda(first, t)
            raise RuntimeError(f"all tensors of a call must be on one device: got {first.device} and {t.device}")
    if index < 0:
        L.require_cuda(first)


def _rows(t: Optional[Tensor]) -> Optional[Tensor]:
    """`t` with unit stride along its last axis (itself where it has that already)."""
    return t if t is None or t.stride()[-1] == 1 else t.contiguous()


def _maps(t: Tensor) -> Tensor:
    """[..., G, N] with the last two axes packed."""
    st = t.stride()
    return t if st[-1] == 1 and (t.shape[-2] == 1 or st[-2] == t.shape[-1]) else t.contiguous()


def _packed(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None else t.contiguous()


def _call(name: str, dev: torch.device, *args) -> None:
    """One entry of the C ABI on the current stream of `dev`.  (torch.cuda.current_stream builds a Stream object: 5 us of a call that takes 15.)"""
    fn = getattr(L.lib(), name)
    index = dev.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        L.check(rc, name)


def _wants_grad(*ts) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangents(name: str, *ts) -> None:
    """A dual tensor asks for no gradient: past this check its tangent would be dropped without a word."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} has no forward-mode derivative")


def _no_grad_step(name: str, whole: str, *ts) -> None:
    if _wants_grad(*ts):
        raise RuntimeError(f"{name} updates its state in place and has no gradient: call it under torch.no_grad(), or use {whole}")


def _moved_on(state: Tensor) -> None:
    """A state was written in place: a graph that had saved it refuses to go backwards through the new values."""
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)


def _state_rows(name: str, t: Tensor, inner: int) -> int:
    """The batch stride of a state that a step updates in place: any, as long as its items are packed and apart."""
    if t.is_contiguous():
        return inner
    want, n = [], 1
    for s in reversed(t.shape[1:]):
        want.append(n)
        n *= s
    got = [st for st, s in zip(reversed(t.stride()[1:]), reversed(t.shape[1:])) if s > 1]
    if got != [w for w, s in zip(want, reversed(t.shape[1:])) if s > 1] or (t.shape[0] > 1 and t.stride(0) < inner):
        raise ValueError(f"{name}: items must be packed and must not overlap (strides {tuple(t.stride())})")
    return t.stride(0) if t.shape[0] > 1 else inner


# ------------------------------------------------------------------------------------------------ short causal convolution
def _conv_fwd(x, weight, bias, act, state, lengths, want_last):
    B, T, Cn = x.shape
    K = weight.shape[1]
    y = x.new_empty(B, T, Cn)
    last = x.new_empty(B, K - 1, Cn) if want_last else None
    p = _pack_conv(x.data_ptr(), weight.data_ptr(), L.ptr(bias), L.ptr(state) if K > 1 else 0, L.ptr(lengths), y.data_ptr(),
                   L.ptr(last) if K > 1 else 0, x.stride(0), x.stride(1), B, T, Cn, K, act)
    _call("ga_causal_conv_fwd", x.device, p, L.dt(x))
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, act, lengths, want_last):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.act = act
        return _conv_fwd(x, weight, bias, act, state, lengths, want_last)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        if dy is None and dlast is None:
            return (None,) * 7
        B, T, Cn = x.shape
        K = weight.shape[1]
        dy = x.new_zeros(B, T, Cn) if dy is None else dy.contiguous()
        dlast = None if dlast is None or K == 1 else dlast.contiguous()
        dx = x.new_empty(B, T, Cn)
        dstate = torch.empty_like(state) if state is not None else None
        dw = weight.new_empty(Cn, K)
        db = weight.new_empty(Cn) if bias is not None else None
        ws = weight.new_empty(L.lib().ga_causal_conv_bwd_ws_elems(B, T, Cn, K))
        p = _pack_conv_bwd(x.data_ptr(), weight.data_ptr(), L.ptr(bias), L.ptr(state) if K > 1 else 0, L.ptr(lengths), dy.data_ptr(),
                           L.ptr(dlast), dx.data_ptr(), L.ptr(dstate) if K > 1 else 0, dw.data_ptr(), L.ptr(db), ws.data_ptr(),
                           x.stride(0), x.stride(1), B, T, Cn, K, ctx.act)
        _call("ga_causal_conv_bwd", x.device, p, L.dt(x))
        return dx, dw, db, dstate, None, None, None


def _conv_weight(weight: Tensor, Cn: int) -> Tensor:
    if weight.dim() == 3 and weight.shape[1] == 1:  # nn.Conv1d(C, C, K, groups=C).weight
        weight = weight.squeeze(1)
    if weight.dim() != 2 or weight.shape[0] != Cn or not 1 <= weight.shape[1] <= L.CCONV_MAX_TAPS:
        raise ValueError(f"weight: expected [C, K] or [C, 1, K] with C = {Cn} and 1 <= K <= {L.CCONV_MAX_TAPS}, got {tuple(weight.shape)}")
    _vec("weight", weight, Cn, weight.shape[1])
    return weight


def _conv_act(act: int) -> None:
    if act not in (L.ACT_NONE, L.ACT_SILU):
        raise ValueError(f"act: ACT_NONE or ACT_SILU expected, got {act}")


def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: int = L.ACT_NONE, state: Optional[Tensor] = None,
                lengths: Optional[Tensor] = None, return_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Depthwise causal convolution along time with at most 8 taps:
        y[b, t, c] = act(bias[c] + sum_k weight[c, k] * x[b, t - (K - 1) + k, c])

    x [B, T, C]; weight [C, K] or [C, 1, K] and bias [C], float32; act ACT_NONE or ACT_SILU.  `state` [B, K - 1, C] in x's type: the rows before
    row 0 (zero without it).  `lengths` (int32 [B], on the device): item b ends at row lengths[b]; values outside 0 .. T count as the nearer
    of the two.  Rows behind an item's end may hold anything, give y = 0 and get no gradient.  With `return_state` also the K - 1 rows
    that end each item: the state of a call that goes on, or of causal_conv_step.  Differentiable in x, weight, bias and state."""
    if x.dim() != 3 or 0 in x.shape:
        raise ValueError(f"x: expected a non-empty [B, T, C], got {tuple(x.shape)}")
    B, T, Cn = x.shape
    L.dt(x)
    weight = _conv_weight(weight, Cn)
    _vec("bias", bias, Cn)
    _conv_act(act)
    _act("state", state, (B, weight.shape[1] - 1, Cn), x.dtype)
    _lengths(lengths, B)
    _no_tangents("causal_conv", x, weight, bias, state)
    _one_device(x, weight, bias, state, lengths)
    x, weight, bias, state, lengths = _rows(x), _packed(weight), _packed(bias), _packed(state), _packed(lengths)
    if _wants_grad(x, weight, bias, state):
        y, last = _CausalConv.apply(x, weight, bias, state, act, lengths, bool(return_state))
    else:
        y, last = _conv_fwd(x, weight, bias, act, state, lengths, bool(return_state))
    return (y, last) if return_state else y


def causal_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: int = L.ACT_NONE) -> Tensor:
    """causal_conv for one more row of every item: x [B, C], state [B, K - 1, C] (moved on by a row IN PLACE; its items may lie apart, as in a
    slice of a larger buffer) -> y [B, C].  No gradient."""
    if x.dim() != 2 or 0 in x.shape:
        raise ValueError(f"x: expected a non-empty [B, C], got {tuple(x.shape)}")
    B, Cn = x.shape
    dt = L.dt(x)
    weight = _conv_weight(weight, Cn)
    K = weight.shape[1]
    _vec("bias", bias, Cn)
    _conv_act(act)
    if state is None:
        raise ValueError("state: a [B, K - 1, C] tensor expected")
    _act("state", state, (B, K - 1, Cn), x.dtype)
    bs = _state_rows("state", state, (K - 1) * Cn) if K > 1 else 0
    _no_tangents("causal_conv_step", x, weight, bias, state)
    _no_grad_step("causal_conv_step", "causal_conv", x, weight, bias, state)
    _one_device(x, weight, bias, state)
    x, weight, bias = _rows(x), _packed(weight), _packed(bias)
    y = x.new_empty(B, Cn)
    p = _pack_conv_step(x.data_ptr(), weight.data_ptr(), L.ptr(bias), state.data_ptr() if K > 1 else 0, y.data_ptr(), x.stride(0), bs, B, Cn,
                        K, act)
    _call("ga_causal_conv_step", x.device, p, dt)
    _moved_on(state)
    return y


# ------------------------------------------------------------------------------------------------ selective scan
@lru_cache(maxsize=256)
def _scan_sizes(B, T, Cn, N, G):
    """(maps, hs, ends, ends_step, dmaps, dparams): elements of ga_scan_buffers, each rounded up to 16 bytes"""
    s = L.ScanBuffers()
    L.check(L.lib().ga_scan_sizes(B, T, Cn, N, G, C.byref(s)), "ga_scan_sizes")
    return tuple((n + 3) & ~3 for n in (s.maps, s.hs, s.ends, s.ends_step, s.dmaps, s.dparams))


def _scan_fwd(u, delta, A, Bm, Cm, D, z, delta_bias, softplus, state, lengths, want_last, want_hs):
    B, T, Cn = u.shape
    G, N = Bm.shape[2:]
    n_maps, n_hs, n_ends, n_step, _, _ = _scan_sizes(B, T, Cn, N, G)
    y = u.new_empty(B, T, Cn)
    last = A.new_empty(B, Cn, N) if want_last else None
    keep = A.new_empty(n_maps + n_hs if want_hs else n_maps + n_ends + n_step)  # maps and hs for the backward pass, or maps and what ends here
    maps = keep.data_ptr()
    hs = maps + 4 * n_maps if want_hs else 0
    ends = 0
    if n_ends:
        tmp = A.new_empty(n_ends + n_step) if want_hs else None
        ends = maps + 4 * n_maps if tmp is None else tmp.data_ptr()
    p = _pack_scan(u.data_ptr(), delta.data_ptr(), L.ptr(z), Bm.data_ptr(), Cm.data_ptr(), A.data_ptr(), L.ptr(D), L.ptr(delta_bias),
                   L.ptr(state), L.ptr(lengths), y.data_ptr(), L.ptr(last), maps, hs, ends, ends + 4 * n_ends, *u.stride()[:2], *delta.stride()[:2],
                   *((0, 0) if z is None else z.stride()[:2]), *Bm.stride()[:2], *Cm.stride()[:2], B, T, Cn, N, G, softplus)
    _call("ga_scan_fwd", u.device, p, L.dt(u))
    return y, last, keep


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, Bm, Cm, D, z, delta_bias, state, softplus, lengths, want_last):
        ctx.set_materialize_grads(False)
        y, last, keep = _scan_fwd(u, delta, A, Bm, Cm, D, z, delta_bias, softplus, state, lengths, want_last, True)
        ctx.save_for_backward(u, delta, A, D, z, delta_bias, lengths, keep)
        ctx.cfg = (*Bm.shape, softplus, state is not None)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        u, delta, A, D, z, delta_bias, lengths, keep = ctx.saved_tensors
        B, T, G, N, softplus, has_state = ctx.cfg
        if dy is None and dlast is None:
            return (None,) * 12
        Cn = u.shape[2]
        dy = u.new_zeros(B, T, Cn) if dy is None else dy.contiguous()
        dlast = _packed(dlast)
        n_maps, _, n_ends, n_step, n_dmaps, n_dparams = _scan_sizes(B, T, Cn, N, G)
        du = u.new_empty(B, T, Cn)
        ddelta = u.new_empty(B, T, Cn)
        dz = u.new_empty(B, T, Cn) if z is not None else None
        dB = u.new_empty(B, T, G, N)
        dC = u.new_empty(B, T, G, N)
        dA = A.new_empty(Cn, N)
        dD = A.new_empty(Cn) if D is not None else None
        dbias = A.new_empty(Cn) if delta_bias is not None else None
        dstate = A.new_empty(B, Cn, N) if has_state else None
        ws = A.new_empty(n_ends + n_step + n_dmaps + n_dparams)
        ends = ws.data_ptr()
        step, maps = ends + 4 * n_ends, keep.data_ptr()
        dmaps = step + 4 * n_step
        p = _pack_scan_bwd(u.data_ptr(), delta.data_ptr(), L.ptr(z), A.data_ptr(), L.ptr(D), L.ptr(delta_bias), L.ptr(lengths), dy.data_ptr(),
                           L.ptr(dlast), maps, maps + 4 * n_maps, du.data_ptr(), ddelta.data_ptr(), L.ptr(dz), dB.data_ptr(), dC.data_ptr(),
                           dA.data_ptr(), L.ptr(dD), L.ptr(dbias), L.ptr(dstate), ends, step, dmaps, dmaps + 4 * n_dmaps, *u.stride()[:2],
                           *delta.stride()[:2], *((0, 0) if z is None else z.stride()[:2]), B, T, Cn, N, G, softplus)
        _call("ga_scan_bwd", u.device, p, L.dt(u))
        return du, ddelta, dA, dB, dC, dD, dz, dbias, dstate, None, None, None


def _scan_maps(name: str, t: Tensor, lead, Cn: int, dtype) -> Tensor:
    if t.dim() == len(lead) + 1:
        t = t.unsqueeze(-2)
    if t.dim() != len(lead) + 2 or t.shape[:-2] != lead:
        raise ValueError(f"{name}: expected {tuple(lead)} + [G, N] (or + [N]), got {tuple(t.shape)}")
    G, N = t.shape[-2:]
    if not 1 <= N <= L.SCAN_MAX_STATES or G < 1 or Cn % G:
        raise ValueError(f"{name}: 1 <= N <= {L.SCAN_MAX_STATES} states and groups that divide the {Cn} channels expected, got G = {G}, N = {N}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    return t


def _scan_rows(t: Optional[Tensor]) -> Optional[Tensor]:
    """_rows, with rows no further apart than the kernels' 32-bit offsets go."""
    if t is None or (t.stride(2) == 1 and t.stride(1) <= L.SCAN_MAX_STRIDE):
        return t
    return t.clone(memory_format=torch.contiguous_format)  # (contiguous() leaves the stride of a single row as it is)


def _scan_checks(u, delta, A, Bm, Cm, D, z, delta_bias, state):
    lead, Cn = u.shape[:-1], u.shape[-1]
    L.dt(u)
    if Cn > L.SCAN_MAX_STRIDE:
        raise ValueError(f"u: at most {L.SCAN_MAX_STRIDE} channels, got {Cn}")
    _act("delta", delta, u.shape, u.dtype)
    _act("z", z, u.shape, u.dtype)
    like = Bm.shape == Cm.shape and Bm.dtype == Cm.dtype
    Bm = _scan_maps("Bm", Bm, lead, Cn, u.dtype)
    Cm = (Cm if Cm.dim() == Bm.dim() else Cm.unsqueeze(-2)) if like else _scan_maps("Cm", Cm, lead, Cn, u.dtype)
    if Bm.shape != Cm.shape:
        raise ValueError(f"Bm and Cm differ in shape: {tuple(Bm.shape)} and {tuple(Cm.shape)}")
    N = Bm.shape[-1]
    _vec("A", A, Cn, N)
    _vec("D", D, Cn)
    _vec("delta_bias", delta_bias, Cn)
    _vec("state", state, lead[0], Cn, N)
    return Bm, Cm


def selective_scan(u: Tensor, delta: Tensor, A: Tensor, Bm: Tensor, Cm: Tensor, D: Optional[Tensor] = None, z: Optional[Tensor] = None,
                   delta_bias: Optional[Tensor] = None, softplus: bool = True, state: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                   return_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """A linear recurrence over N states per channel whose decay and input weights depend on the input:
        step[b, t, c] = softplus(delta[b, t, c] + delta_bias[c])             (the sum itself with softplus=False)
        h[b, t, c, n] = exp(step * A[c, n]) * h[b, t-1, c, n] + step * u[b, t, c] * Bm[b, t, g, n]
        y[b, t, c]    = (sum_n Cm[b, t, g, n] * h[b, t, c, n] + D[c] * u[b, t, c]) * silu(z[b, t, c])

    u, delta, z [B, T, C]; Bm, Cm [B, T, G, N] (or [B, T, N]), channel c reads group g = c // (C / G), N <= 64; A [C, N] (negative for a decay; a
    single row's factor exp(step * A) has to be inside float32, the product over many rows need not), D, delta_bias [C], state [B, C, N] (the
    states before row 0, zero without it): float32.  `lengths` as in causal_conv: rows behind an item's end leave its state alone, give y = 0 and
    get no gradient.  With `return_state` also the states at each item's end, float32 [B, C, N].
    Differentiable in every tensor but `lengths`; for the backward pass C * P / 16 + 2 * G * P floats a row are kept (the state at every 16th row, B
    and C), with P = 8, 16, 32 or 64 for N up to that."""
    if u.dim() != 3 or 0 in u.shape:
        raise ValueError(f"u: expected a non-empty [B, T, C], got {tuple(u.shape)}")
    Bm, Cm = _scan_checks(u, delta, A, Bm, Cm, D, z, delta_bias, state)
    _lengths(lengths, u.shape[0])
    _no_tangents("selective_scan", u, delta, A, Bm, Cm, D, z, delta_bias, state)
    _one_device(u, delta, A, Bm, Cm, D, z, delta_bias, state, lengths)
    u, delta, z, Bm, Cm = _scan_rows(u), _scan_rows(delta), _scan_rows(z), _maps(Bm), _maps(Cm)
    A, D, delta_bias, state, lengths = _packed(A), _packed(D), _packed(delta_bias), _packed(state), _packed(lengths)
    if _wants_grad(u, delta, A, Bm, Cm, D, z, delta_bias, state):
        y, last = _SelectiveScan.apply(u, delta, A, Bm, Cm, D, z, delta_bias, state, int(bool(softplus)), lengths, bool(return_state))
    else:
        y, last, _ = _scan_fwd(u, delta, A, Bm, Cm, D, z, delta_bias, int(bool(softplus)), state, lengths, bool(return_state), False)
    return (y, last) if return_state else y


def selective_scan_step(u: Tensor, delta: Tensor, A: Tensor, Bm: Tensor, Cm: Tensor, state: Tensor, D: Optional[Tensor] = None,
                        z: Optional[Tensor] = None, delta_bias: Optional[Tensor] = None, softplus: bool = True) -> Tensor:
    """selective_scan for one more row of every item: u, delta, z [B, C], Bm, Cm [B, G, N] (or [B, N]); state [B, C, N] float32, updated
    IN PLACE (its items may lie apart, as in a slice of a larger buffer) -> y [B, C].  No gradient."""
    if u.dim() != 2 or 0 in u.shape:
        raise ValueError(f"u: expected a non-empty [B, C], got {tuple(u.shape)}")
    if state is None:
        raise ValueError("state: a [B, C, N] float32 tensor expected")
    Bm, Cm = _scan_checks(u, delta, A, Bm, Cm, D, z, delta_bias, state)
    B, Cn = u.shape
    G, N = Bm.shape[1:]
    bs = _state_rows("state", state, Cn * N)
    _no_tangents("selective_scan_step", u, delta, A, Bm, Cm, D, z, delta_bias, state)
    _no_grad_step("selective_scan_step", "selective_scan", u, delta, A, Bm, Cm, D, z, delta_bias, state)
    _one_device(u, delta, A, Bm, Cm, D, z, delta_bias, state)
    u, delta, z, Bm, Cm, A, D, delta_bias = _rows(u), _rows(delta), _rows(z), _maps(Bm), _maps(Cm), _packed(A), _packed(D), _packed(delta_bias)
    y = u.new_empty(B, Cn)
    p = _pack_scan_step(u.data_ptr(), delta.data_ptr(), L.ptr(z), Bm.data_ptr(), Cm.data_ptr(), A.data_ptr(), L.ptr(D), L.ptr(delta_bias),
                        state.data_ptr(), y.data_ptr(), u.stride(0), delta.stride(0), 0 if z is None else z.stride(0), Bm.stride(0), Cm.stride(0), bs,
                        B, Cn, N, G, int(softplus))
    _call("ga_scan_step", u.device, p, L.dt(u))
    _moved_on(state)
    return y


# ------------------------------------------------------------------------------------------------ norms at a block's edges
def _gate_rows(gate: Optional[Tensor]) -> int:
    return int(gate is not None and gate.dim() == 3)


def _norm_fwd(x, branch, gate, w, b, wp, bp, scale, ab, post, layer, eps, dtype, want_stats):
    B, T, Cn = x.shape
    y = x.new_empty((B, T, Cn), dtype=dtype)
    r = x.new_empty(B, T, Cn) if branch is not None else None
    stats = x.new_empty((B * T, 4), dtype=torch.float32) if want_stats else None
    p = _pack_norm(x.data_ptr(), L.ptr(branch), L.ptr(gate), L.ptr(w), L.ptr(b), L.ptr(wp), L.ptr(bp), L.ptr(scale), L.ptr(ab), L.ptr(r),
                   y.data_ptr(), L.ptr(stats), B, T, Cn, int(post), int(layer), _gate_rows(gate), eps)
    _call("ga_block_norm_fwd", x.device, p, L.dt(x), L.dt(y))
    return r, y, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, w, b, wp, bp, scale, ab, post, layer, eps, dtype):
        ctx.set_materialize_grads(False)
        r, y, stats = _norm_fwd(x, branch, gate, w, b, wp, bp, scale, ab, post, layer, eps, dtype, True)
        ctx.save_for_backward(x, branch, gate, w, b, wp, bp, scale, ab, stats)
        ctx.cfg = (post, layer, dtype)
        return r, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dy):
        x, branch, gate, w, b, wp, bp, scale, ab, stats = ctx.saved_tensors
        post, layer, dtype = ctx.cfg
        if dr is None and dy is None:
            return (None,) * 13
        B, T, Cn = x.shape
        dr, dy = _packed(dr), _packed(dy)
        dx, dbranch, dgate, dw, db, dwp, dbp, dscale, dab = (None if t is None else torch.empty_like(t)  # (all packed)
                                                             for t in (x, branch, gate, w, b, wp, bp, scale, ab))
        rows = _gate_rows(gate)
        by_item = ab is not None or (gate is not None and not rows)
        ws = stats.new_empty(L.lib().ga_block_norm_bwd_ws_elems(B, T, Cn, int(by_item)))
        p = _pack_norm_bwd(x.data_ptr(), L.ptr(branch), L.ptr(gate), L.ptr(w), L.ptr(b), L.ptr(wp), L.ptr(bp), L.ptr(scale), L.ptr(ab),
                           stats.data_ptr(), L.ptr(dr), L.ptr(dy), dx.data_ptr(), L.ptr(dbranch), L.ptr(dgate), L.ptr(dw), L.ptr(db), L.ptr(dwp),
                           L.ptr(dbp), L.ptr(dscale), L.ptr(dab), ws.data_ptr(), B, T, Cn, int(post), int(layer), rows)
        _call("ga_block_norm_bwd", x.device, p, L.dt(x), L.DT_BF16 if dtype == torch.bfloat16 else L.DT_F32)
        return dx, dbranch, dgate, dw, db, dwp, dbp, dscale, dab, None, None, None, None


def block_norm(x: Tensor, branch: Optional[Tensor] = None, *, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               post_norm: bool = False, post_weight: Optional[Tensor] = None, post_bias: Optional[Tensor] = None, gate: Optional[Tensor] = None,
               scale: Optional[Tensor] = None, ab: Optional[Tensor] = None, kind: str = "rms", eps: float = 1e-6,
               dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """What stands between two residual blocks, in one pass: the norm behind a block, its gate and residual scale, the residual sum, and the
    norm in front of the next block with its conditional scale and shift.  Returns (r, y):
        n = norm(branch) * post_weight + post_bias        with post_norm, else the branch itself
        r = x + scale * gate * n
        y = (norm(r) * weight + bias) * (1 + a) + s       ab = (a | s)

    norm(v) = v / sqrt(mean(v^2) + eps) (kind "rms") or (v - mean) / sqrt(var + eps) (kind "layer") over the C <= 4096 channels (|v| up to
    1e18: mean squares are float32).
    x [B, T, C] is the residual stream, float32 or the branch's type, and r has x's type; branch and y are in the activations' type (`dtype` names
    it when there is no branch; x's by default).  weight, bias, post_weight, post_bias, scale: float32 [C] or None (1 or 0).  gate: float32 [B, C]
    (one vector an item) or [B, T, C] in the branch's type.  ab: float32 [B, 2C], as GnFilmAct takes it.  Without a branch (the first block) r is x.
    Differentiable in every tensor."""
    if x.dim() != 3 or 0 in x.shape:
        raise ValueError(f"x: expected a non-empty [B, T, C], got {tuple(x.shape)}")
    B, T, Cn = x.shape
    if Cn > L.BNORM_MAX_C:
        raise ValueError(f"x: at most {L.BNORM_MAX_C} channels, got {Cn}")
    L.dt(x)
    if kind not in ("rms", "layer"):
        raise ValueError(f"kind: 'rms' or 'layer' expected, got {kind!r}")
    if not 1e-30 <= eps <= FLOAT_MAX:
        raise ValueError(f"eps: a positive number that float32 holds expected (1e-30 or more), got {eps}")
    if branch is None:
        if post_norm or post_weight is not None or post_bias is not None or gate is not None or scale is not None:
            raise ValueError("post_norm, post_weight, post_bias, gate and scale belong to a branch")
        dtype = x.dtype if dtype is None else dtype
    else:
        if dtype is not None and dtype != branch.dtype:
            raise TypeError(f"dtype: y has the branch's type {branch.dtype}, got {dtype}")
        dtype = branch.dtype
        _act("branch", branch, x.shape)
        L.dt(branch)
    if dtype not in (torch.float32, torch.bfloat16) or (x.dtype != dtype and x.dtype != torch.float32):
        raise TypeError(f"x must be float32 or of the activations' type ({dtype}), got {x.dtype}")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need post_norm=True")
    for name, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias), ("scale", scale)):
        _vec(name, t, Cn)
    if gate is not None:
        if gate.dim() == 2:
            _vec("gate", gate, B, Cn)
        else:
            _act("gate", gate, (B, T, Cn), dtype)
    _vec("ab", ab, B, 2 * Cn)
    ts = (branch, gate, weight, bias, post_weight, post_bias, scale, ab)
    _no_tangents("block_norm", x, *ts)
    _one_device(x, *ts)
    ts = tuple(_packed(t) for t in ts)
    xc = x.contiguous()
    args = (xc, *ts, bool(post_norm), kind == "layer", float(eps), dtype)
    if _wants_grad(xc, *ts):
        r, y = _BlockNorm.apply(*args)
    else:
        r, y, _ = _norm_fwd(*args, False)
    return (x if branch is None else r), y
