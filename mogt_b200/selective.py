"""Selective state space layer operators: the short causal convolution, the
selective scan, and the single-token forms of both.

    pre_t = bias + sum_j weight[:, j] x_{t-K+1+j},          y_t = silu(pre_t)

    dt_t = softplus(delta_t + delta_bias)
    h_t  = exp(dt_t A) h_{t-1} + dt_t u_t B_t               per channel and state
    y_t  = (C_t h_t + D u_t) silu(z_t)

Unlike the headed gated scan (one decay per head and step) every channel here
has N states with decays of their own, which depend on the input through
delta.  Activations are [batch, time, channels] and may be strided views (a
half of an input projection, a slice of a projection to (delta, B, C)); only
the last dimension has to be dense, anything else is copied.  States are
[batch, K-1, channels] inputs for the convolution and [batch, channels, N]
fp32 for the scan.

``lengths`` (one integer per sequence, on the device, clamped to [0, L]) makes
a batch ragged: what lies behind a sequence's end is not read into the
arithmetic, its outputs and gradients are zero, and the returned state is the
state after the sequence's last token.

The prompt forms are differentiable in every floating tensor, the states
included.  The single-token forms are for generation: they record no gradient
and update the state in place, or into ``new_state``.  What they write counts
as modified in place: a recorded call that still needs it raises in its
backward, and a state that itself requires grad is not written while gradients
are recorded.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _native as N

__all__ = ["causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step"]

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_MAX_STATES = 128


def _cuda(what, *ts):
    """The device of all of ts.  The kernels carry no tangents, so that dual
    tensors are refused as well (their derivative would come out as none)."""
    index = ts[0].get_device()   # -1 on the CPU
    for t in ts:
        if t is not None and (index < 0 or t.get_device() != index):
            if not t.is_cuda or index < 0:
                raise ValueError(f"{what} requires CUDA tensors")
            raise ValueError(f"{what}: all tensors must be on one device")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in ts):
        raise NotImplementedError(f"{what} has no forward-mode derivative")
    return ts[0].device


_MAX_STRIDE = 1 << 27   # the scan's kernels step over a tile's tokens with 32-bit offsets


def _dense_last(t):
    """t itself when its last dimension is dense (and its rows are not absurdly
    far apart), else a contiguous copy."""
    if t is None or ((t.stride(-1) == 1 or t.shape[-1] == 1)
                     and (t.stride(-2) <= _MAX_STRIDE or t.shape[-2] == 1)):
        return t
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


_CODE = {torch.float32: N.F32, torch.bfloat16: N.BF16, torch.float16: N.F16}


def _lengths(lengths, B, what):
    if lengths is None:
        return None
    if lengths.shape != (B,) or lengths.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: lengths must be [B] int64 or int32")
    return lengths if lengths.dtype == torch.int64 and lengths.is_contiguous() else lengths.to(torch.int64).contiguous()


def _f32(t):
    """Dense and in float32; complex values would lose their imaginary part."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    if t.is_complex():
        raise ValueError(f"parameters, states and token values must be real, not {t.dtype}")
    return t.to(torch.float32).contiguous()


def _writable(what, state, new_state):
    if new_state is not state:
        apart = abs(new_state.data_ptr() - state.data_ptr())
        if 0 < apart < state.numel() * state.element_size():
            raise ValueError(f"{what}: state and new_state overlap")
    if new_state.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: the state to write requires grad, and the call records none: "
                         "detach it, or call under torch.no_grad()")


def _written(new_state):
    """The kernels write through a pointer; autograd sees it by the version."""
    if not new_state.is_inference():
        torch.autograd.graph.increment_version(new_state)


def _activation(activation):
    if activation not in ("silu", None):
        raise ValueError("activation must be 'silu' or None")
    return int(activation == "silu")


# --------------------------------------------------------------------------
# causal convolution
# --------------------------------------------------------------------------
def _conv_params(weight, bias, D, what):
    if weight.ndim != 2 or weight.shape[0] != D:
        raise ValueError(f"{what}: weight must be [D, K]")
    if weight.shape[1] not in (2, 3, 4):
        raise ValueError(f"{what}: K must be 2, 3 or 4")
    if weight.dtype not in _DTYPES:
        raise ValueError(f"{what}: weight must be bfloat16, float16 or float32")
    if bias is not None and (bias.shape != (D,) or bias.dtype != weight.dtype):
        raise ValueError(f"{what}: bias must be [D] in weight's dtype")
    return weight.contiguous(), None if bias is None else bias.contiguous()


class _CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, lengths, silu, return_state):
        with N.tag("mogt.causal_conv.forward"):
            y, fin = _conv_fwd(x, weight, bias, initial_state, lengths, silu, return_state)
        ctx.save_for_backward(x, weight, bias, initial_state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return (y, fin) if return_state else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dfinal=None):
        x, weight, bias, init, lengths = ctx.saved_tensors
        B, L, D = x.shape
        K = weight.shape[1]
        dev = x.device
        dy = torch.zeros(B, L, D, dtype=x.dtype, device=dev) if dy is None else _dense_last(dy.to(x.dtype))
        dfinal = None if dfinal is None else dfinal.to(x.dtype).contiguous()
        dx = torch.empty(B, L, D, dtype=x.dtype, device=dev)
        dw = torch.zeros_like(weight) if B * D == 0 else torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias) if B * D else torch.zeros_like(bias)
        dinit = None
        if init is not None and ctx.needs_input_grad[3]:
            dinit = torch.empty(B, K - 1, D, dtype=x.dtype, device=dev)
        nbytes = max(16, N.lib().mogt_causal_conv_bwd_scratch_bytes(B, L, D, K))
        with N.tag("mogt.causal_conv.backward"):
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            N.launch("mogt_causal_conv_bwd", dev, x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _ptr(bias),
                     _ptr(init), _ptr(lengths), dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dfinal), dx.data_ptr(),
                     dw.data_ptr(), _ptr(db), _ptr(dinit), B, L, D, K, ctx.silu, _CODE[x.dtype], _CODE[weight.dtype],
                     scratch.data_ptr(), nbytes)
        return dx, dw, db, dinit, None, None, None


def _conv_fwd(x, weight, bias, init, lengths, silu, return_state):
    B, L, D = x.shape
    K = weight.shape[1]
    dev = x.device
    y = torch.empty(B, L, D, dtype=x.dtype, device=dev)
    fin = torch.empty(B, K - 1, D, dtype=x.dtype, device=dev) if return_state else None
    N.launch("mogt_causal_conv_fwd", dev, x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), _ptr(bias),
             _ptr(init), _ptr(lengths), y.data_ptr(), _ptr(fin), B, L, D, K, silu, _CODE[x.dtype], _CODE[weight.dtype])
    return y, fin


def causal_conv(x, weight, bias=None, *, activation="silu", initial_state=None, lengths=None, return_state=False):
    """Depthwise causal convolution over time with K in {2, 3, 4} taps.

    x: [B, L, D]; weight: [D, K] (the last tap meets the newest input); bias:
    [D].  x_{-1}, x_{-2}, ... are ``initial_state`` [B, K-1, D] (oldest first)
    or zeros.  Returns y [B, L, D] in x's dtype, with ``return_state`` also the
    last K-1 inputs [B, K-1, D], which a later call or causal_conv_step takes."""
    what = "causal_conv"
    if x.ndim != 3 or x.dtype not in _DTYPES:
        raise ValueError(f"{what}: x must be [B, L, D] bfloat16, float16 or float32")
    _cuda(what, x, weight, bias, initial_state, lengths)
    B, L, D = x.shape
    silu = _activation(activation)
    weight, bias = _conv_params(weight, bias, D, what)
    if initial_state is not None:
        if initial_state.shape != (B, weight.shape[1] - 1, D) or initial_state.dtype != x.dtype:
            raise ValueError(f"{what}: initial_state must be [B, K-1, D] in x's dtype")
        initial_state = initial_state.contiguous()
    lengths = _lengths(lengths, B, what)
    x = _dense_last(x)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, initial_state)):
        return _CausalConvFn.apply(x, weight, bias, initial_state, lengths, silu, bool(return_state))
    with N.tag("mogt.causal_conv"):
        y, fin = _conv_fwd(x, weight, bias, initial_state, lengths, silu, return_state)
    return (y, fin) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, activation="silu", new_state=None):
    """One token of causal_conv: x [B, D], state [B, K-1, D] (dense).  Returns
    y [B, D]; the state shifted by x goes into ``new_state`` (default: state;
    another buffer must lie apart from it)."""
    what = "causal_conv_step"
    if x.ndim != 2 or x.dtype not in _DTYPES:
        raise ValueError(f"{what}: x must be [B, D] bfloat16, float16 or float32")
    new_state = state if new_state is None else new_state
    dev = _cuda(what, x, state, new_state, weight, bias)
    B, D = x.shape
    silu = _activation(activation)
    weight, bias = _conv_params(weight, bias, D, what)
    K = weight.shape[1]
    for s in (state, new_state):
        if s.shape != (B, K - 1, D) or s.dtype != x.dtype or not s.is_contiguous():
            raise ValueError(f"{what}: state must be a contiguous [B, K-1, D] in x's dtype")
    _writable(what, state, new_state)
    x = _dense_last(x)
    y = torch.empty(B, D, dtype=x.dtype, device=dev)
    N.launch("mogt_causal_conv_step", dev, x.data_ptr(), x.stride(0), state.data_ptr(), weight.data_ptr(), _ptr(bias),
             y.data_ptr(), new_state.data_ptr(), B, D, K, silu, _CODE[x.dtype], _CODE[weight.dtype])
    _written(new_state)
    return y


# --------------------------------------------------------------------------
# selective scan
# --------------------------------------------------------------------------
def _grouped(t, what, lead):
    """B or C as [..., G, N] with dense states."""
    if t.ndim == len(lead) + 1:
        t = t.unsqueeze(-2)
    if t.ndim != len(lead) + 2 or t.shape[:len(lead)] != lead:
        raise ValueError(f"{what}: B and C must be {list(lead)} + [N] or [G, N]")
    if (t.stride(-1) == 1 or t.shape[-1] == 1) and (t.stride(-3) <= _MAX_STRIDE or t.shape[-3] == 1):
        return t
    return t.contiguous()


def _check_scan(what, u, delta, A, Bm, Cm, D, z, delta_bias):
    """B and C as [..., G, N]; every operand's shape and dtype checked."""
    shape, dtype = u.shape, u.dtype
    lead, ch = shape[:-1], shape[-1]
    if dtype not in _DTYPES:
        raise ValueError(f"{what}: u must be bfloat16, float16 or float32")
    if A.ndim != 2 or A.shape[0] != ch:
        raise ValueError(f"{what}: A must be [D, N]")
    n = A.shape[1]
    if not 1 <= n <= _MAX_STATES:
        raise ValueError(f"{what}: N must be in [1, {_MAX_STATES}]")
    if delta.shape != shape or delta.dtype != dtype:
        raise ValueError(f"{what}: delta must have u's shape and dtype")
    if z is not None and (z.shape != shape or z.dtype != dtype):
        raise ValueError(f"{what}: z must have u's shape and dtype")
    Bm, Cm = _grouped(Bm, what, lead), _grouped(Cm, what, lead)
    if Bm.shape != Cm.shape or Bm.shape[-1] != n:
        raise ValueError(f"{what}: B and C must have one shape, with A's N states")
    if Bm.dtype != dtype or Cm.dtype != dtype:
        raise ValueError(f"{what}: B and C must have u's dtype")
    if Bm.shape[-2] < 1 or ch % Bm.shape[-2]:
        raise ValueError(f"{what}: the number of channels must be a multiple of the number of groups")
    if D is not None and D.shape != (ch,):
        raise ValueError(f"{what}: D must be [D]")
    if delta_bias is not None and delta_bias.shape != (ch,):
        raise ValueError(f"{what}: delta_bias must be [D]")
    return Bm, Cm


def _token_stride(t, dim=1):
    """A token's stride; that of a single token can be anything."""
    return t.stride(dim) if t.shape[dim] > 1 else 0


def _scan_args(u, delta, A, Bm, Cm, D, z, bias, init, lengths, softplus, *rest):
    """mogt_selective_args in the order of its fields; rest: from `out` on."""
    B, L, ch = u.shape
    z_sb, z_sl = (0, 0) if z is None else (z.stride(0), _token_stride(z))
    return N.SelectiveArgs(
        u.data_ptr(), delta.data_ptr(), _ptr(z), Bm.data_ptr(), Cm.data_ptr(),
        u.stride(0), _token_stride(u), delta.stride(0), _token_stride(delta), z_sb, z_sl,
        Bm.stride(0), _token_stride(Bm), Bm.stride(2), Cm.stride(0), _token_stride(Cm), Cm.stride(2),
        A.data_ptr(), _ptr(D), _ptr(bias), _ptr(init), _ptr(lengths),
        B, L, ch, A.shape[1], Bm.shape[2], int(softplus), _CODE[u.dtype], *rest)


def _scan_fwd(u, delta, A, Bm, Cm, D, z, bias, init, lengths, softplus, return_state, save):
    B, L, ch = u.shape
    n = A.shape[1]
    dev = u.device
    lib = N.lib()
    out = u.new_empty((B, L, ch))
    fin = A.new_empty((B, ch, n)) if return_state else None
    saved = A.new_empty(lib.mogt_selective_saved_bytes(B, L, ch, n) // 4) if save else None
    nbytes = lib.mogt_selective_fwd_scratch_bytes(B, L, ch, n, Bm.shape[2])
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    a = _scan_args(u, delta, A, Bm, Cm, D, z, bias, init, lengths, softplus, out.data_ptr(), _ptr(fin), _ptr(saved),
                   None, 0, 0, None, None, None, None, None, None, None, None, None, None, _ptr(scratch), nbytes)
    N.launch("mogt_selective_scan_fwd", dev, ctypes.byref(a))
    return out, fin, saved


class _SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, Bm, Cm, D, z, bias, init, lengths, softplus, return_state):
        f = tuple(_f32(t) for t in (A, D, bias, init))
        with N.tag("mogt.selective_scan.forward"):
            out, fin, saved = _scan_fwd(u, delta, f[0], Bm, Cm, f[1], z, f[2], f[3], lengths, softplus, return_state,
                                        True)
        ctx.save_for_backward(u, delta, A, Bm, Cm, D, z, bias, lengths, saved)
        ctx.softplus = softplus
        ctx.init_dtype = None if init is None else init.dtype
        ctx.set_materialize_grads(False)
        return (out, fin) if return_state else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal=None):
        u, delta, A, Bm, Cm, D, z, bias, lengths, saved = ctx.saved_tensors
        B, L, ch = u.shape
        dev, dt, n, G = u.device, u.dtype, A.shape[1], Bm.shape[2]
        lib = N.lib()
        if B * ch == 0:
            return (torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(A), torch.zeros_like(Bm),
                    torch.zeros_like(Cm), None if D is None else torch.zeros_like(D),
                    None if z is None else torch.zeros_like(u), None if bias is None else torch.zeros_like(bias),
                    None if ctx.init_dtype is None else torch.zeros(B, ch, n, dtype=ctx.init_dtype, device=dev),
                    None, None, None)
        if dout is None:
            dout = torch.zeros(B, L, ch, dtype=dt, device=dev)
        else:
            dout = _dense_last(dout if dout.dtype == dt else dout.to(dt))
        dfinal = _f32(dfinal)
        Af, Df, bf = _f32(A), _f32(D), _f32(bias)
        du, ddelta = u.new_empty((B, L, ch)), u.new_empty((B, L, ch))
        dz = None if z is None else u.new_empty((B, L, ch))
        dB, dC = u.new_empty((B, L, G, n)), u.new_empty((B, L, G, n))
        dA = Af.new_empty((ch, n))
        dD = None if D is None else Af.new_empty(ch)
        dbias = None if bias is None else Af.new_empty(ch)
        dinit = None
        if ctx.init_dtype is not None and ctx.needs_input_grad[8]:
            dinit = Af.new_empty((B, ch, n))
        nbytes = lib.mogt_selective_bwd_scratch_bytes(B, L, ch, n, G)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        a = _scan_args(u, delta, Af, Bm, Cm, Df, z, bf, None, lengths, ctx.softplus, None, None, saved.data_ptr(),
                       dout.data_ptr(), dout.stride(0), _token_stride(dout), _ptr(dfinal), du.data_ptr(),
                       ddelta.data_ptr(), _ptr(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _ptr(dD), _ptr(dbias),
                       _ptr(dinit), scratch.data_ptr(), nbytes)
        with N.tag("mogt.selective_scan.backward"):
            N.launch("mogt_selective_scan_bwd", dev, ctypes.byref(a))
        cast = lambda g, t: g if g is None or t.dtype == torch.float32 else g.to(t.dtype)
        return (du, ddelta, cast(dA, A), dB, dC, cast(dD, D), dz, cast(dbias, bias),
                dinit if dinit is None or ctx.init_dtype == torch.float32 else dinit.to(ctx.init_dtype),
                None, None, None)


def selective_scan(u, delta, A, B, C, *, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
                   lengths=None, return_state=False):
    """The selective scan over a prompt or a training batch.

    u, delta, z: [B, L, D]; A: [D, N] (negative for a decaying state); B, C:
    [B, L, N], or [B, L, G, N] when channels form G equal groups; D,
    delta_bias: [D]; initial_state: [B, D, N].  u, delta, z, B and C share one
    of bfloat16, float16 and float32; the others are used in float32; N <= 128,
    at most 65535 sequences.
    Returns y [B, L, D] in u's dtype, with ``return_state`` also the state
    after the last token, [B, D, N] float32, which a later call or
    selective_scan_step takes."""
    what = "selective_scan"
    if u.ndim != 3:
        raise ValueError(f"{what}: u must be [B, L, D]")
    _cuda(what, u, delta, A, B, C, D, z, delta_bias, initial_state, lengths)
    Bm, Cm = _check_scan(what, u, delta, A, B, C, D, z, delta_bias)
    if initial_state is not None and initial_state.shape != (u.shape[0], u.shape[2], A.shape[1]):
        raise ValueError(f"{what}: initial_state must be [B, D, N]")
    lengths = _lengths(lengths, u.shape[0], what)
    u, delta, z = _dense_last(u), _dense_last(delta), _dense_last(z)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (u, delta, A, Bm, Cm, D, z, delta_bias, initial_state)):
        return _SelectiveScanFn.apply(u, delta, A, Bm, Cm, D, z, delta_bias, initial_state, lengths,
                                      bool(delta_softplus), bool(return_state))
    with N.tag("mogt.selective_scan"):
        out, fin, _ = _scan_fwd(u, delta, _f32(A), Bm, Cm, _f32(D), z, _f32(delta_bias), _f32(initial_state), lengths,
                                delta_softplus, return_state, False)
    return (out, fin) if return_state else out


def selective_scan_step(state, u, delta, A, B, C, *, D=None, z=None, delta_bias=None, delta_softplus=False,
                        new_state=None):
    """One token of selective_scan: state [B, D, N] float32 (dense), u, delta,
    z [B, D], B and C [B, N] or [B, G, N].  Returns y [B, D] in u's dtype; the
    state after the token goes into ``new_state`` (default: state; another
    buffer must lie apart from it)."""
    what = "selective_scan_step"
    if u.ndim != 2:
        raise ValueError(f"{what}: u must be [B, D]")
    new_state = state if new_state is None else new_state
    dev = _cuda(what, u, state, new_state, delta, A, B, C, D, z, delta_bias)
    Bm, Cm = _check_scan(what, u, delta, A, B, C, D, z, delta_bias)
    bs, ch = u.shape
    n = A.shape[1]
    for s in (state, new_state):
        if s.shape != (bs, ch, n) or s.dtype != torch.float32 or not s.is_contiguous():
            raise ValueError(f"{what}: state must be a contiguous [B, D, N] float32")
    _writable(what, state, new_state)
    u, delta, z = _dense_last(u), _dense_last(delta), _dense_last(z)
    A, D, delta_bias = _f32(A), _f32(D), _f32(delta_bias)
    y = torch.empty(bs, ch, dtype=u.dtype, device=dev)
    b_sb, b_sg, _ = Bm.stride()
    c_sb, c_sg, _ = Cm.stride()
    N.launch("mogt_selective_step", dev, state.data_ptr(), new_state.data_ptr(), u.data_ptr(), u.stride(0),
             delta.data_ptr(), delta.stride(0), _ptr(z), 0 if z is None else z.stride(0), Bm.data_ptr(), b_sb, b_sg,
             Cm.data_ptr(), c_sb, c_sg, A.data_ptr(), _ptr(D), _ptr(delta_bias), y.data_ptr(), bs, ch, n, Bm.shape[1],
             int(delta_softplus), _CODE[u.dtype])
    _written(new_state)
    return y
