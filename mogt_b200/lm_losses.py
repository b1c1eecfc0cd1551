"""Losses of post-training on logits: the log-probabilities of labels, the
clipped policy loss with a KL term, and the paired preference loss.

Next to ``chunked_lm_loss`` (plain cross-entropy from hidden states) these
take logits [B, L, V] in bfloat16, float16 or float32 as a head produces them
(rows of a wider, padded head are fine as a view) and labels [B, L] aligned
with them: ``labels[b, l]`` is scored by ``logits[b, l]``.

A token counts when ``mask`` (bool, default: all) is set and its label is not
negative (-100 by convention).  Rows that do not count are not read, whatever
they hold; their log-probability, loss and gradient are zero, and a batch
without any counting token has loss 0.  A counting label >= V gives NaN (it
is not checked on the host, which would have to wait for the device).

Statistics are fp32, sums over tokens and pairs fp64 in a fixed order, so
results do not vary between runs.  Only the logits receive a gradient.
"""
from __future__ import annotations

import warnings

import torch

from . import _native as N
from .selective import _CODE, _DTYPES, _cuda, _f32, _ptr

__all__ = ["token_logprobs", "policy_loss", "preference_loss"]


def _rows(what, logits, labels, mask):
    if logits.ndim != 3 or logits.dtype not in _DTYPES:
        raise ValueError(f"{what}: logits must be [B, L, V] bfloat16, float16 or float32")
    if logits.shape[2] < 1:
        raise ValueError(f"{what}: the vocabulary is empty")
    if labels.shape != logits.shape[:2] or labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: labels must be [B, L] int64 or int32")
    if mask is not None and (mask.shape != labels.shape or mask.dtype != torch.bool):
        raise ValueError(f"{what}: mask must be [B, L] bool")
    if logits.stride(2) != 1 and logits.shape[2] > 1:
        logits = logits.contiguous()
    if labels.dtype != torch.int64 or not labels.is_contiguous():
        labels = labels.to(torch.int64).contiguous()
    return logits, labels, None if mask is None else mask.contiguous()


def _grad_like(logits):
    """An empty [B, L, V] whose rows start at the same offsets from a 16-byte
    boundary as those of logits (slices of a wider head or of the tokens
    included), so that both are accessed 16 bytes at a time; rows are as close
    together as that allows."""
    B, L, V = logits.shape
    sb, sl, _ = logits.stride()
    e = logits.element_size()
    first = logits.data_ptr() % 16 // e
    row = V + (sl - V) % (16 // e) if L > 1 else V
    batch = L * row + (sb - L * row) % (16 // e) if B > 1 else L * row
    if first == 0 and row == V and batch == L * V:
        return torch.empty(B, L, V, dtype=logits.dtype, device=logits.device)
    room = torch.empty(first + B * batch, dtype=logits.dtype, device=logits.device)
    return room.as_strided((B, L, V), (batch, row, 1), first)


def _logprob_fwd(logits, labels, mask, want_stats):
    B, L, V = logits.shape
    dev = logits.device
    lp = torch.empty(B, L, dtype=torch.float32, device=dev)
    stats = torch.empty(B, L, 2, dtype=torch.float32, device=dev) if want_stats else None
    N.launch("mogt_logprob_fwd", dev, logits.data_ptr(), logits.stride(0), logits.stride(1), labels.data_ptr(),
             _ptr(mask), B, L, V, _CODE[logits.dtype], lp.data_ptr(), _ptr(stats))
    return lp, stats


def _logprob_bwd(logits, labels, mask, stats, coef, coef_div, scale, d=None):
    """stats, coef: addresses of f32 [B, L, 2] and [B * L / coef_div].  d: a
    gradient that is right already if scale is 1; a new one otherwise."""
    B, L, V = logits.shape
    dev = logits.device
    unless_one = d is not None
    d = d if unless_one else _grad_like(logits)
    scale = _f32(scale)
    N.launch("mogt_logprob_bwd", dev, logits.data_ptr(), logits.stride(0), logits.stride(1), labels.data_ptr(),
             _ptr(mask), stats, coef, coef_div, _ptr(scale), unless_one, d.data_ptr(), d.stride(0), d.stride(1), B, L, V,
             _CODE[logits.dtype])
    return d


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, mask):
        lp, stats = _logprob_fwd(logits, labels, mask, True)
        ctx.save_for_backward(logits, labels, mask, stats)
        return lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, labels, mask, stats = ctx.saved_tensors
        g = _f32(g)
        return _logprob_bwd(logits, labels, mask, stats.data_ptr(), g.data_ptr(), 1, None), None, None


def token_logprobs(logits, labels, *, mask=None):
    """log softmax(logits)[label] per token, fp32 [B, L]; 0 where a token does
    not count.  Differentiable in logits."""
    what = "token_logprobs"
    _cuda(what, logits, labels, mask)
    logits, labels, mask = _rows(what, logits, labels, mask)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobsFn.apply(logits, labels, mask)
    return _logprob_fwd(logits, labels, mask, False)[0]


def _policy(logits, labels, mask, old, ref, adv, lo, hi, kl, want_grad):
    """loss, lp, work, dlogits.  work (f32, n = B L) holds the rows' statistics
    [n, 2] (with a gradient), the coefficients [n] and the kernels' scratch."""
    B, L, V = logits.shape
    n = B * L
    dev = logits.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    lp = torch.empty(B, L, dtype=torch.float32, device=dev)
    nbytes = N.lib().mogt_policy_loss_scratch_bytes(B, L)
    off = 2 * n if want_grad else 0
    work = torch.empty(off + n + nbytes // 4, dtype=torch.float32, device=dev)
    d = _grad_like(logits) if want_grad else None
    a_sb, a_sl = (adv.stride(0), 0) if adv.ndim == 1 else adv.stride()
    d_sb, d_sl = (d.stride(0), d.stride(1)) if want_grad else (0, 0)
    at = work.data_ptr()
    N.launch("mogt_policy_loss", dev, logits.data_ptr(), logits.stride(0), logits.stride(1), labels.data_ptr(),
             _ptr(mask), old.data_ptr(), _ptr(ref), adv.data_ptr(), a_sb, a_sl, lo, hi, kl, loss.data_ptr(),
             lp.data_ptr(), at if want_grad else None, at + 4 * off, _ptr(d), d_sb, d_sl, B, L, V,
             _CODE[logits.dtype], at + 4 * (off + n), nbytes)
    return loss, lp, work, d


class _PolicyLossFn(torch.autograd.Function):
    """The forward also writes the gradient for d loss = 1 (the rows are on the
    chip at that moment) and the backward hands it out.  For another incoming
    gradient (a scaled loss) it is formed again from the logits, so that it is
    rounded once, with the scale: an fp16 gradient scaled afterwards would have
    lost what the scale is there to save.  So is that of a second backward
    (retain_graph), since the first one may have been changed by its receiver."""

    @staticmethod
    def forward(ctx, logits, labels, mask, old, ref, adv, lo, hi, kl):
        with N.tag("mogt.policy_loss.forward"):
            loss, lp, work, d = _policy(logits, labels, mask, old, ref, adv, lo, hi, kl, True)
        ctx.save_for_backward(logits, labels, mask, work)
        ctx.grad = d
        ctx.mark_non_differentiable(lp)
        ctx.set_materialize_grads(False)
        return loss, lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _glp):
        if g is None:
            return (None,) * 9
        d, ctx.grad = ctx.grad, None
        logits, labels, mask, work = ctx.saved_tensors
        at = work.data_ptr()
        with N.tag("mogt.policy_loss.backward"):
            d = _logprob_bwd(logits, labels, mask, at, at + 8 * labels.numel(), 1, g, d)
        return d, None, None, None, None, None, None, None, None


def _token_f32(what, name, t, shape):
    if t.shape != shape:
        raise ValueError(f"{what}: {name} must be {list(shape)}")
    return _f32(t.detach() if t.requires_grad else t)


def policy_loss(logits, labels, old_logprobs, advantages, *, ref_logprobs=None, mask=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, return_logprobs=False):
    """Clipped policy loss with a KL term, the mean over the counting tokens of

        -min(r a, clip(r, 1 - clip_low, 1 + clip_high) a) + kl_coef (e^d - d - 1)

    with lp = log softmax(logits)[label], r = exp(lp - old_logprobs),
    d = ref_logprobs - lp and a the advantage.  old_logprobs, ref_logprobs:
    [B, L] (without ref_logprobs there is no KL term, whatever kl_coef is; a
    weight left unused that way is warned of); advantages: [B] or [B, L].
    Returns the loss (fp32 scalar), with ``return_logprobs`` also lp [B, L]."""
    what = "policy_loss"
    _cuda(what, logits, labels, old_logprobs, advantages, ref_logprobs, mask)
    logits, labels, mask = _rows(what, logits, labels, mask)
    shape = labels.shape
    old = _token_f32(what, "old_logprobs", old_logprobs, shape)
    ref = None if ref_logprobs is None else _token_f32(what, "ref_logprobs", ref_logprobs, shape)
    if advantages.shape not in (shape, shape[:1]):
        raise ValueError(f"{what}: advantages must be [B] or [B, L]")
    adv = advantages.detach() if advantages.requires_grad else advantages
    adv = adv if adv.dtype == torch.float32 else _f32(adv)
    if ref_logprobs is None and kl_coef != 0:
        warnings.warn(f"{what}: kl_coef has no effect without ref_logprobs", stacklevel=2)
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"{what}: clip_low and clip_high must not be negative")
    if torch.is_grad_enabled() and logits.requires_grad:
        loss, lp = _PolicyLossFn.apply(logits, labels, mask, old, ref, adv, float(clip_low), float(clip_high),
                                       float(kl_coef))
    else:
        with N.tag("mogt.policy_loss"):
            loss, lp = _policy(logits, labels, mask, old, ref, adv, float(clip_low), float(clip_high), float(kl_coef),
                               False)[:2]
    return (loss, lp) if return_logprobs else loss


def _preference(logits, labels, mask, ref, beta, eps, want_grad):
    """loss, seq, coef, stats."""
    B, L, _ = logits.shape
    dev = logits.device
    lp, stats = _logprob_fwd(logits, labels, mask, want_grad)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    seq = torch.empty(B, dtype=torch.float32, device=dev)
    coef = torch.empty(B, dtype=torch.float32, device=dev)
    N.launch("mogt_preference_pairs_f64" if ref.dtype == torch.float64 else "mogt_preference_pairs", dev,
             lp.data_ptr(), ref.data_ptr(), B // 2, L, beta, eps, loss.data_ptr(), seq.data_ptr(), coef.data_ptr())
    return loss, seq, coef, stats


class _PreferenceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, mask, ref, beta, eps):
        with N.tag("mogt.preference_loss.forward"):
            loss, seq, coef, stats = _preference(logits, labels, mask, ref, beta, eps, True)
        ctx.save_for_backward(logits, labels, mask, stats, coef)
        ctx.mark_non_differentiable(seq)
        ctx.set_materialize_grads(False)
        return loss, seq

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _gseq):
        if g is None:
            return (None,) * 6
        logits, labels, mask, stats, coef = ctx.saved_tensors
        with N.tag("mogt.preference_loss.backward"):
            d = _logprob_bwd(logits, labels, mask, stats.data_ptr(), coef.data_ptr(), max(logits.shape[1], 1), g)
        return d, None, None, None, None, None


def preference_loss(logits, labels, ref_logprobs, *, beta=0.1, label_smoothing=0.0, mask=None, return_logprobs=False):
    """Paired preference loss.  Sequences 0..P-1 of the batch are preferred
    over sequences P..2P-1.  With s the sum of a sequence's counting label
    log-probabilities and ref_logprobs [2P] the reference model's sums (float64
    sums are used as they are, any other type in float32),

        x = beta ((s_p - ref_p) - (s_{P+p} - ref_{P+p}))
        loss = mean_p [-(1 - eps) log sigmoid(x) - eps log sigmoid(-x)]

    (eps = label_smoothing).  Returns the loss (fp32 scalar), with
    ``return_logprobs`` also s [2P]."""
    what = "preference_loss"
    _cuda(what, logits, labels, ref_logprobs, mask)
    logits, labels, mask = _rows(what, logits, labels, mask)
    if logits.shape[0] % 2 or logits.shape[0] == 0:
        raise ValueError(f"{what}: the batch must hold preferred sequences and as many others after them")
    if ref_logprobs.dtype == torch.float64 and ref_logprobs.shape == labels.shape[:1]:
        ref = ref_logprobs.detach().contiguous()
    else:
        ref = _token_f32(what, "ref_logprobs", ref_logprobs, labels.shape[:1])
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"{what}: label_smoothing must lie in [0, 1]")
    if torch.is_grad_enabled() and logits.requires_grad:
        loss, seq = _PreferenceLossFn.apply(logits, labels, mask, ref, float(beta), float(label_smoothing))
    else:
        with N.tag("mogt.preference_loss"):
            loss, seq = _preference(logits, labels, mask, ref, float(beta), float(label_smoothing), False)[:2]
    return (loss, seq) if return_logprobs else loss
