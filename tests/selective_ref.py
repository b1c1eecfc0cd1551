"""Plain float64 forms of the selective state space operators and of the
post-training losses, one token after another; gradients by autograd."""
import torch
import torch.nn.functional as F


def live_tokens(lengths, B, L, device):
    if lengths is None:
        return torch.ones(B, L, dtype=torch.bool, device=device)
    n = lengths.to(torch.int64).clamp(0, L)
    return torch.arange(L, device=device)[None] < n[:, None]


def conv_ref(x, w, b, init, lengths, silu=True):
    B, L, D = x.shape
    K = w.shape[1]
    if init is None:
        init = x.new_zeros(B, K - 1, D)
    n = [L] * B if lengths is None else lengths.clamp(0, L).tolist()
    ys, fin = [], []
    for i in range(B):
        h = torch.cat([init[i], x[i, :n[i]]])
        pre = sum(h[j:j + n[i]] * w[:, j] for j in range(K))
        if b is not None:
            pre = pre + b
        ys.append(F.pad(pre * torch.sigmoid(pre) if silu else pre, (0, 0, 0, L - n[i])))
        fin.append(h[n[i]:])
    return torch.stack(ys), torch.stack(fin)


def scan_ref(u, delta, A, Bm, Cm, D=None, z=None, bias=None, softplus=True, init=None, lengths=None):
    """Bm, Cm: [B, L, G, N]."""
    B, L, ch = u.shape
    live = live_tokens(lengths, B, L, u.device)
    rep = ch // Bm.shape[2]
    raw = delta if bias is None else delta + bias
    dt = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    h = init if init is not None else u.new_zeros(B, ch, A.shape[1])
    ys = []
    for t in range(L):
        on = live[:, t, None]
        d = torch.where(on, dt[:, t], 0.0)
        x = torch.where(on, d * u[:, t], 0.0)
        Bt = torch.where(on[..., None], Bm[:, t].repeat_interleave(rep, 1), 0.0)
        h = torch.exp(d[..., None] * A) * h + x[..., None] * Bt
        y = (h * torch.where(on[..., None], Cm[:, t].repeat_interleave(rep, 1), 0.0)).sum(-1)
        if D is not None:
            y = y + D * u[:, t]
        if z is not None:
            y = y * z[:, t] * torch.sigmoid(z[:, t])
        ys.append(torch.where(on, y, 0.0))
    out = torch.stack(ys, 1) if L else u.new_zeros(B, 0, ch)
    return out, h


def logprobs_ref(logits, labels, counts):
    x = torch.where(counts[..., None], logits, 0.0)
    lab = torch.where(counts, labels, 0)
    return torch.where(counts, F.log_softmax(x, -1).gather(-1, lab[..., None])[..., 0], 0.0)


def policy_ref(logits, labels, counts, old, adv, ref, lo, hi, kl):
    lp = logprobs_ref(logits, labels, counts)
    r = torch.exp(lp - old)
    a = adv[:, None] if adv.ndim == 1 else adv
    tok = -torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
    if ref is not None:
        d = ref - lp
        tok = tok + kl * (torch.expm1(d) - d)
    return torch.where(counts, tok, 0.0).sum() / max(1, int(counts.sum())), lp


def preference_ref(logits, labels, counts, ref, beta, eps):
    seq = logprobs_ref(logits, labels, counts).sum(-1)
    P = seq.shape[0] // 2
    d = seq - ref
    x = beta * (d[:P] - d[P:])
    return -((1 - eps) * F.logsigmoid(x) + eps * F.logsigmoid(-x)).mean(), seq


# One rounding to the output type: half a unit in the last place of the largest value.
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def scan_tol(dtype, steps):
    """Every step multiplies the state by an exponential good to about 2^-22 and
    adds a product; the errors add up to at most one such unit a step."""
    return ROUND[dtype] + (steps + 64) * 2.0 ** -22


def max_err(got, ref):
    """max|got - ref| / max|ref| (0 for empty tensors)."""
    if ref.numel() == 0:
        return 0.0
    got, ref = got.detach().double(), ref.detach().double()
    assert bool(torch.isfinite(got).all())
    return float((got - ref).abs().max() / ref.abs().max().clamp(min=1e-30))
