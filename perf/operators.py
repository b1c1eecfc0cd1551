"""Operators of the selective state space path and of post-training, as cases.

Five operators, each in a plain form (elementary torch operations in 32 bits)
and through the framework's public entry points:

  conv        short depthwise causal convolution with SiLU (train, prompts)
  scan        selective state space scan (train, prompts)
  step        the single-token forms of both, one after the other
  policy      clipped policy loss with a KL term on logits, and its gradient
  preference  paired preference loss on logits, and its gradient

Sizes: model width 768 (inner width 2 x 768 = 1536), sequences up to 32768,
vocabulary 32000, as in the backbone benchmark and its tests; the odd sizes
are generic.
"""
import math

import torch
import torch.nn.functional as F

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # a training step's convolution: the first half of an input projection of width 2 x 1536
        dict(name="conv_train", op="conv", dtype="bf16", B=4, L=8192, D=1536, K=4, train=True, ragged=False,
             state=False),
        # a ragged batch of prompts that continue earlier ones (history in, history out), odd width
        dict(name="conv_ragged", op="conv", dtype="fp32", B=7, L=1021, D=770, K=3, train=False, ragged=True,
             state=True),
        # one long prompt: the states a generation starts from
        dict(name="scan_prefill_long", op="scan", dtype="bf16", B=1, L=32768, D=1536, N=16, G=1, train=False,
             ragged=False, state=True, gate=True),
        # an ordinary training batch
        dict(name="scan_train", op="scan", dtype="bf16", B=8, L=2048, D=1536, N=16, G=1, train=True,
             ragged=False, state=False, gate=True),
        # training on one long sequence
        dict(name="scan_train_long", op="scan", dtype="bf16", B=1, L=8192, D=1536, N=16, G=1, train=True,
             ragged=False, state=False, gate=True),
        # a ragged batch carried over segments (state in and out, gradients through both), two groups, odd sizes
        dict(name="scan_ragged_train", op="scan", dtype="fp32", B=4, L=509, D=202, N=13, G=2, train=True,
             ragged=True, state=True, gate=True),
        # one request's token: latency
        dict(name="step_one", op="step", dtype="bf16", B=1, D=1536, N=16, G=1, K=4),
        # a serving batch's token
        dict(name="step_batch", op="step", dtype="bf16", B=256, D=1536, N=16, G=1, K=4),
        # a policy update on 8 responses of 1024 tokens
        dict(name="policy_train", op="policy", dtype="bf16", B=8, L=1024, V=32000, pad=0, train=True, kl=True),
        # a small odd one: a sequence with no counted token, NaN in the masked places, rows of a padded head
        dict(name="policy_small", op="policy", dtype="fp32", B=5, L=37, V=1021, pad=3, train=True, kl=True),
        # preference training on 4 pairs of 512 tokens, one added token in the vocabulary
        dict(name="preference_train", op="preference", dtype="bf16", B=8, L=512, V=32001, pad=0, train=True),
        # a few short pairs, odd sizes
        dict(name="preference_small", op="preference", dtype="fp16", B=6, L=65, V=4099, pad=0, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "step", "policy", "preference"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "conv":
        B, D = _log(rng, 1, 16), _log(rng, 64, 4096)
        L = min(_log(rng, 1, 8192), max(1, 4 * 8192 * 1536 // (B * D)))
        return dict(op=op, dtype=dtype, B=B, L=L, D=D, K=rng.choice([2, 3, 4]), train=rng.random() < 0.5,
                    ragged=rng.random() < 0.4, state=rng.random() < 0.5)
    if op == "scan":
        train = rng.random() < 0.6
        B, G = _log(rng, 1, 8), rng.choice([1, 1, 2])
        D, N = G * (_log(rng, 64, 2048) // G), rng.choice([4, 8, 13, 16, 16, 32, 64])
        top = 8192 if train else 32768
        L = min(_log(rng, 1, top), max(1, (8192 if train else 32768) * 1536 * 16 // (B * D * N)))
        return dict(op=op, dtype=dtype, B=B, L=L, D=D, N=N, G=G, train=train, ragged=rng.random() < 0.4,
                    state=rng.random() < 0.5, gate=rng.random() < 0.7)
    if op == "step":
        G = rng.choice([1, 1, 2])
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 256), D=G * (_log(rng, 64, 1536) // G),
                    N=rng.choice([4, 8, 13, 16]), G=G, K=rng.choice([2, 3, 4]))
    V = _log(rng, 100, 131072)
    rows = max(2, min(_log(rng, 2, 8192), 8192 * 32000 // (V * (2 if dtype == "fp32" else 1))))
    B = 2 * max(1, min(rows // 2, _log(rng, 1, 8)))
    L = max(1, rows // B)
    c = dict(op=op, dtype=dtype, B=B, L=L, V=V, pad=rng.choice([0, 0, 5, 8]), train=rng.random() < 0.7)
    if op == "policy":
        c["kl"] = rng.random() < 0.6
    return c


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _lengths(case, g):
    """Lengths of a ragged batch: from none (the last row) and one token (the first) to all L."""
    B, L = case["B"], case["L"]
    n = torch.randint(1, L + 1, (B,), generator=g, device="cuda")
    n[0] = 1
    if B > 1:
        n[1] = L
        n[-1] = 0
    return n


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    s = {"case": case}
    op = case["op"]
    if op in ("conv", "scan"):
        B, L, D = case["B"], case["L"], case["D"]
        s["lengths"] = _lengths(case, g) if case["ragged"] else None
        pad = None
        if case["ragged"]:
            pad = torch.arange(L, device="cuda")[None] >= s["lengths"][:, None]
    if op == "conv":
        K = case["K"]
        xz = _rn(g, B, L, 2 * D).to(dt)            # the input projection's output: x is its first half
        if pad is not None:
            xz[pad] = float("nan")                 # what lies behind a sequence's end is not data
        s["x"] = xz[..., :D]
        s["weight"] = _rn(g, D, K, scale=1.0 / math.sqrt(K))
        s["bias"] = _rn(g, D, scale=0.1)
        s["init"] = _rn(g, B, K - 1, D).to(dt) if case["state"] else None
        s["dy"] = _rn(g, B, L, D).to(dt) if case["train"] else None
        s["dfinal"] = _rn(g, B, K - 1, D).to(dt) if case["train"] and case["state"] else None
        wrt = ["x", "weight", "bias"] + (["init"] if case["state"] and case["train"] else [])
    elif op == "scan":
        N, G = case["N"], case["G"]
        rank = max(1, D // 32)
        s["u"] = F.silu(_rn(g, B, L, D)).to(dt)
        s["delta"] = _rn(g, B, L, D, scale=0.5).to(dt)
        s["z"] = _rn(g, B, L, 2 * D).to(dt)[..., D:] if case["gate"] else None   # second half of the projection
        dbc = _rn(g, B, L, rank + 2 * G * N).to(dt)                              # one projection: rank, B, C
        s["B"] = dbc[..., rank:rank + G * N].unflatten(-1, (G, N))
        s["C"] = dbc[..., rank + G * N:].unflatten(-1, (G, N))
        if pad is not None:
            for k in ("u", "delta", "z", "B", "C"):
                if s[k] is not None:
                    s[k].masked_fill_(pad.view(B, L, *([1] * (s[k].ndim - 2))), float("nan"))
        s["A"] = -(torch.arange(1, N + 1, device="cuda") * torch.exp(_rn(g, D, N, scale=0.2)))
        step = torch.exp(torch.rand(D, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["bias"] = step + torch.log(-torch.expm1(-step))                        # softplus(bias) = step
        s["D"] = 1.0 + _rn(g, D, scale=0.1)
        s["init"] = _rn(g, B, D, N) if case["state"] and case["train"] else None
        s["dy"] = _rn(g, B, L, D).to(dt) if case["train"] else None
        s["dfinal"] = _rn(g, B, D, N) if case["train"] and case["state"] else None
        wrt = ["u", "delta", "A", "B", "C", "D", "bias"] + (["z"] if case["gate"] else []) + \
            (["init"] if case["state"] and case["train"] else [])
    elif op == "step":
        B, D, N, G, K = (case[k] for k in ("B", "D", "N", "G", "K"))
        s["x"] = _rn(g, B, 2 * D).to(dt)[:, :D]
        s["z"] = _rn(g, B, 2 * D).to(dt)[:, D:]
        s["weight"] = _rn(g, D, K, scale=1.0 / math.sqrt(K)).to(dt)
        s["cbias"] = _rn(g, D, scale=0.1).to(dt)
        s["conv_state"] = _rn(g, B, K - 1, D).to(dt)
        s["delta"] = _rn(g, B, D, scale=0.5).to(dt)
        bc = _rn(g, B, 2 * G * N).to(dt)
        s["B"], s["C"] = bc[:, :G * N].unflatten(-1, (G, N)), bc[:, G * N:].unflatten(-1, (G, N))
        s["A"] = -(torch.arange(1, N + 1, device="cuda") * torch.exp(_rn(g, D, N, scale=0.2)))
        step = torch.exp(torch.rand(D, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
        s["bias"] = step + torch.log(-torch.expm1(-step))
        s["D"] = 1.0 + _rn(g, D, scale=0.1)
        s["state"] = _rn(g, B, D, N)
        # the states after the token go into a second pair of buffers, as a program that may take a token back keeps them
        s["new_conv_state"], s["new_state"] = torch.empty_like(s["conv_state"]), torch.empty_like(s["state"])
        wrt = []
    else:
        B, L, V = case["B"], case["L"], case["V"]
        s["logits"] = _rn(g, B, L, V + case["pad"], scale=2.0).to(dt)[..., :V]
        s["labels"] = torch.randint(0, V, (B, L), generator=g, device="cuda")
        # prompts in front and padding behind do not count; one sequence counts nowhere
        first = torch.randint(0, max(1, L // 4) + 1, (B, 1), generator=g, device="cuda")
        last = L - torch.randint(0, max(1, L // 4) + 1, (B, 1), generator=g, device="cuda")
        pos = torch.arange(L, device="cuda")[None]
        mask = (pos >= first) & (pos < last)
        if op == "policy":
            mask[-1] = False
        s["mask"] = mask
        if case["pad"] == 3:
            s["logits"].masked_fill_(~mask[..., None], float("nan"))
        s["labels"][~mask] = -100
        lp = torch.zeros(B, L, device="cuda")
        for b in range(B):
            x = s["logits"][b].float()
            lab = s["labels"][b].clamp(min=0)
            lp[b] = x.gather(-1, lab[:, None])[:, 0] - torch.logsumexp(x, -1)
        lp = torch.where(mask, lp, 0.0)
        if op == "policy":
            s["old"] = lp + _rn(g, B, L, scale=0.2)
            s["ref"] = lp + _rn(g, B, L, scale=0.3) if case["kl"] else None
            s["adv"] = _rn(g, B)
        else:
            s["ref"] = lp.sum(-1) + _rn(g, B, scale=5.0)
        wrt = ["logits"] if case["train"] else []
    if case.get("train"):
        for k in wrt:
            s[k] = s[k].detach().requires_grad_(True)
    s["wrt"] = wrt
    return s


CLIP_LOW, CLIP_HIGH, KL, BETA, SMOOTH = 0.2, 0.28, 0.05, 0.1, 0.05


# --------------------------------------------------------------------------
# through the framework
# --------------------------------------------------------------------------
def _run_own(s):
    import mogt_b200
    case = s["case"]
    op = case["op"]
    if op == "conv":
        with torch.set_grad_enabled(case["train"]):
            r = mogt_b200.causal_conv(s["x"], s["weight"], s["bias"], activation="silu", initial_state=s["init"],
                                      lengths=s["lengths"], return_state=case["state"])
        outs = tuple(r) if case["state"] else (r,)
        if not case["train"]:
            return list(outs)
        douts = [s["dy"]] + ([s["dfinal"]] if case["state"] else [])
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [s[k] for k in s["wrt"]], douts))
    if op == "scan":
        with torch.set_grad_enabled(case["train"]):
            r = mogt_b200.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                         delta_bias=s["bias"], delta_softplus=True, initial_state=s["init"],
                                         lengths=s["lengths"], return_state=case["state"])
        outs = tuple(r) if case["state"] else (r,)
        if not case["train"]:
            return list(outs)
        douts = [s["dy"]] + ([s["dfinal"]] if case["state"] else [])
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [s[k] for k in s["wrt"]], douts))
    if op == "step":
        u = mogt_b200.causal_conv_step(s["x"], s["conv_state"], s["weight"], s["cbias"], activation="silu",
                                       new_state=s["new_conv_state"])
        y = mogt_b200.selective_scan_step(s["state"], u, s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                          delta_bias=s["bias"], delta_softplus=True, new_state=s["new_state"])
        return [u, y, s["new_conv_state"], s["new_state"]]
    with torch.set_grad_enabled(case["train"]):
        if op == "policy":
            loss, lp = mogt_b200.policy_loss(s["logits"], s["labels"], s["old"], s["adv"], ref_logprobs=s["ref"],
                                             mask=s["mask"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL,
                                             return_logprobs=True)
        else:
            loss, lp = mogt_b200.preference_loss(s["logits"], s["labels"], s["ref"], beta=BETA,
                                                 label_smoothing=SMOOTH, mask=s["mask"], return_logprobs=True)
    if not case["train"]:
        return [loss, lp]
    return [loss.detach(), lp] + list(torch.autograd.grad(loss, [s["logits"]]))


# --------------------------------------------------------------------------
# plain forms: 32 bits throughout, rounded once at the end
# --------------------------------------------------------------------------
def _valid(s):
    if s["lengths"] is None:
        return None
    L = s["case"]["L"]
    return torch.arange(L, device="cuda")[None] < s["lengths"][:, None]


def _plain_conv(s):
    case = s["case"]
    B, L, D, K = case["B"], case["L"], case["D"], case["K"]
    x = s["x"].float()
    valid = _valid(s)
    if valid is not None:
        x = torch.where(valid[..., None], x, 0.0)
    w, b = s["weight"].float(), s["bias"].float()
    init = s["init"].float() if s["init"] is not None else torch.zeros(B, K - 1, D, device="cuda")
    h = torch.cat([init, x], 1)
    pre = b + w[:, 0] * h[:, :L]
    for j in range(1, K):
        pre = pre + w[:, j] * h[:, j:j + L]
    sg = 1.0 / (1.0 + torch.exp(-pre))
    y = pre * sg
    if valid is not None:
        y = torch.where(valid[..., None], y, 0.0)
    outs = [y.to(s["x"].dtype)]
    n = s["lengths"] if valid is not None else torch.full((B,), L, device="cuda")
    idx = (n[:, None] + torch.arange(K - 1, device="cuda")[None])[..., None].expand(B, K - 1, D)
    if case["state"]:
        outs.append(h.gather(1, idx).to(s["x"].dtype))
    if not case["train"]:
        return outs
    gp = s["dy"].float() * (sg + y * (1.0 - sg))
    if valid is not None:
        gp = torch.where(valid[..., None], gp, 0.0)
    dh = torch.zeros(B, L + K - 1, D, device="cuda")
    dw = torch.zeros(D, K, device="cuda")
    for j in range(K):
        dh[:, j:j + L] += w[:, j] * gp
        dw[:, j] = (gp * h[:, j:j + L]).sum((0, 1))
    if case["state"]:
        dh.scatter_add_(1, idx, s["dfinal"].float())
    dx = dh[:, K - 1:]
    if valid is not None:
        dx = torch.where(valid[..., None], dx, 0.0)
    outs += [dx.to(s["x"].dtype), dw.to(s["weight"].dtype), gp.sum((0, 1)).to(s["bias"].dtype)]
    if case["state"]:
        outs.append(dh[:, :K - 1].to(s["init"].dtype))
    return outs


def _plain_scan(s):
    case = s["case"]
    B, L, D, N, G = (case[k] for k in ("B", "L", "D", "N", "G"))
    train, dt_ = case["train"], s["u"].dtype
    valid = _valid(s)

    def clean(t):
        t = t.float()
        return t if valid is None else torch.where(valid.view(B, L, *([1] * (t.ndim - 2))), t, 0.0)

    u, A, Dv = clean(s["u"]), s["A"].float(), s["D"].float()
    Bg, Cg = clean(s["B"]), clean(s["C"])
    raw = clean(s["delta"]) + s["bias"].float()
    dt = torch.where(raw > 20.0, raw, torch.log1p(torch.exp(raw.clamp(max=20.0))))
    if valid is not None:
        dt = torch.where(valid[..., None], dt, 0.0)
    z = clean(s["z"]) if case["gate"] else None
    x = dt * u
    h = s["init"].float() if s["init"] is not None else torch.zeros(B, D, N, device="cuda")
    step = max(1, min(L, 2 ** 26 // (B * D * N)))
    hs = torch.empty(L, B, D, N, device="cuda") if train else None
    y = torch.empty(B, L, D, device="cuda")

    def wide(t, i, j):                       # [B, l, G, N] -> [l, B, G, 1, N]
        return t[:, i:j].transpose(0, 1).unsqueeze(3)

    def grouped(t):                          # [l, B, D, N] -> [l, B, G, D/G, N]
        return t.view(t.shape[0], B, G, D // G, N)

    for i in range(0, L, step):
        j = min(L, i + step)
        a = torch.exp(dt[:, i:j].transpose(0, 1)[..., None] * A)
        xb = (x[:, i:j].transpose(0, 1).reshape(j - i, B, G, D // G, 1) * wide(Bg, i, j)).view(j - i, B, D, N)
        hc = hs[i:j] if train else xb
        for t in range(j - i):
            h = torch.addcmul(xb[t], a[t], h, out=hc[t])
        y[:, i:j] = (grouped(hc) * wide(Cg, i, j)).sum(-1).view(j - i, B, D).transpose(0, 1)
        h = h.clone()
    y = y + Dv * u
    sg = 1.0 / (1.0 + torch.exp(-z)) if z is not None else None
    out = y * (z * sg) if z is not None else y
    if valid is not None:
        out = torch.where(valid[..., None], out, 0.0)
    outs = [out.to(dt_)] + ([h] if case["state"] else [])
    if not train:
        return outs
    do = clean(s["dy"])
    dy = do * (z * sg) if z is not None else do
    dz = do * y * (sg + z * sg * (1.0 - sg)) if z is not None else None
    g = s["dfinal"].float().clone() if case["state"] else torch.zeros(B, D, N, device="cuda")
    dA = torch.zeros(D, N, device="cuda")
    dB, dC = torch.zeros_like(Bg), torch.zeros_like(Cg)
    sB, Aq = torch.empty_like(u), torch.empty_like(u)
    h0 = s["init"].float() if s["init"] is not None else torch.zeros(B, D, N, device="cuda")
    for j in range(L, 0, -step):
        i = max(0, j - step)
        a = torch.exp(dt[:, i:j].transpose(0, 1)[..., None] * A)
        gs = (dy[:, i:j].transpose(0, 1).reshape(j - i, B, G, D // G, 1) * wide(Cg, i, j)).view(j - i, B, D, N)
        for t in range(j - i - 1, -1, -1):
            gs[t] += g                       # adjoint of h_t
            g = a[t] * gs[t]                 # what it hands to h_{t-1}
        hc = hs[i:j]
        hp = torch.cat([(hs[i - 1] if i else h0)[None], hs[i:j - 1]], 0)
        q = gs * (a * hp)
        tr = lambda v: v.transpose(0, 1)
        dC[:, i:j] = tr((tr(dy[:, i:j]).reshape(j - i, B, G, D // G, 1) * grouped(hc)).sum(3))
        dB[:, i:j] = tr((tr(x[:, i:j]).reshape(j - i, B, G, D // G, 1) * grouped(gs)).sum(3))
        sB[:, i:j] = tr((grouped(gs) * wide(Bg, i, j)).sum(-1).view(j - i, B, D))
        Aq[:, i:j] = tr((q * A).sum(-1))
        dA += (tr(dt[:, i:j])[..., None] * q).sum((0, 1))
    du = dt * sB + Dv * dy
    ddel = (u * sB + Aq) * (1.0 / (1.0 + torch.exp(-raw)))
    dD = (dy * u).sum((0, 1))
    if valid is not None:
        du, ddel = (torch.where(valid[..., None], t, 0.0) for t in (du, ddel))
    outs += [du.to(dt_), ddel.to(dt_), dA, dB.to(dt_), dC.to(dt_), dD, ddel.sum((0, 1))]
    if z is not None:
        outs.append(dz.to(dt_))
    return outs + ([g] if case["state"] else [])


def _plain_step(s):
    case = s["case"]
    B, D, N, G = (case[k] for k in ("B", "D", "N", "G"))
    dt_ = s["x"].dtype
    h = torch.cat([s["conv_state"].float(), s["x"].float()[:, None]], 1)
    pre = s["cbias"].float() + (h * s["weight"].float().t()).sum(1)
    u = (pre / (1.0 + torch.exp(-pre))).to(dt_)
    uf = u.float()
    raw = s["delta"].float() + s["bias"]
    dt = torch.where(raw > 20.0, raw, torch.log1p(torch.exp(raw.clamp(max=20.0))))
    xb = ((dt * uf).view(B, G, D // G, 1) * s["B"].float()[:, :, None]).view(B, D, N)
    st = torch.exp(dt[..., None] * s["A"]) * s["state"] + xb
    y = (st.view(B, G, D // G, N) * s["C"].float()[:, :, None]).sum(-1).view(B, D) + s["D"] * uf
    z = s["z"].float()
    return [u, (y * (z / (1.0 + torch.exp(-z)))).to(dt_), h[:, 1:].to(dt_), st]


def _plain_rows(s):
    """Per token: log-probability of its label, and the softmax (rows that do not count are cleared first)."""
    x = torch.where(s["mask"][..., None], s["logits"].detach().float(), 0.0)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    t = e.sum(-1, keepdim=True)
    lab = s["labels"].clamp(min=0)[..., None]
    lp = (x.gather(-1, lab) - m - torch.log(t))[..., 0]
    return torch.where(s["mask"], lp, 0.0), e.div_(t), lab


def _plain_loss(s):
    case = s["case"]
    mask = s["mask"].float()
    lp, p, lab = _plain_rows(s)
    if case["op"] == "policy":
        cnt = mask.sum().clamp(min=1.0)
        r = torch.exp(lp - s["old"])
        adv = s["adv"][:, None]
        s1, s2 = r * adv, r.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
        tok = -torch.minimum(s1, s2)
        g = -torch.where(s1 <= s2, s1, 0.0)
        if s["ref"] is not None:
            d = s["ref"] - lp
            tok = tok + KL * (torch.exp(d) - d - 1.0)
            g = g + KL * (1.0 - torch.exp(d))
        loss = torch.where(s["mask"], tok, 0.0).sum() / cnt
        outs = [loss, lp]
        g = torch.where(s["mask"], g, 0.0) / cnt
    else:
        seq = lp.sum(-1)
        P = case["B"] // 2
        d = seq - s["ref"]
        x = BETA * (d[:P] - d[P:])
        sp = lambda v: torch.where(v > 0, v, 0.0) + torch.log1p(torch.exp(-v.abs()))
        loss = ((1.0 - SMOOTH) * sp(-x) + SMOOTH * sp(x)).mean()
        outs = [loss, seq]
        gx = BETA / P * (1.0 / (1.0 + torch.exp(-x)) - (1.0 - SMOOTH))
        g = torch.cat([gx, -gx])[:, None] * mask
    if case["train"]:
        dl = p.mul_(-g[..., None])
        dl.scatter_add_(-1, lab, g[..., None])
        outs.append(dl.to(s["logits"].dtype))
    return outs


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        if op == "conv":
            return _plain_conv(state)
        if op == "scan":
            return _plain_scan(state)
        if op == "step":
            return _plain_step(state)
        return _plain_loss(state)


# --------------------------------------------------------------------------
# the definitions in 64 bits: one token after another, gradients by differentiating them
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = lambda t: None if t is None else t.detach().double()
    op = case["op"]
    if op == "step":
        u = None
        w, x = f64(s["weight"]), f64(s["x"])
        hist = torch.cat([f64(s["conv_state"]), x[:, None]], 1)
        pre = f64(s["cbias"]) + torch.einsum("bkd,dk->bd", hist, w)
        u = pre * torch.sigmoid(pre)
        ur = u.to(s["x"].dtype).double()       # the scan takes the convolution's rounded output
        dt = F.softplus(f64(s["delta"]) + f64(s["bias"]), threshold=1e9)
        rep = case["D"] // case["G"]
        Bm, Cm = (f64(s[k]).repeat_interleave(rep, 1) for k in ("B", "C"))
        st = torch.exp(dt[..., None] * f64(s["A"])) * f64(s["state"]) + (dt * ur)[..., None] * Bm
        z = f64(s["z"])
        y = ((st * Cm).sum(-1) + f64(s["D"]) * ur) * z * torch.sigmoid(z)
        return [u, y, hist[:, 1:], st]
    leaves = {k: f64(s[k]).requires_grad_(bool(case.get("train"))) for k in s["wrt"]}
    get = lambda k: leaves.get(k, f64(s.get(k)))
    with torch.set_grad_enabled(bool(case.get("train"))):
        if op == "conv":
            B, L, D, K = (case[k] for k in ("B", "L", "D", "K"))
            init = get("init")
            if init is None:
                init = torch.zeros(B, K - 1, D, dtype=torch.float64, device="cuda")
            n = s["lengths"].tolist() if s["lengths"] is not None else [L] * B
            ys, fin = [], []
            for b in range(B):
                h = torch.cat([init[b], get("x")[b, :n[b]]])
                pre = sum(h[j:j + n[b]] * get("weight")[:, j] for j in range(K)) + get("bias")
                ys.append(F.pad(F.silu(pre), (0, 0, 0, L - n[b])))
                fin.append(h[n[b]:])
            outs = [torch.stack(ys)] + ([torch.stack(fin)] if case["state"] else [])
        elif op == "scan":
            B, L, D, N, G = (case[k] for k in ("B", "L", "D", "N", "G"))
            live = _valid(s)
            if live is None:
                live = torch.ones(B, L, dtype=torch.bool, device="cuda")
            u, Bm, Cm, delta = (torch.where(live.view(B, L, *([1] * (get(k).ndim - 2))), get(k), 0.0)
                                for k in ("u", "B", "C", "delta"))
            dt = F.softplus(delta + get("bias"), threshold=1e9) * live[..., None]
            h = get("init")
            if h is None:
                h = torch.zeros(B, D, N, dtype=torch.float64, device="cuda")
            A, rep, ys = get("A"), D // G, []
            dts, xs, Bs, Cs = dt.unbind(1), (dt * u).unbind(1), Bm.unbind(1), Cm.unbind(1)
            for t in range(L):
                h = torch.exp(dts[t][..., None] * A) * h + xs[t][..., None] * Bs[t].repeat_interleave(rep, 1)
                if G == 1:
                    ys.append(torch.bmm(h, Cs[t].transpose(1, 2))[..., 0])
                else:
                    ys.append((h * Cs[t].repeat_interleave(rep, 1)).sum(-1))
            y = torch.stack(ys, 1) + get("D") * u
            if case["gate"]:
                z = torch.where(live[..., None], get("z"), 0.0)
                y = y * z * torch.sigmoid(z)
            outs = [torch.where(live[..., None], y, 0.0)] + ([h] if case["state"] else [])
        else:
            mask = s["mask"]
            x = torch.where(mask[..., None], get("logits") if case["train"] else f64(s["logits"]), 0.0)
            lab = torch.where(mask, s["labels"], 0)
            lp = F.log_softmax(x, -1).gather(-1, lab[..., None])[..., 0] * mask
            if op == "policy":
                r = torch.exp(lp - f64(s["old"]))
                adv = f64(s["adv"])[:, None]
                tok = -torch.minimum(r * adv, torch.clamp(r, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv)
                if s["ref"] is not None:
                    d = f64(s["ref"]) - lp
                    tok = tok + KL * (torch.expm1(d) - d)
                loss = (tok * mask).sum() / max(1, int(mask.sum()))
                outs = [loss, lp]
            else:
                P = case["B"] // 2
                d = lp.sum(-1) - f64(s["ref"])
                x = BETA * (d[:P] - d[P:])
                loss = -((1.0 - SMOOTH) * F.logsigmoid(x) + SMOOTH * F.logsigmoid(-x)).mean()
                outs = [loss, lp.sum(-1)]
        if not case.get("train"):
            return outs
        if op in ("conv", "scan"):
            live = _valid(s)
            dy = f64(s["dy"])
            if live is not None:
                dy = torch.where(live[..., None], dy, 0.0)
            douts = [dy] + ([f64(s["dfinal"])] if case["state"] else [])
            grads = torch.autograd.grad(outs, [leaves[k] for k in s["wrt"]], douts)
        else:
            grads = torch.autograd.grad([outs[0]], [leaves["logits"]])
    # padding and masked places hold NaN inputs: their gradients are zero by definition
    return [o.detach() for o in outs] + [torch.nan_to_num(gr) for gr in grads]


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    e, op, B = _ESIZE[case["dtype"]], case["op"], case["B"]
    if op == "conv":
        n, K = B * case["L"] * case["D"], case["K"]
        if case["train"]:                    # x, dy in; y, dx out
            return {"bytes": 4 * n * e, "flops": n * (2 * K + 4 + 4 * K + 6)}
        return {"bytes": 2 * n * e, "flops": n * (2 * K + 4)}
    if op == "scan":
        D, N, t = case["D"], case["N"], B * case["L"]
        bc = 2 * case["G"] * N
        state = 4 * B * D * N if case["state"] else 0
        gate = 1 if case["gate"] else 0
        if case["train"]:                    # u, delta, z, dy, B, C in; y and their gradients out
            return {"bytes": t * e * ((6 + 2 * gate) * D + 2 * bc) + 4 * state, "flops": t * D * (N * 26 + 20)}
        return {"bytes": t * e * ((3 + gate) * D + bc) + state, "flops": t * D * (N * 7 + 10)}
    if op == "step":
        D, N, K = case["D"], case["N"], case["K"]
        return {"bytes": B * D * (8 * N + e * (2 * (K - 1) + 5)) + 4 * D * (N + 2) + e * D * (K + 1),
                "flops": B * D * (7 * N + 2 * K + 16)}
    n = B * case["L"] * case["V"]
    return {"bytes": n * e * (2 if case["train"] else 1), "flops": n * (8 if case["train"] else 4)}
