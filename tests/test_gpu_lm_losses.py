"""Post-training losses against their float64 forms: values, log-probabilities
and logit gradients over types, row counts and alignments, masks that leave
rows, sequences or everything empty, and values at the ends of the range."""
import pytest
import torch

from .selective_ref import ROUND, logprobs_ref, max_err, policy_ref, preference_ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# Log-probabilities are differences of values up to about 20 with an fp32
# logarithm; a coefficient multiplies a few exponentials good to 2^-22 each.
TOL32 = 2.0 ** -19


def make(B, L, V, dtype, seed=0, pad=0, mask=True, nan=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    t = dict(logits=(2 * rn(B, L, V + pad)).to(dtype)[..., :V], old=None,
             labels=torch.randint(0, V, (B, L), generator=g, device="cuda"), mask=None)
    counts = torch.ones(B, L, dtype=torch.bool, device="cuda")
    if mask:
        t["mask"] = torch.rand(B, L, generator=g, device="cuda") < 0.7
        t["mask"][-1] = False
        counts &= t["mask"]
        t["labels"][0, ::3] = -100
        counts[0, ::3] = False
    if nan:
        t["logits"][~counts] = float("nan")
    t["counts"] = counts
    lp = logprobs_ref(t["logits"].double(), t["labels"], counts).float()
    t["old"], t["ref"], t["adv"] = lp + 0.2 * rn(B, L), lp + 0.3 * rn(B, L), rn(B)
    t["sref"] = lp.sum(-1) + rn(B)
    return t


def policy(t, dtype, kl=0.05, adv=None, **kw):
    import mogt_b200
    adv = t["adv"] if adv is None else adv
    x = t["logits"].detach().requires_grad_(True)
    loss, lp = mogt_b200.policy_loss(x, t["labels"], t["old"], adv, ref_logprobs=t["ref"] if kl else None,
                                     mask=t["mask"], clip_low=0.2, clip_high=0.3, kl_coef=kl, return_logprobs=True)
    x64 = torch.nan_to_num(t["logits"].detach().double()).requires_grad_(True)
    loss64, lp64 = policy_ref(x64, t["labels"], t["counts"], t["old"].double(), adv.double(),
                              t["ref"].double() if kl else None, 0.2, 0.3, kl)
    return x, loss, lp, x64, loss64, lp64


SHAPES = [(2, 1, 1, F32, {}), (2, 3, 7, F32, {}), (4, 5, 100, BF16, dict(pad=3)), (2, 9, 1021, F32, dict(pad=2, nan=True)),
          (6, 4, 4099, F16, {}), (2, 3, 32001, BF16, dict(nan=True)), (2, 2, 70000, F32, dict(pad=1)),
          (4, 70, 513, BF16, dict(mask=False))]


@pytest.mark.parametrize("B,L,V,dtype,opt", SHAPES)
@pytest.mark.parametrize("kl", [0.0, 0.05])
def test_policy_against_definition(B, L, V, dtype, opt, kl):
    t = make(B, L, V, dtype, **opt)
    x, loss, lp, x64, loss64, lp64 = policy(t, dtype, kl)
    assert abs(float(loss.detach()) - float(loss64.detach())) <= TOL32 * max(1.0, abs(float(loss64.detach())))
    assert max_err(lp, lp64) <= TOL32
    g, = torch.autograd.grad(loss, x)
    g64, = torch.autograd.grad(loss64, x64)
    # fp16 keeps gradients below 2^-14 with an absolute step of 2^-24
    floor = 2.0 ** -25 / max(float(g64.abs().max()), 1e-30) if dtype == F16 else 0.0
    assert max_err(g, g64) <= TOL32 + ROUND[dtype] + floor
    assert bool((g[~t["counts"]] == 0).all())


@pytest.mark.parametrize("B,L,V,dtype,opt", SHAPES)
def test_preference_against_definition(B, L, V, dtype, opt):
    import mogt_b200
    t = make(B, L, V, dtype, **opt)
    x = t["logits"].detach().requires_grad_(True)
    loss, seq = mogt_b200.preference_loss(x, t["labels"], t["sref"], beta=0.1, label_smoothing=0.1, mask=t["mask"],
                                          return_logprobs=True)
    x64 = torch.nan_to_num(t["logits"].detach().double()).requires_grad_(True)
    loss64, seq64 = preference_ref(x64, t["labels"], t["counts"], t["sref"].double(), 0.1, 0.1)
    assert abs(float(loss.detach()) - float(loss64.detach())) <= TOL32 * L * 10
    assert max_err(seq, seq64) <= TOL32
    g, = torch.autograd.grad(loss, x)
    g64, = torch.autograd.grad(loss64, x64)
    floor = 2.0 ** -25 / max(float(g64.abs().max()), 1e-30) if dtype == F16 else 0.0
    # the pair's logit moves by the error of its sums of L log-probabilities
    assert max_err(g, g64) <= TOL32 * (L + 2) + ROUND[dtype] + floor


@pytest.mark.parametrize("B,L,V,dtype,opt", SHAPES)
def test_logprobs_and_their_gradient(B, L, V, dtype, opt):
    import mogt_b200
    t = make(B, L, V, dtype, **opt)
    x = t["logits"].detach().requires_grad_(True)
    lp = mogt_b200.token_logprobs(x, t["labels"], mask=t["mask"])
    x64 = torch.nan_to_num(t["logits"].detach().double()).requires_grad_(True)
    lp64 = logprobs_ref(x64, t["labels"], t["counts"])
    assert max_err(lp, lp64) <= TOL32
    with torch.no_grad():
        assert torch.equal(lp, mogt_b200.token_logprobs(x, t["labels"], mask=t["mask"]))
    w = torch.randn(B, L, device="cuda")
    g, = torch.autograd.grad(lp, x, w)
    g64, = torch.autograd.grad(lp64, x64, w.double())
    assert max_err(g, g64) <= TOL32 + ROUND[dtype]


def test_nothing_counts():
    import mogt_b200
    t = make(4, 6, 50, F32)
    mask = torch.zeros(4, 6, dtype=torch.bool, device="cuda")
    x = torch.full_like(t["logits"], float("nan")).requires_grad_(True)
    loss = mogt_b200.policy_loss(x, t["labels"], t["old"], t["adv"], mask=mask)
    g, = torch.autograd.grad(loss, x)
    assert float(loss) == 0.0 and bool((g == 0).all())
    loss = mogt_b200.preference_loss(x, t["labels"], torch.zeros(4, device="cuda"), mask=mask)
    g, = torch.autograd.grad(loss, x)
    assert abs(float(loss) - 0.6931472) <= 1e-6 and bool((g == 0).all())
    empty = mogt_b200.policy_loss(x[:, :0], t["labels"][:, :0], t["old"][:, :0], t["adv"])
    assert float(empty) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ends_of_the_range(dtype):
    """Vocabulary entries masked by -inf or by the type's lowest value, rows
    that hold one value everywhere (the lowest one too), large logits."""
    import mogt_b200
    t = make(2, 6, 300, dtype, mask=False)
    low = torch.finfo(dtype).min
    x = t["logits"].clone()
    lab = t["labels"].clone()
    lab[:] = 7
    x[0, 0, 20:] = float("-inf")
    x[0, 1, 20:] = low
    x[0, 2, :] = low
    x[0, 3, :] = 3.0
    x[0, 4, :] = 1e4 + 64 * (torch.arange(300, device="cuda") % 4)
    x[0, 5, :200] = float("-inf")
    lab[0, 5] = 250
    xg = x.requires_grad_(True)
    lp = mogt_b200.token_logprobs(xg, lab)
    x64 = x.detach().double().requires_grad_(True)
    lp64 = torch.log_softmax(x64, -1).gather(-1, lab[..., None])[..., 0]
    assert max_err(lp, lp64) <= TOL32
    g, = torch.autograd.grad(lp.sum(), xg)
    g64, = torch.autograd.grad(lp64.sum(), x64)
    assert max_err(g, g64) <= TOL32 + ROUND[dtype]


def test_nan_and_bad_labels_show():
    import mogt_b200
    t = make(2, 4, 100, F32, mask=False)
    x = t["logits"].clone()
    x[0, 1, 99] = float("nan")
    lab = t["labels"].clone()
    lab[1, 2] = 100
    lp = mogt_b200.token_logprobs(x, lab)
    bad = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 2] = True
    assert torch.equal(torch.isnan(lp), bad)
    assert bool(torch.isnan(mogt_b200.policy_loss(x, lab, t["old"], t["adv"])))


def test_scaled_and_repeated_backward():
    """d loss other than 1, and a second backward after the first gradient
    was changed in place by its receiver."""
    t = make(2, 5, 1000, F32, pad=5)
    x, loss, _, x64, loss64, _ = policy(t, F32)
    g64, = torch.autograd.grad(loss64, x64)
    a, = torch.autograd.grad(loss, x, torch.tensor(-2.5, device="cuda"), retain_graph=True)
    assert max_err(a, -2.5 * g64) <= TOL32
    a.zero_()
    b, = torch.autograd.grad(loss, x, torch.tensor(3.0, device="cuda"), retain_graph=True)
    assert max_err(b, 3.0 * g64) <= TOL32
    (2 * loss).backward()
    assert max_err(x.grad, 2.0 * g64) <= TOL32


@pytest.mark.parametrize("dtype,scale", [(F16, 65536.0), (BF16, 1.0 / 3.0), (F16, 1.0), (BF16, 1.0)])
def test_a_scaled_loss_is_rounded_once(dtype, scale):
    """Gradients of a mean over many tokens are below fp16's smallest number
    before a loss scale brings them up: the scale goes in before the rounding."""
    t = make(4, 64, 500, dtype, pad=4)
    x, loss, _, x64, loss64, _ = policy(t, dtype)
    g, = torch.autograd.grad(loss * scale, x)
    g64, = torch.autograd.grad(loss64 * scale, x64)
    floor = 2.0 ** -25 / float(g64.abs().max()) if dtype == F16 else 0.0
    assert max_err(g, g64) <= TOL32 + ROUND[dtype] + floor
    big = g64.abs() > 2.0 ** -14          # normal numbers of either type: one rounding each
    err = (g.double() - g64).abs()[big] / g64.abs()[big]
    # beyond the rounding: p carries the fp32 error of its exponential and, as 1 - p at the label, a cancellation
    assert float(err.max()) <= ROUND[dtype] + 2.0 ** -16


def test_per_token_advantages_and_views():
    t = make(4, 6, 200, F32)
    adv = torch.randn(4, 12, device="cuda")[:, ::2]
    x, loss, _, x64, loss64, _ = policy(t, F32, adv=adv)
    g, g64 = torch.autograd.grad(loss, x)[0], torch.autograd.grad(loss64, x64)[0]
    assert abs(float(loss.detach()) - float(loss64.detach())) <= TOL32 and max_err(g, g64) <= TOL32
    # logits whose tokens come first in memory, and whose vocabulary is not dense
    for view in (t["logits"].transpose(0, 1).contiguous().transpose(0, 1),
                 t["logits"].transpose(1, 2).contiguous().transpose(1, 2)):
        s = dict(t, logits=view)
        x2, loss2, _, _, _, _ = policy(s, F32, adv=adv)
        g2, = torch.autograd.grad(loss2, x2)
        assert torch.equal(loss, loss2) and torch.equal(g, g2)


def test_rows_beyond_32_bit_offsets():
    import mogt_b200
    t = make(2, 3, 1000, BF16, mask=False)
    step = 2 ** 31 + 64
    x = torch.empty(step + 3000, dtype=BF16, device="cuda").as_strided((2, 3, 1000), (step, 1000, 1))
    x.copy_(t["logits"])
    assert torch.equal(mogt_b200.token_logprobs(x, t["labels"]), mogt_b200.token_logprobs(t["logits"], t["labels"]))


def test_two_runs_agree_to_the_bit_and_on_another_stream():
    t = make(4, 100, 3001, BF16)
    res = []
    s = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), torch.cuda.current_stream(), s):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            x, loss, lp, *_ = policy(t, BF16)
            res.append((loss, lp, torch.autograd.grad(loss, x)[0]))
    torch.cuda.synchronize()
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], r))


def test_gradient_against_differences():
    """Central differences along the gradient: 1e-2 relative (the loss is kept
    to about 1e-7, its change over the step is about 1e-4)."""
    import mogt_b200
    t = make(2, 4, 50, F32, mask=False)
    t["old"] = t["old"] * 0 + logprobs_ref(t["logits"].double(), t["labels"], t["counts"]).float()
    x, loss, *_ = policy(t, F32)
    g, = torch.autograd.grad(loss, x)
    v = g / g.norm()
    f = lambda s: float(mogt_b200.policy_loss(t["logits"] + s * v, t["labels"], t["old"], t["adv"],
                                              ref_logprobs=t["ref"], mask=t["mask"], clip_low=0.2, clip_high=0.3,
                                              kl_coef=0.05))
    num, ana = (f(0.02) - f(-0.02)) / 0.04, float((g * v).sum())
    assert abs(num - ana) <= 1e-2 * abs(ana)


def test_no_kl_term_without_reference():
    import mogt_b200
    t = make(2, 5, 60, F32)
    args = (t["logits"], t["labels"], t["old"], t["adv"])
    assert torch.equal(mogt_b200.policy_loss(*args, mask=t["mask"], kl_coef=0.3),
                       mogt_b200.policy_loss(*args, mask=t["mask"]))


def test_refusals():
    import mogt_b200
    x, lab = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    f = torch.zeros(2, 3, device="cuda")
    p = torch.zeros(2, device="cuda")
    for match, call in [
            ("logits must be", lambda: mogt_b200.token_logprobs(x[0], lab)),
            ("logits must be", lambda: mogt_b200.token_logprobs(x.double(), lab)),
            ("vocabulary", lambda: mogt_b200.token_logprobs(x[..., :0], lab)),
            ("labels must be", lambda: mogt_b200.token_logprobs(x, lab[:, :2])),
            ("labels must be", lambda: mogt_b200.token_logprobs(x, f)),
            ("mask must be", lambda: mogt_b200.token_logprobs(x, lab, mask=lab)),
            ("CUDA", lambda: mogt_b200.token_logprobs(x, lab.cpu())),
            ("old_logprobs", lambda: mogt_b200.policy_loss(x, lab, p, p)),
            ("advantages", lambda: mogt_b200.policy_loss(x, lab, f, f[:, :2])),
            ("ref_logprobs", lambda: mogt_b200.policy_loss(x, lab, f, p, ref_logprobs=p, kl_coef=0.1)),
            ("clip", lambda: mogt_b200.policy_loss(x, lab, f, p, clip_low=-0.1)),
            ("preferred", lambda: mogt_b200.preference_loss(x[:1], lab[:1], p[:1])),
            ("ref_logprobs", lambda: mogt_b200.preference_loss(x, lab, p[:1])),
            ("label_smoothing", lambda: mogt_b200.preference_loss(x, lab, p, label_smoothing=1.5)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
