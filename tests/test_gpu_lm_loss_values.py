"""Post-training losses where their values are delicate: sums of thousands that
nearly cancel, terms without weight, logits that are slices of larger tensors."""
import pytest
import torch

from .selective_ref import ROUND, max_err, preference_ref
from .test_gpu_lm_losses import TOL32, make, policy

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("seed", range(4))
def test_preference_of_long_responses(seed):
    """Two sums of about -4000 whose difference is a few tens.  A token's
    log-probability is off by at most 2^-19 (a difference of values below 16
    and a logarithm below 16, each rounded to 24 bits), independently from
    token to token: over the 2 L tokens of a pair sqrt(2 L) 2^-19, times beta,
    and the loss moves by no more than its logit does.  Sums kept in 32 bits
    would be off by 2^-13 each before anything else."""
    import mogt_b200
    B, L, V, beta = 8, 512, 32001, 0.1
    t = make(B, L, V, BF16, seed=seed)
    ref = (t["sref"] + 5 * torch.randn(B, generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
    loss, seq = mogt_b200.preference_loss(t["logits"], t["labels"], ref, beta=beta, label_smoothing=0.05,
                                          mask=t["mask"], return_logprobs=True)
    loss64, seq64 = preference_ref(t["logits"].double(), t["labels"], t["counts"], ref.double(), beta, 0.05)
    assert abs(float(loss) - float(loss64)) <= (2 * L) ** 0.5 * 2.0 ** -19 * beta
    assert max_err(seq, seq64) <= TOL32


def test_no_kl_weight_is_no_kl_term():
    """exp(ref - lp) overflows for a label that the model all but excludes; with kl_coef = 0 that is no term at all."""
    import mogt_b200
    x = torch.zeros(1, 3, 10, device="cuda")
    x[0, 1, 4] = -200.0
    lab = torch.full((1, 3), 4, device="cuda")
    lp = mogt_b200.token_logprobs(x, lab)
    adv = torch.ones(1, device="cuda")
    a = x.clone().requires_grad_(True)
    b = x.clone().requires_grad_(True)
    la = mogt_b200.policy_loss(a, lab, lp, adv, ref_logprobs=torch.zeros_like(lp))
    lb = mogt_b200.policy_loss(b, lab, lp, adv)
    assert torch.equal(la, lb) and float(lb.detach()) == -1.0
    assert torch.equal(torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0])


def test_an_impossible_response_of_a_pair():
    """A response with a label at -inf has probability zero: rejected, its pair
    is settled (x = inf, loss 0 without smoothing); preferred, its loss is inf,
    and 0 where the smoothing of 1 swaps the pair."""
    import mogt_b200
    lab = torch.full((2, 3), 4, device="cuda")
    ref = torch.zeros(2, device="cuda")
    for rejected, eps, want in ((True, 0.0, 0.0), (False, 1.0, 0.0), (False, 0.0, float("inf")),
                                (True, 0.25, float("inf"))):
        x = torch.randn(2, 3, 10, device="cuda")
        x[int(rejected), 1, 4] = float("-inf")
        x.requires_grad_(True)
        loss = mogt_b200.preference_loss(x, lab, ref, label_smoothing=eps)
        assert float(loss.detach()) == want, (rejected, eps, float(loss.detach()))
        g, = torch.autograd.grad(loss, x)
        assert bool(torch.isfinite(g).all())
        if want == 0.0:
            assert bool((g == 0).all())


def _address(t):
    """Offsets from a 16-byte boundary of every row."""
    e = t.element_size()
    at = torch.arange(t.shape[0])[:, None] * t.stride(0) + torch.arange(t.shape[1])[None] * t.stride(1)
    return (t.data_ptr() + at * e) % 16


@pytest.mark.parametrize("dtype,V", [(BF16, 1001), (F32, 1001), (F16, 515), (BF16, 1024)])
@pytest.mark.parametrize("cut", ["last", "first", "vocabulary", "every_fourth", "one_row", "expanded"])
def test_gradients_of_sliced_logits(dtype, V, cut):
    """The gradient's rows start at the logits' offsets from a 16-byte boundary
    (both are then accessed 16 bytes at a time), in no more memory than its own
    rows with up to 15 bytes between them take; its values are those of a dense
    copy."""
    import mogt_b200
    g = torch.Generator(device="cuda").manual_seed(3)
    full = torch.randn(4, 12, V, generator=g, device="cuda").to(dtype)
    x = {"last": lambda: full[:, :-1], "first": lambda: full[:, 1:], "vocabulary": lambda: full[..., 7:107],
         "every_fourth": lambda: full[:, ::4], "one_row": lambda: full[:, 5:6],
         "expanded": lambda: full[:1].expand(4, -1, -1)}[cut]()
    B, L, n = x.shape
    lab = torch.randint(0, n, (B, L), generator=g, device="cuda")
    adv = torch.randn(B, generator=g, device="cuda")
    old = torch.full((B, L), -7.0, device="cuda")

    def grads(v):
        v = v.detach().requires_grad_(True)
        out = [torch.autograd.grad(mogt_b200.policy_loss(v, lab, old, adv), v)[0],
               torch.autograd.grad(mogt_b200.token_logprobs(v, lab).sum(), v)[0],
               torch.autograd.grad(mogt_b200.preference_loss(v, lab, adv), v)[0]]
        return out

    dense = grads(x.contiguous())
    for a, b in zip(grads(x), dense):
        # sums over a row go by its alignment: each side is good to TOL32 and one rounding
        assert max_err(a, b) <= TOL32 + 2 * ROUND[dtype]
        assert torch.equal(_address(a), _address(x))
        assert a.untyped_storage().nbytes() <= (B * L * n) * a.element_size() + 16 * (B * L + B + 1)


def test_reference_sums_in_float64():
    """Sums near -40000, where one unit of 32 bits is 4e-3: given in float64
    they are used as they are.  The pair's logits are then good to the
    log-probabilities' own errors (see above)."""
    import mogt_b200
    B, L, V, beta = 4, 3000, 50, 0.1
    t = make(B, L, V, F32, seed=5, mask=False)
    t["logits"] = t["logits"] - 10 * torch.nn.functional.one_hot(t["labels"], V)
    x = t["logits"].detach().requires_grad_(True)
    x64 = t["logits"].double().requires_grad_(True)
    s = torch.log_softmax(x64.detach(), -1).gather(-1, t["labels"][..., None])[..., 0].sum(-1)
    ref = s + torch.tensor([3.001, -1.002, 0.5003, 2.0004], dtype=torch.float64, device="cuda")
    loss = mogt_b200.preference_loss(x, t["labels"], ref, beta=beta)
    loss64, _ = preference_ref(x64, t["labels"], t["counts"], ref, beta, 0.0)
    tol = (2 * L) ** 0.5 * 2.0 ** -19 * beta
    assert abs(float(loss.detach()) - float(loss64.detach())) <= tol
    g, g64 = torch.autograd.grad(loss, x)[0], torch.autograd.grad(loss64, x64)[0]
    assert max_err(g, g64) <= tol + TOL32
