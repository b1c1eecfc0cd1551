"""The selective operators' and losses' plans for larger calls against their
float64 forms: runs of tokens longer than the shortest, sequences split into
segments (ragged, unaligned, many states), four sequences a thread, row kernels
of every CTA size and the counting launch."""
import pytest
import torch

from .selective_ref import ROUND, logprobs_ref, max_err, preference_ref, scan_ref, scan_tol
from .test_gpu_causal_conv import both, tol
from .test_gpu_causal_conv import make as make_conv
from .test_gpu_lm_losses import TOL32, make as make_rows, policy
from .test_gpu_selective_scan import compare, make, ref, run

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# --------------------------------------------------------------------------
# convolution: a run is a 148 x CTAs x 128-th of all (token, access) pairs, 24 at least
# --------------------------------------------------------------------------
@pytest.mark.parametrize("B,L,D,K,dtype,opt", [
    (2, 3200, 2048, 4, BF16, {}),                                   # 8-byte accesses, runs of 29 and 58 tokens
    (4, 1777, 770, 3, F32, dict(init=True, wide=2)),                # 8-byte accesses, runs of 25 and 49
    (3, 1201, 1021, 2, F16, dict(init=True)),                       # single elements, runs of 33 and 65
    (5, 1301, 2044, 4, BF16, dict(init=True, lengths=[1301, 0, 1, 59, 1300])),
])
def test_long_runs(B, L, D, K, dtype, opt):
    got, want, names = both(make_conv(B, L, D, K, dtype, F32, **opt))
    for a, b, n in zip(got, want, names):
        assert a.shape == b.shape and max_err(a, b) <= tol(a.dtype, B * L), (n, max_err(a, b))


# --------------------------------------------------------------------------
# scan: few channels and many tokens make segments
# --------------------------------------------------------------------------
def _split(t):
    """Whether a forward of these sizes is split (its scratch holds the segments' carries)."""
    from mogt_b200 import _native as N
    B, L, D = t["u"].shape
    return N.lib().mogt_selective_fwd_scratch_bytes(B, L, D, t["A"].shape[1], t["B"].shape[2]) > 0


@pytest.mark.parametrize("D,N,G,dtype,opt", [
    (24, 16, 1, F32, {}),
    (24, 16, 1, BF16, dict(wide=True)),
    (33, 13, 1, F32, dict(z=False)),          # a channel without a neighbour
    (34, 4, 2, BF16, dict(skip=False)),       # groups of 17
    (12, 1, 3, F16, {}),
    (20, 33, 2, F32, {}),
    (12, 64, 1, BF16, {}),
    (9, 128, 1, F32, dict(wide=True)),
])
def test_segments_of_a_ragged_batch(D, N, G, dtype, opt):
    """Sequences that are empty, end in the first tile, inside a segment, at a
    segment's start, and behind it; states in and out, gradients through both."""
    t = make(6, 600, D, N, G, dtype, init=True, lengths=[0, 1, 130, 160, 599, 600], **opt)
    assert _split(t)
    got = run(t)
    compare(got, ref(t), 600)
    assert torch.equal(got["state"][0], t["init"][0]) and bool((got["y"][0] == 0).all())
    assert bool((got["du"][2, 130:] == 0).all()) and bool((got["ddelta"][3, 160:] == 0).all())
    assert bool((got["dB"][2, 130:] == 0).all()) and bool((got["dC"][1, 1:] == 0).all())


@pytest.mark.parametrize("N", [4, 16, 64])
def test_a_step_of_zero_keeps_every_bit(N):
    """dt = 0 is a decay of exactly 1: over thousands of tokens, over segment
    chains and in the adjoint, a state and its gradient pass unchanged."""
    L = 5000
    t = make(2, L, 16, N, 1, F32, init=True, bias=False)
    t["delta"][:] = -200.0            # softplus(-200) is 0 in 32 bits
    t["A"] *= 1000.0
    t["dout"][:] = 0
    assert _split(t)
    got = run(t)
    assert torch.equal(got["state"], t["init"]) and torch.equal(got["dinit"], t["dfinal"])


def test_long_memories():
    """A state that remembers m tokens adds up what m steps are off by.  An
    exponential and a multiply-add, each rounded to 24 bits and to either side
    alike, leave sqrt(2 m) 2^-24 / sqrt(3); four standard deviations of it are
    the bar.  An exponential that is low by 2e-8 on average, as the
    instruction is near 1, would be off by m times that, five times the bar.
    dD sums 4096 terms of both signs to about 64 times one: 256 tiles' sums of
    16 (about 4 terms large, off by 4 x 2^-25 of that each), 16 x 16 x 2^-25 /
    64, again four times that."""
    t = make(1, 4096, 64, 16, 1, F32, init=True, z=False)
    t["bias"] = torch.full_like(t["bias"], -6.0)
    t["delta"] *= 0.2
    t["A"] = -0.2 - 0.3 * torch.rand_like(t["A"])     # dt A of 5e-4 to 1.2e-3
    got, want = run(t), ref(t)
    bar = 4 * (2 * 2000) ** 0.5 * 2.0 ** -24 / 3 ** 0.5
    for k, most in dict(y=bar, state=bar, dA=bar, dbias=bar, dD=16 * 2.0 ** -25).items():
        assert max_err(got[k], want[k]) <= most, (k, max_err(got[k], want[k]), most)


@pytest.mark.parametrize("B,D,N,G,dtype", [
    (401, 300, 13, 1, F32),       # 4010 CTAs' worth of sequences: four at a time, one left over
    (1202, 256, 4, 2, BF16),      # two left over
    (203, 768, 16, 1, BF16),      # three left over, 16-byte states
    (100, 200, 64, 1, F16),
    (97, 100, 128, 1, F32),
])
@pytest.mark.parametrize("in_place", [True, False])
def test_step_of_a_large_batch(B, D, N, G, dtype, in_place):
    import mogt_b200
    t = make(B, 1, D, N, G, dtype, init=True)
    y64, h64 = scan_ref(*[t[k].double() for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")], True,
                        t["init"].double())
    state = t["init"].clone()
    new = state if in_place else torch.full_like(state, float("nan"))
    y = mogt_b200.selective_scan_step(state, t["u"][:, 0], t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0],
                                      D=t["D"], z=t["z"][:, 0], delta_bias=t["bias"], delta_softplus=True,
                                      new_state=None if in_place else new)
    assert max_err(y, y64[:, 0]) <= scan_tol(dtype, 1) and max_err(new, h64) <= scan_tol(F32, 1)
    if not in_place:
        assert torch.equal(state, t["init"])


# --------------------------------------------------------------------------
# losses: CTAs of 256 or 512 threads from 296 rows on, a counting launch from 1025 rows on
# --------------------------------------------------------------------------
ROWS = [(6, 61, 513, F32, dict(pad=3)), (6, 61, 4099, F16, dict(nan=True)), (4, 300, 257, BF16, dict(pad=1)),
        (4, 300, 1021, F32, dict(nan=True)), (2, 1500, 8200, BF16, {}), (4, 256, 100, F32, {}), (4, 257, 100, F32, {})]


@pytest.mark.parametrize("B,L,V,dtype,opt", ROWS)
def test_policy_of_many_rows(B, L, V, dtype, opt):
    import mogt_b200
    t = make_rows(B, L, V, dtype, **opt)
    x, loss, lp, x64, loss64, lp64 = policy(t, dtype)
    assert abs(float(loss.detach()) - float(loss64.detach())) <= TOL32 * max(1.0, abs(float(loss64.detach())))
    assert max_err(lp, lp64) <= TOL32
    with torch.no_grad():   # the row kernel without a gradient
        other = mogt_b200.policy_loss(t["logits"], t["labels"], t["old"], t["adv"], ref_logprobs=t["ref"],
                                      mask=t["mask"], clip_low=0.2, clip_high=0.3, kl_coef=0.05)
    assert abs(float(other) - float(loss64.detach())) <= TOL32 * max(1.0, abs(float(loss64.detach())))
    g64, = torch.autograd.grad(loss64, x64)
    floor = 2.0 ** -25 / float(g64.abs().max()) if dtype == F16 else 0.0
    for scale in (1.0, 3.0):   # the forward's gradient, and the one formed again
        g, = torch.autograd.grad(loss, x, torch.tensor(scale, device="cuda"), retain_graph=True)
        assert max_err(g, scale * g64) <= TOL32 + ROUND[dtype] + floor, scale
        assert bool((g[~t["counts"]] == 0).all())


@pytest.mark.parametrize("B,L,V,dtype,opt", ROWS)
def test_preference_and_logprobs_of_many_rows(B, L, V, dtype, opt):
    import mogt_b200
    t = make_rows(B, L, V, dtype, **opt)
    x = t["logits"].detach().requires_grad_(True)
    x64 = torch.nan_to_num(t["logits"].detach().double()).requires_grad_(True)
    lp, lp64 = mogt_b200.token_logprobs(x, t["labels"], mask=t["mask"]), logprobs_ref(x64, t["labels"], t["counts"])
    assert max_err(lp, lp64) <= TOL32
    w = torch.randn(B, L, device="cuda")
    g, g64 = torch.autograd.grad(lp, x, w)[0], torch.autograd.grad(lp64, x64, w.double())[0]
    assert max_err(g, g64) <= TOL32 + ROUND[dtype]
    loss, seq = mogt_b200.preference_loss(x, t["labels"], t["sref"], beta=0.1, label_smoothing=0.1, mask=t["mask"],
                                          return_logprobs=True)
    loss64, seq64 = preference_ref(x64, t["labels"], t["counts"], t["sref"].double(), 0.1, 0.1)
    # the errors of 2 L log-probabilities add up like independent ones
    moved = (2 * L) ** 0.5 * 2.0 ** -19 * 0.1
    assert abs(float(loss.detach()) - float(loss64.detach())) <= moved and max_err(seq, seq64) <= TOL32
    g, g64 = torch.autograd.grad(loss, x)[0], torch.autograd.grad(loss64, x64)[0]
    floor = 2.0 ** -25 / float(g64.abs().max()) if dtype == F16 else 0.0
    assert max_err(g, g64) <= moved + TOL32 + ROUND[dtype] + floor
