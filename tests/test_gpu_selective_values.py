"""Selective scan where its values are delicate: steps masked by the lowest
values there are, states that grow, and decays that are remembered for long."""
import pytest
import torch

from .selective_ref import max_err, scan_ref, scan_tol
from .test_gpu_selective_scan import compare, make, ref, run

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_steps_masked_by_the_lowest_value(dtype, low):
    """delta = -inf or the type's lowest value: no step, no gradient."""
    t = make(2, 70, 24, 16, 1, dtype, init=True)
    t["delta"][:, 3::7] = float("-inf") if low == "inf" else torch.finfo(dtype).min
    t["delta"][1, 16:48] = t["delta"][0, 3]      # whole tiles
    got = run(t)
    want = ref_masked(t)
    assert bool((got["ddelta"][:, 3::7] == 0).all())
    compare(got, want, 70)


def ref_masked(t):
    """The definition, with -1e4 (a step of exactly 0 in 64 bits) for the masks: inf - inf is not formed."""
    return ref(dict(t, delta=t["delta"].double().clamp(min=-1e4)))


def test_single_token_masked_by_the_lowest_value():
    import mogt_b200
    t = make(2, 1, 24, 16, 1, BF16, init=True)
    t["delta"][0] = float("-inf")
    t["delta"][1] = torch.finfo(BF16).min
    st = t["init"].clone()
    mogt_b200.selective_scan_step(st, t["u"][:, 0], t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0],
                                  delta_bias=t["bias"], delta_softplus=True)
    assert torch.equal(st, t["init"])


def test_a_step_as_large_as_the_type_allows():
    """softplus(x) = x up to the largest value: the state becomes dt u B, at once."""
    import mogt_b200
    big = torch.finfo(F32).max
    one = torch.ones(1, 1, 1, device="cuda")
    y, h = mogt_b200.selective_scan(one * 2.0 ** -20, one * big, -one[0], one, one, delta_softplus=True,
                                    return_state=True)
    assert float(y) == float(h) == big * 2.0 ** -20


def _growing(L, G=1):
    """exp(dt A) = e^2 a token: over a segment of 64 tokens or more the decay alone overflows."""
    t = make(1, L, 8, 4, G, F32, z=False, skip=False, bias=False)
    t["A"] = torch.full_like(t["A"], 2.0)
    t["delta"] = torch.ones_like(t["delta"])
    return t


def test_growing_states_start_from_nothing():
    """Zero inputs up to the last 20 tokens, and gradients of the first 20
    outputs only: all values are far from the largest, on either way."""
    t = _growing(4096)
    t["u"][:, :-20] = 0
    t["dout"][:, 20:] = 0
    t["dfinal"] = torch.zeros_like(t["dfinal"])
    compare(run(t, softplus=False), ref(t, softplus=False), 20)


def test_growing_states_that_fit():
    """A state of 1e-30 that grows by e^128 over a segment, and stays below
    3e38.  The exponents' rounding (2^-17 of exponents up to 256) is all of the
    error beyond the steps'."""
    import mogt_b200
    L = 4040
    t = _growing(4096)
    t["u"][:] = 0
    t["u"][:, 3967] = 1e-30
    lengths = torch.tensor([L], device="cuda")
    args = [t[k] for k in ("u", "delta", "A", "B", "C")]
    y, h = mogt_b200.selective_scan(*args, lengths=lengths, return_state=True)
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(h).all())
    y64, h64 = scan_ref(*[a.double() for a in args], softplus=False, lengths=lengths)
    assert max_err(y, y64) <= 2.0 ** -15 and max_err(h, h64) <= 2.0 ** -15
