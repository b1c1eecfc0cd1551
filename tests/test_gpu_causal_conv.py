"""Short causal convolution against its float64 form: outputs, last inputs
and gradients over types, widths, lengths and layouts; the single-token form."""
import pytest
import torch

from .selective_ref import ROUND, conv_ref, max_err

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(B, L, D, K, dtype, pdtype, seed=0, bias=True, init=False, lengths=None, wide=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    t = dict(x=rn(B, L, D + wide).to(dtype)[..., wide:], w=rn(D, K).to(pdtype), b=rn(D).to(pdtype) if bias else None,
             init=rn(B, K - 1, D).to(dtype) if init else None, dy=rn(B, L, D + wide).to(dtype)[..., wide:],
             dfinal=rn(B, K - 1, D).to(dtype), lengths=None)
    if lengths is not None:
        t["lengths"] = torch.tensor(lengths, device="cuda")
        dead = torch.arange(L, device="cuda")[None] >= t["lengths"].clamp(0, L)[:, None]
        t["x"].masked_fill_(dead[..., None], float("nan"))
        t["dy"].masked_fill_(dead[..., None], float("nan"))
    return t


def both(t, activation="silu"):
    import mogt_b200
    names = [k for k in ("x", "w", "b", "init") if t[k] is not None]
    leaf = {k: t[k].detach().requires_grad_(True) if t[k] is not None else None for k in ("x", "w", "b", "init")}
    y, f = mogt_b200.causal_conv(leaf["x"], leaf["w"], leaf["b"], activation=activation, initial_state=leaf["init"],
                                 lengths=t["lengths"], return_state=True)
    g = torch.autograd.grad((y, f), [leaf[k] for k in names], (t["dy"], t["dfinal"]))
    clean = lambda v: torch.nan_to_num(v.detach().double())
    l64 = {k: clean(t[k]).requires_grad_(True) if t[k] is not None else None for k in ("x", "w", "b", "init")}
    y64, f64 = conv_ref(l64["x"], l64["w"], l64["b"], l64["init"], t["lengths"], activation == "silu")
    g64 = torch.autograd.grad((y64, f64), [l64[k] for k in names], (clean(t["dy"]), clean(t["dfinal"])),
                              allow_unused=True)
    g64 = [torch.zeros_like(l64[k]) if v is None else v for k, v in zip(names, g64)]
    return [y, f] + list(g), [y64, f64] + list(g64), ["y", "final"] + ["d" + k for k in names]


def tol(dtype, tokens):
    # K products per value; a weight's gradient sums `tokens` of them
    return ROUND[dtype] + (16 + tokens ** 0.5) * 2.0 ** -22


@pytest.mark.parametrize("B,L,D,K,dtype,pdtype,opt", [
    (1, 1, 1, 2, F32, F32, {}),
    (2, 1, 16, 4, BF16, BF16, dict(init=True)),
    (2, 2, 24, 4, F32, F32, dict(init=True)),
    (1, 3, 9, 3, F16, F32, dict(bias=False)),
    (3, 17, 770, 3, F32, F32, dict(init=True, wide=2)),
    (2, 129, 1536, 4, BF16, F32, dict(wide=8)),
    (2, 300, 100, 2, F16, F16, dict(init=True, wide=1)),
    (1, 5000, 64, 4, BF16, F32, {}),
    (4, 1000, 12, 4, F32, F32, dict(init=True, wide=3)),
])
def test_against_definition(B, L, D, K, dtype, pdtype, opt):
    got, want, names = both(make(B, L, D, K, dtype, pdtype, **opt))
    for a, b, n in zip(got, want, names):
        assert a.shape == b.shape and max_err(a, b) <= tol(a.dtype, B * L), (n, max_err(a, b))


@pytest.mark.parametrize("K", [2, 3, 4])
def test_ragged_batch(K):
    t = make(7, 40, 20, K, F32, F32, init=True, lengths=[0, 1, 2, 3, 16, 40, 99])
    got, want, names = both(t)
    for a, b, n in zip(got, want, names):
        assert max_err(a, b) <= tol(F32, 280), n
    assert torch.equal(got[1][0], t["init"][0])


def test_no_activation_and_no_tokens():
    got, want, names = both(make(2, 50, 33, 4, F32, F32), activation=None)
    for a, b, n in zip(got, want, names):
        assert max_err(a, b) <= tol(F32, 100), n
    t = make(2, 0, 8, 4, F32, F32, init=True)
    got, want, names = both(t)
    assert torch.equal(got[1], t["init"]) and torch.equal(got[-1], t["dfinal"]) and bool((got[3] == 0).all())


def test_dense_copy_of_other_layouts():
    import mogt_b200
    t = make(2, 60, 24, 4, BF16, F32)
    x = t["x"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(mogt_b200.causal_conv(x, t["w"], t["b"]), mogt_b200.causal_conv(t["x"], t["w"], t["b"]))


def test_rows_beyond_32_bit_offsets():
    import mogt_b200
    step, L, D = 2 ** 31 + 64, 50, 32
    t = make(2, L, D, 4, BF16, F32)
    x = torch.empty(step + L * D, dtype=BF16, device="cuda").as_strided((2, L, D), (step, D, 1))
    x.copy_(t["x"])
    assert torch.equal(mogt_b200.causal_conv(x, t["w"], t["b"]), mogt_b200.causal_conv(t["x"], t["w"], t["b"]))


def test_prompt_then_single_tokens():
    import mogt_b200
    t = make(3, 40, 50, 4, BF16, BF16)
    full, last = mogt_b200.causal_conv(t["x"], t["w"], t["b"], return_state=True)
    for start in (0, 1, 2, 37):
        y, st = mogt_b200.causal_conv(t["x"][:, :start], t["w"], t["b"], return_state=True)
        for s in range(start, 40):
            before = st.clone()
            kept = torch.empty_like(st)
            y2 = mogt_b200.causal_conv_step(t["x"][:, s], st, t["w"], t["b"], new_state=kept)
            assert torch.equal(before, st)
            y = mogt_b200.causal_conv_step(t["x"][:, s], st, t["w"], t["b"])
            assert torch.equal(y, y2) and torch.equal(st, kept)
            assert torch.equal(y, full[:, s])
        assert torch.equal(st, last)


def test_two_runs_agree_to_the_bit():
    t = make(4, 900, 192, 4, BF16, F32, init=True)
    a, b = both(t)[0], both(t)[0]
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradients_against_differences():
    """Central differences over 1e-2 of the kernel's fp32 forward: 1e-3."""
    import mogt_b200
    t = make(1, 30, 16, 4, F32, F32, init=True)
    got, _, names = both(t)
    g = dict(zip(names, got))
    for k in ("x", "w", "b", "init"):
        v = g["d" + k] / g["d" + k].norm()

        def value(s):
            p = {n: t[n] + s * v if n == k else t[n] for n in ("x", "w", "b", "init")}
            y, f = mogt_b200.causal_conv(p["x"], p["w"], p["b"], initial_state=p["init"], return_state=True)
            return float((y.double() * t["dy"].double()).sum() + (f.double() * t["dfinal"].double()).sum())

        num = (value(1e-2) - value(-1e-2)) / 2e-2
        ana = float((g["d" + k].double() * v.double()).sum())
        assert abs(num - ana) <= 1e-3 * abs(ana), (k, num, ana)


def test_refusals():
    import mogt_b200
    conv, step = mogt_b200.causal_conv, mogt_b200.causal_conv_step
    x, w, b = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(8, 4, device="cuda"), torch.zeros(8, device="cuda")
    st = torch.zeros(2, 3, 8, device="cuda")
    for match, call in [
            ("x must be", lambda: conv(x[0], w)),
            ("x must be", lambda: conv(x.double(), w)),
            ("weight must be", lambda: conv(x, w[:4])),
            ("K must be", lambda: conv(x, torch.zeros(8, 5, device="cuda"))),
            ("bias must be", lambda: conv(x, w, b[:3])),
            ("bias must be", lambda: conv(x, w, b.bfloat16())),
            ("activation", lambda: conv(x, w, b, activation="gelu")),
            ("initial_state", lambda: conv(x, w, b, initial_state=st[:, :2])),
            ("initial_state", lambda: conv(x, w, b, initial_state=st.bfloat16())),
            ("lengths", lambda: conv(x, w, b, lengths=torch.zeros(2, device="cuda"))),
            ("CUDA", lambda: conv(x, w.cpu(), b)),
            ("x must be", lambda: step(x, st, w)),
            ("state must be", lambda: step(x[:, 0], st[:, :2].contiguous(), w)),
            ("state must be", lambda: step(x[:, 0], torch.zeros(2, 8, 3, device="cuda").transpose(1, 2), w)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
