"""Selective scan against its float64 token-by-token form: outputs, states and
every gradient, over types, group and state counts, lengths from none to many
tiles, ragged batches, strided operands, and the single-token form."""
import pytest
import torch

from .selective_ref import max_err, scan_ref, scan_tol

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(B, L, D, N, G, dtype, seed=0, z=True, skip=True, bias=True, init=False, lengths=None, wide=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    extra = 3 if wide else 0                     # strided rows: views of wider tensors
    act = lambda scale=1.0: (rn(B, L, D + extra) * scale).to(dtype)[..., extra:]
    grp = lambda: rn(B, L, G * N + extra).to(dtype)[..., extra:].unflatten(-1, (G, N))
    t = dict(u=act(), delta=act(0.5), A=-torch.rand(D, N, generator=g, device="cuda") * 4 - 0.1, B=grp(), C=grp())
    t["D"] = rn(D) if skip else None
    t["z"] = act() if z else None
    t["bias"] = rn(D) - 2.0 if bias else None
    t["init"] = rn(B, D, N) if init else None
    t["dout"], t["dfinal"] = rn(B, L, D).to(dtype), rn(B, D, N)
    if lengths is not None:
        lengths = torch.tensor(lengths, device="cuda")
        dead = torch.arange(L, device="cuda")[None] >= lengths.clamp(0, L)[:, None]
        for k in ("u", "delta", "B", "C", "z", "dout"):
            if t[k] is not None:
                t[k].masked_fill_(dead.view(B, L, *([1] * (t[k].ndim - 2))), float("nan"))
    t["lengths"] = lengths
    return t


def run(t, softplus=True, grads=True):
    import mogt_b200
    names = [k for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "init") if t[k] is not None]
    leaf = {k: t[k].detach().requires_grad_(grads) if t[k] is not None else None for k in
            ("u", "delta", "A", "B", "C", "D", "z", "bias", "init")}
    y, h = mogt_b200.selective_scan(leaf["u"], leaf["delta"], leaf["A"], leaf["B"], leaf["C"], D=leaf["D"], z=leaf["z"],
                                    delta_bias=leaf["bias"], delta_softplus=softplus, initial_state=leaf["init"],
                                    lengths=t["lengths"], return_state=True)
    out = {"y": y.detach(), "state": h.detach()}
    if grads:
        for k, v in zip(names, torch.autograd.grad((y, h), [leaf[k] for k in names], (t["dout"], t["dfinal"]))):
            out["d" + k] = v
    return out


def ref(t, softplus=True):
    names = [k for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "init") if t[k] is not None]
    clean = lambda v: torch.nan_to_num(v.detach().double())
    leaf = {k: clean(t[k]).requires_grad_(True) if t[k] is not None else None for k in
            ("u", "delta", "A", "B", "C", "D", "z", "bias", "init")}
    y, h = scan_ref(leaf["u"], leaf["delta"], leaf["A"], leaf["B"], leaf["C"], leaf["D"], leaf["z"], leaf["bias"],
                    softplus, leaf["init"], t["lengths"])
    g = torch.autograd.grad((y, h), [leaf[k] for k in names], (clean(t["dout"]), t["dfinal"].double()),
                            allow_unused=True)
    out = {"y": y, "state": h}
    for k, v in zip(names, g):
        out["d" + k] = torch.zeros_like(leaf[k]) if v is None else v
    return out


def compare(got, want, steps):
    for k in want:
        assert got[k].shape == want[k].shape, k
        tol = scan_tol(got[k].dtype, steps)
        assert max_err(got[k], want[k]) <= tol, (k, max_err(got[k], want[k]), tol)


SHAPES = [
    # B, L, D, N, G, dtype, options
    (1, 1, 1, 1, 1, F32, {}),
    (2, 1, 64, 16, 1, BF16, dict(init=True)),
    (2, 7, 33, 4, 1, F32, dict(init=True)),
    (1, 16, 8, 5, 2, F32, dict(z=False)),
    (3, 17, 130, 16, 1, BF16, dict(wide=True)),
    (2, 33, 6, 8, 3, F16, dict(skip=False)),
    (2, 100, 96, 13, 2, F32, dict(init=True, wide=True)),
    (1, 300, 200, 16, 1, F32, dict(bias=False)),
    (1, 1025, 40, 16, 1, BF16, dict(init=True)),
    (2, 65, 20, 33, 1, F32, dict(init=True)),
    (1, 50, 24, 64, 2, BF16, dict(z=False, skip=False)),
    (1, 40, 9, 128, 1, F32, dict(init=True)),
    (2, 515, 256, 2, 2, F32, {}),
]


@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "-".join(str(v) for v in c[:5]) + f"-{c[5]}"[-9:])
def test_against_definition(case):
    B, L, D, N, G, dtype, opt = case
    t = make(B, L, D, N, G, dtype, **opt)
    compare(run(t), ref(t), L)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ragged_batch(dtype):
    t = make(7, 70, 36, 16, 2, dtype, init=True, lengths=[0, 1, 15, 16, 17, 70, 100])
    got, want = run(t), ref(t)
    compare(got, want, 70)
    assert bool((got["y"][0] == 0).all()) and torch.equal(got["state"][0], t["init"][0])
    assert bool((got["du"][1, 1:] == 0).all()) and bool((got["dB"][2, 15:] == 0).all())


def test_lengths_int32_and_negative_are_clamped():
    t = make(2, 20, 16, 4, 1, F32, init=True)
    t["lengths"] = torch.tensor([-5, 9], dtype=torch.int32, device="cuda")
    compare(run(t), ref(t), 20)


def test_no_tokens():
    t = make(2, 0, 24, 16, 1, BF16, init=True)
    got = run(t)
    assert torch.equal(got["state"], t["init"]) and torch.equal(got["dinit"], t["dfinal"])
    assert got["y"].shape == (2, 0, 24) and bool((got["dA"] == 0).all()) and bool((got["dD"] == 0).all())
    empty = make(0, 5, 24, 16, 1, BF16)
    assert run(empty)["y"].shape == (0, 5, 24)


def test_without_softplus():
    t = make(1, 60, 48, 16, 1, F32, bias=False)
    t["delta"] = t["delta"].abs() * 0.2
    compare(run(t, softplus=False), ref(t, softplus=False), 60)


def test_extreme_steps():
    """delta far out on both sides: no decay at all, and a state that is
    forgotten at once (exp underflows to 0)."""
    t = make(2, 64, 32, 16, 1, F32, init=True, bias=False)
    t["delta"][:, ::3] = -80.0
    t["delta"][:, 1::3] = 60.0
    compare(run(t), ref(t), 64)


def test_layouts_are_copied_when_not_dense():
    t = make(2, 40, 32, 16, 1, F32, init=True)
    want = run(t)
    for k in ("u", "delta", "z"):
        t[k] = t[k].transpose(1, 2).contiguous().transpose(1, 2)     # [B, D, L] in memory
    t["B"] = t["B"].transpose(2, 3).contiguous().transpose(2, 3)
    t["C"] = t["C"].flip(-1).flip(-1).transpose(1, 3).contiguous().transpose(1, 3)
    t["dout"] = t["dout"].transpose(1, 2).contiguous().transpose(1, 2)
    got = run(t)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_expanded_operands():
    """B and C broadcast over the batch (stride 0) and one row for all tokens."""
    t = make(3, 30, 16, 4, 1, F32)
    t["B"], t["C"] = t["B"][:1].expand(3, -1, -1, -1), t["C"][:, :1].expand(-1, 30, -1, -1)
    compare(run(t), ref(t), 30)


def test_rows_beyond_32_bit_offsets():
    """The second sequence starts more than 2^31 elements behind the first."""
    import mogt_b200
    L, D, N = 20, 32, 16
    step = 2 ** 31 + 64
    t = make(2, L, D, N, 1, BF16, lengths=None)
    base = torch.empty(step + L * D, dtype=BF16, device="cuda")
    far = {}
    for i, k in enumerate(("u", "delta", "z")):
        far[k] = base.as_strided((2, L, D), (step, D, 1))
        far[k].copy_(t[k])
        y = mogt_b200.selective_scan(*[far[k] if n == k else t[n] for n in ("u", "delta", "A", "B", "C")], D=t["D"],
                                     z=far[k] if k == "z" else t["z"], delta_bias=t["bias"], delta_softplus=True)
        w = mogt_b200.selective_scan(*[t[n] for n in ("u", "delta", "A", "B", "C")], D=t["D"], z=t["z"],
                                     delta_bias=t["bias"], delta_softplus=True)
        assert torch.equal(y, w), k


def test_segments_of_a_long_sequence_join():
    """Two calls with the state handed over equal one call; so do prompts
    followed by single tokens."""
    import mogt_b200
    t = make(2, 700, 64, 16, 1, F32)
    kw = dict(D=t["D"], delta_bias=t["bias"], delta_softplus=True)
    cut = lambda a, b: [t["u"][:, a:b], t["delta"][:, a:b], t["A"], t["B"][:, a:b], t["C"][:, a:b]]
    full, hf = mogt_b200.selective_scan(*cut(0, 700), z=t["z"], return_state=True, **kw)
    y1, h1 = mogt_b200.selective_scan(*cut(0, 333), z=t["z"][:, :333], return_state=True, **kw)
    y2, h2 = mogt_b200.selective_scan(*cut(333, 700), z=t["z"][:, 333:], initial_state=h1, return_state=True, **kw)
    tol = scan_tol(F32, 700)
    assert max_err(torch.cat([y1, y2], 1), full) <= tol and max_err(h2, hf) <= tol
    y, h = mogt_b200.selective_scan(*cut(0, 690), z=t["z"][:, :690], return_state=True, **kw)
    for s in range(690, 700):
        y = mogt_b200.selective_scan_step(h, t["u"][:, s], t["delta"][:, s], t["A"], t["B"][:, s], t["C"][:, s],
                                          z=t["z"][:, s], **kw)
        assert max_err(y, full[:, s]) <= tol
    assert max_err(h, hf) <= tol


@pytest.mark.parametrize("B,D,N,G,dtype", [(1, 1, 1, 1, F32), (3, 70, 16, 1, BF16), (2, 48, 13, 2, F32),
                                           (5, 36, 64, 3, F16), (1, 8, 128, 1, F32), (2, 20, 6, 1, BF16)])
def test_step_against_definition(B, D, N, G, dtype):
    import mogt_b200
    t = make(B, 1, D, N, G, dtype, init=True, wide=True)
    y64, h64 = scan_ref(*[t[k].double() for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")], True,
                        t["init"].double())
    state, keep = t["init"].clone(), torch.empty_like(t["init"])
    kw = dict(D=t["D"], z=t["z"][:, 0], delta_bias=t["bias"], delta_softplus=True)
    args = [t["u"][:, 0], t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0]]
    y = mogt_b200.selective_scan_step(state, *args, new_state=keep, **kw)
    assert torch.equal(state, t["init"])
    assert max_err(y, y64[:, 0]) <= scan_tol(dtype, 1) and max_err(keep, h64) <= scan_tol(F32, 1)
    y2 = mogt_b200.selective_scan_step(state, *args, **kw)
    assert torch.equal(y, y2) and torch.equal(state, keep)


def test_gradients_against_differences():
    """Directional derivative by central differences of the kernel's own
    forward.  The forward's error of about 2^-20 of the sum over a step of
    2e-3 gives 5e-4, the truncation about as much: 5e-3 relative."""
    import mogt_b200
    t = make(1, 48, 64, 16, 1, F32, init=True)
    g = run(t)
    gen = torch.Generator(device="cuda").manual_seed(9)
    names = ("u", "delta", "A", "B", "C", "D", "z", "bias", "init")

    def value(s):
        p = {k: t[k] + s * v[k] for k in names}
        y, h = mogt_b200.selective_scan(p["u"], p["delta"], p["A"], p["B"], p["C"], D=p["D"], z=p["z"],
                                        delta_bias=p["bias"], delta_softplus=True, initial_state=p["init"],
                                        return_state=True)
        return float((y.double() * t["dout"].double()).sum() + (h.double() * t["dfinal"].double()).sum())

    for k in names:
        v = {n: torch.zeros_like(t[n]) for n in names}
        # along the gradient itself: the derivative is its squared norm
        v[k] = g["d" + k] / g["d" + k].norm()
        eps = 2e-3 if k != "A" else 1e-2
        num = (value(eps) - value(-eps)) / (2 * eps)
        ana = float((g["d" + k].double() * v[k].double()).sum())
        assert abs(num - ana) <= 5e-3 * abs(ana), (k, num, ana)


def test_two_runs_agree_to_the_bit_and_on_another_stream():
    t = make(4, 300, 192, 16, 1, BF16, init=True)
    a, b = run(t), run(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = run(t)
    torch.cuda.current_stream().wait_stream(s)
    for k in a:
        assert torch.equal(a[k], b[k]) and torch.equal(a[k], c[k]), k


def test_gradient_of_one_output_alone():
    import mogt_b200
    t = make(1, 30, 16, 4, 1, F32)
    u = t["u"].clone().requires_grad_(True)
    y, h = mogt_b200.selective_scan(u, t["delta"], t["A"], t["B"], t["C"], return_state=True, delta_softplus=True)
    u64 = t["u"].double().requires_grad_(True)
    y64, h64 = scan_ref(u64, *[t[k].double() for k in ("delta", "A", "B", "C")])
    for got, want in ((h, h64), (y, y64)):
        a, = torch.autograd.grad(got.sum(), u, retain_graph=True)
        b, = torch.autograd.grad(want.sum(), u64, retain_graph=True)
        assert max_err(a, b) <= scan_tol(F32, 30)


def test_refusals():
    import mogt_b200
    t = make(2, 5, 8, 4, 1, F32)
    scan, step = mogt_b200.selective_scan, mogt_b200.selective_scan_step
    ok = [t[k] for k in ("u", "delta", "A", "B", "C")]

    def bad(match, i=None, v=None, **kw):
        a = list(ok)
        if i is not None:
            a[i] = v
        with pytest.raises(ValueError, match=match):
            scan(*a, **kw)

    bad("u must be", 0, t["u"][0])
    bad("u must be", 0, t["u"].double())
    bad("delta must have", 1, t["delta"][:, :4])
    bad("delta must have", 1, t["delta"].bfloat16())
    bad("A must be", 2, t["A"][:7])
    bad("N must be", 2, torch.zeros(8, 129, device="cuda"))
    bad("B and C must", 3, t["B"][:, :4])
    bad("one shape", 3, t["B"][..., :3])
    bad("B and C must have u's dtype", 4, t["C"].bfloat16())
    with pytest.raises(ValueError, match="number of groups"):
        scan(t["u"], t["delta"], t["A"], t["B"].repeat(1, 1, 3, 1), t["C"].repeat(1, 1, 3, 1))
    bad("z must have", z=t["z"][..., :4])
    bad("D must be", D=t["D"][:3])
    bad("delta_bias must be", delta_bias=t["bias"][:3])
    bad("initial_state must be", initial_state=torch.zeros(2, 8, 3, device="cuda"))
    bad("lengths must be", lengths=torch.zeros(3, dtype=torch.int64, device="cuda"))
    bad("lengths must be", lengths=torch.zeros(2, device="cuda"))
    bad("CUDA", 1, t["delta"].cpu())
    st = torch.zeros(2, 8, 4, device="cuda")
    a1 = [t["u"][:, 0], t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0]]
    for s in (st[:1], st.bfloat16(), st.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(ValueError, match="state must be"):
            step(s, *a1)
    with pytest.raises(ValueError, match="u must be"):
        step(st, *ok)
