"""The selective state space operators together: training form, prompts and
single tokens of the small language model agree, a training step's gradients
match the same model on the float64 forms, blocks stack in the MOGT backbone,
and the post-training example runs."""
import importlib.util
from pathlib import Path

import pytest
import torch

from .selective_ref import conv_ref, max_err, policy_ref, scan_ref

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


def _model(seed=0, **kw):
    from mogt_b200.selective_lm import SelectiveLM
    torch.manual_seed(seed)
    return SelectiveLM(97, 48, 2, **kw).cuda()


def test_prompts_and_tokens_match_the_training_form():
    """fp32 projections in different shapes, then the scan: 1e-4 of the
    largest logit (the repository's fp32 bar)."""
    m = _model()
    ids = torch.randint(0, 97, (3, 40), device="cuda")
    with torch.no_grad():
        full = m(ids)
        n = torch.tensor([1, 17, 33], device="cuda")
        logits, caches = m.prefill(ids[:, :33], n)
        for b in range(3):
            assert max_err(logits[b], full[b, n[b] - 1]) <= 1e-4
        for t in range(7):
            tok = ids[torch.arange(3, device="cuda"), n + t]
            logits = m.step(tok, caches)
            for b in range(3):
                assert max_err(logits[b], full[b, n[b] + t]) <= 1e-4, (t, b)


def test_a_token_step_in_a_cuda_graph():
    """A captured step replays on the same buffers like the calls themselves."""
    m = _model(2)
    ids = torch.randint(0, 97, (2, 12), device="cuda")
    _, caches = m.prefill(ids[:, :4])
    _, want = m.prefill(ids[:, :4])
    tok = ids[:, 4].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # warm-up on copies: a step changes the caches
        m.step(tok, [tuple(t.clone() for t in c) for c in caches])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = m.step(tok, caches)
    for t in range(4, 12):
        tok.copy_(ids[:, t])
        graph.replay()
        direct = m.step(ids[:, t], want)
        assert max_err(logits, direct) <= 1e-6
        for a, b in zip(caches, want):
            assert max_err(a[0], b[0]) <= 1e-6 and max_err(a[1], b[1]) <= 1e-6


def test_training_gradients_against_float64():
    """Every parameter's gradient of a policy step against the same network in
    float64 (token by token); fp32 projections dominate: 1e-4 relative."""
    import mogt_b200
    m = _model(1, d_state=5)
    ids = torch.randint(0, 97, (2, 21), device="cuda")
    labels = torch.randint(0, 97, (2, 21), device="cuda")
    mask = torch.rand(2, 21, device="cuda") < 0.8
    adv = torch.tensor([1.0, -0.5], device="cuda")
    with torch.no_grad():
        old = mogt_b200.token_logprobs(m(ids), labels, mask=mask) + 0.05
    loss = mogt_b200.policy_loss(m(ids), labels, old, adv, ref_logprobs=old - 0.1, mask=mask, kl_coef=0.1)
    got = dict(zip([n for n, _ in m.named_parameters()], torch.autograd.grad(loss, list(m.parameters()))))

    import copy
    d = copy.deepcopy(m).double()
    norm = lambda x, mod: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + mod.eps) * mod.weight
    x = d.embedding(ids)
    for blk in d.blocks:
        xz = blk.in_proj(norm(x, blk.norm))
        u, _ = conv_ref(xz[..., :blk.d_inner], blk.conv_weight, blk.conv_bias, None, None)
        dbc = blk.x_proj(u)
        delta, B, C = dbc.split([blk.rank, blk.d_state, blk.d_state], -1)
        y, _ = scan_ref(u, blk.dt_proj(delta), -torch.exp(blk.A_log), B[:, :, None], C[:, :, None], blk.D,
                        xz[..., blk.d_inner:], blk.dt_bias)
        x = x + blk.out_proj(y)
    logits = norm(x, d.norm_f) @ d.embedding.weight.t()
    loss64, _ = policy_ref(logits, labels, mask, old.double(), adv.double(), old.double() - 0.1, 0.2, 0.2, 0.1)
    want = torch.autograd.grad(loss64, list(d.parameters()))
    assert abs(float(loss.detach()) - float(loss64.detach())) <= 1e-5
    for (name, _), w in zip(d.named_parameters(), want):
        assert max_err(got[name], w) <= 1e-4, (name, max_err(got[name], w))


def test_blocks_stack_in_the_backbone():
    from mogt_b200.backbone import MOGTModel, configure_identity_coupled
    from mogt_b200.selective_lm import SelectiveBlock
    torch.manual_seed(0)
    m = configure_identity_coupled(MOGTModel(50, 64, 2, 16).cuda())
    ids = torch.randint(0, 50, (2, 30), device="cuda")
    before = m(ids)
    m.blocks.insert(1, SelectiveBlock(64).cuda())
    after = m(ids)
    assert after.shape == before.shape and bool(torch.isfinite(after).all())
    after.sum().backward()
    assert all(p.grad is not None for p in m.blocks[1].parameters())


def test_example_runs():
    spec = importlib.util.spec_from_file_location("posttrain", ROOT / "examples" / "posttrain_selective_lm.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    h = mod.main(["--steps", "3", "--batch", "8", "--prompt", "9", "--new-tokens", "12", "--vocab", "64",
                  "--d-model", "32"])
    assert len(h) == 3 and all(abs(v) < 1e3 for s in h for v in s.values())
