"""What the single-token forms write is known to autograd: a state that a
recorded call still needs cannot be changed unnoticed, and one that takes part
in a recorded computation is not written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _conv(B=2, D=8, K=4):
    rn = lambda *s: torch.randn(*s, device="cuda")
    return rn(B, 5, D), rn(D, K), rn(B, K - 1, D)


def _scan(B=2, D=8, N=4):
    rn = lambda *s: torch.randn(*s, device="cuda")
    return rn(B, 5, D), rn(B, 5, D), -torch.rand(D, N, device="cuda"), rn(B, 5, N), rn(B, 5, N), rn(B, D, N)


@pytest.mark.parametrize("separate", [False, True])
def test_backward_after_a_step_over_its_history_raises(separate):
    import mogt_b200
    x, w, st = _conv()
    w.requires_grad_(True)
    y = mogt_b200.causal_conv(x, w, initial_state=st)
    if separate:   # the state goes into the recorded call's buffer
        mogt_b200.causal_conv_step(x[:, 0], torch.zeros_like(st), w.detach(), new_state=st)
    else:
        mogt_b200.causal_conv_step(x[:, 0], st, w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("separate", [False, True])
def test_backward_after_a_step_over_a_saved_state_raises(separate):
    import mogt_b200
    u, delta, A, B, C, st = _scan()
    p = torch.ones_like(st, requires_grad=True)
    y = (p * st).sum()
    step = [u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0]]
    if separate:
        mogt_b200.selective_scan_step(torch.zeros_like(st), *step, new_state=st)
    else:
        mogt_b200.selective_scan_step(st, *step)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_recorded_state_is_not_written():
    import mogt_b200
    x, w, st = _conv()
    w.requires_grad_(True)
    _, last = mogt_b200.causal_conv(x.requires_grad_(True), w, initial_state=st, return_state=True)
    x = x.detach()
    with pytest.raises(ValueError, match="requires grad"):
        mogt_b200.causal_conv_step(x[:, 0], last, w)
    with torch.no_grad():   # as in torch, without recording it may be
        mogt_b200.causal_conv_step(x[:, 0], last, w)
    mogt_b200.causal_conv_step(x[:, 0], last.detach(), w)
    kept = torch.empty_like(st)
    mogt_b200.causal_conv_step(x[:, 0], last, w, new_state=kept)   # only read

    u, delta, A, B, C, st = _scan()
    _, last = mogt_b200.selective_scan(u, delta, A.requires_grad_(True), B, C, return_state=True)
    step = [u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0]]
    with pytest.raises(ValueError, match="requires grad"):
        mogt_b200.selective_scan_step(last, *step)
    mogt_b200.selective_scan_step(last.detach(), *step)
    mogt_b200.selective_scan_step(last, *step, new_state=torch.empty_like(st))


def test_steps_in_inference_mode():
    import mogt_b200
    with torch.inference_mode():
        x, w, st = _conv()
        before = st.clone()
        mogt_b200.causal_conv_step(x[:, 0], st, w)
        assert torch.equal(st[:, :-1], before[:, 1:]) and torch.equal(st[:, -1], x[:, 0])
        u, delta, A, B, C, st = _scan()
        mogt_b200.selective_scan_step(st, u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0])


def test_overlapping_states_are_refused():
    """A new state may be the old one or lie apart from it: threads of one sequence would write what others still read."""
    import mogt_b200
    x, w, _ = _conv()
    buf = torch.randn(3, 3, 8, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        mogt_b200.causal_conv_step(x[:, 0], buf[:2], w, new_state=buf[1:])
    mogt_b200.causal_conv_step(x[:, 0], buf[:2], w, new_state=buf[:2])
    u, delta, A, B, C, _ = _scan()
    buf = torch.randn(4, 8, 4, device="cuda")
    step = [u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0]]
    for state, new in ((buf[:2], buf[1:3]), (buf[1:3], buf[:2])):
        with pytest.raises(ValueError, match="overlap"):
            mogt_b200.selective_scan_step(state, *step, new_state=new)
    mogt_b200.selective_scan_step(buf[:2], *step, new_state=buf[2:])
