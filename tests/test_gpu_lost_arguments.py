"""Arguments that would lose a part of themselves are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _z(*s, **kw):
    return torch.zeros(*s, device="cuda", **kw)


C64 = torch.complex64


def test_complex_arguments_are_refused():
    """This layer family also comes with complex A; the kernels' states are real."""
    import mogt_b200 as m
    u, A, B = _z(2, 5, 8), _z(8, 4), _z(2, 5, 4)
    st = _z(2, 8, 4)
    for call in (lambda: m.selective_scan(u, u, A.to(C64), B, B),
                 lambda: m.selective_scan(u, u, A, B, B, D=_z(8, dtype=C64)),
                 lambda: m.selective_scan(u, u, A, B, B, delta_bias=_z(8, dtype=C64)),
                 lambda: m.selective_scan(u, u, A, B, B, initial_state=st.to(C64)),
                 lambda: m.selective_scan_step(st, u[:, 0], u[:, 0], A.to(C64), B[:, 0], B[:, 0])):
        with pytest.raises(ValueError, match="must be real"):
            call()
    x, lab, f, p = _z(2, 3, 10), _z(2, 3, dtype=torch.int64), _z(2, 3), _z(2)
    for call in (lambda: m.policy_loss(x, lab, f.to(C64), p),
                 lambda: m.policy_loss(x, lab, f, p.to(C64)),
                 lambda: m.policy_loss(x, lab, f, p, ref_logprobs=f.to(C64), kl_coef=0.1),
                 lambda: m.preference_loss(x, lab, p.to(C64))):
        with pytest.raises(ValueError, match="must be real"):
            call()


def test_real_arguments_of_other_types_are_taken():
    import mogt_b200 as m
    u, A, B = torch.randn(1, 5, 8, device="cuda"), -torch.ones(8, 4, device="cuda"), torch.randn(1, 5, 4, device="cuda")
    want = m.selective_scan(u, u, A, B, B)
    for dt in (torch.float64, torch.bfloat16, torch.int64):
        assert torch.equal(m.selective_scan(u, u, A.to(dt), B, B), want)
    x, lab, f = torch.randn(2, 3, 10, device="cuda"), _z(2, 3, dtype=torch.int64), _z(2, 3)
    assert torch.equal(m.policy_loss(x, lab, f, torch.tensor([1, -1], device="cuda")),
                       m.policy_loss(x, lab, f, torch.tensor([1.0, -1.0], device="cuda")))


def test_forward_mode_is_refused():
    """The kernels carry no tangents: a dual tensor must not come out as if its derivative were zero."""
    import mogt_b200 as m
    import torch.autograd.forward_ad as fw
    x, w, u, A, B = _z(2, 5, 8), _z(8, 4), _z(2, 5, 8), -torch.ones(8, 4, device="cuda"), _z(2, 5, 4)
    lg, lab, f, p = _z(2, 3, 10), _z(2, 3, dtype=torch.int64), _z(2, 3), _z(2)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        for call in (lambda: m.causal_conv(dual(x), w), lambda: m.causal_conv(x, dual(w)),
                     lambda: m.causal_conv_step(dual(x[:, 0]), _z(2, 3, 8), w),
                     lambda: m.selective_scan(u, dual(u), A, B, B), lambda: m.selective_scan(u, u, A, dual(B), B),
                     lambda: m.selective_scan(u, u, A, B, B, initial_state=dual(_z(2, 8, 4))),
                     lambda: m.selective_scan_step(_z(2, 8, 4), u[:, 0], u[:, 0], dual(A), B[:, 0], B[:, 0]),
                     lambda: m.token_logprobs(dual(lg), lab), lambda: m.policy_loss(dual(lg), lab, f, p),
                     lambda: m.preference_loss(dual(lg), lab, p)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        # tensors without a tangent pass through a dual level
        assert m.causal_conv(x, w).shape == x.shape and m.token_logprobs(lg, lab).shape == lab.shape


def test_a_kl_weight_without_reference_is_said():
    """Without ref_logprobs there is no KL term, whatever its weight; that a weight is left unused is not kept silent."""
    import warnings

    import mogt_b200 as m
    x, lab, f, p = _z(2, 3, 10), _z(2, 3, dtype=torch.int64), _z(2, 3), _z(2)
    with pytest.warns(UserWarning, match="ref_logprobs"):
        m.policy_loss(x, lab, f, p, kl_coef=0.05)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        m.policy_loss(x, lab, f, p)
        m.policy_loss(x, lab, f, p, ref_logprobs=f, kl_coef=0.05)
