"""CPU checks of the selective state space and loss entry points: CPU tensors
are refused before the library is asked for anything, and the C ABI checks
its own arguments (no GPU is touched by a refused call)."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    import mogt_b200
    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    u, A, B = torch.zeros(1, 4, 8), torch.zeros(8, 2), torch.zeros(1, 4, 2)
    lab = torch.zeros(1, 4, dtype=torch.int64)
    f = torch.zeros(1, 4)
    for call in (lambda: mogt_b200.causal_conv(x, w),
                 lambda: mogt_b200.causal_conv_step(x[:, 0], torch.zeros(1, 3, 8), w),
                 lambda: mogt_b200.selective_scan(u, u, A, B, B),
                 lambda: mogt_b200.selective_scan_step(torch.zeros(1, 8, 2), u[:, 0], u[:, 0], A, B[:, 0], B[:, 0]),
                 lambda: mogt_b200.token_logprobs(x, lab),
                 lambda: mogt_b200.policy_loss(x, lab, f, torch.zeros(1)),
                 lambda: mogt_b200.preference_loss(torch.zeros(2, 4, 8), lab.expand(2, 4), torch.zeros(2))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_c_abi_checks_its_arguments():
    from mogt_b200 import _native as N
    lib = N.lib()
    p = ctypes.c_void_p(16)   # never dereferenced: every call below is refused first
    conv = lambda B, L, D, K, dt, pd, w=p: lib.mogt_causal_conv_fwd(p, 0, 0, w, None, None, None, p, None, B, L, D, K,
                                                                  1, dt, pd, None)
    assert conv(-1, 1, 1, 4, 0, 0) == N.ERR_SHAPE
    assert conv(1, 1, 1, 5, 0, 0) == N.ERR_UNSUPPORTED
    assert conv(1, 1, 1, 4, 3, 0) == N.ERR_DTYPE
    assert conv(1, 1, 1, 4, 0, 0, None) == N.ERR_ARG
    assert conv(0, 1, 1, 4, 0, 0) == N.OK
    assert lib.mogt_causal_conv_bwd(p, 0, 0, p, None, None, None, p, 0, 0, None, p, p, None, None, 1, 8, 4, 4, 1, 0, 0,
                                    None, 0, None) == N.ERR_WORKSPACE
    a = N.SelectiveArgs()
    a.B, a.L, a.D, a.N, a.G = 1, 4, 6, 16, 4
    fwd = lambda: lib.mogt_selective_scan_fwd(ctypes.byref(a), None)
    assert fwd() == N.ERR_SHAPE            # 6 channels in 4 groups
    a.G, a.N = 2, 129
    assert fwd() == N.ERR_UNSUPPORTED
    a.N, a.dtype = 16, 7
    assert fwd() == N.ERR_DTYPE
    a.dtype = 1
    assert fwd() == N.ERR_ARG
    a.u_sl = 1 << 40
    assert fwd() == N.ERR_UNSUPPORTED
    assert lib.mogt_selective_scan_fwd(None, None) == N.ERR_ARG
    assert lib.mogt_selective_scan_bwd(None, None) == N.ERR_ARG
    lp = lambda B, L, V, dt, x=p: lib.mogt_logprob_fwd(x, 0, 0, p, None, B, L, V, dt, p, None, None)
    assert lp(1, 1, 0, 0) == N.ERR_SHAPE and lp(1, 1, 5, 9) == N.ERR_DTYPE and lp(1, 1, 5, 0, None) == N.ERR_ARG
    assert lp(1 << 20, 1 << 20, 5, 0) == N.ERR_UNSUPPORTED and lp(0, 3, 5, 0) == N.OK
    assert lib.mogt_policy_loss(p, 0, 0, p, None, p, None, p, 0, 0, 0.2, 0.2, 0.0, p, p, None, p, None, 0, 0, 1, 1, 5, 0,
                                None, 0, None) == N.ERR_WORKSPACE
    assert lib.mogt_preference_pairs(p, None, 1, 1, 0.1, 0.0, p, p, p, None) == N.ERR_ARG
    bwd = lambda scale, unless: lib.mogt_logprob_bwd(p, 0, 0, p, None, p, p, 1, scale, unless, None, 0, 0, 1, 1, 5, 0,
                                                    None)
    assert bwd(p, 0) == N.ERR_ARG and bwd(None, 1) == N.ERR_ARG


def test_scratch_sizes():
    from mogt_b200 import _native as N
    lib = N.lib()
    assert lib.mogt_selective_saved_bytes(2, 33, 8, 16) == 2 * 3 * 8 * 16 * 4
    assert lib.mogt_selective_saved_bytes(2, 33, 8, 5) == 2 * 3 * 8 * 8 * 4      # states padded to 8
    assert lib.mogt_selective_fwd_scratch_bytes(64, 64, 1536, 16, 1) == 0        # channels fill the GPU
    assert lib.mogt_selective_fwd_scratch_bytes(1, 32768, 1536, 16, 1) > 0       # one long sequence is split
    assert lib.mogt_selective_bwd_scratch_bytes(1, 64, 9, 4, 2) == 0             # refused by the call itself
    assert lib.mogt_causal_conv_bwd_scratch_bytes(1, 100, 64, 4) > 0
    assert lib.mogt_policy_loss_scratch_bytes(2, 3) == 7 * 4
