"""CPU checks of the loss entry points' own argument checks (no GPU is touched by a refused call)."""
import ctypes


def test_pairs_with_float64_reference_sums():
    from mogt_b200 import _native as N
    lib = N.lib()
    p = ctypes.c_void_p(16)   # never dereferenced
    call = lambda ref, P, L, lp=p: lib.mogt_preference_pairs_f64(lp, ref, P, L, 0.1, 0.0, p, p, p, None)
    assert call(None, 1, 1) == N.ERR_ARG and call(p, -1, 1) == N.ERR_SHAPE and call(p, 1, 1, None) == N.ERR_ARG
