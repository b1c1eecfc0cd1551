"""Limits of the selective scan's C ABI that keep its 32-bit indexes in range
(no GPU is touched by a refused call)."""
import ctypes


def test_channels_whose_threads_pass_32_bits_are_refused():
    from mogt_b200 import _native as N
    lib = N.lib()
    p = ctypes.c_void_p(16)   # never dereferenced

    def step(D, n):
        return lib.mogt_selective_step(p, p, p, D, p, D, None, 0, p, n, n, p, n, n, p, None, None, p, 1, D, n, 1, 1,
                                       N.BF16, None)

    # a channel takes ceil(N / 4) threads, rounded up to a power of two; they are counted in 32 bits
    assert step(1 << 26, 128) == N.ERR_UNSUPPORTED
    assert step(1 << 27, 64) == N.ERR_UNSUPPORTED
    assert step((1 << 27) + 1, 1) == N.ERR_UNSUPPORTED
