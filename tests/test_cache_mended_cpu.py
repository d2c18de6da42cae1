"""Refusals and rules of the paged-cache entry points that came after their first tests, without a GPU."""
import ctypes

from kernelcodegen_b200 import _lib


def test_more_requests_than_a_limited_wait_can_walk_past(lib):
    st2, st3 = (ctypes.c_int64 * 2)(64, 64), (ctypes.c_int64 * 3)(4096, 1024, 64)
    for T, cu in ((1, 16), (2 ** 20 + 1, None)):
        rc = lib.kcg_fmha_cached_fwd(_lib.BF16, T, 2 ** 20 + 1, 2, 1, 64, 1, 1.0, 1, 16, st2, 16, st3, 16, 16, st3, 16, 4, 16, 16, 2, 2, 16, cu,
                                     16, st2, 16, 1 << 30, None)
        assert rc == _lib.ERR_UNSUPPORTED and "requests" in lib.kcg_last_error().decode()
