"""Sizes that the ragged products' C entry points refuse before anything is launched."""
import ctypes as C

import pytest

INVALID_ARGUMENT = 4
MOST = 2 ** 31 - 257


@pytest.mark.parametrize("N,K", [(MOST + 1 - (MOST + 1) % 8 + 8, 8), (8, 2 ** 31 - 8), (2 ** 31 - 8, 64), (12, 8), (8, 20), (0, 8), (8, -8)])
def test_widths(lib, N, K):
    # the pointers are looked at for their alignment alone
    p, i64 = (lambda: C.c_void_p(4096)), C.c_int64
    tail = (p(), C.c_int(0), C.c_int(2), i64(16), C.c_int(N), C.c_int(K), C.c_void_p(0))
    assert lib.mcclGroupedGemm(p(), i64(K), p(), p(), *tail) == INVALID_ARGUMENT
    assert lib.mcclGroupedGemmBackwardData(p(), i64(N), p(), p(), *tail) == INVALID_ARGUMENT
    assert lib.mcclGroupedGemmBackwardWeight(p(), i64(N), p(), i64(K), p(), *tail) == INVALID_ARGUMENT
    assert lib.mcclGroupedGemmBackward(p(), i64(N), p(), i64(K), p(), p(), p(), *tail) == INVALID_ARGUMENT
