"""Which kernels 4-bit weights go to, without a GPU."""

import ctypes

import pytest

from linear_shapes import KERNELS

I64, BOOL = ctypes.c_int64, ctypes.c_bool


@pytest.fixture(scope="module")
def launches():
    from feather_ops import _lib

    call = ctypes.CDLL(str(_lib.LIBRARY)).feather_linear_launches
    call.restype = ctypes.c_int
    call.argtypes = [I64] * 3 + [BOOL] * 3 + [ctypes.POINTER(I64)]

    def of(m, n, k, gated, fine):
        out = (I64 * 16)()
        return [tuple(out[4 * i:4 * i + 4]) for i in range(call(m, n, k, gated, True, fine, out))]

    return of


@pytest.mark.parametrize("fine", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k", [512, 2048, 4096, 5120, 8192, 16384])
def test_up_to_64_rows_have_one_launch_that_takes_codes_as_they_are(launches, k, gated, fine):
    for m in (1, 16, 17, 32, 33, 48, 64):
        for n in [*range(1, 1 << 18, 3331), 53248, 128256, 151936, 1 << 18]:
            (launch,) = launches(m, n, k, gated, fine)
            assert KERNELS[launch[0]].startswith("few"), (m, n)
