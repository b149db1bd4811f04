"""Which kernels the block-scaled product runs a shape on, without a GPU: the shapes of the kernels' tests reach them all."""

import ctypes
import pathlib
import re

import pytest

from block_mm_shapes import IN_FLIGHT, KERNELS, LAUNCHES, NEVER_LONG, NEVER_SPLIT

HEADER = pathlib.Path(__file__).resolve().parents[1] / "feather-ops_amd" / "csrc" / "block_mm_launch.h"


@pytest.fixture(scope="module")
def launches():
    from feather_ops import _lib

    call = ctypes.CDLL(str(_lib.LIBRARY)).feather_block_scaled_mm_launches
    call.restype = ctypes.c_int
    call.argtypes = [ctypes.c_int64] * 3 + [ctypes.POINTER(ctypes.c_int64)]

    def of(m, n, k):
        out = (ctypes.c_int64 * 16)()
        return [tuple(out[4 * i:4 * i + 4]) for i in range(call(m, n, k, out))]

    return of


def test_names_are_those_of_the_kernels():
    body = re.search(r"enum BlockMmKernel \{(.*?)\};", HEADER.read_text(), re.S).group(1)
    assert re.findall(r"^\s*k(\w+),", body, re.M) == [
        name.title().replace(" ", "").replace("X", "x") for name in KERNELS]


@pytest.mark.parametrize("shape", LAUNCHES, ids=str)
def test_shape_goes_to_its_kernels(launches, shape):
    got = launches(*shape)
    assert [(KERNELS[kernel], splits > 1) for kernel, splits, _, _ in got] == LAUNCHES[shape]
    m, n, k = shape
    assert k % 16 and sum(rows * cols for _, _, rows, cols in got) == m * n
    if len(got) == 1 and LAUNCHES[shape][0] not in NEVER_LONG:
        kernel, splits = got[0][:2]
        assert -(-k // 128) // splits >= IN_FLIGHT[KERNELS[kernel]] and -(-k // 128) / splits > IN_FLIGHT[KERNELS[kernel]]


def test_every_kernel_is_reached():
    reached = {launch for listed in LAUNCHES.values() for launch in listed}
    want = {(kernel, split) for kernel in KERNELS for split in (False, True)} - {(kernel, True) for kernel in NEVER_SPLIT}
    assert reached == want


def test_products_are_cut_along_both_axes(launches):
    cuts = [{(len({rows for _, _, rows, _ in got}) > 1, len({cols for _, _, _, cols in got}) > 1)}
            for got in map(lambda shape: launches(*shape), LAUNCHES) if len(got) > 1]
    assert set.union(*cuts) == {(True, False), (False, True), (True, True)}


def test_shapes_without_a_plan(launches):
    assert launches(0, 5, 128) == launches(5, 0, 128) == launches(5, 5, -1) == launches(5, 5, 1 << 23) == []
    assert len(launches(1, 1, 0)) == 1


def test_launches_have_fewer_than_2_32_threads():
    """A grid of more would be cut off without an error: such shapes are refused."""
    from feather_ops import _lib

    need = _lib.c_library().feather_block_scaled_mm_workspace_bytes
    assert need(1, (1 << 26) - 16, 16) >= 0 and need(64, (1 << 26) - 16, 16) >= 0 and need((1 << 29) - 1, 1, 16) >= 0
    for m, n, k in ((1, 1 << 27, 16), (8, 1 << 27, 16), (1, (1 << 29) - 1, 16), (1, 1 << 26, 4096), ((1 << 21) + 1, 1 << 17, 16)):
        assert need(m, n, k) == -1
