"""The gated block's elementwise backward through the C ABI: its values, its padding and what lies behind it."""

import ctypes

import pytest
import torch

import linear_ref as ref

P, I64, INT = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int


@pytest.fixture(scope="module")
def backward():
    from feather_ops import _lib

    call = ctypes.CDLL(str(_lib.LIBRARY)).feather_gated_backward
    call.restype = ctypes.c_bool
    call.argtypes = [P, I64, P, I64, INT, INT, P, I64, P, I64, I64, P]
    return call


@pytest.mark.parametrize("f", [1, 4, 9, 12, 20])
def test_rows_without_room_for_the_padding_are_refused(backward, f):
    if torch.cuda.is_available():
        pytest.skip("without a GPU: nothing is behind the addresses")
    f8 = -(-f // 8) * 8
    assert not backward(0x10000, f, 0x20000, 2 * f8, 0, 0, 0x30000, 2 * f8 - 8, None, 4, f, None)


@pytest.mark.gpu
@pytest.mark.parametrize("act", range(3))
@pytest.mark.parametrize("dtype", ref.HALVES)
@pytest.mark.parametrize("m,f", [(1, 1), (3, 4), (2, 9), (5, 12), (600, 13), (2, 16), (3, 2043)])
def test_columns_behind_the_gradients_are_zero(backward, m, f, dtype, act):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    f8 = -(-f // 8) * 8
    g = torch.Generator("cuda").manual_seed(f)
    gy = torch.randn((m, f), generator=g, device="cuda").to(dtype)
    kept = torch.full((m, 2 * f8), float("nan"), device="cuda")
    gate, up = (torch.randn((m, f), generator=g, device="cuda") for _ in range(2))
    kept[:, :f], kept[:, f8:f8 + f] = gate, up
    grad = torch.full((m + 1, 2 * f8 + 8), 77.0, dtype=dtype, device="cuda")
    assert backward(gy.data_ptr(), f, kept.data_ptr(), 2 * f8, 0 if dtype == torch.bfloat16 else 1, act, grad.data_ptr(),
                    grad.stride(0), None, m, f, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    value, slope = ref.activation(gate.double(), ref.ACTIVATIONS[act])
    want = torch.cat((gy.double() * slope * up.double(), gy.double() * value), 1)
    # the slope is a difference of two terms of up to |g| in size
    off = gy.double().abs() * (1 + gate.double().abs()) * (1 + up.double().abs()) * ref.ACT
    ref.check(grad[:m, :2 * f], want, off.repeat(1, 2))
    assert (grad[:m, 2 * f:2 * f8] == 0).all()
    assert (grad[:m, 2 * f8:] == 77.0).all() and (grad[m] == 77.0).all()
