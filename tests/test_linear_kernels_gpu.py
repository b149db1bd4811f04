"""Every kernel of the 16-bit and 4-bit products through the C ABI, against 64 bits: unsplit and split K, products in parts, operands
along and across their sums, strides, workspaces that are left as they were found, and outputs beyond their ends."""

import ctypes

import pytest
import torch

import linear_ref as ref
from linear_shapes import GATED, INT4, INT4_GATED, PRODUCT

pytestmark = pytest.mark.gpu
P, I64, INT, BOOL = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_bool
TYPES = {torch.bfloat16: 0, torch.float16: 1}


@pytest.fixture(scope="module")
def lib():
    from feather_ops import _lib

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    handle = ctypes.CDLL(str(_lib.LIBRARY))
    for name, args in {
        "feather_gated_linear": [P, I64, P, I64, P, INT, INT, P, I64, P, I64, I64, I64, I64, P, I64, P],
        "feather_product": [P, I64, BOOL, P, I64, BOOL, P, INT, P, I64, I64, I64, I64, P, I64, P],
        "feather_int4_linear": [P, I64, P, I64, P, I64, P, I64, INT, P, INT, BOOL, INT, P, I64, I64, I64, I64, P, I64, P],
    }.items():
        getattr(handle, name).restype = BOOL
        getattr(handle, name).argtypes = args
        need = getattr(handle, name + "_workspace_bytes")
        need.restype = I64
        need.argtypes = [I64] * 3 + ([BOOL] if "int4" in name else [])
    return handle


def _type(dtype):
    """The C ABI's number of a type."""
    return TYPES[dtype]


def _randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _wide(t, zeros=True):
    """A matrix with its rows a piece further apart than they have to be, behind their columns zeros up to the next 8 (or not) and
    then values that would show."""
    rows, cols = t.shape
    whole = -(-cols // 8) * 8
    out = torch.full((rows, whole + 8), float("nan"), dtype=t.dtype, device="cuda")
    if zeros:
        out[:, cols:whole] = 0
    out[:, :cols] = t
    return out[:, :cols]


def _workspace(need):
    return torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda") if need else None


def _at(t):
    return None if t is None else t.data_ptr()


def _output(m, n, dtype):
    """[m, n] inside a larger matrix of a value that a stray store would change."""
    whole = torch.full((m + 2, n + 5), 77.0, dtype=dtype, device="cuda")
    return whole, whole[1:m + 1, 2:n + 2]


def _untouched(whole, m, n):
    edge = torch.ones_like(whole, dtype=torch.bool)
    edge[1:m + 1, 2:n + 2] = False
    return (whole[edge] == 77.0).all()


def _twice(call, need):
    """Runs a call two times on one workspace, whose counters it leaves at zero."""
    ws = _workspace(need)
    results = []
    for _ in range(2):
        results.append(call(_at(ws), need))
        torch.cuda.synchronize()
        if ws is not None:
            assert not ws[:64 * 1024].any()
    assert torch.equal(*results)
    return results[0]


@pytest.mark.parametrize("across", ["neither", "b", "both"])
@pytest.mark.parametrize("shape", PRODUCT, ids=str)
def test_product(lib, shape, across):
    m, n, k = shape
    dtype = torch.bfloat16 if (m + n) % 4 else torch.float16
    a, b = _randn((m, k), dtype, 1), _randn((n, k), dtype, 2, k**-0.5)
    bias = _randn((n,), dtype, 3)
    a_across, b_across = across == "both", across != "neither"
    # rows across are read up to a multiple of 8 values, whatever those are
    pa = _wide(a.t(), False) if a_across else _wide(a)
    pb = _wide(b.t(), False) if b_across else _wide(b)

    def call(ws, size):
        whole, c = _output(m, n, dtype)
        assert lib.feather_product(_at(pa), pa.stride(0), a_across, _at(pb), pb.stride(0), b_across, _at(bias), _type(dtype), _at(c),
                                   c.stride(0), m, n, k, ws, size, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert _untouched(whole, m, n)
        return c

    c = _twice(call, lib.feather_product_workspace_bytes(m, n, k))
    a, b, bias = a.double(), b.double(), bias.double()
    ref.check(c, a @ b.t() + bias, ref.sum_error(k, a.abs() @ b.abs().t() + bias.abs()))


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("shape", GATED, ids=str)
def test_gated(lib, shape, keep):
    m, f, k = shape
    dtype = torch.bfloat16 if (m + f) % 4 else torch.float16
    act = (m + k) % 3
    x, w, bias = _randn((m, k), dtype, 1), _randn((2 * f, k), dtype, 2, k**-0.5), _randn((2 * f,), dtype, 3)
    px, pw = _wide(x), _wide(w)
    f8 = -(-f // 8) * 8
    kept = torch.full((m + 1, 2 * f8 + 4), 55.0, device="cuda") if keep else None

    def call(ws, size):
        whole, y = _output(m, f, dtype)
        assert lib.feather_gated_linear(_at(px), px.stride(0), _at(pw), pw.stride(0), _at(bias), _type(dtype), act, _at(y), y.stride(0), _at(kept),
                                        0 if kept is None else kept.stride(0), m, f, k, ws, size, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert _untouched(whole, m, f)
        return y

    y = _twice(call, lib.feather_gated_linear_workspace_bytes(m, f, k))
    ref.check(y, *ref.gated(x, w, bias, ref.ACTIVATIONS[act]))
    if keep:
        x, w, bias = x.double(), w.double(), bias.double()
        h, bound = x @ w.t() + bias, ref.sum_error(k, x.abs() @ w.abs().t() + bias.abs())
        for half in range(2):
            got = kept[:m, half * f8:half * f8 + f].double()
            assert ((got - h[:, half * f:(half + 1) * f]).abs() <= bound[:, half * f:(half + 1) * f]).all()
        assert (kept[m] == 55.0).all() and (kept[:, 2 * f8:] == 55.0).all()


def _int4_weight(n, k, group, zeros, dtype):
    g = torch.Generator("cuda").manual_seed(5)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
    scale = (torch.rand((groups, n), generator=g, device="cuda") * 0.01 + 0.001).to(dtype)
    zero = torch.randint(0, 16, (groups, n), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return codes, scale, zero


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_int4(lib, gated, group, zeros):
    for shape in INT4_GATED if gated else INT4:
        m, n, k = shape
        dtype = torch.bfloat16 if (m + n + group // 32) % 4 else torch.float16
        act = (m + k) % 3
        rows = 2 * n if gated else n
        codes, scale, zero = _int4_weight(rows, k, group, zeros, dtype)
        x, bias = _randn((m, k), dtype, 1), _randn((rows,), dtype, 3)
        px = _wide(x)
        # rows 16 bytes apart and behind them codes of other values; the last ends with its memory, up to 16 bytes
        pitch = -(-codes.shape[1] // 16) * 16
        wide = torch.randint(0, 256, (rows, pitch), device="cuda", dtype=torch.uint8)
        wide[:, :codes.shape[1]] = codes
        framed = torch.full((scale.shape[0], rows + 5), float("nan"), dtype=dtype, device="cuda")
        framed[:, :rows] = scale

        def call(ws, size):
            whole, y = _output(m, n, dtype)
            assert lib.feather_int4_linear(_at(px), px.stride(0), _at(wide), pitch, _at(framed), rows + 5, _at(zero), rows, group, _at(bias),
                                           _type(dtype), gated, act, _at(y), y.stride(0), m, n, k, ws, size,
                                           torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            assert _untouched(whole, m, n), shape
            return y

        y = _twice(call, lib.feather_int4_linear_workspace_bytes(m, n, k, gated))
        weight = (codes, scale.t(), None if zero is None else zero.t())
        h, bound = ref.int4(x, *weight, bias)
        if m > 64:   # the weight is rounded to x's dtype first
            bound = bound + x.double().abs() @ ref.half_step(dtype, ref.int4_values(*weight, k)).t()
        if gated:
            gate, up = h.chunk(2, 1)
            d_gate, d_up = bound.chunk(2, 1)
            value, slope = ref.activation(gate, ref.ACTIVATIONS[act])
            h, bound = value * up, ((slope.abs() + 2 * d_gate) * d_gate * up.abs() + value.abs() * d_up + d_gate * d_up +
                                    ref.ACT * (value * up).abs())
        print(shape, flush=True)
        ref.check(y, h, bound)


@pytest.mark.parametrize("m", [70, 300])
def test_int4_rows_of_codes_off_16_bytes(m):
    """They are dequantized first; the sums are the same but for their order."""
    import feather_ops as fo

    codes, scale, zero = _int4_weight(150, 648, 128, True, torch.bfloat16)
    x = _randn((m, 648), torch.bfloat16, 1)
    wide = torch.zeros(150, 332, dtype=torch.uint8, device="cuda")
    wide[:, 4:328] = codes
    want, bound = ref.int4(x, codes, scale.t(), zero.t(), None)
    bound = bound + x.double().abs() @ ref.half_step(x.dtype, ref.int4_values(codes, scale.t(), zero.t(), 648)).t()
    for c in (codes, wide[:, 4:328]):
        ref.check(fo.int4_linear(x, c, scale.t(), zero.t()), want, bound)
