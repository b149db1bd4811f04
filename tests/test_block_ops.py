"""The operators with one scale for each block of 128, without a GPU: the C ABI's declarations and refusals, shapes under
fake tensors, and the layer's relabelling."""

import ctypes
import pathlib
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import feather_ops as fo

HEADER = pathlib.Path(__file__).resolve().parents[1] / "include" / "feather_block_ops.h"
P, I64, INT, BOOL, F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_bool, ctypes.c_float
# Fake, aligned device addresses: every call below is refused before anything dereferences them.
X, Y, Z, W, S, T = (0x10000 * (i + 1) for i in range(6))


@pytest.fixture(scope="module")
def lib():
    from feather_ops import _lib

    handle = ctypes.CDLL(str(_lib.LIBRARY))
    for name, args in {
        "feather_block_scaled_mm": [P, I64, BOOL, P, I64, I64] * 2 + [BOOL, P, P, I64, INT, I64, I64, I64, P, I64, P],
        "feather_quantize_blocks": [P, INT, I64, P, I64, P, I64, I64, BOOL, I64, I64, P],
        "feather_quantize_tiles": [P, INT, I64, BOOL] + [P, I64, P, I64, I64] * 2 + [P, BOOL, I64, I64, P],
        "feather_sum_rows": [P, P, INT, I64, I64, P],
        "feather_rms_norm": [P, I64, P, I64, P, BOOL, F32, INT, P, I64, P, I64, P, I64, P, I64, I64, BOOL, P, I64, I64, P],
        "feather_rms_norm_backward": [P, I64, P, I64, P, I64, P, BOOL, P, INT, P, I64, P, I64, I64, P],
        "feather_silu_mul": [P, I64, INT, P, I64, P, I64, P, I64, I64, BOOL, I64, I64, P],
        "feather_silu_mul_backward": [P, I64, P, I64, INT, P, I64, I64, I64, P],
    }.items():
        getattr(handle, name).restype = BOOL
        getattr(handle, name).argtypes = args
    handle.feather_block_scaled_mm_workspace_bytes.restype = I64
    handle.feather_block_scaled_mm_workspace_bytes.argtypes = [I64, I64, I64]
    handle.feather_rms_norm_backward_parts.restype = I64
    handle.feather_rms_norm_backward_parts.argtypes = [I64, I64]
    return handle


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = re.findall(r"^\s*(?:bool|int64_t)\s+(\w+)\s*\(", text, flags=re.M)
    assert len(names) == len(set(names)) == 10
    for name in names:
        assert hasattr(lib, name), name


def _mm(lib, a=X, lda=256, b=Y, ldb=256, bias=None, c=Z, ldc=64, out=0, M=8, N=64, K=256, sa=S, sb=T, ws=None, ws_bytes=0):
    return lib.feather_block_scaled_mm(a, lda, False, sa, 1, 8, b, ldb, False, sb, 1, 1, False, bias, c, ldc, out, M, N, K,
                                       ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(M=0), dict(N=0), dict(K=-1), dict(M=-5), dict(K=300), dict(lda=255), dict(lda=264), dict(ldb=248), dict(a=X + 8),
    dict(b=Y + 1), dict(a=None), dict(b=None), dict(c=None), dict(sa=None), dict(sb=None), dict(sa=S + 2), dict(ldc=63),
    dict(out=3), dict(out=-1), dict(c=Z + 1), dict(out=2, c=Z + 2), dict(bias=W + 1), dict(K=1 << 23, lda=1 << 23, ldb=1 << 23),
    dict(M=1 << 31), dict(N=1 << 31),
])
def test_product_refuses(lib, bad):
    assert not _mm(lib, **bad)


def test_workspace_bytes(lib):
    need = lib.feather_block_scaled_mm_workspace_bytes
    assert need(0, 5, 128) == -1 and need(5, 5, -1) == -1 and need(1, 1 << 31, 128) == -1
    seen = set()
    for m, n, k in [(1, 4096, 4096), (64, 1024, 16384), (512, 512, 8192), (4096, 4096, 4096), (128, 300, 16000),
                    (1, 128, 16384), (24, 4096, 14336), (1, 1 << 20, 128), (1 << 20, 1 << 14, 1 << 14), (300, 300, 4 << 20)]:
        nbytes = need(m, n, k)
        assert 0 <= nbytes < 1 << 31
        seen.add(nbytes > 0)
        if nbytes:   # a short, missing or unaligned one is refused
            for ws, size in ((None, nbytes), (W, nbytes - 1), (W + 16, nbytes)):
                assert not _mm(lib, lda=k, ldb=k, ldc=n, M=m, N=n, K=k, ws=ws, ws_bytes=size)
    assert seen == {False, True}


def _norm(lib, x=X, ldx=64, res=None, h=None, ldh=64, w=W, type=0, y=Y, ldy=64, codes=None, ldq=64, s=None, rows=4, cols=64):
    return lib.feather_rms_norm(x, ldx, res, 64, w, False, 1e-6, type, h, ldh, y, ldy, codes, ldq, s, 1, 4, False, None, rows,
                                cols, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w=None), dict(y=None), dict(ldx=63), dict(ldy=63), dict(type=3), dict(rows=0), dict(cols=0),
    dict(res=Z), dict(h=Z), dict(res=Z, h=T, ldh=3), dict(codes=T, s=S), dict(y=None, codes=T), dict(y=None, s=S),
    dict(y=None, codes=T, s=S, ldq=63), dict(x=X + 1), dict(w=W + 1), dict(type=2, y=Y + 2), dict(y=None, codes=T, s=S + 1),
])
def test_norm_refuses(lib, bad):
    assert not _norm(lib, **bad)


def test_other_functions_refuse(lib):
    def back(gy=X, gh=None, ld_gh=64, h=Y, w=W, r=S, type=0, out=Z, ld=64, rows=4, cols=64):
        return lib.feather_rms_norm_backward(gy, 64, gh, ld_gh, h, 64, w, False, r, type, out, ld, None, rows, cols, None)

    for bad in (dict(gy=None), dict(h=None), dict(w=None), dict(r=None), dict(out=None), dict(ld=63), dict(rows=0),
                dict(cols=-1), dict(type=9), dict(gh=T, ld_gh=2), dict(h=Y + 1)):
        assert not back(**bad), bad
    assert lib.feather_rms_norm_backward_parts(0, 5) == 0 and lib.feather_rms_norm_backward_parts(1, 5) == 1

    def gate(x=X, ldx=128, type=1, y=Y, ldy=64, codes=None, s=None, rows=4, cols=64):
        return lib.feather_silu_mul(x, ldx, type, y, ldy, codes, 64, s, 1, 4, False, rows, cols, None)

    for bad in (dict(x=None), dict(ldx=127), dict(type=5), dict(y=None), dict(ldy=63), dict(codes=T, s=S), dict(rows=0),
                dict(cols=0), dict(x=X + 1), dict(y=None, codes=T)):
        assert not gate(**bad), bad
    assert not lib.feather_silu_mul_backward(X, 64, Y, 127, 0, Z, 128, 4, 64, None)
    assert not lib.feather_silu_mul_backward(X, 63, Y, 128, 0, Z, 128, 4, 64, None)
    assert not lib.feather_silu_mul_backward(X, 64, Y, 128, 0, Z, 127, 4, 64, None)
    assert not lib.feather_quantize_blocks(None, 0, 64, Y, 64, S, 1, 4, False, 4, 64, None)
    assert not lib.feather_quantize_blocks(X, 0, 64, Y, 63, S, 1, 4, False, 4, 64, None)
    assert not lib.feather_quantize_blocks(X, 0, 64, Y, 64, None, 1, 4, False, 4, 64, None)

    def tiles(x=X, codes=Y, s=S, codes_t=Z, s_t=T, sums=W, rows=4, cols=64):
        return lib.feather_quantize_tiles(x, 0, 64, False, codes, 64, s, 1, 4, codes_t, 16, s_t, 1, 64, sums, False, rows, cols,
                                          None)

    for bad in (dict(x=None), dict(codes=None), dict(s=None), dict(codes_t=None), dict(s_t=None), dict(rows=0), dict(rows=17),
                dict(codes=None, s=None, codes_t=None, s_t=None, sums=None)):
        assert not tiles(**bad), bad
    assert not lib.feather_sum_rows(None, Y, 0, 4, 4, None) and not lib.feather_sum_rows(X, Y, 0, 0, 4, None)
    assert not lib.feather_sum_rows(X, Y + 1, 0, 4, 4, None) and not lib.feather_sum_rows(X, Y, 7, 4, 4, None)


@pytest.mark.parametrize("mode", ["fake", "symbolic"])
def test_shapes_under_fake_tensors(mode):
    from torch.fx.experimental.symbolic_shapes import ShapeEnv

    def mlp(x, res, w, wide, narrow, wide_scale, narrow_scale):
        codes, scale, h = fo.rms_norm_quantized(x, w, res)
        gate_up = fo.block_scaled_mm(codes, scale, wide, wide_scale)
        codes, scale = fo.silu_mul_quantized(gate_up)
        return fo.block_scaled_mm(codes, scale, narrow, narrow_scale, None, torch.float16), h

    with FakeTensorMode(shape_env=ShapeEnv()):
        def new(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, dtype=dtype, device="cuda")

        f8 = torch.float8_e4m3fn
        args = (new(7, 256), new(7, 256), new(256), new(1024, 256, dtype=f8), new(256, 512, dtype=f8),
                new(8, 2, dtype=torch.float32), new(2, 4, dtype=torch.float32))
        y, h = mlp(*args)
        assert y.shape == (7, 256) and y.dtype == torch.float16 and h.shape == (7, 256) and h.dtype == torch.bfloat16
        x = new(3, 5, 130)
        codes, scale = fo.quantize_blocks(x)
        assert codes.shape == x.shape and scale.shape == (3, 5, 2)
        codes, scale = fo.quantize_blocks(new(300, 130), torch.float8_e5m2, square=True)
        assert codes.stride() == (192, 1) and codes.dtype == torch.float8_e5m2 and scale.shape == (3, 2)
        assert fo.block_scaled_linear(x, new(77, 130), new(77)).shape == (3, 5, 77)
        assert fo.rms_norm(x, new(130)).shape == x.shape and fo.silu_mul(x).shape == (3, 5, 65)
    nodes = [n for n in make_fx(mlp, tracing_mode=mode)(*args).graph.nodes if "feather_ops" in str(n.target)]
    assert len(nodes) == 4


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for call in (lambda: fo.quantize_blocks(x), lambda: fo.rms_norm(x, x[0]), lambda: fo.silu_mul(x),
                 lambda: fo.block_scaled_linear(x, x)):
        with pytest.raises(NotImplementedError):
            call()


def test_relabelling_leaves_trained_layers_to_each_pass():
    model = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.ReLU(), torch.nn.Linear(32, 16))
    keys = set(model.state_dict())
    assert fo.to_block_scaled_linear(model, accept=lambda m: isinstance(m, torch.nn.Linear) and m.in_features == 64) == 1
    assert isinstance(model[0], fo.BlockScaledLinear) and not isinstance(model[2], fo.BlockScaledLinear)
    assert not hasattr(model[0], "weight_fp8") and set(model.state_dict()) == keys
    with pytest.raises(ValueError, match="fp8 dtype"):
        fo.to_block_scaled_linear(model, torch.float16)


def test_tracing_with_symbolic_sizes():
    """Sizes that the tracer makes symbolic: each call goes into the graph; a product's own are fixed by its plan."""
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype)

    f8, f32 = torch.float8_e4m3fn, torch.float32
    for call, args, want in (
            (fo.block_scaled_mm, (empty(20, 256, dtype=f8), empty(20, 2, dtype=f32), empty(64, 256, dtype=f8),
                                  empty(1, 2, dtype=f32)), 1),
            (fo.block_scaled_linear, (empty(2, 20, 256), empty(64, 256), empty(64)), 3),
            (fo.quantize_blocks, (empty(3, 20, 256),), 1), (fo.rms_norm, (empty(3, 20, 256), empty(256)), 1),
            (fo.rms_norm_quantized, (empty(3, 20, 256), empty(256)), 1), (fo.silu_mul, (empty(3, 20, 256),), 1),
            (fo.silu_mul_quantized, (empty(3, 20, 256),), 1)):
        graph = make_fx(lambda *a: call(*a), tracing_mode="symbolic")(*args).graph
        assert len([n for n in graph.nodes if "feather_ops" in str(n.target)]) == want, call
