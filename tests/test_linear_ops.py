"""The feed-forward operators without a GPU: the C ABI's declarations, plans and refusals, shapes under fake tensors, the layer's
relabelling, and the package without its autograd nodes."""

import ctypes
import pathlib
import re
import shutil
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import feather_ops as fo
from linear_shapes import GATED, INT4, INT4_GATED, KERNELS, NEVER_SPLIT, PRODUCT

ROOT = pathlib.Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "feather_linear_ops.h"
LAUNCHES = ROOT / "feather-ops_amd" / "csrc" / "linear_launch.h"
PACKAGE = ROOT / "feather-ops_amd" / "feather_ops"
P, I64, INT, BOOL = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_bool
# Fake, aligned device addresses: every call below is refused before anything dereferences them.
X, Y, Z, W, S, T = (0x10000 * (i + 1) for i in range(6))


@pytest.fixture(scope="module")
def lib():
    from feather_ops import _lib

    handle = ctypes.CDLL(str(_lib.LIBRARY))
    for name, args in {
        "feather_gated_linear": [P, I64, P, I64, P, INT, INT, P, I64, P, I64, I64, I64, I64, P, I64, P],
        "feather_gated_backward": [P, I64, P, I64, INT, INT, P, I64, P, I64, I64, P],
        "feather_product": [P, I64, BOOL, P, I64, BOOL, P, INT, P, I64, I64, I64, I64, P, I64, P],
        "feather_int4_linear": [P, I64, P, I64, P, I64, P, I64, INT, P, INT, BOOL, INT, P, I64, I64, I64, I64, P, I64, P],
        "feather_int4_linear_direct": [P, I64, I64, I64, I64, BOOL],
        "feather_int4_dequantize": [P, I64, P, I64, P, I64, INT, INT, P, I64, I64, I64, P],
        "feather_int4_quantize": [P, I64, INT, INT, P, I64, P, I64, P, I64, I64, I64, P],
    }.items():
        getattr(handle, name).restype = BOOL
        getattr(handle, name).argtypes = args
    for name, args in {"gated_linear_workspace_bytes": [I64] * 3, "product_workspace_bytes": [I64] * 3,
                       "int4_linear_workspace_bytes": [I64] * 3 + [BOOL], "gated_backward_parts": [I64] * 2}.items():
        getattr(handle, "feather_" + name).restype = I64
        getattr(handle, "feather_" + name).argtypes = args
    return handle


@pytest.fixture(scope="module")
def launches(lib):
    call = lib.feather_linear_launches
    call.restype = INT
    call.argtypes = [I64] * 3 + [BOOL] * 3 + [ctypes.POINTER(I64)]

    def of(m, n, k, gated=False, int4=False, fine=False):
        out = (I64 * 16)()
        return [tuple(out[4 * i:4 * i + 4]) for i in range(call(m, n, k, gated, int4, fine, out))]

    return of


def test_library_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = re.findall(r"^\s*(?:bool|int64_t)\s+(\w+)\s*\(", text, flags=re.M)
    assert len(names) == len(set(names)) == 11
    for name in names:
        assert hasattr(lib, name), name


def test_names_are_those_of_the_kernels():
    body = re.search(r"enum LinearKernel : int \{(.*?)\};", LAUNCHES.read_text(), re.S).group(1)
    names = re.findall(r"\bk(\w+),", body)
    want = [n.replace("tile 256x256", "Tile256").replace("tile 256x128", "Tile256x128").replace("tile 128x128", "Tile128")
            .replace("int4 256x256", "Int4Tile256").replace("int4 128x256", "Int4Tile128").replace("few ", "Few")
            .replace(" ", "_").replace("/", "_") for n in KERNELS]
    assert names == want


@pytest.mark.parametrize("kind", ["product", "gated", "int4", "int4 gated"])
def test_shapes_go_to_their_kernels(launches, kind):
    gated, int4 = "gated" in kind, "int4" in kind
    for (m, n, k), want in {"product": PRODUCT, "gated": GATED, "int4": INT4, "int4 gated": INT4_GATED}[kind].items():
        got = launches(m, n, k, gated, int4)
        assert [(KERNELS[kernel], splits > 1) for kernel, splits, _, _ in got] == want, (m, n, k)
        columns = 2 * -(-n // 16) * 16 if gated else n
        assert sum(rows * cols for _, _, rows, cols in got) == m * columns


def test_every_kernel_is_reached():
    reached = {launch for listed in (PRODUCT, GATED, INT4, INT4_GATED) for shape in listed.values() for launch in shape}
    assert reached == {(kernel, split) for kernel in KERNELS for split in (False, True)} - {(kernel, True) for kernel in NEVER_SPLIT}


def test_fine_groups_with_zero_points_take_fewer_waves(launches, lib):
    """Their workspace is asked for without knowing the groups: it is enough for both."""
    for shape in INT4_GATED:
        coarse, fine = launches(*shape, True, True), launches(*shape, True, True, True)
        for (kernel, _, *size), (other, splits, *same) in zip(coarse, fine):
            assert KERNELS[other] not in ("few 16 2/16/1", "few 32 2/4/4") and size == same
            assert kernel == other or KERNELS[kernel] in ("few 16 2/16/1", "few 32 2/4/4")
            assert splits == 1 or lib.feather_int4_linear_workspace_bytes(*shape, True) > 0
        assert launches(*shape, False, True) == launches(*shape, False, True, True)


def test_which_codes_are_dequantized(lib):
    """Many rows, whose product is in 16 bits, and rows of codes that do not start on 16-byte boundaries; never few rows."""
    direct = lib.feather_int4_linear_direct
    assert direct(Y, 2560, 512, 13824, 5120, False) and not direct(Y, 2560, 16384, 13824, 5120, False)
    assert not direct(Y + 4, 2560, 512, 13824, 5120, False) and not direct(Y, 2564, 512, 13824, 5120, False)
    assert direct(Y + 4, 2052, 64, 4096, 4096, False) and direct(Y + 4, 2052, 1, 4096, 4096, True)


def test_launches_have_fewer_than_2_32_threads(launches, lib):
    """Sizes whose grid would be cut off without an error are refused by their workspace or the call."""
    assert launches(0, 5, 128) == launches(5, 0, 128) == launches(5, 5, 0) == launches(5, 5, (1 << 21) + 1) == []
    for m, n, k in ((1 << 29, 1 << 10, 64), (1 << 20, 1 << 28, 64), (1, 1 << 29, 64)):
        assert lib.feather_product_workspace_bytes(m, n, k) == -1
        assert not _product(lib, M=m, N=n, K=k, lda=k, ldb=k, ldc=n)
        assert not _int4(lib, M=m, N=n, K=k, ldx=k, ldy=n, ld_codes=k, ld_scale=n, ld_zero=n)


def _gated(lib, x=X, ldx=64, w=W, ldw=64, bias=None, type=0, act=0, y=Y, ldy=40, kept=None, ld_kept=80, M=4, F=40, K=64, ws=None,
           ws_bytes=0):
    return lib.feather_gated_linear(x, ldx, w, ldw, bias, type, act, y, ldy, kept, ld_kept, M, F, K, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=X + 2), dict(w=None), dict(w=W + 8), dict(y=None), dict(y=Y + 1), dict(ldx=56), dict(ldx=68), dict(ldw=56),
    dict(ldx=(1 << 21) + 8), dict(bias=S + 1), dict(type=2), dict(type=-1), dict(act=3), dict(act=-1), dict(ldy=39), dict(M=0),
    dict(F=0), dict(K=0), dict(K=60), dict(M=-1), dict(F=1 << 30), dict(kept=T + 4), dict(kept=T, ld_kept=76), dict(kept=T, ld_kept=82),
    dict(kept=T, ld_kept=1 << 22),
])
def test_gated_refuses(lib, bad):
    assert not _gated(lib, **bad)


def test_gated_backward_refuses(lib):
    def back(gy=X, ld_gy=40, kept=W, ld_kept=80, type=0, act=0, grad=Y, ld=80, sums=None, M=4, F=40):
        return lib.feather_gated_backward(gy, ld_gy, kept, ld_kept, type, act, grad, ld, sums, M, F, None)

    for bad in (dict(gy=None), dict(gy=X + 1), dict(ld_gy=39), dict(kept=None), dict(kept=W + 4), dict(ld_kept=76), dict(ld_kept=82),
                dict(type=2), dict(act=3), dict(grad=None), dict(grad=Y + 2), dict(ld=72), dict(ld=84), dict(M=0), dict(F=0),
                dict(F=1 << 30), dict(M=1 << 32)):
        assert not back(**bad), bad
    assert lib.feather_gated_backward_parts(0, 5) == 0 and lib.feather_gated_backward_parts(1, 5) == 1


def _product(lib, a=X, lda=64, a_across=False, b=W, ldb=64, b_across=False, bias=None, type=0, c=Y, ldc=40, M=8, N=40, K=64, ws=None,
             ws_bytes=0):
    return lib.feather_product(a, lda, a_across, b, ldb, b_across, bias, type, c, ldc, M, N, K, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(a=None), dict(a=X + 8), dict(b=None), dict(b=W + 2), dict(c=None), dict(c=Y + 1), dict(lda=56), dict(lda=66), dict(ldb=56),
    dict(a_across=True), dict(a_across=True, b_across=True, lda=4), dict(b_across=True, ldb=32), dict(bias=S + 1), dict(type=2),
    dict(ldc=39), dict(M=0), dict(N=0), dict(K=0), dict(K=-8), dict(N=1 << 30), dict(K=1 << 22, lda=1 << 22, ldb=1 << 22),
])
def test_product_refuses(lib, bad):
    assert not _product(lib, **bad)


def _int4(lib, x=X, ldx=64, codes=W, ld_codes=32, scale=S, ld_scale=40, zero=None, ld_zero=40, group=32, bias=None, type=0, gated=False,
          act=0, y=Y, ldy=40, M=4, N=40, K=64, ws=None, ws_bytes=0):
    return lib.feather_int4_linear(x, ldx, codes, ld_codes, scale, ld_scale, zero, ld_zero, group, bias, type, gated, act, y, ldy,
                                   M, N, K, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=X + 2), dict(ldx=56), dict(ldx=68), dict(codes=None), dict(codes=W + 2), dict(ld_codes=28), dict(ld_codes=34),
    dict(ld_codes=(1 << 22) + 4), dict(scale=None), dict(scale=S + 1), dict(ld_scale=39), dict(zero=T, ld_zero=39), dict(group=16),
    dict(group=48), dict(group=256), dict(bias=Z + 1), dict(type=2), dict(gated=True), dict(act=3), dict(y=None), dict(y=Y + 1),
    dict(ldy=39), dict(M=0), dict(N=0), dict(K=0), dict(M=100, codes=W + 4), dict(M=100, ld_codes=36), dict(N=2, ld_scale=2),
])
def test_int4_refuses(lib, bad):
    assert not _int4(lib, **bad)


def test_int4_weights_refuse(lib):
    def dequantize(codes=W, ld_codes=32, scale=S, ld_scale=40, zero=None, ld_zero=40, group=32, type=0, w=Y, ldw=64, N=40, K=64):
        return lib.feather_int4_dequantize(codes, ld_codes, scale, ld_scale, zero, ld_zero, group, type, w, ldw, N, K, None)

    for bad in (dict(codes=None), dict(codes=W + 1), dict(ld_codes=28), dict(ld_codes=33), dict(scale=None), dict(ld_scale=39), dict(zero=T, ld_zero=3),
                dict(group=100), dict(type=2), dict(w=None), dict(w=Y + 2), dict(ldw=60), dict(ldw=56), dict(N=0), dict(K=0)):
        assert not dequantize(**bad), bad

    def quantize(w=Y, ldw=64, type=0, group=32, codes=W, ld_codes=32, scale=S, ld_scale=40, zero=None, ld_zero=40, N=40, K=64):
        return lib.feather_int4_quantize(w, ldw, type, group, codes, ld_codes, scale, ld_scale, zero, ld_zero, N, K, None)

    for bad in (dict(w=None), dict(w=Y + 1), dict(ldw=63), dict(type=2), dict(group=0), dict(codes=None), dict(codes=W + 2), dict(ld_codes=28),
                dict(scale=None), dict(ld_scale=39), dict(zero=T, ld_zero=39), dict(N=0), dict(K=0)):
        assert not quantize(**bad), bad


def test_workspaces(lib):
    """Those of split products: a short, missing or unaligned one is refused."""
    calls = {
        "product": (lambda m, n, k: lib.feather_product_workspace_bytes(m, n, k),
                    lambda m, n, k, ws, size: _product(lib, M=m, N=n, K=k, lda=k, ldb=k, ldc=n, ws=ws, ws_bytes=size)),
        "gated": (lambda m, n, k: lib.feather_gated_linear_workspace_bytes(m, n, k),
                  lambda m, n, k, ws, size: _gated(lib, M=m, F=n, K=k, ldx=k, ldw=k, ldy=n, ws=ws, ws_bytes=size)),
        "int4": (lambda m, n, k: lib.feather_int4_linear_workspace_bytes(m, n, k, False),
                 lambda m, n, k, ws, size: _int4(lib, M=m, N=n, K=k, ldx=k, ldy=n, ld_codes=k, ld_scale=n, ws=ws, ws_bytes=size)),
    }
    for need, call in calls.values():
        assert need(0, 8, 64) == -1 and need(8, 0, 64) == -1 and need(8, 8, 0) == -1
        seen = set()
        for m, n, k in ((1, 64, 16384), (64, 512, 8192), (100, 256, 4096), (1000, 1000, 8192), (4096, 16384, 512), (4, 40, 64)):
            size = need(m, n, k)
            assert 0 <= size < 1 << 31
            seen.add(size > 0)
            if size:
                for ws, given in ((None, size), (T, size - 1), (T + 16, size)):
                    assert not call(m, n, k, ws, given)
        assert seen == {False, True}


@pytest.mark.parametrize("mode", ["fake", "symbolic"])
def test_shapes_under_fake_tensors(mode):
    from torch.fx.experimental.symbolic_shapes import ShapeEnv

    def block(x, norm, wide, codes, scale, zero):
        y = fo.gated_linear(fo.rms_norm(x, norm), wide, None, "gelu")
        return fo.int4_linear(y, codes, scale, zero)

    with FakeTensorMode(shape_env=ShapeEnv()):
        def new(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, dtype=dtype, device="cuda")

        u8 = torch.uint8
        args = (new(2, 7, 256), new(256), new(160, 256), new(72, 40, dtype=u8), new(72, 3), new(72, 3, dtype=u8))
        y = block(*args)
        assert y.shape == (2, 7, 72) and y.dtype == torch.bfloat16
        assert fo.int4_gated_linear(new(5, 80), *args[3:]).shape == (5, 36)
        codes, scale, zero = fo.quantize_int4(new(21, 130), 64, zeros=True)
        assert codes.shape == (21, 65) and scale.shape == zero.shape == (21, 3) and scale.stride(0) == 1
        assert fo.dequantize_int4(codes, scale, zero, 129).shape == (21, 129) and fo.quantize_int4(new(4, 8))[2] is None
    nodes = [n for n in make_fx(block, tracing_mode=mode)(*args).graph.nodes if "feather_ops" in str(n.target)]
    assert len(nodes) >= 3


def test_cpu_tensors_are_refused():
    x, codes = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.uint8)
    scale = torch.ones(8, 1, dtype=torch.bfloat16)
    for call in (lambda: fo.gated_linear(x, x), lambda: fo.int4_linear(x, codes, scale), lambda: fo.int4_gated_linear(x, codes, scale),
                 lambda: fo.quantize_int4(x), lambda: fo.dequantize_int4(codes, scale)):
        with pytest.raises(NotImplementedError):
            call()


def test_arguments_are_checked_without_a_gpu():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    codes, scale = torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1, dtype=torch.bfloat16)
    for call in (lambda: fo.gated_linear(x.float(), w.float()), lambda: fo.gated_linear(x, w.half()), lambda: fo.gated_linear(x, w[:3]),
                 lambda: fo.gated_linear(x, w[:, :8]), lambda: fo.gated_linear(x, w, x[0, :3]), lambda: fo.gated_linear(x, w, None, "relu"),
                 lambda: fo.int4_linear(x.float(), codes, scale), lambda: fo.int4_linear(x[:, :32], codes, scale),
                 lambda: fo.int4_linear(x, codes.int(), scale), lambda: fo.int4_linear(x, codes, scale[:4]),
                 lambda: fo.int4_linear(x, codes, scale, scale), lambda: fo.int4_gated_linear(x, codes[:7], scale[:7]),
                 lambda: fo.quantize_int4(x, 48), lambda: fo.quantize_int4(x.float()), lambda: fo.dequantize_int4(codes, scale.float())):
        with pytest.raises(ValueError):
            call()


def test_relabelling():
    model = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.ReLU(), torch.nn.Linear(32, 16))
    assert fo.to_int4_linear(model) == 0 and type(model[0]) is torch.nn.Linear   # fp32 weights stay
    with FakeTensorMode():
        kw = dict(device="cuda", dtype=torch.bfloat16)
        model = torch.nn.Sequential(torch.nn.Linear(64, 32, **kw), torch.nn.ReLU(), torch.nn.Linear(32, 16, **kw))
        keys = list(model.state_dict())
        assert fo.to_int4_linear(model, 32, accept=lambda m: isinstance(m, torch.nn.Linear) and m.in_features == 64) == 1
        assert isinstance(model[0], fo.Int4Linear) and not isinstance(model[2], fo.Int4Linear)
        assert list(model.state_dict()) == keys and model(torch.empty(3, 64, dtype=torch.bfloat16, device="cuda")).shape == (3, 16)


PROGRAM = """
import torch
import feather_ops as fo
from torch._subclasses.fake_tensor import FakeTensorMode

with FakeTensorMode():
    new = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="cuda")
    x, w = new(4, 256), new(128, 256)
    int4 = fo.quantize_int4(w)
    print(int4[0].shape, fo.dequantize_int4(*int4).shape, fo.int4_gated_linear(x, *int4).shape)
    for call in (lambda: fo.gated_linear(x, w), lambda: fo.int4_linear(x, *int4)):
        try:
            call()
            print("no error")
        except ImportError as error:
            print("ImportError", "_autograd.so" in str(error), "make -C feather-ops_amd" in str(error))
"""


def test_without_the_library_of_autograd_nodes(tmp_path):
    copy = tmp_path / "feather_ops"
    copy.mkdir()
    for file in PACKAGE.iterdir():
        if file.suffix == ".py":
            shutil.copy(file, copy)
        elif file.suffix == ".so" and file.name != "_autograd.so":
            (copy / file.name).symlink_to(file)
    run = subprocess.run([sys.executable, "-c", PROGRAM], cwd=tmp_path, capture_output=True, text=True, timeout=110)
    assert run.returncode == 0, run.stderr[-2000:]
    assert run.stdout.splitlines() == ["torch.Size([128, 128]) torch.Size([128, 256]) torch.Size([4, 64])"] + ["ImportError True True"] * 2
