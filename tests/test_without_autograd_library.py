"""The package without the library of autograd nodes (torch's unstable C++ interface), without a GPU: what does not need it
works, what does says so."""

import pathlib
import shutil
import subprocess
import sys

import pytest

PACKAGE = pathlib.Path(__file__).resolve().parents[1] / "feather-ops_amd" / "feather_ops"

PROGRAM = """
import torch
import feather_ops as fo
from torch._subclasses.fake_tensor import FakeTensorMode

with FakeTensorMode():
    new = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="cuda")
    x, w = new(4, 256), new(128, 256)
    f8 = torch.float8_e4m3fn
    print(fo.scaled_mm_hip(x, new(16, 128, 16, dtype=f8), new(dtype=torch.float32), None, torch.bfloat16).shape)
    codes, scale = fo.quantize_blocks(x)
    print(fo.block_scaled_mm(codes, scale, *fo.quantize_blocks(w, square=True)).shape)
    print(fo.rms_norm_quantized(x, w[0])[0].shape, fo.silu_mul_quantized(x)[0].shape)
    leaf = x.clone().requires_grad_()
    for call in (lambda t: fo.silu_mul(t), lambda t: fo.rms_norm(t, w[0]), lambda t: fo.block_scaled_linear(t, w)):
        for t in (x, leaf):
            try:
                call(t)
                print("no error")
            except ImportError as error:
                print("ImportError", "_autograd.so" in str(error), "make -C feather-ops_amd" in str(error))
"""


@pytest.fixture(params=["missing", "unloadable"])
def package(request, tmp_path):
    copy = tmp_path / "feather_ops"
    copy.mkdir()
    for file in PACKAGE.iterdir():
        if file.suffix == ".py":
            shutil.copy(file, copy)
        elif file.suffix == ".so" and file.name != "_autograd.so":
            (copy / file.name).symlink_to(file)
    if request.param == "unloadable":
        (copy / "_autograd.so").write_bytes(b"built for another torch")
    return tmp_path


def _run(package, program):
    return subprocess.run([sys.executable, "-c", program], cwd=package, capture_output=True, text=True, timeout=110)


def test_only_what_needs_it_fails(package):
    run = _run(package, PROGRAM)
    assert run.returncode == 0, run.stderr[-2000:]
    lines = run.stdout.splitlines()
    assert lines[:3] == ["torch.Size([4, 128])", "torch.Size([4, 128])", "torch.Size([4, 256]) torch.Size([4, 128])"]
    assert lines[3:] == ["ImportError True True"] * 6


def test_the_build_asks_for_it(package):
    run = _run(package, "import feather_ops; feather_ops._lib.require_autograd()")
    assert run.returncode != 0 and "ImportError" in run.stderr and "_autograd.so" in run.stderr


def test_other_libraries_are_needed(package):
    (package / "feather_ops" / "_C.so").unlink()
    run = _run(package, "import feather_ops")
    assert run.returncode != 0 and "native extension missing" in run.stderr
