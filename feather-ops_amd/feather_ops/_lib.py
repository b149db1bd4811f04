"""Loading of the native code: `_C` (the torch library), through it `libfeather_ops_gfx950.so`, and `_autograd.so` (the
autograd nodes of its ops). The first keeps to torch's stable interface, the last cannot, and may fail to load beside another
torch than it was built for: then the operators that need it (`rms_norm`, `silu_mul`, `block_scaled_linear`) raise, and
everything else works.

There is no fallback: if the extension is not built, importing `feather_ops` fails with the build
command, and the ops only have a CUDA (HIP) dispatch key, so CPU tensors are rejected by the dispatcher.
"""

import ctypes
import pathlib

import torch

HERE = pathlib.Path(__file__).resolve().parent
LIBRARY = HERE / "libfeather_ops_gfx950.so"
EXTENSION = HERE / "_C.so"
AUTOGRAD = HERE / "_autograd.so"
BUILD_HINT = "build it with `make -C feather-ops_amd -j8` or `python -c 'import __graft_entry__ as g; g.build()'`"

_loaded = False


def load() -> None:
    """Import `_C`, which registers `torch.ops.feather_ops.*` and loads the HIP library, and load `_autograd.so`."""
    global _loaded
    if _loaded:
        return
    if not EXTENSION.exists() or not LIBRARY.exists():
        raise ImportError(f"feather_ops native extension missing ({EXTENSION.name}, {LIBRARY.name}): {BUILD_HINT}")
    from . import _C  # noqa: F401  registers the feather_ops torch library

    try:
        torch.ops.load_library(str(AUTOGRAD))
    except OSError as error:
        _refuse_autograd(error)

    _loaded = True


_autograd_error: OSError | None = None
_refusals: list[torch.library.Library] = []


def require_autograd(*_args, **_kwargs) -> None:
    """Raise unless `_autograd.so` is loaded."""
    if _autograd_error is not None:
        raise ImportError(f"feather_ops: {AUTOGRAD.name} is missing or does not load ({_autograd_error}): "
                          f"{BUILD_HINT}") from _autograd_error


def _refuse_autograd(error: OSError) -> None:
    """In place of the nodes: ops that raise, rather than results that autograd would lose sight of."""
    global _autograd_error
    _autograd_error = error
    define = torch.library.Library("feather_ops", "FRAGMENT")
    define.define("block_scaled_linear(Tensor x, Tensor weight, Tensor? bias, bool e5m2, Tensor? weight_codes, "
                  "Tensor? weight_scale, Tensor? workspace) -> Tensor")
    define.impl("block_scaled_linear", require_autograd, "CompositeImplicitAutograd")
    nodes = torch.library.Library("feather_ops", "IMPL", "AutogradCUDA")
    for name in ("silu_mul", "rms_norm"):
        nodes.impl(name, require_autograd)
    _refusals.extend((define, nodes))


_c_library = None


def c_library() -> ctypes.CDLL:
    """The HIP library's C ABI through ctypes, for the entry points no torch op wraps (the handle is the one
    `_C` already loaded: the same file)."""
    global _c_library
    if _c_library is None:
        load()
        lib = ctypes.CDLL(str(LIBRARY))
        lib.feather_set_weight_streaming.restype = ctypes.c_int
        lib.feather_set_weight_streaming.argtypes = [ctypes.c_int]
        lib.feather_linear_backward_workspace_bytes.restype = ctypes.c_int64
        lib.feather_linear_backward_workspace_bytes.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_bool]
        lib.feather_linear_backward_depth.restype = ctypes.c_int64
        lib.feather_linear_backward_depth.argtypes = [ctypes.c_int64, ctypes.c_bool]
        lib.feather_linear_backward_split_bytes.restype = ctypes.c_int64
        lib.feather_linear_backward_split_bytes.argtypes = ([ctypes.c_int64] * 3 + [ctypes.c_bool] + [ctypes.c_int] * 5 +
                                                            [ctypes.c_bool, ctypes.c_int])
        lib.feather_block_scaled_mm_workspace_bytes.restype = ctypes.c_int64
        lib.feather_block_scaled_mm_workspace_bytes.argtypes = [ctypes.c_int64] * 3
        _c_library = lib
    return _c_library


def require_native() -> None:
    """Raise unless the HIP extension is loaded (the product path has no CPU fallback)."""
    if not _loaded:
        load()
