"""B200 (sm_100a) execution backend for Tila's typed TIR.

Importing this package installs the backend into the installed Tila runtime:
launches of ``@ti.jit`` kernels on CUDA tensors are code-generated to CUDA
C++, compiled with NVRTC for sm_100a and launched through the native C ABI
(``libtila_b200.so``).  CPU arrays still run on Tila's NumPy interpreter.

``tila_b200.ops`` holds hand-written operators that stand around a model's
attention (rotary positions, query/key norms, a paged cache and the attention
that reads it).  They need no Tila: where it is not installed, the package
offers them alone, and every other name raises the ImportError that says so.
"""

import importlib

try:
    from ._reference import tila
except ImportError as _missing:
    _no_tila = str(_missing)
else:
    _no_tila = None
    from .plugin import B200, install, installed, uninstall
    from .backend import check_device_errors, program_range, read_device_errors, generated_source

    install()

__all__ = ["tila", "B200", "install", "uninstall", "installed", "program_range",
           "read_device_errors", "check_device_errors", "generated_source"]


def __getattr__(name):
    if name == "ops":                      # imports torch, which a Tila program may do without
        return importlib.import_module(".ops", __name__)
    if _no_tila is not None and name in __all__:
        raise ImportError(_no_tila)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
