"""The PyTorch functions of lib/mm_torch_ops.so (csrc/torch/ops.cpp): layer norm, routing and the experts' products with
their autograd nodes.  Built in-tree by mace-million_amd/build.py against the installed torch; there is no fallback."""
import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (its libraries are loaded before the extension's)

from . import _lib

PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "mm_torch_ops.so")
_ops = None


def ops():
    global _ops
    if _ops is None:
        _lib.lib()                                    # refuses a library of other argument conventions
        if not os.path.exists(PATH):
            raise RuntimeError(f"MI355X operators not built: {PATH} is missing (run python mace-million_amd/build.py)")
        loader = importlib.machinery.ExtensionFileLoader("mm_torch_ops", PATH)
        mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("mm_torch_ops", loader))
        try:
            loader.exec_module(mod)
        except ImportError as e:
            raise RuntimeError(f"{PATH} does not load with this torch {torch.__version__}: rebuild it "
                               f"(python mace-million_amd/build.py): {e}") from e
        _ops = mod
    return _ops
