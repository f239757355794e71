"""Loads an operator shim (csrc/train_op.cpp, csrc/serve_op.cpp) and binds it to the kernel library that the package has loaded."""
import ctypes as C
import os

import torch

from . import _lib


def load(path: str, bind: str, names):
    """The operators `names` of torch.ops.albatross_b200, from the shim at `path`."""
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -m albatross_b200.build`")
    torch.ops.load_library(path)
    missing = C.c_char_p()
    f = getattr(C.CDLL(path), bind)
    f.argtypes = [C.c_char_p, C.POINTER(C.c_char_p)]
    if f(_lib.LIB_PATH.encode(), C.byref(missing)):
        raise ImportError(f"{_lib.LIB_PATH} does not have {missing.value.decode()}: build both again with `python -m albatross_b200.build`")
    ops = torch.ops.albatross_b200
    return [getattr(ops, n).default for n in names]
