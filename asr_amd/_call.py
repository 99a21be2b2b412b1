"""The operators bound through torch_binding.cpp (asr_amd/_torch_ops.so): argument checks, outputs, workspaces and autograd
functions in C++ around the C ABI of the library that asr_amd/_lib.py has loaded."""
from __future__ import annotations

import ctypes
import os

import torch  # noqa: F401  (its libraries have to be loaded first)

from . import _lib

if not os.path.exists(os.path.join(os.path.dirname(os.path.abspath(__file__)), "_torch_ops.so")):
    raise ImportError("asr_amd/_torch_ops.so is missing: build it with `make -C asr_amd/csrc` "
                      "(or `python -c 'import __graft_entry__ as g; g.build()'`). asr_amd has no CPU or eager fallback.")
from . import _torch_ops as ops  # noqa: E402

# the entry points are bound by name: only the version tells that their arguments are those the binding was compiled for
if getattr(ops, "abi_version", None) != _lib.ABI_VERSION:
    raise ImportError(f"asr_amd/_torch_ops.so: ABI version {getattr(ops, 'abi_version', None)}, expected {_lib.ABI_VERSION}; "
                      "rebuild it (`make -C asr_amd/csrc`)")
ops.bind({name: ctypes.cast(getattr(_lib.lib, name), ctypes.c_void_p).value for name in ops.entries if name})
