"""Builds (in-tree, under build/torch_ext) and loads the torch extensions.

``cail_torch`` is the GIL-free MPI_Allreduce on tensors; ``cail_ops_torch``
binds the language-model operators of ``libcail_ops.so``.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
import threading

from .. import _lib

_SRC_DIR = os.path.join(_lib.ROOT, "csrc", "torch_ext")
_SRC = os.path.join(_SRC_DIR, "cail_torch.cpp")
_OPS_SRC = os.path.join(_SRC_DIR, "cail_ops_torch.cpp")
_OPS_H = os.path.join(_lib.ROOT, "csrc", "lmops", "include", "cail_ops.h")
_BUILD = os.path.join(_lib.BUILD, "torch_ext")
_OPS_BUILD = os.path.join(_lib.BUILD, "torch_ext_ops")
_mod = None
_ops_mod = None
_ops_lock = threading.Lock()


def build(verbose: bool = False):
    """Compiles cail_torch into build/torch_ext (no-op when up to date)."""
    from torch.utils.cpp_extension import load

    os.makedirs(_BUILD, exist_ok=True)
    return load(name="cail_torch", sources=[_SRC], build_directory=_BUILD, extra_cflags=["-O2"],
                verbose=verbose)


def get():
    """The loaded cail_torch, wired to the interposer chosen by cail_b200.init()."""
    global _mod
    if _mod is None:
        libs = _lib.loaded()
        if libs is None:
            raise RuntimeError("cail_b200.init() must run before the extension is used")
        _mod = build()
        addr = ctypes.cast(libs.cail.MPI_Allreduce, ctypes.c_void_p).value
        _mod.set_allreduce(addr, _lib.H["MPI_IN_PLACE"])
    return _mod


def build_ops(verbose: bool = False):
    """Compiles cail_ops_torch into build/torch_ext_ops (a finished build that
    is newer than its sources is loaded as it is)."""
    so = os.path.join(_OPS_BUILD, "cail_ops_torch.so")
    if os.path.exists(so) and os.path.getmtime(so) >= max(os.path.getmtime(_OPS_SRC), os.path.getmtime(_OPS_H)):
        spec = importlib.util.spec_from_file_location("cail_ops_torch", so)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        return mod
    from torch.utils.cpp_extension import load

    os.makedirs(_OPS_BUILD, exist_ok=True)
    return load(name="cail_ops_torch", sources=[_OPS_SRC], build_directory=_OPS_BUILD, extra_cflags=["-O2"],
                with_cuda=True, verbose=verbose)


def get_ops():
    """The loaded cail_ops_torch, wired to build/lib/libcail_ops.so.  Needs no
    cail_b200.init(): these operators do not communicate."""
    global _ops_mod
    if _ops_mod is None:
        with _ops_lock:
            if _ops_mod is None:
                path = _lib.lib_path("libcail_ops.so")
                if not os.path.exists(path):
                    raise FileNotFoundError(f"{path} missing: run cail_b200.build.build_native() first")
                import torch  # noqa: F401  (the extension links against it)

                mod = build_ops()
                mod.load(path)
                _ops_mod = mod
    return _ops_mod
