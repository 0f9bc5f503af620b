"""Loads ``libs/_d3d_host.so`` (csrc/host), the native path of a plugin's ``enqueue`` and of the operators without a plugin.

The module gets the addresses of the C-ABI entry points from the library that ``_lib`` has loaded, so that the checked
and the tuning builds go through the same path.  There is no interpreted fallback: a missing module is an error.
"""
import ctypes
import importlib.machinery
import importlib.util
import os

from . import _lib

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libs", "_d3d_host.so")
_MODULE = None


def module():
    global _MODULE
    if _MODULE is None:
        import torch  # noqa: F401  (its libraries must be in the process before the module is)
        if not os.path.exists(PATH):
            raise RuntimeError("%s is missing: build it with `python -m deploy3d_b200.build`" % PATH)
        loader = importlib.machinery.ExtensionFileLoader("_d3d_host", PATH)
        mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("_d3d_host", loader))
        loader.exec_module(mod)
        mod.set_check(_lib.check)
        _MODULE = mod
    return _MODULE


def _address(name):
    fn = getattr(_lib.lib(), name) if name in _lib.SIGNATURES else None
    return ctypes.cast(fn, ctypes.c_void_p).value if fn is not None else 0


def call(name, prefix):
    """Native enqueue of the plugin `name` whose C-ABI functions start with `prefix`."""
    return module().Call(name, prefix, _address(prefix + "_output_desc"), _address(prefix + "_workspace"),
                         _address(prefix + "_enqueue"))


_SEQUENCE = ("d3d_layer_norm", "d3d_layer_norm_int8", "d3d_layer_norm_backward", "d3d_layer_norm_backward_workspace",
             "d3d_quantize_rows", "d3d_int8_linear", "d3d_int8_linear_workspace", "d3d_gated_recurrence",
             "d3d_gated_recurrence_backward", "d3d_gated_recurrence_step", "d3d_gated_recurrence_state_rows",
             "d3d_gated_recurrence_workspace")  # in the order of csrc/host/sequence.cpp
_BOUND = False


def sequence():
    """The module with the voxel-sequence operators' entry points in place."""
    global _BOUND
    mod = module()
    if not _BOUND:
        mod.bind_sequence(tuple(_address(name) for name in _SEQUENCE))
        _BOUND = True
    return mod
