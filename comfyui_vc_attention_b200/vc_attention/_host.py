"""The extension with the host side of the block operators (csrc/host_ops.cpp):
argument checks, strided views, output and workspace buffers and the call of
the C ABI.  Built by ``comfyui_vc_attention_b200.build`` beside this file;
loading is lazy and loud, and the entry points it calls are those of the
library that ``_native`` has loaded."""

from __future__ import annotations

import ctypes
import importlib.util
import os

import torch  # noqa: F401  (its libraries are loaded before the extension's)

from . import _native as N

HOST_OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_host_ops.so")

_ENTRY_POINTS = ("vcattn_qk_norm_rope", "vcattn_quantize_blocks", "vcattn_matmul_blocks",
                 "vcattn_matmul_blocks_workspace_bytes", "vcattn_attn_packed")
_mod = None


def host_ops():
    """The loaded extension; raises NativeUnavailable (never falls back)."""
    global _mod
    if _mod is None:
        lib = N.lib()
        if not os.path.exists(HOST_OPS_PATH):
            raise N.NativeUnavailable(f"{HOST_OPS_PATH} not found; build it with "
                                      f"`python -m comfyui_vc_attention_b200.build`")
        try:
            spec = importlib.util.spec_from_file_location(__package__ + "._host_ops", HOST_OPS_PATH)
            mod = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(mod)
        except ImportError as e:
            raise N.NativeUnavailable(f"failed to load {HOST_OPS_PATH}: {e}") from e
        mod.bind(mod, {name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRY_POINTS}, N.check)
        _mod = mod
    return _mod
