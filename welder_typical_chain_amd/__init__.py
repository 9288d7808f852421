"""MI355X-native (gfx950) fused Matmul -> row-Softmax, the hot path of the
Welder typical chain, behind the reference's compile / solver C entry points,
and the operators of a transformer layer around it (``layer.py``).

Importing the package needs neither a GPU nor the built library; the first
call into the kernels loads ``libwtc_hip.so`` and fails loudly if it is
missing.
"""
from . import _lib  # noqa: F401

_CHAIN = ["matmul_softmax", "workspace_size", "new_workspace", "read_error_flags"]
_LAYER = ["matmul_epilogue", "matmul_epilogue_backward", "window_attention", "window_attention_backward",
          "window_attention_decode"]
__all__ = _CHAIN + _LAYER


def __getattr__(name):
    if name in _CHAIN:
        from . import chain
        return getattr(chain, name)
    if name in _LAYER:
        from . import layer
        return getattr(layer, name)
    raise AttributeError(name)
