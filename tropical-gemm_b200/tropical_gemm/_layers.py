"""The torch binding of layer norm, 8-bit floating point layers and token log probabilities."""
import os

from . import _native as N

_ext = None


def ext():
    """The binding (raises if it has not been built)."""
    global _ext
    if _ext is None:
        N.lib()
        path = os.path.join(os.path.dirname(N.LIB_PATH), "_layers_torch.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} not found: build it with `python __graft_entry__.py build` "
                              "(or `make -C tropical-gemm_b200 torch`)")
        from . import _layers_torch
        _ext = _layers_torch
    return _ext
