"""The compiled binding of the operators for language models (binding/fa2_native.cpp): tensors straight to the C ABI."""
from __future__ import annotations

import ctypes as C

from . import _capi

# the functions the module calls, in the order of its `Abi`
_FUNCTIONS = (
    "fa2_document_layout_bytes", "fa2_document_layout", "fa2_fwd_workspace_bytes", "fa2_scored_bwd_workspace_bytes",
    "fa2_scored_fwd", "fa2_scored_bwd", "fa2_paged_work_bytes", "fa2_paged_plan", "fa2_paged_cache_write",
    "fa2_paged_workspace_bytes", "fa2_paged_attention", "fa2_last_error",
)
_module = None


def load():
    """The module, bound to the library that `_capi.load` has loaded. Its functions return None for calls they do not
    take; the Python function of the same name goes on then."""
    global _module
    if _module is None:
        lib = _capi.load()
        try:
            from . import _fa2_native
        except ImportError as e:
            raise ImportError(f"the binding _fa2_native cannot be loaded ({e}): build it with "
                              f"`python {_capi._PKG_ROOT}/build.py`. There is no fallback implementation.") from e
        _fa2_native.bind(*(C.cast(getattr(lib, name), C.c_void_p).value for name in _FUNCTIONS))
        _module = _fa2_native
    return _module
