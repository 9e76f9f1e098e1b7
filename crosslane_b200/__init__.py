"""crosslane_b200: B200-native (sm_100a) routed-expert decode lane for crosslane.

The product is the C ABI in include/crosslane_b200.h, implemented by
libcrosslane_b200.so (CUDA kernels + C++ host runtime). This package binds it for
Python callers; importing it fails if the library is not built.
"""
from ._capi import ClbError, lib  # noqa: F401  (raises ImportError if the .so is missing)
from .bank import (BLOCK_BYTES, IQ1_M, IQ2_XS, IQ2_XXS, Q8K_BLOCK_BYTES, ROLE_DOWN, ROLE_GATE,  # noqa: F401
                   ROLE_UP, ExpertBank, lane_config_parse, pack, packed_bytes, q8k_activate, q8k_mv, q8k_quantize,
                   route_b_device, route_device, route_host, router_device, unpack)

_NAMES = ["ExpertBank", "ClbError", "pack", "unpack", "packed_bytes", "route_host", "route_device",
          "router_device", "route_b_device", "lane_config_parse",
          "q8k_quantize", "q8k_mv", "q8k_activate", "IQ2_XXS", "IQ2_XS", "IQ1_M", "BLOCK_BYTES",
          "ROLE_GATE", "ROLE_UP", "ROLE_DOWN", "Q8K_BLOCK_BYTES"]
# these take torch tensors; the rest of the package works without importing torch
_BLOCK_OPS = ["ExpertRoute", "BlockNorm", "Int8Linear", "int8_quantize"]


def __getattr__(name):
    if name == "__all__":  # `import *` brings them where they load
        try:
            from . import block_ops  # noqa: F401
        except (ImportError, OSError):
            return _NAMES
        return _BLOCK_OPS + _NAMES
    if name in _BLOCK_OPS:
        from . import block_ops
        return getattr(block_ops, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__():
    return sorted(set(globals()) | set(_BLOCK_OPS))
