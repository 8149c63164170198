"""Loads _trips_host.so, the host side of adamw.py and lookup.py (trips_amd/csrc/torch_shim/trips_host.cpp)."""
import functools

from . import _lib


@functools.lru_cache(maxsize=None)
def host():
    """The extension; raises if it has not been built."""
    _lib.load()
    try:
        from . import _trips_host
    except ImportError as e:
        raise RuntimeError("trips_amd/_trips_host.so cannot be loaded: build it with `python -m trips_amd.build`") from e
    return _trips_host
