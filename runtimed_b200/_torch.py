"""The binding that hands torch tensors to the C ABI (csrc/rtd_torch.cpp): it reads the
tensors' fields, checks them and calls the library without ctypes' conversions, on the
current stream of the tensors' device.  Loading fails loudly when it is not built."""
from __future__ import annotations

import torch  # noqa: F401  (its libraries come first)

from . import _lib
from .errors import ConfigError, ShapeError
from .weights import Context, _raise

_lib.lib()
try:
    from . import _rtd_torch as binding
except ImportError as e:
    raise ImportError(f"runtimed_b200/_rtd_torch.so cannot be loaded ({e}): run `python -m runtimed_b200.build`; "
                      "there is no fallback path") from e


def _fail(status: int, device: int) -> None:
    if status == _lib.RTD_ERR_SHAPE:  # the binding has checked the shapes: what is left is a bound of the call's numbers
        msg = _lib.lib().rtd_last_error(Context.for_device(device).handle)
        raise ConfigError(msg.decode() if msg else "rtd: shape")
    _raise(status, Context.for_device(device).handle)


def _address(device: int) -> int:
    h = Context.for_device(device).handle
    return 0 if h is None else h.value


binding.setup(ConfigError, ShapeError, _fail, _address)
