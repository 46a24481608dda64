"""ssla_hip: host side of the MI355X drain of SSLA-S s2 + s3 + YOLOX head.

  abi     numpy / ctypes mirrors of include/ssla_abi.h
  lib     ctypes binding of libssla_hip.so (include/ssla_hip.h)
  ops     sequence operators on torch tensors: linear attention, group norm, and,
          with gradients, the layers' recurrence and layer norm
  hybrid  device buffers, weight packing, HybridS2S3Config, drain calls
  stub    weight-directory generator (tools/make_ssla_stub.py schema)
  events  seeded synthetic event / ring-record streams
"""
from importlib.util import find_spec as _find

from . import abi, events, stub  # noqa: F401  (no GPU needed)

__all__ = ["abi", "events", "stub", "lib", "hybrid"]
# the operators are on torch's tensors, and built where there is a torch
if _find("torch") and _find(__name__ + "._ops"):
    __all__.append("ops")
