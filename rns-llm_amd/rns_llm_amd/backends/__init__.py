from .hip_backend import (
    AdaptiveMetadata,
    HipRNSBackend,
    PreparedAdaptiveRNSWeight,
    PreparedRNSWeight,
    RNSRequestBatchWorkspace,
    RNSWorkspace,
    hip_extension_available,
)
from .kv_cache import KVBatch, KVCache
from .kv_pool import KVPool, KVStep
from .rotary import Rotary

__all__ = [
    "AdaptiveMetadata",
    "HipRNSBackend",
    "KVBatch",
    "KVCache",
    "KVPool",
    "KVStep",
    "PreparedAdaptiveRNSWeight",
    "PreparedRNSWeight",
    "RNSRequestBatchWorkspace",
    "RNSWorkspace",
    "Rotary",
    "hip_extension_available",
]
