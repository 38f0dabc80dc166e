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

__all__ = [
    "AdaptiveMetadata",
    "HipRNSBackend",
    "KVBatch",
    "KVCache",
    "PreparedAdaptiveRNSWeight",
    "PreparedRNSWeight",
    "RNSRequestBatchWorkspace",
    "RNSWorkspace",
    "hip_extension_available",
]
