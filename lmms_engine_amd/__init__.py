"""MI355X-native Muon optimizer step (drop-in for lmms_engine.utils.muon_utils)."""
from .layers import gated_linear, linear  # noqa: F401
from .muon_utils import (  # noqa: F401
    Muon,
    SingelDeviceWork,
    Work,
    adam_update,
    apply_momentum,
    apply_scaling,
    fast_newtonschulz,
    matmul_transpose,
    matmul_transpose_assign,
    muon_update,
)
from .rows import dropout, embedding, layer_norm, rms_norm  # noqa: F401

__all__ = [
    "Muon",
    "SingelDeviceWork",
    "Work",
    "adam_update",
    "apply_momentum",
    "apply_scaling",
    "dropout",
    "embedding",
    "fast_newtonschulz",
    "gated_linear",
    "layer_norm",
    "linear",
    "matmul_transpose",
    "matmul_transpose_assign",
    "muon_update",
    "rms_norm",
]
