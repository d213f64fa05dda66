"""B200-native (sm_100a) path-ordered geometric attention: forward, generation and training.

Drop-in for SiddhiMali/HolonomyAwareAttention's PathOrderedGeometricMHA
(core/attention.py, core/attention_fast_chunked.py): same constructor,
parameters and forward signature; the causal forward runs in hand-written
CUDA kernels behind the C ABI of libhoa.so (include/hoa.h).
"""
from .attention import PathOrderedGeometricMHA
from . import ops
from .cache import PathCache, decode, prefill
from .training import AdamW, train_step

__all__ = ["PathOrderedGeometricMHA", "PathCache", "prefill", "decode", "AdamW", "train_step", "ops"]
