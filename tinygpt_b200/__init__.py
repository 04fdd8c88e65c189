"""tinygpt_b200 -- B200-native batched logits processing and sampling.

The product is the CUDA library libtgsample.so behind the C ABI in
include/tgsample.h; this package builds it, binds it with ctypes and offers a
host API with the reference sampler's parameter names (tinygpt_b200.sampler).
"""
from .beam import BeamSearch  # noqa: F401
from .cache import PagedCache, tree_masks  # noqa: F401
from .sampler import Sampler, SpecVerifier, sample_next, row_params  # noqa: F401

__all__ = ["BeamSearch", "PagedCache", "Sampler", "SpecVerifier", "sample_next", "row_params", "tree_masks"]
