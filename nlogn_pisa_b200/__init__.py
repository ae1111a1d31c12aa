"""B200 (sm_100a) implementation of PISA's hot path: hierarchical LSE block
selection over a mean-pooled key pyramid, then attention over the selected
key blocks.

The operators keep the reference package's names and signatures
(``pisa.ops``: select_blocks / top_k_pyramid_fn, sparse_attention /
sparse_attn_fn, mean_pool, build_pyramid; ``xmixers`` PyramidCache /
TensorCache).  All computation runs in the hand-written CUDA library
``libpisa_b200.so`` through its C ABI (include/pisa_b200.h).
"""

from .attention import sparse_attention, sparse_attn_fn
from .cache import PyramidCache, TensorCache
from .dense import full_attention, prefix_attention
from ._lib import set_status_checks
from .int8 import Int8Linear, checkpoint_int8, int8_linear, quantize_int8, restore_int8
from .norm_rotary import qk_norm_rotary
from .residual_norm import residual_norm
from .selection import (bsa_fn, build_pyramid, decode_select_attend, grouped_leaf_scores, mean_pool,
                        routing_geometry, select_blocks, top_k_pyramid_fn)
from .swiglu import swiglu, swiglu_ffn

mean_pooling_fn = mean_pool

__all__ = [
    "select_blocks", "top_k_pyramid_fn", "sparse_attention", "sparse_attn_fn", "mean_pool",
    "mean_pooling_fn", "build_pyramid", "routing_geometry", "PyramidCache", "TensorCache",
    "grouped_leaf_scores", "set_status_checks", "decode_select_attend", "bsa_fn",
    "full_attention", "prefix_attention", "qk_norm_rotary", "residual_norm", "swiglu", "swiglu_ffn", "quantize_int8",
    "int8_linear", "Int8Linear", "checkpoint_int8", "restore_int8",
]
