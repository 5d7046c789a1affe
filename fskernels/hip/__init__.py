"""The single HIP backend of the decode hot path (gfx950): it replaces the
reference's fskernels.triton, fskernels.cuda and fskernels.tilelang decode
modules, and has operators beside them that the reference leaves to torch or lacks
(the norm and rotation of queries and keys, the shared-prefix decode).  The HF
attention and rotary patches are in fskernels.hip.hf."""
from .decode import (FP8_DTYPE, FP8_MAX, flash_decode_gqa_hf_dense_optimized,
                     flash_decode_gqa_hf_fp8, flash_decode_gqa_varlen, fp8_decode_table,
                     paged_flash_decode, paged_flash_decode_shared, paged_gather, quantize_to_fp8, set_num_splits,
                     set_num_splits_fp8)
from .kv_write import paged_kv_write
from .rotary import paged_kv_write_rope, qk_norm_rope

__all__ = [
    "FP8_DTYPE", "FP8_MAX", "flash_decode_gqa_varlen", "flash_decode_gqa_hf_dense_optimized",
    "flash_decode_gqa_hf_fp8", "paged_flash_decode", "paged_flash_decode_shared",
    "quantize_to_fp8", "set_num_splits",
    "set_num_splits_fp8", "paged_gather", "fp8_decode_table", "paged_kv_write",
    "paged_kv_write_rope", "qk_norm_rope",
]
