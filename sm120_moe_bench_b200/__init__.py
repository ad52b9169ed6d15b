"""B200 (sm_100a) fused NVFP4 MoE expert layer: PyTorch host side over a C-ABI CUDA library.

Public surface:
  * ``ops``          -- thin torch wrappers of the C entry points (routing, permutation tables,
                        activation quantiser, decoder, the fused layer);
  * ``token_sort``   -- token rows sorted by expert and back, with weights applied, differentiable;
  * ``int8``         -- 8-bit integer rows and products (dense and per expert), the expert layer on 8-bit weights;
  * ``verdict_moe``  -- ``VerdictMoEExperts`` / ``VerdictMoEMonolithic``, the operator classes with the
                        reference's method set and argument meaning;
  * ``synth``        -- seeded synthetic NVFP4 layers in the reference's tensor layout.
"""
from . import _lib  # noqa: F401  (fails loudly when the CUDA library is absent)
from .ops import (MoEShape, MoEWeights, Workspace, build_tables, dequantize, fused_moe,  # noqa: F401
                  quantize, route)
from .int8 import Int8Rows, int8_experts, int8_linear, int8_matmul, int8_status, quantize_int8  # noqa: F401
from .token_sort import TokenPlan, plan_tokens, sort_tokens, unsort_tokens  # noqa: F401
