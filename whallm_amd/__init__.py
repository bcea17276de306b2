"""MI355X-native (gfx950) MoE expert path: HIP kernels behind a C ABI, with a
torch-facing layer that keeps the reference runtime's expert-FFN operator
signatures (runtime/deepseek_v4_ssd/qwen4_exp.py:763-1051, model.py:318-546)."""

from . import _lib
from .ops import (BlockNormGrads, FP8Experts, MXFP4Experts, Permutation, block_norm, block_norm_backward, combine_pairs, combine_rows, combine_rows_backward, dequant_mxfp4, dequant_fp8_blocks, dequant_fp8_e8m0, experts_fp8, experts_mxfp4,
                  linear_bf16, linear_fp8, mlp_bf16, moe_fp8, moe_mxfp4, mtp_verify_greedy, mtp_verify_rejection, norm_fp8, norm_router, permute, prefill_layout, process_logits, quantize_fp8, repack_router,
                  route_scored, route_softmax_topk, sample_logits, sort_tokens, sort_tokens_backward, split_rows_e2m3, split_rows_e4m3, swiglu_fp8)

__all__ = [
    "BlockNormGrads", "FP8Experts", "MXFP4Experts", "Permutation", "block_norm", "block_norm_backward", "combine_pairs", "combine_rows", "combine_rows_backward", "dequant_mxfp4", "dequant_fp8_blocks", "dequant_fp8_e8m0", "experts_fp8", "experts_mxfp4",
    "linear_bf16", "linear_fp8", "mlp_bf16", "moe_fp8", "moe_mxfp4",
    "mtp_verify_greedy", "mtp_verify_rejection", "norm_fp8", "norm_router", "permute", "repack_router", "prefill_layout", "process_logits", "quantize_fp8", "route_scored", "route_softmax_topk", "sample_logits",
    "sort_tokens", "sort_tokens_backward", "split_rows_e2m3", "split_rows_e4m3", "swiglu_fp8",
]
