"""HIP kernels for the codec/vocoder decode path, with the reference kernels' Python API."""

from .bias_snake_beta import SnakeBetaCoefficients, fused_bias_snake_beta
from .block_fp8 import (
    BlockFp8Rows,
    BlockFp8Weight,
    block_fp8_linear,
    block_fp8_weight,
    pack_block_fp8,
    quantize_block_rows,
)
from .channel_embedding import ChannelEmbeddingTables
from .codec_state import history_exchange, overlap_exchange
from .conv import (
    PackedConv,
    ResidualUnitWeights,
    fused_conv,
    pack_conv1d,
    pack_conv_transpose1d,
    residual_stack,
)
from .gated_norm import gated_residual_norm
from .logits import adjust_logits
from .rotary import apply_rotary, rotary_frequencies
from .rvq import rvq_gather_sum
from .single_output_conv import clamped_single_output_conv, single_output_conv

__all__ = [
    "BlockFp8Rows",
    "BlockFp8Weight",
    "ChannelEmbeddingTables",
    "PackedConv",
    "ResidualUnitWeights",
    "SnakeBetaCoefficients",
    "adjust_logits",
    "apply_rotary",
    "block_fp8_linear",
    "block_fp8_weight",
    "clamped_single_output_conv",
    "fused_bias_snake_beta",
    "fused_conv",
    "gated_residual_norm",
    "history_exchange",
    "overlap_exchange",
    "pack_block_fp8",
    "pack_conv1d",
    "pack_conv_transpose1d",
    "quantize_block_rows",
    "residual_stack",
    "rotary_frequencies",
    "rvq_gather_sum",
    "single_output_conv",
]
