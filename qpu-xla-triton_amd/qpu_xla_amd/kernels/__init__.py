"""gfx950 kernels of the quantized-linear path, one module per reference kernel module."""

from qpu_xla_amd.kernels.add_rms_norm import (  # noqa: F401
    ADD_RMS_NORM_KERNEL,
    AddRmsNormOptions,
    add_rms_norm,
    add_rms_norm_grid,
    add_rms_norm_int8,
    add_rms_norm_mxfp4,
    add_rms_norm_mxfp8,
    add_rms_norm_q8_0,
)
from qpu_xla_amd.kernels.gemm_int8 import (  # noqa: F401
    TILED_W8A8_GEMM_DEQUANTIZE_KERNEL,
    TILED_W8A8_GEMM_KERNEL,
    pack_int8_gemm_operands,
    pack_int8_quads,
    supports_tiled_w8a8_gemm,
    supports_tiled_w8a8_gemm_dequantize,
    w8a8_gemm_dequantize,
    w8a8_gemm_i32,
)
from qpu_xla_amd.kernels.gemv_int8 import W8A8_GEMV_KERNEL, supports_w8a8_gemv  # noqa: F401
from qpu_xla_amd.kernels.ggml_geglu_q8 import (  # noqa: F401
    GGML_GEGLU_Q8_0_KERNEL,
    GGML_GEGLU_Q8_0_SPLIT_KERNEL,
    ggml_geglu_q8_0,
    ggml_geglu_q8_0_split,
    ggml_gelu_fp16_table,
    supports_ggml_geglu_q8_0,
    supports_ggml_geglu_q8_0_split,
)
from qpu_xla_amd.kernels.ggml_q4_0 import (  # noqa: F401
    GGML_Q4_0_Q8_0_LINEAR_KERNEL,
    GGML_Q4_0_Q8_0_TILED_LINEAR_KERNEL,
    Q4_0LaneWeights,
    Q4_0LinearBatch,
    ggml_q4_0_q8_0_block_dots,
    ggml_q4_0_q8_0_lane_linear,
    ggml_q4_0_q8_0_linear,
    ggml_q4_0_q8_0_tiled_linear,
    pack_ggml_q4_0_blocks,
    pack_ggml_q4_0_lane_weights,
    pack_ggml_q4_0_tiled_weights,
    pack_ggml_q8_0_blocks,
    split_ggml_q8_0_blocks,
    supports_ggml_q4_0_q8_0_linear,
    supports_ggml_q4_0_q8_0_tiled_linear,
    unpack_ggml_q4_0_blocks,
    unpack_ggml_q8_0_blocks,
)
from qpu_xla_amd.kernels.ggml_q8_0 import (  # noqa: F401
    GGML_Q8_0_Q8_0_LINEAR_M4_KERNEL,
    ggml_q8_0_q8_0_linear,
    supports_ggml_q8_0_q8_0_linear_m4,
)
from qpu_xla_amd.kernels.mxfp4 import (  # noqa: F401
    MXFP4_GATED_GEMM_KERNEL,
    MXFP4_GEMM_KERNEL,
    Mxfp4GatedOptions,
    dequantize_mxfp4,
    dequantize_mxfp8,
    mxfp4_gated_gemm,
    mxfp4_gated_linear,
    mxfp4_gemm,
    mxfp4_gemm_grid,
    mxfp4_linear,
    quantize_mxfp4,
    quantize_mxfp8,
)
from qpu_xla_amd.kernels.paged_attention import (  # noqa: F401
    PAGED_ATTENTION_KERNEL,
    PAGED_ATTENTION_SCORES_KERNEL,
    PagedAttentionOptions,
    paged_attention,
    paged_attention_grid,
    paged_attention_scores,
)
from qpu_xla_amd.kernels.paged_eviction import (  # noqa: F401
    PAGED_CACHE_EVICT_KERNEL,
    PagedEvictionOptions,
    paged_cache_evict,
    paged_cache_evict_grid,
)
from qpu_xla_amd.kernels.qk_norm_rope import (  # noqa: F401
    QK_NORM_ROPE_CACHE_KERNEL,
    QkNormRopeOptions,
    qk_norm_rope,
    qk_norm_rope_cache,
    qk_norm_rope_grid,
)
from qpu_xla_amd.kernels.quantize import quantize_q4_0, quantize_q8_0, quantize_rows_int8  # noqa: F401
from qpu_xla_amd.kernels.w8a8_epilogue import W8A8_DEQUANTIZE_KERNEL, supports_w8a8_dequantize, w8a8_dequantize  # noqa: F401
