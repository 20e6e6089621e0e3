"""tensorcache_b200: the AMO-BQ feature-cache hot path of TensorCache on NVIDIA B200.

Drop-in for the reference's API on that path -- ``compress`` / ``decompress``,
``BlockwiseInt8Codec``, ``quantize_int8_amo_bq`` / ``dequantize_int8_amo_bq``, the symmetric
``quantize_int8_g32`` / ``quantize_int8_adaptive`` / ``dequantize_int8_g32``,
``FusedDequantLinear``, ``ZeroCopyTensorStreamer``, ``FeatureCacheWriter`` /
``FeatureCacheDataset`` -- on hand-written sm_100a CUDA kernels behind a C ABI
(``include/tcb200.h``, ``libtcb200.so``).  Beside it stand low-bit operators the reference does
not have: the MXFP4 codec and product (``quantize_mxfp4``, ``dequantize_mxfp4``, ``mxfp4_matmul``),
linear layers that train with their input kept in 8 bits (``int8_checkpoint_linear``,
``fused_dequant_linear``) and the device-resident ``DeviceFeatureCache``.  There is no Triton, no backend switch
and no CPU implementation: without the built library or a CUDA device the
compute calls raise.
"""
from .checkpoint import Int8CheckpointLinear, fused_dequant_linear, int8_checkpoint_linear
from .codec import (AMO_BQ_PRESETS, BlockwiseInt8Codec, dequantize_int8_amo_bq, dequantize_int8_g32,
                    quantize_int8_adaptive, quantize_int8_amo_bq, quantize_int8_g32)
from .device_cache import DeviceFeatureCache
from .feature_cache import FeatureCacheDataset, FeatureCacheWriter
from .fused_linear import FusedDequantLinear, fused_dequant_matmul
from .mxfp4 import dequantize_mxfp4, mxfp4_matmul, mxfp4_scales_from_rows, mxfp4_scales_to_rows, quantize_mxfp4
from .streamer import ZeroCopyTensorStreamer
from .utils import auto_select_mode, benchmark_tensor, compress, decompress, estimate_compression, selftest_sum_order

__version__ = "0.1.0"
__all__ = [
    "AMO_BQ_PRESETS", "BlockwiseInt8Codec", "quantize_int8_amo_bq", "dequantize_int8_amo_bq",
    "quantize_int8_g32", "quantize_int8_adaptive", "dequantize_int8_g32",
    "compress", "decompress", "estimate_compression", "benchmark_tensor", "auto_select_mode", "selftest_sum_order",
    "FusedDequantLinear", "fused_dequant_matmul",
    "fused_dequant_linear", "int8_checkpoint_linear", "Int8CheckpointLinear",
    "quantize_mxfp4", "dequantize_mxfp4", "mxfp4_matmul", "mxfp4_scales_to_rows", "mxfp4_scales_from_rows",
    "DeviceFeatureCache", "FeatureCacheWriter", "FeatureCacheDataset", "ZeroCopyTensorStreamer",
]
