"""sm_100a (B200) MedNeXt training operators behind the mednext-accel API.

Public names mirror the reference package ``mednext_accel``: the v1 factories,
``MedNeXtV1`` / ``MedNeXtV1Config`` / ``get_mednext_v1_config``,
``CheckpointConfig``, the adaptive operator wrappers and the
``PolicyResolver`` / ``PolicyDecision`` selection API.  The CUDA kernels live in
``lib/libmednext_b200.so`` (C ABI declared in ``include/mednext_b200.h``) and are
loaded on first use.
"""

from .adaptive import (
    AdaptiveDepthwise3d,
    AdaptivePointwise3d,
    ModelOptimizationContext,
    install_adaptive_operators,
)
from .drop import dropout
from .grn import (
    AdaptiveGlobalResponseNorm3d,
    GlobalResponseNorm3d,
    fused_global_response_norm3d,
    global_response_norm3d_reference,
    install_adaptive_grn,
)
from .loss import cross_entropy
from .mixer import ChannelMixer3d, Int8ChannelMixer3d
from .network import (
    CheckpointConfig,
    MedNeXtBlock,
    MedNeXtDownBlock,
    MedNeXtUpBlock,
    MedNeXtV1,
    MedNeXtV1Config,
    OutputHead,
    get_mednext_v1_config,
    mednext_base,
    mednext_large,
    mednext_medium,
    mednext_small,
)
from .norm import LayerNorm3d, layer_norm
from .optimization import (
    ExecutionContext,
    ImplementationRegistry,
    ImplementationSpec,
    OperatorDescriptor,
    OptimizationReport,
    PolicyDecision,
    PolicyResolver,
    default_implementation_registry,
)
from .quant import Int8Pointwise3d, int8_linear, quantize_int8

__version__ = "0.1.0"

__all__ = [
    "AdaptiveDepthwise3d",
    "AdaptiveGlobalResponseNorm3d",
    "GlobalResponseNorm3d",
    "fused_global_response_norm3d",
    "global_response_norm3d_reference",
    "install_adaptive_grn",
    "AdaptivePointwise3d",
    "ChannelMixer3d",
    "CheckpointConfig",
    "ExecutionContext",
    "ImplementationRegistry",
    "ImplementationSpec",
    "Int8ChannelMixer3d",
    "Int8Pointwise3d",
    "LayerNorm3d",
    "MedNeXtBlock",
    "MedNeXtDownBlock",
    "MedNeXtUpBlock",
    "MedNeXtV1",
    "MedNeXtV1Config",
    "ModelOptimizationContext",
    "OperatorDescriptor",
    "OptimizationReport",
    "OutputHead",
    "PolicyDecision",
    "PolicyResolver",
    "cross_entropy",
    "default_implementation_registry",
    "dropout",
    "get_mednext_v1_config",
    "install_adaptive_operators",
    "int8_linear",
    "layer_norm",
    "mednext_base",
    "mednext_large",
    "mednext_medium",
    "mednext_small",
    "quantize_int8",
]
