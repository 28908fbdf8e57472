"""ffn_kernel_amd — mask-routed linear / SwiGLU FFN for AMD MI355X (gfx950).

Drop-in for the `ffn_kernel` package of wenhaoli-xmu/ffn_kernel (ffn_kernel/__init__.py:1):
    from ffn_kernel_amd import MaskedLinear, MaskedFFN
"""
from .modules import MaskedFFNModule, MaskedFFNMXFP4Module, MaskedLinearModule, MaskedLinearMXFP4Module
from .mxfp4 import (MXFP4, MaskedFFNMXFP4, MaskedLinearMXFP4, masked_ffn_mxfp4_backward, masked_ffn_mxfp4_forward,
                    masked_linear_mxfp4_backward, masked_linear_mxfp4_forward, mxfp4_dequantise, mxfp4_quantise)
from .ops import (MaskedFFN, MaskedLinear, Routing, masked_ffn_backward, masked_ffn_forward, masked_linear_backward,
                  masked_linear_forward, route, set_route_cache, shared_routing)

__all__ = ["MaskedLinear", "MaskedFFN", "MaskedLinearModule", "MaskedFFNModule", "masked_linear_forward",
           "masked_linear_backward", "masked_ffn_forward", "masked_ffn_backward", "Routing", "route", "shared_routing",
           "set_route_cache", "MXFP4", "mxfp4_quantise", "mxfp4_dequantise", "MaskedLinearMXFP4", "MaskedFFNMXFP4",
           "masked_linear_mxfp4_forward", "masked_linear_mxfp4_backward", "masked_ffn_mxfp4_forward", "masked_ffn_mxfp4_backward",
           "MaskedLinearMXFP4Module", "MaskedFFNMXFP4Module"]
