"""MI355X-native MoMoE: SwiGLU mixture-of-experts layer on hand-written gfx950 kernels.

The public names of the reference package (momoe/__init__.py:1-5), `balance_loss` and `MoMoEFP8`.
"""
from .experts import MoMoE, MoEFunction
from .experts_fp8 import MoMoEFP8
from .router import TopKRouter, TopKRouterFunction
from .moe import MoE
from .balance import balance_loss

__all__ = ["MoMoE", "MoE", "TopKRouter", "MoEFunction", "TopKRouterFunction", "balance_loss",
           "MoMoEFP8"]
