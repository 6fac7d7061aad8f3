"""MI355X-native MoMoE: SwiGLU mixture-of-experts layer on hand-written gfx950 kernels.

The public names of the reference package (momoe/__init__.py:1-5), `balance_loss`, `FeedForward`, and for serving
`MoMoEFP8`, `MoMoEInt4` and `FeedForwardInt4`.
"""
from .experts import MoMoE, MoEFunction
from .experts_fp8 import MoMoEFP8
from .feed_forward import FeedForward, FeedForwardFunction
from .int4 import FeedForwardInt4, MoMoEInt4
from .router import TopKRouter, TopKRouterFunction
from .moe import MoE
from .balance import balance_loss

__all__ = ["MoMoE", "MoE", "TopKRouter", "MoEFunction", "TopKRouterFunction", "balance_loss",
           "FeedForward", "FeedForwardFunction", "MoMoEFP8", "MoMoEInt4", "FeedForwardInt4"]
