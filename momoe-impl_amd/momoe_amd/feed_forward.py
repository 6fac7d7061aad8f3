"""`FeedForward`: a dense SwiGLU block, forward and backward, for the layers beside the mixture that have no router.

What `MoMoE` does for one expert that takes every token with a gate weight of 1 (momoe/momoe.py:847-972), without the routing.
The kernels are in csrc/feed_forward.hip (the weights' gradients in csrc/wgrad.hip), the host path in csrc/layer_binding.cpp.
"""
import torch
import torch.nn as nn

from . import _layer
from .int4 import FeedForwardInt4


class FeedForwardFunction:
    """(x, Wl1_D2H, Wl2_HD, save_percent) -> y: the autograd function of the block, native (csrc/layer_binding.cpp).

    Forward: a | b = x Wl1, h = a * b * sigmoid(b), y = h Wl2.  With save_percent > 0 the a | b of that share of the rows are kept for
    the backward, in fp32; those of the others are computed again there.  No second derivative."""

    @staticmethod
    def apply(x, Wl1_D2H, Wl2_HD, save_percent=0):
        return _layer.feed_forward(x, Wl1_D2H, Wl2_HD, save_percent)


class FeedForward(nn.Module):
    """y = (a * b * sigmoid(b)) Wl2 with a | b = x Wl1.

    Args:
        embedding_dim: D.  intermediate_dim: H.  Both multiples of 32, and where weights are trained D up to 2^20, H up to 2^19.
        save_percent: share of the rows whose pre-activations are kept for the backward, 0..100: 8 * H bytes a row, for a sixth less to
        compute in a step.
        Wl1_D2H / Wl2_HD: optional initial weights, [D, 2H] and [H, D]; the first H columns of Wl1 are the linear half, the last H go
        through SiLU.
    """

    def __init__(self, embedding_dim, intermediate_dim, save_percent=0, Wl1_D2H=None, Wl2_HD=None):
        assert save_percent >= 0 and save_percent <= 100, (
            "save_percent must be between 0 and 100 inclusive, got {}".format(save_percent))
        super().__init__()
        self.D = embedding_dim
        self.H = intermediate_dim
        self.save_percent = save_percent
        if Wl1_D2H is None:
            Wl1_D2H = torch.randn((self.D, 2 * self.H), device="cuda", dtype=torch.bfloat16) / self.D
        if Wl2_HD is None:
            Wl2_HD = torch.randn((self.H, self.D), device="cuda", dtype=torch.bfloat16) / self.D
        self.Wl1_D2H = nn.Parameter(Wl1_D2H.clone().detach().to(torch.bfloat16), requires_grad=True)
        self.Wl2_HD = nn.Parameter(Wl2_HD.clone().detach().to(torch.bfloat16), requires_grad=True)

    def to_int4(self, group_size=128):
        """The block for serving with its weights in 4 bits (`FeedForwardInt4.from_feed_forward`); forward only."""
        return FeedForwardInt4.from_feed_forward(self, group_size)

    def forward(self, x):
        """x [.., D] (of any floating type, rounded to bf16) -> y bf16 [.., D]."""
        return FeedForwardFunction.apply(x, self.Wl1_D2H, self.Wl2_HD, self.save_percent)
