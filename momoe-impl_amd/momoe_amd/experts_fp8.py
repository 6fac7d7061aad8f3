"""`MoMoEFP8`: the experts of a SwiGLU mixture-of-experts layer for serving, weights and the rows that meet them in 8-bit
floating point (e4m3) with a scale for each 128 values.

The reference's experts are bf16 (momoe/momoe.py:914-972); the call is that of `MoMoE`, without a backward.
The kernels are in csrc/experts_fp8.hip and csrc/quantize.hip, the host path in csrc/layer_binding.cpp.
"""
import torch
import torch.nn as nn

from . import _hip, _layer, experts

BLOCK = 128


def _blocks(n):
    return -(-n // BLOCK)


class MoMoEFP8(nn.Module):
    """Mixture of SwiGLU experts with 8-bit weights; forward only.

    Args:
        embedding_dim: D.  intermediate_dim: H.  num_experts: N.  num_chosen_experts: K per token, as in `MoMoE`.
        Wl1_ND2H, Wl2_NHD: float8_e4m3fn, [N, D, 2H] (the linear half first, then that of the SiLU) and [N, H, D].
        Wl1_scale, Wl2_scale: fp32, [N, ceil(D/128), 2, ceil(H/128)] (the two halves have blocks of their own) and
        [N, ceil(H/128), ceil(D/128)]: a weight is its e4m3 value times the scale of its 128 x 128 block.
    D and H must be multiples of 32.  Each 128 consecutive values of a token (and of its h) are scaled by the least
    power of two that leaves none above 448, e4m3's largest (values below 2^-100 by one of 2^-108); NaN or infinity among
    them make NaN of the token.  x may be bf16, fp32 or fp16; any other type is rounded to bf16 first.

    Calls of few rows (an average below 20 an expert) multiply exactly and add up in fp32.  Larger ones multiply by the 8-bit matrix
    instruction, which of each eight products cuts off what lies 13 binades below the largest: a token's result depends, in its
    third digit, on how many others are in the call.  Results leave the second product in groups of eight columns of 15 bits with a
    shared exponent: one that is NaN or infinite makes NaN of its eight.

    The weights are laid out once, in the order that the kernels read them in; `weights()` gives them back.
    `from_momoe` quantizes the weights of a `MoMoE`.
    """

    def __init__(self, embedding_dim, intermediate_dim, num_experts, num_chosen_experts, Wl1_ND2H, Wl1_scale, Wl2_NHD, Wl2_scale):
        super().__init__()
        D, H, N = embedding_dim, intermediate_dim, num_experts
        self._set_sizes(D, H, N, num_chosen_experts)
        for name, t, dtype, size in (("Wl1_ND2H", Wl1_ND2H, torch.float8_e4m3fn, (N, D, 2 * H)),
                                     ("Wl1_scale", Wl1_scale, torch.float32, (N, _blocks(D), 2, _blocks(H))),
                                     ("Wl2_NHD", Wl2_NHD, torch.float8_e4m3fn, (N, H, D)),
                                     ("Wl2_scale", Wl2_scale, torch.float32, (N, _blocks(H), _blocks(D)))):
            assert t.dtype == dtype and tuple(t.shape) == size, f"{name} must be {dtype} {size}, got {t.dtype} {tuple(t.shape)}"
        self._hold(_hip.fp8_pack_weights(Wl1_ND2H.detach().contiguous(), 2), Wl1_scale.detach().contiguous(),
                   _hip.fp8_pack_weights(Wl2_NHD.detach().contiguous(), 1), Wl2_scale.detach().contiguous())

    @classmethod
    def from_momoe(cls, momoe):
        """The experts of a `MoMoE` in 8 bits, each 128 x 128 block scaled by the least power of two that leaves none of its
        weights above 448."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        self._set_sizes(momoe.D, momoe.H, momoe.N, momoe.K)
        W1, S1 = _hip.fp8_pack_weights(momoe.Wl1_ND2H.detach().contiguous(), 2)
        W2, S2 = _hip.fp8_pack_weights(momoe.Wl2_NHD.detach().contiguous(), 1)
        self._hold(W1, S1, W2, S2.reshape(self.N, _blocks(self.H), _blocks(self.D)))
        return self

    def _set_sizes(self, D, H, N, K):
        assert D % 32 == 0 and H % 32 == 0, f"D and H must be multiples of 32, got {D} and {H}"
        assert 1 <= K <= N, f"num_chosen_experts must be between 1 and {N}, got {K}"
        self.D, self.H, self.N, self.K = D, H, N, K

    def _hold(self, W1, S1, W2, S2):
        self.register_buffer("Wl1_packed", W1)
        self.register_buffer("Wl2_packed", W2)
        # as their bits: `.to(dtype)` of a module that holds this one leaves whole numbers alone
        self.register_buffer("Wl1_scale_bits", S1.view(torch.int32).clone())
        self.register_buffer("Wl2_scale_bits", S2.view(torch.int32).clone())

    @property
    def Wl1_scale(self):
        return self.Wl1_scale_bits.view(torch.float32)

    @property
    def Wl2_scale(self):
        return self.Wl2_scale_bits.view(torch.float32)

    def weights(self):
        """(Wl1_ND2H, Wl1_scale, Wl2_NHD, Wl2_scale) as the constructor takes them."""
        def rows(packed, R, halves):
            groups = packed.numel() // (self.N * _blocks(R) * 2048)
            w = packed.view(self.N, groups // halves, halves, _blocks(R), 2, 4, 16, 16)
            # [expert][k-block][half][lane / 16][byte] x [half of the columns][group][lane % 16]
            w = w.permute(0, 3, 4, 5, 7, 2, 1, 6).reshape(self.N, _blocks(R) * BLOCK, groups * 16)
            return w[:, :R].contiguous().view(torch.float8_e4m3fn)
        return rows(self.Wl1_packed, self.D, 2), self.Wl1_scale, rows(self.Wl2_packed, self.H, 1), self.Wl2_scale

    def forward(self, x_BSD, mask_NM, s_NM):
        """As `MoMoE.forward`: (y_BSD bf16, tokens per expert int64 [N]).  Nothing may require a gradient."""
        return _layer.experts_fp8(x_BSD, self.Wl1_packed, self.Wl1_scale_bits, self.Wl2_packed, self.Wl2_scale_bits, mask_NM, s_NM,
                                  self.K, self.H, experts.CHECK_ROUTING)
