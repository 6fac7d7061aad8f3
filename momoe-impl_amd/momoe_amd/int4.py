"""`MoMoEInt4` and `FeedForwardInt4`: the experts of a SwiGLU mixture-of-experts layer, and the dense block beside them, for serving with
4-bit weights.

The reference's weights are bf16 (momoe/momoe.py:914-972); the calls are those of `MoMoE` and `FeedForward`, without a backward.
The kernels are in csrc/int4.hip, the host path in csrc/layer_binding.cpp.
"""
import torch
import torch.nn as nn

from . import _hip, _layer, experts

GROUPS = (32, 64, 128)


def _groups(n, group):
    return -(-n // group)


def quantize(W, group_size=128):
    """Weights [.., R, C] -> (codes uint8 [.., R / 2, C], scale bf16 and zero uint8 [.., ceil(R / group_size), C]): the 16 values of a group
    of a column reach from the lesser of its least weight and 0 to the greater of its greatest and 0, with 0 among them.  A NaN or an infinity
    leaves no number in its group: the scale is NaN or infinite, too."""
    if W.dim() > 2:
        parts = [quantize(w, group_size) for w in W]
        return tuple(torch.stack(t) for t in zip(*parts))
    R, C = W.shape
    G = _groups(R, group_size)
    w = torch.nn.functional.pad(W.detach().float(), (0, 0, 0, G * group_size - R)).view(G, group_size, C)
    lo, hi = w.amin(1).clamp_max(0), w.amax(1).clamp_min(0)
    scale = ((hi - lo) / 15).to(torch.bfloat16)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    # (what such a scale divides may be NaN, of which no whole number can be made)
    zero = torch.round(-lo / scale.float()).nan_to_num(0).clamp(0, 15)
    q = (torch.round(w / scale.float()[:, None]).nan_to_num(0) + zero[:, None]).clamp(0, 15).to(torch.uint8).view(G * group_size, C)[:R]
    return q[0::2] | (q[1::2] << 4), scale, zero.to(torch.uint8)


class _Int4Block(nn.Module):
    """What both keep: the packed codes and the words of scales and zeros of N blocks."""

    def _set_sizes(self, D, H, N, group_size):
        assert D % 32 == 0 and H % 32 == 0 and D > 0 and H > 0, f"D and H must be multiples of 32, got {D} and {H}"
        assert group_size in GROUPS, f"group_size must be one of {GROUPS}, got {group_size}"
        self.D, self.H, self.N, self.group_size = D, H, N, group_size

    def _lay_out(self, lead, Wl1, Wl1_scale, Wl2, Wl2_scale, Wl1_zero, Wl2_zero):
        """lead: the leading sizes of the arguments, (N,) or (); `self.N` blocks."""
        D, H, G, N = self.D, self.H, self.group_size, self.N
        matrices = (("Wl1", D, 2 * H, Wl1, Wl1_scale, Wl1_zero), ("Wl2", H, D, Wl2, Wl2_scale, Wl2_zero))
        for name, R, C, codes, scale, zero in matrices:
            rows = (*lead, _groups(R, G), C)
            assert codes.dtype == torch.uint8 and tuple(codes.shape) == (*lead, R // 2, C), \
                f"{name} must be torch.uint8 {(*lead, R // 2, C)}, got {codes.dtype} {tuple(codes.shape)}"
            assert scale.dtype in (torch.bfloat16, torch.float16) and tuple(scale.shape) == rows, \
                f"{name}_scale must be torch.bfloat16 or torch.float16 {rows}, got {scale.dtype} {tuple(scale.shape)}"
            assert zero is None or (zero.dtype == torch.uint8 and tuple(zero.shape) == rows), \
                f"{name}_zero must be None or torch.uint8 {rows}, got {None if zero is None else (zero.dtype, tuple(zero.shape))}"
            assert {t.device for t in (Wl1, scale, codes, zero) if t is not None} == {Wl1.device}, "codes, scales and zeros must be on one device"
        for name, R, C, codes, scale, zero in matrices:
            packed, words = _hip.int4_pack_weights(
                codes.detach().reshape(N, R // 2, C).contiguous(), scale.detach().reshape(N, -1, C).contiguous(),
                None if zero is None else zero.detach().reshape(N, -1, C).contiguous(), 2 if name == "Wl1" else 1, G)
            # (whole numbers: `.to(dtype)` of a module that holds this one leaves them alone)
            self.register_buffer(f"{name}_packed", packed)
            self.register_buffer(f"{name}_words", words)
        self.scale_dtypes = (Wl1_scale.dtype, Wl2_scale.dtype)

    def _unpacked(self, packed, words, R, C, halves, scale_dtype):
        KB, SG, cols = _groups(R, 128), 128 // self.group_size, C // halves
        w = packed.view(torch.int32).view(self.N, cols // 16, halves, KB, 4, 16, 4)
        # [expert][columns / 16][half][k-block][lane / 16][column][word] and the byte of a word's k-values 2 i, 2 i + 1
        b = torch.stack([(w >> (4 * i) & 15) | (w >> (16 + 4 * i) & 15) << 4 for i in range(4)], -1).to(torch.uint8)
        codes = b.permute(0, 3, 6, 4, 7, 2, 1, 5).reshape(self.N, KB * 64, C)[:, :R // 2].contiguous()
        s = words.view(self.N, cols // 16, halves, KB, 16, SG).permute(0, 3, 5, 2, 1, 4).reshape(self.N, KB * SG, C)
        s = s[:, :_groups(R, self.group_size)].contiguous()
        return codes, (s & ~15).view(torch.float32).to(scale_dtype), (s & 15).to(torch.uint8)

    def weights(self):
        """(Wl1, Wl1_scale, Wl2, Wl2_scale, Wl1_zero, Wl2_zero) as the constructor takes them."""
        c1, s1, z1 = self._unpacked(self.Wl1_packed, self.Wl1_words, self.D, 2 * self.H, 2, self.scale_dtypes[0])
        c2, s2, z2 = self._unpacked(self.Wl2_packed, self.Wl2_words, self.H, self.D, 1, self.scale_dtypes[1])
        return c1, s1, c2, s2, z1, z2


class MoMoEInt4(_Int4Block):
    """Mixture of SwiGLU experts with 4-bit weights; forward only.

    Args:
        embedding_dim: D.  intermediate_dim: H.  num_experts: N.  num_chosen_experts: K per token, as in `MoMoE`.
        Wl1_ND2H, Wl2_NHD: codes, uint8 [N, D / 2, 2H] (the linear half first, then that of the SiLU) and [N, H / 2, D]: k-value 2 r of a
        column in the low four bits of row r, 2 r + 1 in the high ones.
        Wl1_scale, Wl2_scale: bf16 or fp16 [N, ceil(D / group_size), 2H] and [N, ceil(H / group_size), D].
        Wl1_zero, Wl2_zero: uint8 0..15 (of greater ones the low four bits) of the same sizes; None: 8 throughout.
        group_size: k-values that share a scale and a zero, 32, 64 or 128.
    A weight is (code - zero) * scale, and is multiplied as that, unrounded, with sums in fp32; x and h are bf16 (x of any other type is
    rounded to bf16).  D and H must be multiples of 32.  A NaN or an infinity in a token makes NaN of it; so may a value above
    2^113, or one above 2^111 when it is multiplied by a scale.

    The weights are laid out once, in the order that the kernels read them in; `weights()` gives them back.
    `from_momoe` quantizes the weights of a `MoMoE`.
    """

    def __init__(self, embedding_dim, intermediate_dim, num_experts, num_chosen_experts, Wl1_ND2H, Wl1_scale, Wl2_NHD, Wl2_scale,
                 Wl1_zero=None, Wl2_zero=None, group_size=128):
        super().__init__()
        self._set_sizes(embedding_dim, intermediate_dim, num_experts, group_size)
        assert 1 <= num_chosen_experts <= num_experts, f"num_chosen_experts must be between 1 and {num_experts}, got {num_chosen_experts}"
        self.K = num_chosen_experts
        self._lay_out((num_experts,), Wl1_ND2H, Wl1_scale, Wl2_NHD, Wl2_scale, Wl1_zero, Wl2_zero)

    @classmethod
    def from_momoe(cls, momoe, group_size=128):
        """The experts of a `MoMoE` in 4 bits, by `quantize`."""
        q1, s1, z1 = quantize(momoe.Wl1_ND2H, group_size)
        q2, s2, z2 = quantize(momoe.Wl2_NHD, group_size)
        return cls(momoe.D, momoe.H, momoe.N, momoe.K, q1, s1, q2, s2, z1, z2, group_size)

    def forward(self, x_BSD, mask_NM, s_NM):
        """As `MoMoE.forward`: (y_BSD bf16, tokens per expert int64 [N]).  Nothing may require a gradient."""
        return _layer.experts_int4(x_BSD, self.Wl1_packed, self.Wl1_words, self.Wl2_packed, self.Wl2_words, mask_NM, s_NM, self.K, self.H,
                                   self.group_size, experts.CHECK_ROUTING)


class FeedForwardInt4(_Int4Block):
    """The dense block with 4-bit weights; forward only.  The arguments are those of `MoMoEInt4` without the experts: Wl1_D2H uint8
    [D / 2, 2H], Wl2_HD [H / 2, D], scales and zeros [ceil(D / group_size), 2H] and [ceil(H / group_size), D].
    `from_feed_forward` quantizes the weights of a `FeedForward`."""

    def __init__(self, embedding_dim, intermediate_dim, Wl1_D2H, Wl1_scale, Wl2_HD, Wl2_scale, Wl1_zero=None, Wl2_zero=None, group_size=128):
        super().__init__()
        self._set_sizes(embedding_dim, intermediate_dim, 1, group_size)
        self._lay_out((), Wl1_D2H, Wl1_scale, Wl2_HD, Wl2_scale, Wl1_zero, Wl2_zero)

    @classmethod
    def from_feed_forward(cls, block, group_size=128):
        """The weights of a `FeedForward` in 4 bits, by `quantize`."""
        q1, s1, z1 = quantize(block.Wl1_D2H, group_size)
        q2, s2, z2 = quantize(block.Wl2_HD, group_size)
        return cls(block.D, block.H, q1, s1, q2, s2, z1, z2, group_size)

    def weights(self):
        """(Wl1, Wl1_scale, Wl2, Wl2_scale, Wl1_zero, Wl2_zero) as the constructor takes them."""
        return tuple(t[0] for t in super().weights())

    def forward(self, x):
        """x [.., D] -> y bf16 [.., D].  Nothing may require a gradient."""
        return _layer.feed_forward_int4(x, self.Wl1_packed, self.Wl1_words, self.Wl2_packed, self.Wl2_words, self.H, self.group_size)
