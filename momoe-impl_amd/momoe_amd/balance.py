"""`balance_loss`: the load-balancing loss of a router, with its per-expert counts and its gradient.

The reference balances by the selection bias alone (momoe/sample_moe.py:65-67); a loss can stand beside it or in its place.
The kernels are in csrc/balance.hip, the host path in csrc/layer_binding.cpp.
"""
from . import _layer


def balance_loss(logits, mask_NM, num_shared_experts=0, valid=None, per_sequence=False):
    """(loss fp32 [], counts int64 [N]) of gate logits [M, N] or [B, S, N] (bf16, fp32 or fp16) and the 0/1 mask [N, M] of the
    experts that each token took, as `TopKRouter` returns it.

    With p = softmax over the N - num_shared_experts routed experts (the shared ones are the last), T tokens that count, c_i of
    them at expert i:

        loss = (N - Ks) * sum_i (c_i / sum_j c_j) * (sum over tokens of p_i / T)

    which is 1 where both are even.  The counts are constants of the gradient, which goes to the logits; those of shared experts
    and of tokens that do not count get zeros.  The tensor of counts is the caller's own: summing it over ranks before the backward
    changes no gradient.

    valid: bool [M] or [B, S] (for [M, N] logits any two dimensions that hold M flags in order), False for the tokens that do
    not count (padding); what their logits hold does not matter.
    per_sequence: the loss is taken for each of the B sequences and averaged over those in which a routed expert holds a token;
    counts are then [B, N].  Without any such token the loss is zero.
    A token that counts and has no routed logit above -inf makes the loss NaN.
    No second derivative; up to 512 experts.
    """
    return _layer.balance_loss(logits, mask_NM, num_shared_experts, valid, per_sequence)
