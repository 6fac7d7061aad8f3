"""Plain 64-bit restatements of the operators beside the reference's path: the balance loss of the router."""
import torch


def balance_loss(logits, mask_NM, Ks=0, valid=None, groups=1, weight=1.0):
    """(loss, counts [groups, N], d (weight * loss) / d logits) in 64 bits, group by group from the definition.

    logits [M, N]; groups of M / groups consecutive tokens; valid bool [M] or None."""
    M, N = logits.shape
    Nr, S = N - Ks, M // groups
    l = logits.double()
    grad = torch.zeros(M, N, dtype=torch.float64)
    counts = torch.zeros(groups, N, dtype=torch.int64)
    losses, parts = [], []
    for g in range(groups):
        rows = torch.arange(g * S, (g + 1) * S)
        if valid is not None:
            rows = rows[valid[rows]]
        counts[g] = (mask_NM[:, rows] != 0).sum(1)
        pairs = counts[g, :Nr].sum().item()
        if pairs == 0:
            continue
        share = counts[g, :Nr].double() / pairs
        p = torch.softmax(l[rows, :Nr], -1)
        losses.append(Nr * (share * p.mean(0)).sum())
        parts.append((rows, Nr / len(rows) * p * (share - (share * p).sum(-1, keepdim=True))))
    for rows, part in parts:
        grad[rows, :Nr] = weight * part / len(losses)
    loss = torch.stack(losses).mean() if losses else torch.zeros((), dtype=torch.float64)
    return loss, counts, grad
