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


# ---- 8-bit floating point: e4m3 with a scale for each 128 values ------------------------------------------------------------
BLOCK = 128


def blocks(n):
    return -(-n // BLOCK)


def e4m3(v):
    """64-bit values, none above 448, to the nearest of e4m3 (three bits behind the point, least exponent -6), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def rows_in_8_bits(x):
    """(e4m3 values, exponents of the scales [rows, blocks]) of rows x: a block's scale is the least power of two that leaves none
    of its values above 448, magnitudes below 2^-100 counting as that."""
    x = x.double()
    R, n = x.shape
    part = torch.nn.functional.pad(x, (0, blocks(n) * BLOCK - n)).view(R, -1, BLOCK)
    exponent = torch.ceil(torch.log2(part.abs().amax(-1).clamp_min(2.0 ** -100) / 448))
    q = e4m3(part / torch.exp2(exponent)[..., None])
    return q.reshape(R, -1)[:, :n], exponent.to(torch.int64)


def rounded_rows(x):
    """The values that rows x have in 8 bits."""
    q, e = rows_in_8_bits(x)
    return q * torch.exp2(e.double()).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def block_weights(q, scale):
    """The values, in 64 bits, of e4m3 weights [.., R, C] with scales [.., row blocks, column blocks]."""
    R, C = q.shape[-2:]
    return q.float().double() * scale.double().repeat_interleave(BLOCK, -2)[..., :R, :].repeat_interleave(BLOCK, -1)[..., :C]


def experts_fp8(x_MD, W1, W2, mask_NM, s_NM):
    """y [M, D] in 64 bits of the experts with weights W1 [N, D, 2H], W2 [N, H, D] (the values that their 8 bits stand for)."""
    H = W2.shape[1]
    y = torch.zeros(x_MD.shape, dtype=torch.float64)
    xq = rounded_rows(x_MD)
    for i in range(W2.shape[0]):
        rows = torch.nonzero(mask_NM[i]).flatten()
        if len(rows):
            z = xq[rows] @ W1[i]
            h = z[:, :H] * z[:, H:] * torch.sigmoid(z[:, H:])
            y[rows] += s_NM[i, rows].double()[:, None] * (rounded_rows(h) @ W2[i])
    return y
