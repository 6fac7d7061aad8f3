"""Two operators of a mixture-of-experts layer, in plain form and through `momoe_amd`, and the cases they are timed on.

balance  The load-balancing loss of a router with its counts, forward and gradient: from the gate logits l [tokens, N] and the
         0/1 mask [N, tokens] of the experts that each token took.  Over the Nr = N - Ks routed experts p = softmax(l); for each
         group of tokens (a sequence, or the whole batch) with T tokens that count and c_i of them at expert i,
             loss = Nr * sum_i (c_i / sum_j c_j) * (sum_tokens p_i / T),
         averaged over the groups in which an expert holds a token.  The counts are constants of the gradient.
experts  The experts of the layer for serving, weights in 8-bit floating point (e4m3) with a scale for each 128 x 128 block of the
         linear half, the SiLU half and the down projection.  Each 128 values of a row are brought to 8 bits before a product, with
         the least power of two as their scale that leaves none above 448: a | b = q(x) W1, h = a * b * sigmoid(b),
         y = sum over a token's experts of s * (q(h) W2).
"""
import math
import os
import sys

import torch

own = False  # true: the calls of `momoe_amd`; false: elementary torch operations in 32 bits

DEV = "cuda:0"
BLOCK = 128  # values that share a scale
LARGEST = 448.0  # of e4m3
SMALLEST_AMAX = 2.0 ** -100  # a row of smaller values, zeros too, is scaled as if this were its largest


def _package():
    path = os.path.abspath("momoe-impl_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import momoe_amd
    return momoe_amd


def _experts(name, tokens, D, H, N, K, Ks=0, skew=0.0):
    return {"name": name, "op": "experts", "tokens": tokens, "D": D, "H": H, "N": N, "K": K, "Ks": Ks, "skew": skew}


def _balance(name, B, S, N, K, Ks=0, skew=0.5, dtype="bfloat16", per_sequence=False, padded=False):
    return {"name": name, "op": "balance", "B": B, "S": S, "N": N, "K": K, "Ks": Ks, "skew": skew, "dtype": dtype,
            "per_sequence": per_sequence, "padded": padded}


def listed():
    return [
        # one sequence being decoded: eight experts' weights stream, launches and host work show
        _experts("experts 1 token", 1, 2048, 768, 128, 8),
        # a decode batch: most experts hold one or two tokens
        _experts("experts 16 tokens", 16, 2048, 768, 128, 8),
        # a large decode batch or a short prompt, no multiple of anything: every expert's weights stream
        _experts("experts 131 tokens", 131, 2048, 768, 128, 8),
        # a prompt of ordinary length: between streaming and multiplying
        _experts("experts 1000 tokens", 1000, 2048, 768, 128, 8),
        # batched prefill: bound by the matrix products
        _experts("experts 8192 tokens", 8192, 2048, 768, 128, 8),
        # widths that are no power of two, K that does not divide N
        _experts("experts 7680 tokens ragged", 7680, 2176, 1152, 64, 6),
        # few experts receive ten times the mean load and four see every token
        _experts("experts 16384 tokens skewed", 16384, 2048, 1408, 64, 8, Ks=4, skew=1.8),
        # a layer of a unit test or of a debugging run: launches only, widths below a block
        _experts("experts tiny", 128, 96, 64, 8, 2),
        # the loss beside a training step of that size: launches and host work only
        _balance("balance 128 tokens", 1, 128, 8, 2),
        # the loss beside the headline training layer, over the whole batch
        _balance("balance 8192 tokens", 4, 2048, 128, 8),
        # a padded batch, one loss a sequence, four shared experts that take no part, logits left in 32 bits
        _balance("balance 16 x 1000 padded", 16, 1000, 64, 8, Ks=4, dtype="float32", per_sequence=True, padded=True),
        # the largest batch, 8 x 8192 tokens
        _balance("balance 65536 tokens", 8, 8192, 64, 8, per_sequence=True),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    if rng.random() < 0.4:
        tokens = int(_log_uniform(rng, 1, 65536))
        N = rng.choice((2, 8, 16, 33, 60, 64, 96, 128, 200, 256, 384, 512))
        Ks = rng.choice((0, 0, 0, 1, 2, 4)) if N > 8 else 0
        B = min(tokens, int(_log_uniform(rng, 1, 64)))
        S = tokens // B
        while B * S * N > 65536 * 64:  # no more than the largest listed one
            S = (S + 1) // 2
        case = _balance("", B, S, N, Ks + rng.randint(1, min(8, N - Ks)), Ks, rng.choice((0.0, 0.5, 1.5)),
                        rng.choice(("bfloat16", "bfloat16", "float32", "float16")), rng.random() < 0.5, rng.random() < 0.4)
        del case["name"]
        return case
    most, weights = _flops(listed()[6]), max(_weights(c) for c in listed() if c["op"] == "experts")
    while True:
        step = rng.choice((32, 64, 128))  # D and H are multiples of 32
        Ks = rng.choice((0, 0, 0, 1, 2))
        case = _experts("", int(_log_uniform(rng, 1, 16384)), max(step, int(_log_uniform(rng, 64, 4096)) // step * step),
                        max(step, int(_log_uniform(rng, 32, 2048)) // step * step),
                        rng.choice((4, 8, 16, 32, 48, 64, 96, 128)), Ks + rng.choice((1, 2, 4, 6, 8)), Ks,
                        rng.choice((0.0, 0.0, 0.5, 1.8)))
        del case["name"]
        if case["K"] <= case["N"] // 2 and _flops(case) < most and _weights(case) <= weights:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _routing(logits, K, Ks):
    """The 0/1 mask [N, tokens] of the K - Ks routed experts of the greatest logits (the lower index where they are equal) and
    of the Ks shared ones, and the gate weights: softmax over those chosen, and over the shared ones, [tokens, N]."""
    M, N = logits.shape
    Ng = N - Ks
    order = torch.sort(logits[:, :Ng], dim=-1, descending=True, stable=True).indices[:, :K - Ks]
    chosen = torch.zeros(M, Ng, dtype=torch.bool, device=DEV).scatter_(1, order, True)
    w = torch.softmax(logits[:, :Ng].float(), -1) * chosen
    s_MN = torch.cat([w / w.sum(-1, keepdim=True), torch.softmax(logits[:, Ng:].float(), -1)], -1)
    mask = torch.ones(N, M, dtype=torch.int32, device=DEV)
    mask[:Ng] = chosen.T.to(torch.int32)
    return mask, s_MN.contiguous()


def _logits(M, N, Ks, skew, gen):
    logits = torch.randn(M, N, generator=gen, device=DEV)
    logits[:, :N - Ks] -= skew * torch.log(torch.arange(1, N - Ks + 1, device=DEV, dtype=torch.float32))
    return logits


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _quantized(W):
    """W [N, rows, cols] -> (e4m3 [N, rows, cols], fp32 scales [N, row blocks, column blocks])."""
    N, R, C = W.shape
    scale = torch.empty(N, _blocks(R), _blocks(C), device=DEV)
    q = torch.empty(N, R, C, dtype=torch.float8_e4m3fn, device=DEV)
    for i in range(_blocks(R)):
        rows = slice(i * BLOCK, min(R, (i + 1) * BLOCK))
        part = torch.nn.functional.pad(W[:, rows].float(), (0, _blocks(C) * BLOCK - C))
        part = part.view(N, -1, _blocks(C), BLOCK)
        scale[:, i] = part.abs().amax(dim=(1, 3)).clamp_min(SMALLEST_AMAX) / LARGEST
        part = part / scale[:, i].view(N, 1, -1, 1)
        q[:, rows] = part.reshape(N, -1, _blocks(C) * BLOCK)[:, :, :C].to(torch.float8_e4m3fn)
    return q, scale


def _experts_inputs(case, seed):
    M, D, H, N, K, Ks = (case[k] for k in ("tokens", "D", "H", "N", "K", "Ks"))
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(1, M, D, generator=gen, device=DEV).to(torch.bfloat16)
    mask, s_MN = _routing(_logits(M, N, Ks, case["skew"], gen), K, Ks)
    W1 = torch.empty(N, D, 2 * H, device=DEV, dtype=torch.bfloat16).normal_(0, 0.02, generator=gen)
    qa, sa = _quantized(W1[:, :, :H])
    qb, sb = _quantized(W1[:, :, H:])
    W1 = None
    q2, s2 = _quantized(torch.empty(N, H, D, device=DEV, dtype=torch.bfloat16).normal_(0, 0.02, generator=gen))
    W1 = torch.cat([qa.view(torch.uint8), qb.view(torch.uint8)], -1).view(torch.float8_e4m3fn)
    return {"op": "experts", "x": x, "mask": mask, "s": s_MN.T, "W1": W1, "S1": torch.stack([sa, sb], 2), "W2": q2, "S2": s2}


def _balance_inputs(case, seed):
    B, S, N, K, Ks = (case[k] for k in ("B", "S", "N", "K", "Ks"))
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    logits = _logits(B * S, N, Ks, case["skew"], gen).to(dtype)
    mask, _ = _routing(logits, K, Ks)
    valid = None
    if case["padded"]:  # sequences of any length from none to all of S, padded at the end
        length = torch.randint(0, S + 1, (B, 1), generator=gen, device=DEV)
        valid = torch.arange(S, device=DEV) < length
    # what the loss weighs in the training loss; half precision trains with a scaled loss
    weight = torch.full((), 0.01 * (65536.0 if dtype == torch.float16 else 1.0), device=DEV)
    return {"op": "balance", "logits": logits.view(B, S, N), "mask": mask, "Ks": Ks, "valid": valid,
            "per_sequence": case["per_sequence"], "weight": weight}


def prepare(case, seed):
    if case["op"] == "balance":
        state = _balance_inputs(case, seed)
        if own:
            state["logits"].requires_grad_()
        return state
    state = _experts_inputs(case, seed)
    if own:  # the layer of a program that serves: it lays its weights out once
        state["layer"] = _package().MoMoEFP8(case["D"], case["H"], case["N"], case["K"], state.pop("W1"), state.pop("S1"),
                                             state.pop("W2"), state.pop("S2"))
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------
def run(state):
    if state["op"] == "balance":
        return _run_balance(state) if own else _plain_balance(state)
    if not own:
        return _plain_experts(state)
    with torch.no_grad():
        y, sizes = state["layer"](state["x"], state["mask"], state["s"])
    return [y, sizes]


def _run_balance(state):
    logits = state["logits"]
    logits.grad = None
    loss, counts = _package().balance_loss(logits, state["mask"], num_shared_experts=state["Ks"], valid=state["valid"],
                                           per_sequence=state["per_sequence"])
    loss.backward(state["weight"])
    return [loss.detach(), counts, logits.grad]


def _plain_balance(state):
    logits, mask, valid = state["logits"], state["mask"], state["valid"]
    B, S, N = logits.shape
    Nr = N - state["Ks"]
    ok = torch.ones(B, S, dtype=torch.bool, device=DEV) if valid is None else valid
    groups = (B, S) if state["per_sequence"] else (1, B * S)
    ok = ok.reshape(*groups, 1)
    routed = logits.reshape(*groups, N)[:, :, :Nr].float()
    e = torch.exp(routed - routed.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    held = mask.T.reshape(*groups, N) * ok
    counts = held.sum(1)
    c = counts[:, :Nr].float()
    tokens = ok.sum(1).float()                                            # [groups, 1]
    pairs = c.sum(1, keepdim=True)
    full = pairs > 0
    share = torch.where(full, c / pairs.clamp_min(1), torch.zeros_like(c))
    mean = torch.where(ok, p, torch.zeros_like(p)).sum(1) / tokens.clamp_min(1)
    ngroups = full.sum().clamp_min(1).float()
    loss = Nr * (share * mean).sum() / ngroups
    # d loss / d l_j = weight * Nr / (T * groups) * p_j * (share_j - sum_i share_i p_i)
    inner = share.unsqueeze(1) - (share.unsqueeze(1) * p).sum(-1, keepdim=True)
    grad = p * inner * (state["weight"] * Nr / (tokens.clamp_min(1) * ngroups)).unsqueeze(1)
    grad = torch.where(ok & full.unsqueeze(1), grad, torch.zeros_like(grad))
    grad = torch.nn.functional.pad(grad, (0, N - Nr)).reshape(B, S, N)
    return [loss, counts if state["per_sequence"] else counts[0], grad.to(logits.dtype)]


def _rows_in_8_bits(x):
    """x [rows, n] in fp32 as the values that e4m3 with a scale for each 128 of a row holds."""
    R, n = x.shape
    part = torch.nn.functional.pad(x, (0, _blocks(n) * BLOCK - n)).view(R, -1, BLOCK)
    m, e = torch.frexp(part.abs().amax(-1, keepdim=True).clamp_min(SMALLEST_AMAX))
    e = e - 9 + (m > LARGEST / 512).to(torch.int32)
    q = torch.ldexp(part, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).reshape(R, -1)[:, :n]


def _weights_of(q, scale):
    """The values that one expert's e4m3 [rows, cols] with block scales stand for."""
    R, C = q.shape
    return q.float() * scale.repeat_interleave(BLOCK, 0)[:R].repeat_interleave(BLOCK, 1)[:, :C]


def _plain_experts(state):
    x, mask, s = state["x"], state["mask"], state["s"]
    _, M, D = x.shape
    N, H = state["W2"].shape[:2]
    xq = _rows_in_8_bits(x.view(M, D).float())
    y = torch.zeros(M, D, device=DEV)
    sizes = mask.sum(1)
    for i in torch.nonzero(sizes).flatten().tolist():
        rows = torch.nonzero(mask[i]).flatten()
        xi = xq[rows]
        a = xi @ _weights_of(state["W1"][i, :, :H], state["S1"][i, :, 0])
        b = xi @ _weights_of(state["W1"][i, :, H:], state["S1"][i, :, 1])
        h = _rows_in_8_bits(a * (b / (1 + torch.exp(-b))))
        y[rows] += s[i, rows].unsqueeze(1) * (h @ _weights_of(state["W2"][i], state["S2"][i]))
    return [y.to(torch.bfloat16).view(1, M, D), sizes]


# ---- what the results are, in 64 bits ----------------------------------------------------------------------------------------
def _e4m3(v):
    """v (64 bits) to the nearest value of e4m3, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp_min(-6) - 3)
    return torch.round(v / step) * step  # (|v| <= 448 here)


def _exact_rows(x):
    out = torch.empty_like(x)
    for k in range(0, x.shape[1], BLOCK):
        largest = x[:, k:k + BLOCK].abs().amax(1, keepdim=True).clamp(min=SMALLEST_AMAX)
        scale = torch.exp2(torch.ceil(torch.log2(largest / LARGEST)))
        out[:, k:k + BLOCK] = _e4m3(x[:, k:k + BLOCK] / scale) * scale
    return out


def _exact_experts(case, seed):
    t = _experts_inputs(case, seed)
    x = _exact_rows(t["x"][0].double())
    y = torch.zeros_like(x)
    N, H, D = t["W2"].shape

    def weight(q, scale):
        w = q.double()
        for i in range(scale.shape[0]):
            for j in range(scale.shape[1]):
                w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[i, j].double()
        return w

    for i in range(N):
        tokens = (t["mask"][i] != 0).nonzero()[:, 0]
        if len(tokens) == 0:
            continue
        lin = torch.mm(x[tokens], weight(t["W1"][i, :, :H].contiguous(), t["S1"][i, :, 0]))
        gate = torch.mm(x[tokens], weight(t["W1"][i, :, H:].contiguous(), t["S1"][i, :, 1]))
        out = torch.mm(_exact_rows(lin * gate * torch.sigmoid(gate)), weight(t["W2"][i], t["S2"][i]))
        y.index_add_(0, tokens, out * t["s"][i, tokens].double()[:, None])
    return [y[None], (t["mask"] != 0).sum(1)]


def _exact_balance(case, seed):
    t = _balance_inputs(case, seed)
    B, S, N = t["logits"].shape
    Nr = N - t["Ks"]
    leaf = t["logits"].double().requires_grad_()
    prob = torch.softmax(leaf[..., :Nr], -1)
    held = t["mask"].view(N, B, S).permute(1, 2, 0)
    terms, counts = [], []
    for part in ([slice(b, b + 1) for b in range(B)] if t["per_sequence"] else [slice(0, B)]):
        here = torch.ones_like(held[part, :, 0], dtype=torch.bool) if t["valid"] is None else t["valid"][part]
        c = held[part][here].sum(0)
        counts.append(c)
        if c[:Nr].sum() > 0:
            terms.append(Nr * torch.dot(c[:Nr].double() / c[:Nr].sum().double(), prob[part][here].mean(0)))
    if terms:
        loss = torch.stack(terms).mean()
        grad, = torch.autograd.grad(loss, leaf, t["weight"].double())
    else:
        loss, grad = torch.zeros((), dtype=torch.float64, device=DEV), torch.zeros_like(leaf)
    return [loss.detach(), torch.stack(counts) if t["per_sequence"] else counts[0], grad]


def exact(case, seed):
    return (_exact_balance if case["op"] == "balance" else _exact_experts)(case, seed)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def _weights(case):
    return 3 * case["D"] * case["H"] * case["N"]


def _flops(case):
    return 6 * case["D"] * case["H"] * case["tokens"] * case["K"]


def work(case):
    if case["op"] == "balance":
        M, N = case["B"] * case["S"], case["N"]
        size = 4 if case["dtype"] == "float32" else 2
        counts = 8 * N * (case["B"] if case["per_sequence"] else 1)
        # logits in, their gradient out, the mask; softmax and its gradient are about ten operations an element
        return {"bytes": 2 * size * M * N + 4 * M * N + (M if case["padded"] else 0) + counts, "flops": 10 * M * N}
    M, D, N, K, Ks = (case[k] for k in ("tokens", "D", "N", "K", "Ks"))
    # experts that hold a token, had every routed expert the same chance; a byte for each of their weights
    held = Ks + (N - Ks) * (1 - (1 - (K - Ks) / (N - Ks)) ** M)
    scales = 4 * (2 * _blocks(D) * _blocks(case["H"]) + _blocks(case["H"]) * _blocks(D))
    # the mask, the gate weights of the pairs, x and y in 16 bits, tokens per expert
    return {"bytes": held * (3 * D * case["H"] + scales) + 4 * N * M + 4 * M * K + 4 * M * D + 8 * N, "flops": _flops(case)}
