"""Two operators next to a mixture-of-experts layer, in plain form and through `momoe_amd`, and the cases they are timed on.

ffn   The gated feed-forward block of the layers that have no router: a | b = x W1, h = a * b * sigmoid(b), y = h W2, with the
      gradients of x and of both weights, or forward only.
int4  The same block, or the experts of a mixture of them, for serving, with weights in 4 bits: a weight is (code - zero) * scale,
      with a zero and a scale for each `group` consecutive values of the contraction and each column (zero 8 where none is given).
      Of the mixture, y = sum over a token's experts of s * (its expert's block).
"""
import math
import os
import sys

import torch

own = False  # true: the calls of `momoe_amd`; false: elementary torch operations in 32 bits

DEV = "cuda:0"


def _package():
    path = os.path.abspath("momoe-impl_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import momoe_amd
    return momoe_amd


def _ffn(name, tokens, D, H, train=True, save=0):
    return {"name": name, "op": "ffn", "tokens": tokens, "D": D, "H": H, "train": train, "save": save}


def _int4(name, tokens, D, H, N=0, K=0, group=128, zeros=False, skew=0.0):
    return {"name": name, "op": "int4", "tokens": tokens, "D": D, "H": H, "N": N, "K": K, "group": group, "zeros": zeros, "skew": skew}


def listed():
    return [
        # one sequence being decoded: the weights stream, launches and host work show
        _ffn("ffn serve 1 token", 1, 2048, 8192, train=False),
        # a decode batch through a wide layer, no power of two
        _ffn("ffn serve 24 tokens", 24, 4096, 11264, train=False),
        # a layer of a unit test or of a debugging run: launches only
        _ffn("ffn train tiny", 128, 96, 64),
        # a small step, widths and tokens that are no multiple of a tile; pre-activations kept
        _ffn("ffn train 1000 tokens ragged", 1000, 2176, 1152, save=100),
        # the tokens of the headline training layer, pre-activations recomputed
        _ffn("ffn train 8192 tokens", 8192, 2048, 8192),
        # the largest step: bound by the matrix products
        _ffn("ffn train 16384 tokens", 16384, 4096, 11264, save=100),
        # experts, one sequence being decoded: eight of them, launches and host work show
        _int4("int4 experts 1 token", 1, 2048, 768, 128, 8),
        # a decode batch: most experts hold one or two tokens
        _int4("int4 experts 16 tokens", 16, 2048, 768, 128, 8),
        # a short prompt, zeros given, smaller groups: about 60 tokens an expert
        _int4("int4 experts 1000 tokens", 1000, 2048, 768, 128, 8, group=64, zeros=True),
        # the dense block, one sequence being decoded
        _int4("int4 ffn 1 token", 1, 4096, 11264),
        # a decode batch, smallest groups, widths that fill neither a group of columns nor a tile
        _int4("int4 ffn 50 tokens ragged", 50, 2176, 1152, group=32, zeros=True),
        # a prompt: bound by the matrix products
        _int4("int4 ffn 4096 tokens", 4096, 4096, 11264),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _width(rng, lo, hi):
    step = rng.choice((32, 64, 128))  # widths are multiples of 32
    return max(step, int(_log_uniform(rng, lo, hi)) // step * step)


def draw(rng):
    most = _flops(listed()[5])
    while True:
        if rng.random() < 0.5:
            train = rng.random() < 0.6
            case = _ffn("", int(_log_uniform(rng, 1, 32768)), _width(rng, 64, 4096), _width(rng, 32, 12288), train,
                        rng.choice((0, 0, 50, 100)) if train else 0)
        else:
            N = rng.choice((0, 0, 4, 8, 16, 48, 64, 128))
            case = _int4("", int(_log_uniform(rng, 1, 4096)), _width(rng, 64, 4096), _width(rng, 32, 2048 if N else 12288), N,
                         rng.choice((1, 2, 4, 6, 8)) if N else 0, rng.choice((32, 64, 128, 128)), rng.random() < 0.5,
                         rng.choice((0.0, 0.0, 0.5, 1.8)) if N else 0.0)
            if N and case["K"] > N // 2:
                continue
        del case["name"]
        if _flops(case) <= most and case["D"] * case["H"] * max(1, case.get("N", 0)) <= 2048 * 768 * 128:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _routing(logits, K):
    """The 0/1 mask [N, tokens] of the K greatest logits (the lower index where they are equal), and the softmax over those
    chosen, [tokens, N]."""
    M, N = logits.shape
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :K]
    chosen = torch.zeros(M, N, dtype=torch.bool, device=DEV).scatter_(1, order, True)
    w = torch.softmax(logits, -1) * chosen
    return chosen.T.to(torch.int32).contiguous(), (w / w.sum(-1, keepdim=True)).contiguous()


def _codes(N, R, C, group, zeros, gen):
    """Codes of normal weights of deviation 0.02, two to a byte [N, R / 2, C] (the even k-value in the low four bits), bf16 scales and
    zeros [N, ceil(R / group), C]."""
    packed = torch.empty(N, R // 2, C, dtype=torch.uint8, device=DEV)
    for i in range(N):
        q = torch.empty(R // 2, 2, C, device=DEV).normal_(7.5, 2.7, generator=gen).round_().clamp_(0, 15).to(torch.uint8)
        packed[i] = q[:, 0] | (q[:, 1] << 4)
    G = -(-R // group)
    scale = torch.empty(N, G, C, device=DEV).normal_(0, 0.15, generator=gen).exp_().mul_(0.02 / 2.7).to(torch.bfloat16)
    zero = torch.randint(6, 11, (N, G, C), generator=gen, device=DEV, dtype=torch.uint8) if zeros else None
    return packed, scale, zero


def _inputs(case, seed):
    M, D, H = case["tokens"], case["D"], case["H"]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(1, M, D, generator=gen, device=DEV).to(torch.bfloat16)
    if case["op"] == "ffn":
        W1 = torch.empty(D, 2 * H, device=DEV, dtype=torch.bfloat16).normal_(0, 0.02, generator=gen)
        W2 = torch.empty(H, D, device=DEV, dtype=torch.bfloat16).normal_(0, 0.02, generator=gen)
        gy = torch.randn(1, M, D, generator=gen, device=DEV).to(torch.bfloat16) if case["train"] else None
        return {"op": "ffn", "x": x, "W1": W1, "W2": W2, "gy": gy}
    N = case["N"]
    state = {"op": "int4", "x": x, "group": case["group"]}
    state["W1"], state["S1"], state["Z1"] = _codes(max(1, N), D, 2 * H, case["group"], case["zeros"], gen)
    state["W2"], state["S2"], state["Z2"] = _codes(max(1, N), H, D, case["group"], case["zeros"], gen)
    if N:
        logits = torch.randn(M, N, generator=gen, device=DEV)
        logits -= case["skew"] * torch.log(torch.arange(1, N + 1, device=DEV, dtype=torch.float32))
        mask, s_MN = _routing(logits, case["K"])
        state["mask"], state["s"] = mask, s_MN.T
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:  # the layer that a program keeps; of 4-bit weights it lays them out once
        m, D, H = _package(), case["D"], case["H"]
        if case["op"] == "ffn":
            state["layer"] = m.FeedForward(D, H, save_percent=case["save"], Wl1_D2H=state.pop("W1"), Wl2_HD=state.pop("W2"))
            state["x"].requires_grad_(case["train"])
        else:
            W1, S1, Z1, W2, S2, Z2 = (state.pop(k) for k in ("W1", "S1", "Z1", "W2", "S2", "Z2"))
            if case["N"]:
                state["layer"] = m.MoMoEInt4(D, H, case["N"], case["K"], W1, S1, W2, S2, Z1, Z2, group_size=case["group"])
            else:
                first = [None if t is None else t[0] for t in (W1, S1, W2, S2, Z1, Z2)]
                state["layer"] = m.FeedForwardInt4(D, H, *first, group_size=case["group"])
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_ffn(state) if state["op"] == "ffn" else _run_int4(state)
    return _plain_ffn(state) if state["op"] == "ffn" else _plain_int4(state)


def _run_ffn(state):
    layer, x = state["layer"], state["x"]
    if state["gy"] is None:
        with torch.no_grad():
            return [layer(x)]
    x.grad = layer.Wl1_D2H.grad = layer.Wl2_HD.grad = None
    y = layer(x)
    y.backward(state["gy"])
    return [y.detach(), x.grad, layer.Wl1_D2H.grad, layer.Wl2_HD.grad]


def _run_int4(state):
    with torch.no_grad():
        if "mask" in state:
            return list(state["layer"](state["x"], state["mask"], state["s"]))
        return [state["layer"](state["x"])]


def _gated(x, W1, W2):
    H = W2.shape[0]
    a, b = x @ W1[:, :H], x @ W1[:, H:]
    sig = 1 / (1 + torch.exp(-b))
    h = a * b * sig
    return a, b, sig, h, h @ W2


def _plain_ffn(state):
    x, W1, W2 = state["x"][0].float(), state["W1"].float(), state["W2"].float()
    a, b, sig, h, y = _gated(x, W1, W2)
    out = [y.to(torch.bfloat16)[None]]
    if state["gy"] is None:
        return out
    gy = state["gy"][0].float()
    u = gy @ W2.T
    gz = torch.cat([u * b * sig, u * a * sig * (1 + b * (1 - sig))], -1)
    return out + [(gz @ W1.T).to(torch.bfloat16)[None], (x.T @ gz).to(torch.bfloat16), (h.T @ gy).to(torch.bfloat16)]


def _weights_of(packed, scale, zero, group):
    """The values that one matrix of codes [R / 2, C] stands for, in 32 bits."""
    R, C = 2 * packed.shape[0], packed.shape[1]
    q = torch.stack([packed & 15, packed >> 4], 1).view(R, C).float()
    z = 8.0 if zero is None else zero.float().repeat_interleave(group, 0)[:R]
    return (q - z) * scale.float().repeat_interleave(group, 0)[:R]


def _plain_int4(state):
    x, group = state["x"][0].float(), state["group"]

    def block(i, rows):
        W1 = _weights_of(state["W1"][i], state["S1"][i], None if state["Z1"] is None else state["Z1"][i], group)
        W2 = _weights_of(state["W2"][i], state["S2"][i], None if state["Z2"] is None else state["Z2"][i], group)
        return _gated(rows, W1, W2)[4]

    if "mask" not in state:
        return [block(0, x).to(torch.bfloat16)[None]]
    y, sizes = torch.zeros_like(x), state["mask"].sum(1)
    for i in torch.nonzero(sizes).flatten().tolist():
        rows = torch.nonzero(state["mask"][i]).flatten()
        y[rows] += state["s"][i, rows].unsqueeze(1) * block(i, x[rows])
    return [y.to(torch.bfloat16)[None], sizes]


# ---- what the results are, in 64 bits ----------------------------------------------------------------------------------------
def _exact_block(x, W1, W2):
    lin, gate = torch.mm(x, W1).chunk(2, -1)
    return torch.mm(lin * torch.nn.functional.silu(gate), W2)


def _exact_matrix(packed, scale, zero, group):
    w = torch.empty(2 * packed.shape[0], packed.shape[1], dtype=torch.float64, device=DEV)
    w[0::2], w[1::2] = (packed % 16).double(), (packed // 16).double()
    for g in range(scale.shape[0]):
        k = slice(g * group, (g + 1) * group)
        w[k] = (w[k] - (8.0 if zero is None else zero[g].double())) * scale[g].double()
    return w


def exact(case, seed):
    t = _inputs(case, seed)
    x = t["x"][0].double()
    if case["op"] == "ffn":
        W1, W2 = t["W1"].double(), t["W2"].double()
        if t["gy"] is None:
            return [_exact_block(x, W1, W2)[None]]
        leaves = [x.requires_grad_(), W1.requires_grad_(), W2.requires_grad_()]
        y = _exact_block(*leaves)
        gx, g1, g2 = torch.autograd.grad(y, leaves, t["gy"][0].double())
        return [y.detach()[None], gx[None], g1, g2]

    def block(i, rows):
        zeros = [None if t[z] is None else t[z][i] for z in ("Z1", "Z2")]
        return _exact_block(rows, _exact_matrix(t["W1"][i], t["S1"][i], zeros[0], t["group"]),
                            _exact_matrix(t["W2"][i], t["S2"][i], zeros[1], t["group"]))

    if not case["N"]:
        return [block(0, x)[None]]
    y = torch.zeros_like(x)
    for i in range(case["N"]):
        tokens = (t["mask"][i] != 0).nonzero()[:, 0]
        if len(tokens):
            y.index_add_(0, tokens, block(i, x[tokens]) * t["s"][i, tokens].double()[:, None])
    return [y[None], (t["mask"] != 0).sum(1)]


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def _flops(case):
    return (18 if case.get("train") else 6) * case["tokens"] * max(1, case.get("K", 0)) * case["D"] * case["H"]


def work(case):
    M, D, H = case["tokens"], case["D"], case["H"]
    if case["op"] == "ffn":
        # x, y and the weights in 16 bits; of a step the gradients of all four, too
        return {"bytes": (2 if case["train"] else 1) * (4 * M * D + 6 * D * H), "flops": _flops(case)}
    N, K, G = case["N"], case["K"], case["group"]
    # blocks that hold a token, had every expert the same chance; half a byte a weight, 16 bits a scale, 4 a zero
    held = N * (1 - (1 - K / N) ** M) if N else 1
    groups = -(-D // G) * 2 * H + -(-H // G) * D
    weights = held * (1.5 * D * H + groups * (2.5 if case["zeros"] else 2))
    return {"bytes": weights + 4 * M * D + (4 * N * M + 4 * M * K + 8 * N if N else 0), "flops": _flops(case)}
