"""Operators of gated-MLP models with expert layers: routing that can be trained and balanced, and 8-bit integer products, as cases
that can be timed.

A case is one call of one operator:

    route_balance  a router's training step: the top_k experts of each token with their weights, the tokens that each expert gets,
                   the balance loss, and the gradient of the logits from the gradients of weights and loss
    q8_linear      y = x·Wᵀ + b in 8-bit integers: W with a scale for each row, x with one for each token, found in the call
    q8_mlp         a whole gated MLP whose three matrices are in 8 bits
    q8_moe         a whole mixture-of-experts layer from the router's logits on, its experts gated MLPs in 8 bits

    M tokens, K hidden size, N intermediate size (q8_linear: K inputs, N outputs), E experts, k of them per token

The balance loss is E · sum over experts of f·P, f an expert's share of all choices and P the mean of its softmax probability
over the tokens; f counts as a constant.  Tokens that a mask leaves out, and experts whose logit is -inf, are in neither.

8-bit integers: a row of numbers v becomes n = 127 v / max|v|, rounded half to even, and the scale max|v| / 127.  Token rows are
rows of x; the hidden states of a gated MLP are rounded to x's type and become 8-bit rows again.

The storage of 8-bit weights is the package's documented one.  A weight matrix [rows, cols] is padded with zeros to multiples of
16 rows and 128 columns; codes is int8 [rows/16, cols/128, 2, 4, 16, 16]: tile of 16 rows, block of 128 columns, half s of the
block, quarter q of the half, row r of the tile, and columns 64 s + 16 q + 0..15 of the block.  scales is float32 [rows].
Experts are a leading dimension of both.
"""

from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _route(dtype, M, E, k, normalize=True, masked=0, padded=False):
    return {"kind": "route_balance", "dtype": dtype, "M": M, "E": E, "k": k, "normalize": normalize, "masked": masked, "padded": padded}


def _linear(dtype, M, K, N, bias=False):
    return {"kind": "q8_linear", "dtype": dtype, "M": M, "K": K, "N": N, "bias": bias}


def _mlp(dtype, M, K, N, bias=False, act="silu"):
    return {"kind": "q8_mlp", "dtype": dtype, "M": M, "K": K, "N": N, "bias": bias, "act": act}


def _moe(dtype, M, K, N, E, k, act="silu", normalize=True):
    return {"kind": "q8_moe", "dtype": dtype, "M": M, "K": K, "N": N, "E": E, "k": k, "act": act, "normalize": normalize}


def listed():
    named = [
        # a router's step over a short sequence: launches and host time
        ("route_balance_short", _route("fp32", 64, 8, 2)),
        # over a batch of sequences, many experts of which some are not available to each token, padding at the end
        ("route_balance_batch", _route("fp32", 16384, 128, 8, masked=32, padded=True)),
        # logits in 16 bits, a number of experts that no vector divides, weights that are not normalised
        ("route_balance_half", _route("bf16", 4097, 60, 4, normalize=False)),
        # one sequence through a small projection: launches and latency
        ("q8_linear_single", _linear("bf16", 1, 2048, 2048)),
        # widths that no tile divides, a bias, an odd batch
        ("q8_linear_ragged", _linear("bf16", 77, 1160, 3096, bias=True)),
        # a prompt through a wide projection: the matrix cores
        ("q8_linear_prompt", _linear("fp16", 4096, 4096, 14336)),
        # one sequence through a large MLP: the weights' way from memory
        ("q8_mlp_single", _mlp("bf16", 1, 4096, 14336)),
        # a serving batch through the largest MLP
        ("q8_mlp_batch", _mlp("fp16", 16, 8192, 28672)),
        # a prompt, biases, another activation
        ("q8_mlp_prompt", _mlp("bf16", 2048, 4096, 11008, bias=True, act="gelu")),
        # one sequence through a layer of many small experts: the smallest whole layer
        ("q8_moe_single", _moe("bf16", 1, 2048, 1024, 64, 8)),
        # a batch of drafts through it: every expert has a few tokens
        ("q8_moe_drafts", _moe("fp16", 96, 2048, 1024, 64, 8)),
        # a batch of prompts through a layer of a few large experts
        ("q8_moe_prompt", _moe("bf16", 4096, 4096, 14336, 8, 2)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


_USUAL = (512, 768, 1024, 1408, 1536, 2048, 2560, 2816, 3584, 4096, 5120, 5632, 6144, 7168, 8192, 10240, 11008, 14336, 16384,
          24576, 28672)


def _width(rng, lo, hi):
    """A layer width: as often one of the usual ones as a multiple of 8 that is none of 64."""
    width = _log_uniform(rng, lo, hi)
    if rng.random() < 0.5:
        return min((w for w in _USUAL if lo <= w <= hi), key=lambda w: abs(math.log(w / width)))
    return int(width) // 64 * 64 + 8 * rng.randrange(1, 8)


# products of a matrix of the largest listed case, and its weights' elements per matrix
_MOST_PRODUCTS = 4096 * 2 * 4096 * 14336
_MOST_ELEMENTS = 8 * 4096 * 14336


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["route", "linear", "mlp", "moe"])
    if kind == "route":
        E = rng.choice([4, 8, 16, 24, 60, 64, 96, 128, 160, 256])
        k = min(E, rng.choice([1, 2, 4, 6, 8]))
        M = int(_log_uniform(rng, 1, 16384 * min(1.0, 128 / E))) | 1
        return _route(rng.choice(["fp32", "fp32", "fp16", "bf16"]), M, E, k, rng.random() < 0.7, rng.choice([0, 0, E // 2]),
                      rng.random() < 0.4)
    dtype = rng.choice(["fp16", "bf16"])
    act = rng.choice(["silu", "silu", "gelu", "relu"])
    if kind == "linear":
        K, N = _width(rng, 512, 8192), _width(rng, 512, 14336)
        return _linear(dtype, max(1, round(_log_uniform(rng, 1, 4096))), K, N, bias=rng.random() < 0.4)
    if kind == "mlp":
        K, N = _width(rng, 512, 8192), _width(rng, 512, 28672)
        M = round(_log_uniform(rng, 1, min(4096, _MOST_PRODUCTS / (K * N))))
        return _mlp(dtype, max(1, M), K, N, bias=rng.random() < 0.4, act=act)
    E = rng.choice([4, 8, 16, 32, 60, 64, 128])
    k = min(E, rng.choice([1, 2, 2, 4, 6, 8]))
    M = max(1, round(_log_uniform(rng, 1, 4096)))
    K = _width(rng, 512, 4096)
    most = min(_MOST_PRODUCTS / (M * k), _MOST_ELEMENTS / E) / K - 64
    N = min(_width(rng, 512, 14336), int(most) // 64 * 64 + 8 * rng.randrange(1, 8))
    return _moe(dtype, M, K, N, E, k, act=act, normalize=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _quantized(w):
    """codes and scales of [rows, cols] weights."""
    rows, cols = w.shape
    R, C = -(-rows // 16) * 16, -(-cols // 128) * 128
    w = w.float()
    top = w.abs().amax(-1, keepdim=True)
    n = torch.zeros((R, C), dtype=torch.int8, device=w.device)
    n[:rows, :cols] = torch.round(127.0 * w / torch.where(top > 0, top, 1.0)).to(torch.int8)
    codes = n.view(R // 16, 16, C // 128, 2, 4, 16).permute(0, 2, 3, 4, 1, 5).contiguous()
    return codes, (top / 127.0).squeeze(-1)


def prepare(case, seed):
    dtype = _DTYPES[case["dtype"]]
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(shape, std, kind=dtype):
        return torch.empty(shape, dtype=kind, device=dev).normal_(0.0, std, generator=gen)

    def eight_bits(rows, cols, experts=None):
        if experts is None:
            return _quantized(normal((rows, cols), 0.02)) + (rows, cols)
        each = [_quantized(normal((rows, cols), 0.02)) for _ in range(experts)]
        return torch.stack([c for c, _ in each]), torch.stack([s for _, s in each]), rows, cols

    def bias(n):
        return torch.empty(n, dtype=dtype, device=dev).uniform_(-0.01, 0.01, generator=gen) if case["bias"] else None

    kind, M = case["kind"], case["M"]
    if kind == "route_balance":
        E, k = case["E"], case["k"]
        # some experts are more popular than others: that is what the loss is against
        logits = (normal((M, E), 1.0, torch.float32) + normal((1, E), 0.7, torch.float32)).to(dtype)
        if case["masked"]:
            off = torch.rand((M, E), device=dev, generator=gen).argsort(dim=1)[:, : case["masked"]]
            logits.scatter_(1, off, float("-inf"))
        mask = None
        if case["padded"]:
            length = torch.randint(max(1, M // 2), M + 1, (1,), device=dev, generator=gen)
            mask = torch.arange(M, device=dev) < length
        return {"case": case, "logits": logits.requires_grad_(), "mask": mask, "d_weights": normal((M, k), 0.1, torch.float32),
                "d_loss": torch.rand((), device=dev, generator=gen) * 0.01 + 0.005}
    K, N = case["K"], case["N"]
    state = {"case": case, "x": normal((M, K), 1.0)}
    if kind == "q8_linear":
        state["w"], state["b"] = eight_bits(N, K), bias(N)
    elif kind == "q8_mlp":
        state["gate"], state["up"], state["down"] = eight_bits(N, K), eight_bits(N, K), eight_bits(K, N)
        state["b_gate"], state["b_up"], state["b_down"] = bias(N), bias(N), bias(K)
    else:
        E = case["E"]
        state["logits"] = normal((M, E), 1.5, torch.float32)
        state["gate"], state["up"], state["down"] = eight_bits(N, K, E), eight_bits(N, K, E), eight_bits(K, N, E)
    return state


# ------------------------------------------------------------------ plain forms
def _act(name, g):
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g.clamp(min=0.0) if name == "relu" else g / (1.0 + torch.exp(-g))


def _rows8(x):
    """8-bit integers of rows [..., n], as float32, and their scales [..., 1]."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(127.0 * x / torch.where(top > 0, top, 1.0)), top / 127.0


def _integers(codes, rows, cols):
    """float32 integers [..., rows, cols]."""
    d = codes.dim() - 6
    n = codes.permute(*range(d), d, d + 4, d + 1, d + 2, d + 3, d + 5)
    return n.reshape(*codes.shape[:d], codes.shape[d] * 16, codes.shape[d + 1] * 128)[..., :rows, :cols].float()


def _product(x, w, b=None):
    """float32 x·Wᵀ + b of 8-bit rows and weights."""
    q, s = _rows8(x)
    codes, scales, rows, cols = w
    y = (q @ _integers(codes, rows, cols).T) * (s * scales)
    return y if b is None else y + b.float()


def _plain_softmax(logits):
    logits = logits.float()
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
    return e, e.sum(-1, keepdim=True)


def _plain_route(logits, k, normalize):
    experts = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, :k]
    e, total = _plain_softmax(logits)
    chosen = e.gather(1, experts)
    total = chosen.sum(-1, keepdim=True) if normalize else total
    return torch.where(total > 0, chosen / total, 0.0), experts


def _plain_balance(state):
    case, logits, d_weights = state["case"], state["logits"].detach(), state["d_weights"]
    M, E, k = case["M"], case["E"], case["k"]
    weights, experts = _plain_route(logits, k, case["normalize"])
    e, total = _plain_softmax(logits)
    p = torch.where(total > 0, e / total, 0.0)
    there = total > 0 if state["mask"] is None else (total > 0) & state["mask"].unsqueeze(-1)
    counted = there & (logits.gather(1, experts) > float("-inf"))
    counts = torch.zeros(E, dtype=torch.int64, device=logits.device)
    counts.scatter_add_(0, experts.reshape(-1), counted.reshape(-1).to(torch.int64))
    tokens = there.sum().clamp(min=1)
    share = counts.float() / counts.sum().clamp(min=1)
    loss = E * (share * torch.where(there, p, 0.0).sum(0) / tokens).sum()
    d = torch.where(there, p, 0.0) * (share - (share * p).sum(-1, keepdim=True)) * (state["d_loss"] * E / tokens)
    mixed = (weights * d_weights).sum(-1, keepdim=True)
    if case["normalize"]:
        d.scatter_add_(1, experts, weights * (d_weights - mixed))
    else:
        d.scatter_add_(1, experts, weights * d_weights)
        d -= p * mixed
    return weights, experts, counts, loss, d.to(logits.dtype)


def _plain_moe(state):
    case, x = state["case"], state["x"]
    M, K, N, E, k = case["M"], case["K"], case["N"], case["E"], case["k"]
    weights, experts = _plain_route(state["logits"], k, case["normalize"])
    chosen = experts.reshape(-1)
    pairs = torch.arange(M * k, device=x.device)
    if M * k <= E:
        # fewer choices than experts: each with its expert's matrices
        lanes, place = pairs, torch.zeros_like(pairs)
        rows = x.repeat_interleave(k, dim=0).unsqueeze(1)
        gate, up, down = ((w[0][chosen], w[1][chosen]) + w[2:] for w in (state["gate"], state["up"], state["down"]))
    else:
        # every expert with its tokens, padded to as many as the one that has most
        order = torch.argsort(chosen, stable=True)
        counts = torch.zeros(E, dtype=torch.int64, device=x.device).scatter_add_(0, chosen, torch.ones_like(chosen))
        lanes, place = chosen, torch.empty_like(chosen)
        place[order] = pairs - (counts.cumsum(0) - counts)[chosen[order]]
        rows = torch.zeros((E, int(counts.max()), K), dtype=x.dtype, device=x.device)
        rows[lanes, place] = x.repeat_interleave(k, dim=0)
        gate, up, down = state["gate"], state["up"], state["down"]

    def product(rows, w):
        q, s = _rows8(rows)
        y = torch.bmm(_integers(w[0], *w[2:]), q.transpose(1, 2).contiguous())
        return (y * w[1].unsqueeze(-1)).transpose(1, 2) * s

    h = (_act(case["act"], product(rows, gate)) * product(rows, up)).to(x.dtype)
    y = product(h, down)[lanes, place].reshape(M, k, K)
    return (y * weights.unsqueeze(-1)).sum(1).to(x.dtype)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "route_balance":
        return _plain_balance(state)
    if kind == "q8_moe":
        return _plain_moe(state)
    x = state["x"]
    if kind == "q8_linear":
        return _product(x, state["w"], state["b"]).to(x.dtype)
    h = _act(case["act"], _product(x, state["gate"], state["b_gate"])) * _product(x, state["up"], state["b_up"])
    return _product(h.to(x.dtype), state["down"], state["b_down"]).to(x.dtype)


# ------------------------------------------------------------------ the package's operators
@functools.lru_cache(maxsize=None)
def _ops():
    package = os.path.join(os.getcwd(), "triton-gated-mlp_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from triton_gated_mlp.ops import moe, quant

    return moe, quant


def _own(state):
    moe, quant = _ops()
    case = state["case"]
    kind = case["kind"]
    if kind == "route_balance":
        logits = state["logits"]
        weights, experts, counts, loss = moe.moe_route_balanced(logits, case["k"], normalize=case["normalize"], token_mask=state["mask"])
        (d_logits,) = torch.autograd.grad((weights, loss), logits, (state["d_weights"], state["d_loss"]))
        return weights.detach(), experts, counts, loss.detach(), d_logits
    with torch.no_grad():
        if kind == "q8_linear":
            return quant.q8_linear_fwd(state["x"], quant.Q8Weight(*state["w"]), state["b"])
        gate, up, down = (quant.Q8Weight(*state[n]) for n in ("gate", "up", "down"))
        if kind == "q8_mlp":
            return quant.q8_mlp_fwd(state["x"], gate, state["b_gate"], up, state["b_up"], down, state["b_down"], act_fn=case["act"])
        return moe.moe_mlp_fwd(state["x"], state["logits"], gate, up, down, case["k"], normalize=case["normalize"], act_fn=case["act"])


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size, M = _SIZES[case["dtype"]], case["M"]
    if case["kind"] == "route_balance":
        # logits in and their gradient out; per choice a weight, its gradient and a 64-bit expert number
        E, k = case["E"], case["k"]
        return {"bytes": M * (2 * E * size + 16 * k + (1 if case["padded"] else 0)) + 8 * E, "flops": 12 * M * E}
    K, N = case["K"], case["N"]
    if case["kind"] == "q8_linear":
        return {"bytes": N * (K + 4) + size * (M * (K + N) + (N if case["bias"] else 0)), "flops": 2 * M * N * K}
    if case["kind"] == "q8_mlp":
        return {"bytes": 3 * N * K + 4 * (2 * N + K) + size * (2 * M * K + (2 * N + K if case["bias"] else 0)), "flops": 6 * M * N * K}
    # the experts that M tokens choose between them, if each chooses k of E at random
    read = case["E"] * (1.0 - (1.0 - case["k"] / case["E"]) ** M)
    return {"bytes": read * (3 * N * K + 4 * (2 * N + K)) + 2 * size * M * K + 4 * M * case["E"], "flops": 6 * M * case["k"] * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows8(x):
    """The numbers that rows of 8-bit integers stand for, in float64."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    steps = (x * 127.0 / top.clamp(min=1e-300)).round()
    return steps * top / 127.0


def _exact_weight(codes, scales, rows, cols):
    """float64 weights [rows, cols], each looked up by where it lies."""
    dev = codes.device
    blocks = codes.shape[1]
    flat = codes.reshape(-1)
    c = torch.arange(cols, device=dev)
    out = torch.empty((rows, cols), dtype=torch.float64, device=dev)
    for first in range(0, rows, 2048):
        r = torch.arange(first, min(rows, first + 2048), device=dev).unsqueeze(1)
        at = (((r // 16 * blocks + c // 128) * 2 + c % 128 // 64) * 4 + c % 64 // 16) * 256 + r % 16 * 16 + c % 16
        out[first : first + r.shape[0]] = flat[at].double() * scales[first : first + r.shape[0], None].double()
    return out


def _exact_mlp(x, gate, b_gate, up, b_up, down, b_down, act):
    dtype = x.dtype
    x = _exact_rows8(x)
    g, u = x @ gate.T, x @ up.T
    if b_gate is not None:
        g, u = g + b_gate.double(), u + b_up.double()
    if act == "silu":
        a = g * torch.sigmoid(g)
    else:
        a = torch.nn.functional.gelu(g) if act == "gelu" else torch.relu(g)
    y = _exact_rows8((a * u).to(dtype)) @ down.T
    return y if b_down is None else y + b_down.double()


def _exact_route(logits, k, normalize):
    picks = []
    left = logits.clone()
    for _ in range(k):  # the largest that is left, the lowest index among equals
        best = left == left.amax(-1, keepdim=True)
        if picks:
            best = best & ~torch.zeros_like(best).scatter_(1, torch.stack(picks, 1), True)
        pick = best.int().argmax(-1)
        picks.append(pick)
        left = left.scatter(1, pick.unsqueeze(1), float("-inf"))
    experts = torch.stack(picks, 1)
    p = torch.softmax(logits, -1)
    w = p.gather(1, experts)
    return p, (w / w.sum(-1, keepdim=True) if normalize else w), experts


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "q8_linear":
        y = _exact_rows8(state["x"]) @ _exact_weight(*state["w"]).T
        return y if state["b"] is None else y + state["b"].double()
    if kind == "q8_mlp":
        return _exact_mlp(state["x"], _exact_weight(*state["gate"]), state["b_gate"], _exact_weight(*state["up"]), state["b_up"],
                          _exact_weight(*state["down"]), state["b_down"], case["act"])
    E, k = case["E"], case["k"]
    if kind == "route_balance":
        with torch.enable_grad():
            logits = state["logits"].detach().double().requires_grad_()
            p, weights, experts = _exact_route(logits, k, case["normalize"])
            rows = torch.ones(case["M"], dtype=torch.bool, device=p.device) if state["mask"] is None else state["mask"]
            picked = torch.zeros_like(p).scatter(1, experts, 1.0) * (logits.detach() > float("-inf"))
            share = picked[rows].sum(0)
            loss = E * (share / share.sum() * p[rows].mean(0)).sum()
            (d,) = torch.autograd.grad((weights, loss), logits, (state["d_weights"].double(), state["d_loss"].double()))
        return weights.detach(), None, None, loss.detach(), d
    _, p, experts = _exact_route(state["logits"].double(), k, case["normalize"])
    x = state["x"]
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(E):
        tokens, slots = torch.nonzero(experts == e, as_tuple=True)
        if tokens.numel() == 0:
            continue
        w = [_exact_weight(state[n][0][e], state[n][1][e], *state[n][2:]) for n in ("gate", "up", "down")]
        out = _exact_mlp(x[tokens], w[0], None, w[1], None, w[2], None, case["act"])
        y.index_add_(0, tokens, out * p[tokens, slots].unsqueeze(1))
    return y
