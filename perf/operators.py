"""Serving operators of gated-MLP models with expert layers and 4-bit weights, as cases that can be timed.

A case is one call of one operator:

    q4_linear   y = x·Wᵀ + b, W in 4 bits with group scales (few token rows)
    q4_mlp      a whole gated MLP whose three matrices are in 4 bits
    route       softmax of router logits, the top_k largest of each token, their weights
    moe         a whole mixture-of-experts layer for a few tokens, from the router's logits on; the experts are gated
                MLPs with 16-bit weights (bits = 16) or 4-bit ones (bits = 4)

    M tokens, K hidden size, N intermediate size (q4_linear: K inputs, N outputs), E experts, k of them per token

The 4-bit storage is the package's documented one.  A weight matrix [rows, cols] is padded to multiples of 16 rows and
128 columns.  codes is uint8 [rows/16, cols/128, 4, 16, 4, 4]: tile of 16 rows, block of 128 columns, q, row r of
the tile, step s, byte b, and the four bytes of (q, r, s) hold columns 32 s + 8 q + 0..7 of the block as n + 8 with
-8 <= n <= 7: columns 0, 2, 4, 6 in nibbles 0 to 3, columns 1, 3, 5, 7 in nibbles 4 to 7, a byte's low nibble first.
scales, of the activations' type, is [rows/16, cols/128, 4, 128/g, 4]: tile, block, quarter of the tile's rows, group of g
columns in the block, row in the quarter.  The weight is scale·n.  Experts are a leading dimension of both.
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


def _linear(dtype, M, K, N, g, bias=False):
    return {"kind": "q4_linear", "dtype": dtype, "M": M, "K": K, "N": N, "g": g, "bias": bias}


def _mlp(dtype, M, K, N, g, bias=False, act="silu"):
    return {"kind": "q4_mlp", "dtype": dtype, "M": M, "K": K, "N": N, "g": g, "bias": bias, "act": act}


def _route(dtype, M, E, k, normalize=True, masked=0):
    return {"kind": "route", "dtype": dtype, "M": M, "E": E, "k": k, "normalize": normalize, "masked": masked}


def _moe(dtype, M, K, N, E, k, bits=16, g=128, act="silu", normalize=True):
    return {"kind": "moe", "dtype": dtype, "M": M, "K": K, "N": N, "E": E, "k": k, "bits": bits, "g": g, "act": act,
            "normalize": normalize}


def listed():
    named = [
        # one sequence through a small projection: launch and latency
        ("q4_linear_single", _linear("bf16", 1, 2048, 2048, 128)),
        # a serving batch through a wide projection
        ("q4_linear_batch", _linear("fp16", 16, 4096, 14336, 128)),
        # widths that no tile divides, a bias, the finest groups, an odd batch
        ("q4_linear_ragged", _linear("bf16", 7, 1160, 3096, 32, bias=True)),
        # one sequence through a small model's MLP
        ("q4_mlp_single", _mlp("bf16", 1, 2048, 5632, 128)),
        # a serving batch through the largest MLP
        ("q4_mlp_batch", _mlp("fp16", 16, 8192, 28672, 128)),
        # speculative decoding's drafts of a batch: more tokens than one matrix tile, biases, another activation
        ("q4_mlp_drafts", _mlp("bf16", 48, 4096, 11008, 64, bias=True, act="gelu")),
        # routing of one token, and of a batch of prompts where some experts are not available to each token
        ("route_single", _route("fp32", 1, 8, 2)),
        ("route_prompts", _route("bf16", 16384, 128, 8, masked=32)),
        # one sequence through a layer of a few large experts
        ("moe_single", _moe("bf16", 1, 4096, 14336, 8, 2)),
        # a serving batch through a layer of many small experts: nearly all of them are read
        ("moe_batch", _moe("fp16", 16, 2048, 1024, 64, 8)),
        # the same layer in 4 bits for one sequence: the smallest whole layer
        ("moe_q4_single", _moe("bf16", 1, 2048, 1024, 64, 8, bits=4)),
        # a batch through large experts in 4 bits
        ("moe_q4_batch", _moe("fp16", 16, 4096, 14336, 8, 2, bits=4)),
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


# what the plain form of the largest listed case multiplies (16 tokens, 2 experts each), and its weights' elements per matrix
_MOST_PRODUCTS = 16 * 2 * 4096 * 14336
_MOST_ELEMENTS = 8 * 4096 * 14336


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["q4_linear", "q4_mlp", "route", "moe", "moe"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "route":
        E = rng.choice([8, 16, 24, 60, 64, 96, 128, 160, 256])
        k = rng.choice([1, 2, 4, 6, 8])
        M = int(_log_uniform(rng, 1, 16384)) | 1
        return _route(rng.choice(["fp32", "fp16", "bf16"]), M, E, k, rng.random() < 0.7, rng.choice([0, 0, E // 2]))
    M = round(_log_uniform(rng, 1, 64))
    g = rng.choice([32, 64, 128, 128])
    act = rng.choice(["silu", "silu", "gelu", "relu"])
    if kind == "moe":
        E = rng.choice([4, 8, 16, 32, 60, 64, 128])
        k = min(E, rng.choice([1, 2, 2, 4, 6, 8]))
        K = _width(rng, 512, 4096)
        most = min(_MOST_PRODUCTS / (M * k), _MOST_ELEMENTS / E) / K - 64
        N = min(_width(rng, 512, 14336), int(most) // 64 * 64 + 8 * rng.randrange(1, 8))
        return _moe(dtype, M, K, N, E, k, bits=rng.choice([4, 16]), g=g, act=act, normalize=rng.random() < 0.7)
    K = _width(rng, 512, 8192)
    N = _width(rng, 512, 28672)
    if kind == "q4_linear":
        return _linear(dtype, M, K, N, g, bias=rng.random() < 0.4)
    return _mlp(dtype, M, K, N, g, bias=rng.random() < 0.4, act=act)


# ------------------------------------------------------------------ inputs
def _quantized(w, g):
    """codes and scales of [rows, cols] weights: each group's largest magnitude becomes 7 steps."""
    rows, cols = w.shape
    R, C = -(-rows // 16) * 16, -(-cols // 128) * 128
    full = torch.zeros((R, C), dtype=torch.float32, device=w.device)
    full[:rows, :cols] = w
    groups = full.view(R, C // g, g)
    scale = (groups.abs().amax(-1) / 7).to(w.dtype)
    step = torch.where(scale > 0, scale.float(), 1.0)
    n = (groups / step.unsqueeze(-1)).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    # [tile, row, block, step, q, column pair, odd] -> nibble (odd, pair)
    n = n.view(R // 16, 16, C // 128, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5).reshape(R // 16, C // 128, 4, 16, 4, 4, 2)
    codes = n[..., 0] | (n[..., 1] << 4)
    scales = scale.view(R // 16, 4, 4, C // 128, 128 // g).permute(0, 3, 1, 4, 2).contiguous()
    return codes, scales


def prepare(case, seed):
    dtype = _DTYPES[case["dtype"]]
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(shape, std, kind=dtype):
        return torch.empty(shape, dtype=kind, device=dev).normal_(0.0, std, generator=gen)

    def four_bits(rows, cols, experts=None):
        if experts is None:
            return _quantized(normal((rows, cols), 0.02), case["g"]) + (rows, cols, case["g"])
        each = [_quantized(normal((rows, cols), 0.02), case["g"]) for _ in range(experts)]
        return (torch.stack([c for c, _ in each]), torch.stack([s for _, s in each]), rows, cols, case["g"])

    def bias(n):
        return torch.empty(n, dtype=dtype, device=dev).uniform_(-0.01, 0.01, generator=gen) if case["bias"] else None

    kind, M = case["kind"], case["M"]
    if kind == "route":
        logits = normal((M, case["E"]), 1.5)
        if case["masked"]:
            # experts that are not available to a token: another set for each
            off = torch.rand((M, case["E"]), device=dev, generator=gen).argsort(dim=1)[:, : case["masked"]]
            logits.scatter_(1, off, float("-inf"))
        return {"case": case, "logits": logits}
    K, N = case["K"], case["N"]
    state = {"case": case, "x": normal((M, K), 1.0)}
    if kind == "q4_linear":
        state["w"], state["b"] = four_bits(N, K), bias(N)
    elif kind == "q4_mlp":
        state["gate"], state["up"], state["down"] = four_bits(N, K), four_bits(N, K), four_bits(K, N)
        state["b_gate"], state["b_up"], state["b_down"] = bias(N), bias(N), bias(K)
    else:
        E = case["E"]
        state["logits"] = normal((M, E), 1.5, torch.float32)
        if case["bits"] == 4:
            state["gate"], state["up"], state["down"] = four_bits(N, K, E), four_bits(N, K, E), four_bits(K, N, E)
        else:
            state["gate"], state["up"], state["down"] = normal((E, N, K), 0.02), normal((E, N, K), 0.02), normal((E, K, N), 0.02)
    return state


# ------------------------------------------------------------------ plain forms
def _act(name, g):
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g.clamp(min=0.0) if name == "relu" else g / (1.0 + torch.exp(-g))


def _unpacked(codes, scales, rows, cols, g):
    """float32 weights [..., rows, cols]."""
    lead = codes.shape[:-6]
    RT, KB = codes.shape[-6:-4]
    d = len(lead)
    n = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(*lead, RT, KB, 4, 16, 4, 2, 4).transpose(-1, -2)
    n = n.permute(*range(d), d, d + 3, d + 1, d + 4, d + 2, d + 5, d + 6).reshape(*lead, RT * 16, KB * 128 // g, g)
    s = scales.float().permute(*range(d), d, d + 2, d + 4, d + 1, d + 3).reshape(*lead, RT * 16, KB * 128 // g, 1)
    return ((n.float() - 8.0) * s).reshape(*lead, RT * 16, KB * 128)[..., :rows, :cols]


def _plus(y, b):
    return y if b is None else y + b.float()


def _plain_route(logits, k, normalize):
    logits = logits.float()
    experts = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
    chosen = e.gather(1, experts)
    total = (chosen if normalize else e).sum(-1, keepdim=True)
    return torch.where(total > 0, chosen / total, 0.0), experts


def _plain_moe(state):
    case = state["case"]
    weights, experts = _plain_route(state["logits"], case["k"], case["normalize"])
    chosen = experts.reshape(-1)
    x = state["x"].float().repeat_interleave(case["k"], dim=0).unsqueeze(-1)

    def matrices(w):
        if case["bits"] == 16:
            return w[chosen].float()
        return _unpacked(w[0][chosen], w[1][chosen], *w[2:])

    h = _act(case["act"], torch.bmm(matrices(state["gate"]), x)) * torch.bmm(matrices(state["up"]), x)
    y = torch.bmm(matrices(state["down"]), h).reshape(case["M"], case["k"], case["K"])
    return (y * weights.unsqueeze(-1)).sum(1).to(state["x"].dtype)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "route":
        return _plain_route(state["logits"], case["k"], case["normalize"])
    if kind == "moe":
        return _plain_moe(state)
    x = state["x"].float()
    if kind == "q4_linear":
        return _plus(x @ _unpacked(*state["w"]).T, state["b"]).to(state["x"].dtype)
    g = _plus(x @ _unpacked(*state["gate"]).T, state["b_gate"])
    u = _plus(x @ _unpacked(*state["up"]).T, state["b_up"])
    return _plus((_act(case["act"], g) * u) @ _unpacked(*state["down"]).T, state["b_down"]).to(state["x"].dtype)


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
    if kind == "route":
        return tuple(moe.moe_route(state["logits"], case["k"], normalize=case["normalize"]))
    if kind == "q4_linear":
        return quant.q4_linear_fwd(state["x"], quant.Q4Weight(*state["w"]), state["b"])
    gate, up, down = state["gate"], state["up"], state["down"]
    if kind == "q4_mlp":
        return quant.q4_mlp_fwd(state["x"], quant.Q4Weight(*gate), state["b_gate"], quant.Q4Weight(*up), state["b_up"],
                                quant.Q4Weight(*down), state["b_down"], act_fn=case["act"])
    if case["bits"] == 4:
        gate, up, down = quant.Q4Weight(*gate), quant.Q4Weight(*up), quant.Q4Weight(*down)
    return moe.moe_mlp_fwd(state["x"], state["logits"], gate, up, down, case["k"], normalize=case["normalize"], act_fn=case["act"])


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size, M = _SIZES[case["dtype"]], case["M"]
    if case["kind"] == "route":
        # logits in; a float32 weight and a 64-bit expert number out for each choice
        return {"bytes": M * (case["E"] * size + case["k"] * 12), "flops": 4 * M * case["E"]}
    K, N = case["K"], case["N"]
    per_weight = size if case["kind"] == "moe" and case["bits"] == 16 else 0.5 + size / case["g"]
    if case["kind"] == "q4_linear":
        return {"bytes": N * K * per_weight + size * (M * (K + N) + (N if case["bias"] else 0)), "flops": 2 * M * N * K}
    if case["kind"] == "q4_mlp":
        return {"bytes": 3 * N * K * per_weight + size * (2 * M * K + (2 * N + K if case["bias"] else 0)), "flops": 6 * M * N * K}
    # the experts that M tokens choose between them, if each chooses k of E at random
    read = case["E"] * (1.0 - (1.0 - case["k"] / case["E"]) ** M)
    return {"bytes": 3 * read * N * K * per_weight + 2 * size * M * K + 4 * M * case["E"], "flops": 6 * M * case["k"] * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(codes, scales, rows, cols, g):
    """float64 weights [rows, cols], each looked up by where its nibble and its scale lie."""
    dev = codes.device
    KB = codes.shape[1]
    flat, flat_scales = codes.reshape(-1), scales.reshape(-1)
    c = torch.arange(cols, device=dev)
    out = torch.empty((rows, cols), dtype=torch.float64, device=dev)
    for first in range(0, rows, 2048):
        r = torch.arange(first, min(rows, first + 2048), device=dev).unsqueeze(1)
        block = (r // 16) * KB + c // 128
        nibble = (c % 8) // 2 + 4 * (c % 2)
        at = (((block * 4 + (c % 32) // 8) * 16 + r % 16) * 4 + (c % 128) // 32) * 4 + nibble // 2
        n = ((flat[at] >> (4 * (nibble % 2)).to(torch.uint8)) & 15).double() - 8.0
        at = ((block * 4 + (r % 16) // 4) * (128 // g) + (c % 128) // g) * 4 + r % 4
        out[first : first + r.shape[0]] = n * flat_scales[at].double()
    return out


def _exact_mlp(x, gate, b_gate, up, b_up, down, b_down, act):
    g, u = x @ gate.T, x @ up.T
    if b_gate is not None:
        g, u = g + b_gate.double(), u + b_up.double()
    if act == "silu":
        a = g * torch.sigmoid(g)
    else:
        a = torch.nn.functional.gelu(g) if act == "gelu" else torch.relu(g)
    y = (a * u) @ down.T
    return y if b_down is None else y + b_down.double()


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "q4_linear":
        y = state["x"].double() @ _exact_rows(*state["w"]).T
        return y if state["b"] is None else y + state["b"].double()
    if kind == "q4_mlp":
        return _exact_mlp(state["x"].double(), _exact_rows(*state["gate"]), state["b_gate"], _exact_rows(*state["up"]),
                          state["b_up"], _exact_rows(*state["down"]), state["b_down"], case["act"])
    logits = state["logits"].double()
    k = case["k"]
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
    p = torch.softmax(logits, -1).gather(1, experts)
    if case["normalize"]:
        p = p / p.sum(-1, keepdim=True)
    if kind == "route":
        return p, None
    x = state["x"].double()
    y = torch.zeros_like(x)
    for e in range(case["E"]):
        tokens, slots = torch.nonzero(experts == e, as_tuple=True)
        if tokens.numel() == 0:
            continue
        if case["bits"] == 4:
            w = [_exact_rows(state[n][0][e], state[n][1][e], *state[n][2:]) for n in ("gate", "up", "down")]
        else:
            w = [state[n][e].double() for n in ("gate", "up", "down")]
        out = _exact_mlp(x[tokens], w[0], None, w[1], None, w[2], None, case["act"])
        y.index_add_(0, tokens, out * p[tokens, slots].unsqueeze(1))
    return y
