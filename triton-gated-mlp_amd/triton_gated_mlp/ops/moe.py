"""Mixture-of-experts layers of gated MLPs, for serving (host wrappers over libgmlp.so).

Inference only: no operator here has a backward pass.  The reference has no such operators; an expert is its EagerGatedMLP
(src/triton_gated_mlp/gated_mlp.py:73-98) without biases.
"""

from __future__ import annotations

from typing import NamedTuple, Union

from torch import Tensor

from .. import _cabi
from .quant import Q4Weight


class Routing(NamedTuple):
    weights: Tensor  # float32 [..., top_k]
    experts: Tensor  # int64 [..., top_k], in descending order of the logits


def moe_logits(x: Tensor, W_router: Tensor) -> Tensor:
    """float32 x [..., hidden]·W_routerᵀ, W_router [experts, hidden] in x's dtype; experts a multiple of 4.  Made for a few
    tokens: 64 rows at a time."""
    return _cabi.torch_binding().moe_logits(x, W_router)


def moe_route(logits: Tensor, top_k: int, normalize: bool = True) -> Routing:
    """Softmax over the last dimension of `logits` (float32, float16 or bfloat16; at most 512 experts) and the top_k
    (at most 16) largest of each token, the lowest number first among equals; with `normalize` their weights are divided by
    their sum.  An expert whose logit is -inf is not available to the token and has weight 0."""
    return Routing(*_cabi.torch_binding().moe_route(logits, int(top_k), bool(normalize)))


def moe_mlp_fwd(
    x: Tensor,
    logits: Tensor,
    W_gate: Union[Tensor, Q4Weight],
    W_up: Union[Tensor, Q4Weight],
    W_down: Union[Tensor, Q4Weight],
    top_k: int,
    normalize: bool = True,
    act_fn: str = "silu",
) -> Tensor:
    """y[t] = sum over t's experts e of weight·down_e(act_fn(gate_e(x[t])) * up_e(x[t])), routed as moe_route does.

    x [..., K]; logits [..., E]; W_gate, W_up [E, N, K] and W_down [E, K, N] in x's dtype, or all three as Q4Weight.  Made for a
    few tokens: the weights of every expert that any of 64 token rows chose are read once, and of no other; a longer
    batch runs 64 rows at a time.  Nothing is copied to the host.  Beyond 4 token rows (2 with Q4Weight) the hidden
    states are rounded to x's dtype, as FusedGatedMLP does; the sum over experts is rounded once."""
    binding = _cabi.torch_binding()
    quantized = [isinstance(w, Q4Weight) for w in (W_gate, W_up, W_down)]
    if any(quantized) and not all(quantized):
        raise TypeError("W_gate, W_up and W_down are either all tensors or all Q4Weight")
    call = binding.moe_mlp_q4 if quantized[0] else binding.moe_mlp
    return call(x, logits, W_gate, W_up, W_down, int(top_k), bool(normalize), _cabi.act_code(act_fn))
