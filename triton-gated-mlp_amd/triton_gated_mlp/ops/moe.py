"""Mixture-of-experts layers of gated MLPs (host wrappers over libgmlp.so): routing, for serving and for training, and whole layers, for
serving.

Inference only, but for moe_route_balanced: no other operator here has a backward pass.  The reference has no such operators; an expert is its EagerGatedMLP
(src/triton_gated_mlp/gated_mlp.py:73-98) without biases.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import Tensor

from .. import _cabi
from .quant import Q4Weight, Q8Weight


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


class BalancedRouting(NamedTuple):
    weights: Tensor  # float32 [..., top_k]
    experts: Tensor  # int64 [..., top_k], in descending order of the logits
    counts: Tensor  # int64 [experts]
    loss: Tensor  # float32, a scalar


def moe_route_balanced(logits: Tensor, top_k: int, normalize: bool = True, token_mask: Optional[Tensor] = None) -> BalancedRouting:
    """moe_route for training: the same experts and weights (bit for bit up to 256 experts; beyond, their sums have another order), the number
    of choices that fell on each expert, and the balance loss E · sum_e f_e·P_e, f_e being the expert's share of all choices and P_e the
    mean of its softmax probability over the tokens.  It is 1 where every expert gets as much.

    `weights` and `loss` have gradients for the logits (any of the two may be left unused); f counts as a constant.  `token_mask`
    (bool [...], the logits' leading dimensions) is False for tokens, padding for instance, that are in neither counts nor
    loss; they are routed like the others.  Tokens to which no expert is available (logits -inf) are in neither either, nor
    choices of an expert that is not.  Without a token that counts the loss is 0."""
    if logits.requires_grad and torch.is_grad_enabled() and logits.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            "moe_route_balanced: capturing a step that records an autograd graph into a HIP graph is not supported (as with "
            "FusedGatedMLP); capture it under torch.no_grad() only"
        )
    return BalancedRouting(*_cabi.torch_binding().moe_route_balanced(logits, int(top_k), bool(normalize), token_mask))


def moe_mlp_fwd(
    x: Tensor,
    logits: Tensor,
    W_gate: Union[Tensor, Q4Weight, Q8Weight],
    W_up: Union[Tensor, Q4Weight, Q8Weight],
    W_down: Union[Tensor, Q4Weight, Q8Weight],
    top_k: int,
    normalize: bool = True,
    act_fn: str = "silu",
) -> Tensor:
    """y[t] = sum over t's experts e of weight·down_e(act_fn(gate_e(x[t])) * up_e(x[t])), routed as moe_route does.

    x [..., K]; logits [..., E]; W_gate, W_up [E, N, K] and W_down [E, K, N] in x's dtype, or all three as Q4Weight or Q8Weight.
    Nothing is copied to the host.

    Q8Weight: for any number of tokens.  The hidden states are rounded to x's dtype and become 8-bit integers as q8_mlp_fwd's
    do, the sum over experts is rounded once.  An expert is not run for a token whose weight for it is 0.

    Others: made for a few tokens: the weights of every expert that any of 64 token rows chose are read once, and of no other; a longer
    batch runs 64 rows at a time.  Beyond 4 token rows (2 with Q4Weight) the hidden
    states are rounded to x's dtype, as FusedGatedMLP does; the sum over experts is rounded once."""
    binding = _cabi.torch_binding()
    kinds = {Q4Weight if isinstance(w, Q4Weight) else Q8Weight if isinstance(w, Q8Weight) else Tensor for w in (W_gate, W_up, W_down)}
    if len(kinds) > 1:
        raise TypeError("W_gate, W_up and W_down are either all tensors or all Q4Weight or all Q8Weight")
    call = binding.moe_mlp if Tensor in kinds else binding.moe_mlp_q4 if Q4Weight in kinds else binding.moe_mlp_q8
    return call(x, logits, W_gate, W_up, W_down, int(top_k), bool(normalize), _cabi.act_code(act_fn))
