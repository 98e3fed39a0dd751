"""Serving modules beside FusedGatedMLP: a gated MLP on 4-bit weights, and a mixture of gated-MLP experts.

  Q4GatedMLP.from_float(mlp, group_size)                      a FusedGatedMLP or EagerGatedMLP with its weights in 4 bits
  GatedMoE(hidden_size, intermediate_size, num_experts, top_k)  router and experts, in 16 bits or, after quantize_(), 4

Inference only: both raise where autograd would have to record them.  The reference has no such modules; an expert is its
EagerGatedMLP (src/triton_gated_mlp/gated_mlp.py:73-98) without biases.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor, nn

from . import _cabi
from .gated_mlp import ACT_FWD
from .ops import fwd as _fwd
from .ops import moe as _moe
from .ops import quant as _quant
from .ops.quant import Q4Weight


class _Q4Buffers(nn.Module):
    """A Q4Weight whose tensors move, and are saved, with the module.  (`.half()` and the like convert the scales.)"""

    def __init__(self, weight: Q4Weight):
        super().__init__()
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.rows, self.cols, self.group_size = weight.rows, weight.cols, weight.group_size

    def weight(self) -> Q4Weight:
        return Q4Weight(self.codes, self.scales, self.rows, self.cols, self.group_size)

    def of(self, expert: int) -> Q4Weight:
        return Q4Weight(self.codes[expert], self.scales[expert], self.rows, self.cols, self.group_size)


class Q4GatedMLP(nn.Module):
    """down(act(gate(x)) * up(x)) with the three matrices in 4 bits (see ops.quant) and the biases as they were."""

    def __init__(self, gate: Q4Weight, up: Q4Weight, down: Q4Weight, b_gate: Optional[Tensor] = None, b_up: Optional[Tensor] = None,
                 b_down: Optional[Tensor] = None, hidden_act: str = "silu"):
        super().__init__()
        if hidden_act not in ACT_FWD:
            raise KeyError(hidden_act)
        self.hidden_size, self.intermediate_size, self.act_fn = gate.cols, gate.rows, hidden_act
        self.gate_proj, self.up_proj, self.down_proj = _Q4Buffers(gate), _Q4Buffers(up), _Q4Buffers(down)
        for name, b in (("b_gate", b_gate), ("b_up", b_up), ("b_down", b_down)):
            self.register_buffer(name, None if b is None else b.detach())

    @classmethod
    def from_float(cls, mlp: nn.Module, group_size: int = 128) -> "Q4GatedMLP":
        """From a gated-MLP module on the GPU in float16 or bfloat16.  Its dropout is left out, as in evaluation."""
        layers = (mlp.gate_proj, mlp.up_proj, mlp.down_proj)
        return cls(*(_quant.quantize_q4(layer.weight.detach(), group_size) for layer in layers), *(layer.bias for layer in layers),
                   hidden_act=mlp.act_fn)

    def forward(self, x: Tensor) -> Tensor:
        return _quant.q4_mlp_fwd(x, self.gate_proj.weight(), self.b_gate, self.up_proj.weight(), self.b_up, self.down_proj.weight(),
                                 self.b_down, act_fn=self.act_fn)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, {self.intermediate_size}, group_size={self.gate_proj.group_size}, hidden_act={self.act_fn!r}"


class GatedMoE(nn.Module):
    """y = sum over a token's top_k experts of weight * expert(x), routed by the softmax of router(x).

    `router` [experts, hidden] gives float32 logits, from weights of x's type or float32; gate_proj, up_proj [experts, intermediate,
    hidden] and down_proj [experts, hidden, intermediate] have x's type.  Few tokens run on the weight-streaming
    kernels, nothing goes to the host, and the call can be captured into a HIP graph; from `long_batch` token rows on
    the experts run one after the other on the dense kernels, which needs the number of each expert's tokens on the host
    and rounds each expert's output to x's type ahead of the sum over experts.
    """

    def __init__(self, hidden_size: int, intermediate_size: int, num_experts: int, top_k: int, normalize: bool = True,
                 hidden_act: str = "silu"):
        super().__init__()
        if hidden_act not in ACT_FWD:
            raise KeyError(hidden_act)
        if not 1 <= top_k <= num_experts:
            raise ValueError(f"top_k = {top_k} of {num_experts} experts")
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.num_experts, self.top_k, self.normalize, self.act_fn = num_experts, top_k, normalize, hidden_act
        self.router = nn.Linear(hidden_size, num_experts, bias=False)
        self.gate_proj = nn.Parameter(torch.empty(num_experts, intermediate_size, hidden_size))
        self.up_proj = nn.Parameter(torch.empty(num_experts, intermediate_size, hidden_size))
        self.down_proj = nn.Parameter(torch.empty(num_experts, hidden_size, intermediate_size))
        for p in (self.gate_proj, self.up_proj, self.down_proj):  # as nn.Linear does
            nn.init.uniform_(p, -1 / math.sqrt(p.shape[2]), 1 / math.sqrt(p.shape[2]))

    def quantize_(self, group_size: int = 128) -> "GatedMoE":
        """The experts' weights (on the GPU, float16 or bfloat16) in 4 bits from now on; the router stays as it is."""
        for name in ("gate_proj", "up_proj", "down_proj"):
            weight = _quant.quantize_q4(getattr(self, name).detach(), group_size)
            delattr(self, name)
            setattr(self, name, _Q4Buffers(weight))
        return self

    @property
    def quantized(self) -> bool:
        return isinstance(self.gate_proj, _Q4Buffers)

    def _weights(self, expert: Optional[int] = None):
        for w in (self.gate_proj, self.up_proj, self.down_proj):
            if isinstance(w, _Q4Buffers):
                yield w.weight() if expert is None else w.of(expert)
            else:
                yield w if expert is None else w[expert]

    def route_logits(self, x: Tensor) -> Tensor:
        """float32 router logits of [rows, hidden] tokens."""
        w, E = self.router.weight, self.num_experts
        if x.shape[0] <= 64 and w.dtype == x.dtype and E % 4 == 0:
            return _moe.moe_logits(x, w)
        # a router kept in float32, or many rows: the float32 GEMM (which takes whole rows of 8, and looks at no gradients)
        _cabi.torch_binding().inference_only("GatedMoE", [x, w])
        w = w.float()
        if E % 8:
            w = nn.functional.pad(w, (0, 0, 0, 8 - E % 8))
        return _fwd.linear_fwd(x.float(), w)[:, :E]

    def long_batch(self) -> int:
        """Token rows from which the experts' own passes are the faster way.  The streaming kernels read the experts in use once
        per 64 rows; passes of their own cost 60 to 70 us an expert on the host or, of large experts, their weights' way at
        half the rate, and 4-bit weights of more than 64 tokens are written out in 16 bits first.  ms, streamed and one by one,
        experts of hidden x intermediate size: 16 bits, 8 of 4096 x 14336 128 rows 0.91 0.92, 192 rows 1.37 0.95; 8 of 2048 x 5632
        384 rows 0.66 0.67, 512 rows 0.88 0.67; 64 of 2048 x 1024 1536 rows 3.4 4.0, 2048 rows 4.6 4.0; 4 of 8192 x 28672 65 rows
        1.9 1.3.  4 bits, 8 of 4096 x 14336 512 rows 1.6 2.0, 768 rows 2.3 2.1; 8 of 2048 x 5632 768 rows 0.75 0.78, 1024 rows 0.99
        0.83; 64 of 2048 x 1024 2048 rows 2.1 4.5, 6144 rows 6.4 4.8, but 8 of them 1536 rows 0.71 0.70; 4 of 8192 x 28672 256 rows
        2.4 3.1, 384 rows 3.5 3.3."""
        size = self.hidden_size * self.intermediate_size
        rows = min(9e10 / size, 550 + 4e9 / size) if self.quantized else min(2e10 / (3 * size), 95 + 3.4e9 / size)
        return max(65, int(rows))

    def forward(self, x: Tensor) -> Tensor:
        rows = x.reshape(-1, self.hidden_size)
        logits = self.route_logits(rows)
        if rows.shape[0] < self.long_batch():
            y = _moe.moe_mlp_fwd(rows, logits, *self._weights(), self.top_k, normalize=self.normalize, act_fn=self.act_fn)
        else:
            y = self._one_by_one(rows, logits)
        return y.reshape(x.shape)

    def _one_by_one(self, x: Tensor, logits: Tensor) -> Tensor:
        _cabi.torch_binding().inference_only("GatedMoE", [x, *self.parameters()])
        weights, experts = _moe.moe_route(logits, self.top_k, normalize=self.normalize)
        # (an expert that is not available to the token, logit -inf, is not run for it: behind the others, and not counted)
        experts = experts.masked_fill(logits.gather(-1, experts) == -math.inf, self.num_experts).reshape(-1)
        order = experts.argsort(stable=True)
        counts = torch.bincount(experts, minlength=self.num_experts).tolist()[: self.num_experts]
        y = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
        first = 0
        for e, n in enumerate(counts):
            pairs = order[first : first + n]
            first += n
            if n == 0:
                continue
            tokens = pairs // self.top_k
            gate, up, down = self._weights(e)
            if self.quantized:
                out = _quant.q4_mlp_fwd(x[tokens], gate, None, up, None, down, None, act_fn=self.act_fn)
            else:
                out, _ = _fwd.mlp_fwd(x[tokens], gate, None, up, None, down, None, act_fn=self.act_fn)
            y.index_add_(0, tokens, out.float() * weights.reshape(-1)[pairs, None])
        return y.to(x.dtype)

    def extra_repr(self) -> str:
        return (f"{self.hidden_size}, {self.intermediate_size}, num_experts={self.num_experts}, top_k={self.top_k}, "
                f"normalize={self.normalize}, hidden_act={self.act_fn!r}")

