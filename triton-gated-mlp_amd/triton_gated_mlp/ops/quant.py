"""4-bit weights with group scales, for serving: storage, and the linear layer and gated MLP on it (host wrappers over
libgmlp.so).

A weight is scale·n with -8 <= n <= 7 and one scale per row and group of 32, 64 or 128 columns.  The products are of scale·n
itself, accumulated in fp32.  Inference only: no operator here has a backward pass.  The reference has no such operators; the
math is that of its nn.Linear and EagerGatedMLP (src/triton_gated_mlp/gated_mlp.py:73-98).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

from torch import Tensor

from .. import _cabi


class Q4Weight(NamedTuple):
    """A 4-bit weight matrix [rows, cols], or one per expert with a leading dimension of codes and scales.

    Rows are padded to tiles of 16, columns to blocks of 128.  codes: uint8 [tiles, blocks, 4 q, 16 r, 4 s, 4]; the four
    bytes of (q, r, s) are columns 32 s + 8 q + 0..7 of the tile's row r as n + 8, columns 0, 2, 4, 6 in nibbles 0 to 3 and
    1, 3, 5, 7 in nibbles 4 to 7, a byte's low nibble first.  scales, of the activations' dtype: [tiles, blocks, 4, 128 /
    group_size, 4]: quarter of the tile's rows, group, row of the quarter.  (include/gmlp.h defines the same storage.)
    """

    codes: Tensor
    scales: Tensor
    rows: int
    cols: int
    group_size: int


def quantize_q4(W: Tensor, group_size: int = 128) -> Q4Weight:
    """W [rows, cols] or [experts, rows, cols] in 4 bits: each group's largest magnitude becomes 7 steps."""
    codes, scales = _cabi.torch_binding().q4_quantize(W, int(group_size))
    return Q4Weight(codes, scales, W.shape[-2], W.shape[-1], int(group_size))


def dequantize_q4(weight: Q4Weight) -> Tensor:
    """scale·n rounded to the scales' dtype, [rows, cols] or [experts, rows, cols]."""
    return _cabi.torch_binding().q4_dequantize(weight)


def q4_linear_fwd(x: Tensor, weight: Q4Weight, bias: Optional[Tensor] = None) -> Tensor:
    """x [..., cols]·Wᵀ + bias.  Up to 64 token rows the weights are streamed once in their 4 bits; more rows run on
    the dense GEMM with the weights rounded to 16 bits first, as dequantize_q4 gives them."""
    return _cabi.torch_binding().q4_linear(x, weight, bias)


def q4_mlp_fwd(
    x: Tensor,
    W_gate: Q4Weight,
    b_gate: Optional[Tensor],
    W_up: Q4Weight,
    b_up: Optional[Tensor],
    W_down: Q4Weight,
    b_down: Optional[Tensor],
    act_fn: str = "silu",
) -> Tensor:
    """A whole gated MLP on 4-bit weights: two kernels up to 64 token rows, beyond as q4_linear_fwd.  Beyond
    2 token rows the hidden states are rounded to x's dtype between the two, as FusedGatedMLP does (in float16 one past
    65504 is infinite)."""
    return _cabi.torch_binding().q4_mlp(x, W_gate, b_gate, W_up, b_up, W_down, b_down, _cabi.act_code(act_fn))
