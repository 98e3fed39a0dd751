"""Decoding through a stack of serving layers, in one HIP graph: tokens go through alternating 4-bit (8-bit, 16-bit) gated MLPs and layers of
experts, each behind a normalisation and added to the residual, as a language model's feed-forward halves do.

    PYTHONPATH=triton-gated-mlp_amd python -m triton_gated_mlp.decode_example [--tokens 1] [--layers 8] [--bits 4]
"""

from __future__ import annotations

import argparse
import time

import torch
from torch import Tensor, nn

from .experts import GatedMoE, Q4GatedMLP, Q8GatedMLP
from .gated_mlp import FusedGatedMLP


class DecodeStack(nn.Module):
    def __init__(self, hidden_size: int, intermediate_size: int, expert_size: int, num_experts: int, top_k: int, layers: int, bits: int,
                 group_size: int, dtype: torch.dtype, device: torch.device):
        super().__init__()
        self.blocks = nn.ModuleList()
        for i in range(layers):
            with torch.device(device):
                if i % 2 == 0:
                    layer = FusedGatedMLP(hidden_size, intermediate_size, bias=False).to(dtype).eval()
                    if bits < 16:
                        layer = Q4GatedMLP.from_float(layer, group_size) if bits == 4 else Q8GatedMLP.from_float(layer)
                else:
                    layer = GatedMoE(hidden_size, expert_size, num_experts, top_k).to(dtype)
                    layer = layer.quantize_(group_size, bits) if bits < 16 else layer
            self.blocks.append(layer)

    def forward(self, x: Tensor) -> Tensor:
        for layer in self.blocks:
            x = x + layer(nn.functional.rms_norm(x, x.shape[-1:]))
        return x


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=1, help="sequences decoded together (at most 64)")
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--intermediate", type=int, default=5632)
    ap.add_argument("--expert", type=int, default=1024, help="intermediate size of an expert")
    ap.add_argument("--experts", type=int, default=64)
    ap.add_argument("--top-k", type=int, default=8)
    ap.add_argument("--bits", type=int, default=4, choices=(4, 8, 16))
    ap.add_argument("--group", type=int, default=128, choices=(32, 64, 128))
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args(argv)
    dev, dtype = torch.device("cuda", 0), torch.bfloat16
    torch.manual_seed(0)
    with torch.no_grad():
        model = DecodeStack(a.hidden, a.intermediate, a.expert, a.experts, a.top_k, a.layers, a.bits, a.group, dtype, dev)
        x = torch.randn(a.tokens, a.hidden, dtype=dtype, device=dev)
        eager = model(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(x)
        for _ in range(5):
            graph.replay()
        torch.cuda.synchronize()
        if not torch.equal(y, eager):
            raise AssertionError("the graph gives something else than the eager layers")
        began = time.perf_counter()
        for _ in range(a.steps):
            graph.replay()
        torch.cuda.synchronize()
        us = (time.perf_counter() - began) / a.steps * 1e6
    print(f"{a.layers} layers, {a.bits} bits, {a.tokens} token(s) a step: {us:.1f} us a step, {a.tokens / us * 1e6:.0f} tokens/s")
    return us


if __name__ == "__main__":
    main()
