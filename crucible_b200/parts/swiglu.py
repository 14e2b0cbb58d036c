"""Dense SwiGLU feed-forward: x += (silu(n Wg^T) * (n Wu^T)) Wd^T.

`model.py:240-245`, `engine/src/model.rs:254-273`; SiLU on the gate,
g / (1 + exp(-g)), in fp32 (`engine/kernels/kernels.cu:1038-1047`).  Gate and
up matrices are stored separately in the checkpoint and concatenated at load
into one [2I, d] operand so one matrix product serves both; each output element
is still the same dot product, so numerics per element do not change.
"""
from __future__ import annotations

import torch

from .. import ops
from ..config.model_config import ConfigError, FeedForwardSpec
from ..ops import quantized
from .base import FEED_FORWARDS, FeedForward, TensorDecl


class SwiGLU(FeedForward):
    fuses_norm = True

    def __init__(self, spec: FeedForwardSpec):
        self.spec = spec
        self.gate_up = None
        self.down = None
        self.dtype = None

    def tensors(self):
        d, i = self.spec.width, self.spec.intermediate
        return [TensorDecl("gate", (i, d)), TensorDecl("up", (i, d)), TensorDecl("down", (d, i))]

    def bind(self, tensors, dtype, device):
        self.gate_up = torch.cat([tensors["gate"], tensors["up"]], dim=0).contiguous()
        self.down = tensors["down"]
        ops.declare_weights(self.gate_up, self.down)
        self.dtype = dtype

    def forward(self, ctx, h, residual):
        t, i = h.shape[0], self.spec.intermediate
        act = ctx.scratch("ffn.act", (t, i), self.dtype)
        ops.linear_swiglu(h, self.gate_up, act, ctx)
        ops.linear(act, self.down, residual, accumulate=True, closes=ctx)


class SwiGLU4(SwiGLU):
    """The same with its matrices in 4 bits (`quantized.Weights4`): the checkpoint's are packed once, at load,
    with an e4m3 scale for every `group` weights of a feature (option, 64) and a float32 one a feature.  Rows, sums
    and the gated pair are those of the engine's dtype."""
    fuses_norm = False         # its first product takes normalised rows: nobody is asked to leave others for it

    def __init__(self, spec: FeedForwardSpec):
        super().__init__(spec)
        self.group = int(spec.option("group", 64))
        if self.group <= 0 or self.group % 32 or spec.width % self.group or spec.intermediate % self.group:
            raise ConfigError(f"4-bit feed-forward: a group is a multiple of 32 that divides the widths "
                              f"{spec.width} and {spec.intermediate}, got {self.group}")

    def bind(self, tensors, dtype, device):
        both = torch.cat([tensors["gate"], tensors["up"]], dim=0)
        self.gate_up = quantized.Weights4.pack(both, self.group)
        self.down = quantized.Weights4.pack(tensors["down"], self.group)
        self.dtype = dtype

    def forward(self, ctx, h, residual):
        t, i = h.shape[0], self.spec.intermediate
        both = ctx.scratch("ffn.gate_up", (t, 2 * i), self.dtype)
        act = ctx.scratch("ffn.act", (t, i), self.dtype)
        quantized.linear4(h, self.gate_up, both)
        ops.swiglu(both, act)
        quantized.linear4(act, self.down, residual, add=residual)


FEED_FORWARDS.register("swiglu", SwiGLU)
FEED_FORWARDS.register("swiglu_4bit", SwiGLU4)
