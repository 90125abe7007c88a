"""Channels-first linear layer.

Mirrors `deconver/layers/linear.py:7-58` of the reference: a 1x1 `nn.Conv1d` over the flattened
spatial axes, so the parameters are named `linear.weight` / `linear.bias` and checkpoints move
both ways.  On CUDA the whole layer is one native autograd node (`csrc/ndc_torch.cpp`): the product
and the input gradient are library GEMMs over the tensors as they lie (the convolution route
converts to channels-last and back for some shapes: 256 -> 64 channels over 4 x 128^3 positions take
4.49 ms against 0.98 ms), the bias is added and its gradient reduced by this library's own kernels
(`csrc/ndc_bias.cu`: the library's broadcast add is not vectorised and its reduction uses one block
per output channel, which shows at the small per-GPU batches of a batch-sharded training step), and
the weight gradient is that of the `Deconv` layer's projection.  CPU tensors, other dtypes and
float32 without a bias take the plain `nn.Conv1d`.

`channel_linear` is the same layer as a function.  Both can keep their input for the weight gradient in 8 bits
(``checkpoint="fp8"``), and compute their products from operands held in 8 bits (``products="fp8"``); these
run on CUDA float32 / bfloat16 tensors only.
"""

from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from .fp8 import is_fp8
from .functional import native

_DTYPES = (torch.float32, torch.bfloat16)


def native_operands(x: torch.Tensor, weight: torch.Tensor):
    """``(x, weight)`` in the type the product runs in, or None where the native node does not take
    them.  Under autocast that is its type, as for a convolution."""
    if not x.is_cuda or not weight.is_cuda or x.dim() < 3:
        return None
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight = x.to(dtype), weight.to(dtype)
    return (x, weight) if x.dtype in _DTYPES and x.dtype == weight.dtype else None


def channel_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, checkpoint: str = "exact",
                   products: str = "exact") -> torch.Tensor:
    """``y[b, o] = sum_c weight[o, c, 0] x[b, c] + bias[o]`` for ``x`` (batch, in_channels, spatial...).

    checkpoint="fp8": the backward pass knows the input as it is held in 8 bits (`deconver_b200.fp8`), blocks along the
        positions: the weight's gradient is that of what is held; the result and the other gradients are not touched.
        (Of large bfloat16 layers, 2^18 weights and 10^11 operations, it is read back whole for that gradient.)
    products="fp8": the products are of operands held in 8 bits, in blocks of 128 along what they are summed over:
        y (blocks of input channels), the input's gradient (of output channels), the weight's (of positions, from the
        checkpoint, so that the input is kept in 8 bits here too).  Sums are float32; the bias and its gradient are not
        held in 8 bits.  Up to 2^24 positions per sample.
    """
    eight = is_fp8(checkpoint, "checkpoint"), is_fp8(products, "products")
    operands = native_operands(x, weight)
    if not any(eight):
        if operands is not None and (bias is not None or operands[0].dtype == torch.bfloat16):
            return native("linear", (*operands, bias))
        if x.numel() and weight.numel():
            y = F.conv1d(x.flatten(2), weight, bias)
        else:                                   # a convolution refuses it, or gives no outputs
            y = weight[:, :, 0] @ x.flatten(2)
            y = y if bias is None else y + bias[:, None]
        return y.view(x.shape[0], weight.shape[0], *x.shape[2:])
    if operands is None:
        raise RuntimeError("deconver_b200: linear in 8 bits takes CUDA float32 / bfloat16 tensors (batch, channels, spatial...) and a weight of "
                           f"their type, not {x.dtype} {tuple(x.shape)} on {x.device} and {weight.dtype} on {weight.device}")
    return native("linear_q8", (*operands, bias), eight[1])


class Linear(nn.Module):
    checkpoint, products, eight = "exact", "exact", False

    def __init__(self, in_channels: int, out_channels: int, bias: bool = True,
                 device: Optional[torch.device] = None, dtype: Optional[torch.dtype] = None, *,
                 checkpoint: str = "exact", products: str = "exact"):
        super().__init__()
        self.checkpoint, self.products = checkpoint, products
        self.eight = is_fp8(checkpoint, "checkpoint") | is_fp8(products, "products")
        self.flatten = nn.Flatten(start_dim=2)
        self.linear = nn.Conv1d(in_channels, out_channels, kernel_size=1, bias=bias,
                                device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        bias = self.linear.bias
        if self.eight:
            return channel_linear(x, self.linear.weight, bias, checkpoint=self.checkpoint, products=self.products)
        operands = native_operands(x, self.linear.weight)
        if operands is not None and (bias is not None or operands[0].dtype == torch.bfloat16):
            return native("linear", (*operands, bias))
        shape = x.shape
        return self.linear(self.flatten(x)).view(shape[0], -1, *shape[2:])

    def extra_repr(self) -> str:
        return f"checkpoint={self.checkpoint}, products={self.products}" if self.eight else ""
