"""Layer norm as a module, for models whose batches are too small for the blocks' BatchNorm (train/erfnet_blocks.py:23,44,
50,82): it has no running statistics and is the same in training and in evaluation.  No counterpart in the reference."""
import torch
import torch.nn as nn

from . import functional as hipf

__all__ = ["LayerNorm"]


class LayerNorm(nn.Module):
    """Normalises the last axis (``dim=-1``) or, with ``dim=1``, every pixel of an [N,C,H,W] activation over its channels.

    ``weight`` and ``bias`` ([num_channels], fp32, ones and zeros) exist unless ``affine`` / ``bias`` is False.  GPU tensors
    (fp32 or bf16) run functional.layer_norm; CPU tensors stock torch on the same parameters, as in the blocks."""

    def __init__(self, num_channels, eps=1e-5, affine=True, bias=True, dim=-1):
        super().__init__()
        if dim not in (-1, 1):
            raise ValueError(f"LayerNorm: dim must be -1 or 1 (got {dim})")
        self.num_channels, self.eps, self.dim = num_channels, eps, dim
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine and bias else None

    def forward(self, input):
        if input.dim() < (2 if self.dim == 1 else 1) or input.shape[self.dim] != self.num_channels:
            raise ValueError(f"LayerNorm: {self.num_channels} channels on axis {self.dim} of {tuple(input.shape)}")
        if input.is_cuda:
            return hipf.layer_norm(input, self.weight, self.bias, self.eps, self.dim)
        x = input.movedim(self.dim, -1)
        w, b = (None if p is None else p.float() for p in (self.weight, self.bias))
        y = torch.nn.functional.layer_norm(x.float(), (self.num_channels,), w, b, self.eps)
        return y.to(input.dtype).movedim(-1, self.dim)

    def extra_repr(self):
        return f"{self.num_channels}, eps={self.eps}, affine={self.weight is not None}, bias={self.bias is not None}, dim={self.dim}"
