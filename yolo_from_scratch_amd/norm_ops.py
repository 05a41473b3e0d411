"""Layer norm over the last axis, forward and backward (csrc/norm_kernels.hip, include/yfs.h: yfs_layer_norm_*).

The reference's blocks have no normalisation (yolo_toy_regressor_torch.py:206-211, :258-266); its roadmap names it as the
next step (README.md:30).  ``HipLayerNorm`` is the form that trains: in the head it stands between ``fc.1`` and its
activation (``model.YoloRegressorModel(head_norm=True)``), over channels-last feature maps it normalises each cell.
"""
import torch
import torch.nn as nn

from . import _lib as L


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of ``x`` [..., C] (fp32, bf16 or fp16; rows with any stride) over its last axis, ``weight`` and ``bias``
    [C] or None; the result is a dense tensor of x's dtype.  Statistics, products and sums are fp32.  Differentiable (once) in
    x, weight and bias; the gradients of weight and bias are summed over the rows in a fixed order.

    Capturing forward and backward into a graph works as for any operator of torch: no autograd graph of the same leaves
    that was made outside the capture may be alive, or torch's engine makes the outer stream part of the capture."""
    return (L._binding or L.binding()).layer_norm(x, weight, bias, eps)


class HipLayerNorm(nn.Module):
    """nn.LayerNorm(channels) on the kernels above (same parameter names, fp32).  ``channels_first=True`` normalises the
    channels of an [N, C, H, W] map at each cell, as the conv blocks' channels-last maps hold them (no copy; other layouts
    are rearranged first)."""

    def __init__(self, channels, eps=1e-5, bias=True, channels_first=False):
        super().__init__()
        self.channels, self.eps, self.channels_first = channels, eps, channels_first
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels)) if bias else None

    def forward(self, x):
        if not self.channels_first:
            return layer_norm(x, self.weight, self.bias, self.eps)
        if x.dim() != 4 or x.shape[1] != self.channels:
            raise L.YfsError(f"HipLayerNorm(channels_first): expected [N, {self.channels}, H, W], got {tuple(x.shape)}")
        return layer_norm(x.permute(0, 2, 3, 1), self.weight, self.bias, self.eps).permute(0, 3, 1, 2)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}, bias={self.bias is not None}, channels_first={self.channels_first}"
