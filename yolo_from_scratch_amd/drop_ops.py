"""Dropout from a counter-based generator, without a stored mask (csrc/dropout_kernels.hip, include/yfs.h: yfs_dropout_*).

The reference's head drops with nn.Dropout(0.2) behind a LeakyReLU (yolo_toy_regressor_torch.py:260-261).  ``fc_ops`` does
both in the epilogue of one product and stores a byte per element for the backward pass; this form stands on its own behind
any layer and keeps the seed alone: the backward pass draws the same numbers again.  The rule is the epilogue's, so the
same seed and p keep the same elements.
"""
import torch
import torch.nn as nn

from . import _lib as L


def dropout(x, p, seed, slope=1.0):
    """LeakyReLU(slope) (1.0: none) and dropout of ``x`` (fp32, bf16 or fp16, any shape) as one kernel; element e of the
    row-major tensor is kept iff (philox4x32_10(key=seed, counter=e // 4)[e % 4] >> 8) * 2**-24 >= p (p rounded to
    fp32 for this comparison) and then scaled by 1 / (1 - p).  Differentiable once.  ``seed``: an int (64 bits are used), or an int64 tensor of one element on x's GPU
    that the kernels read when they run (a captured graph then draws a new mask when the tensor is changed between replays;
    it must keep its value from the forward to the backward pass).  Nothing but the seed, and y where there is an
    activation, is kept for the backward pass.  0 <= p <= 1, 0 <= slope <= 1."""
    return (L._binding or L.binding()).dropout(x, p, seed, slope)


class HipDropout(nn.Module):
    """nn.LeakyReLU(slope) (1.0: none) and nn.Dropout(p) as one kernel without a stored mask.  In training each call draws
    its seed from torch's CPU generator, as ``HipLinear`` does (reproducible under torch.manual_seed); while a graph is captured,
    from the GPU's, so that every replay draws a mask of its own.  In eval mode the activation alone is applied."""

    def __init__(self, p=0.5, slope=1.0):
        super().__init__()
        if not 0.0 <= p <= 1.0 or not 0.0 <= slope <= 1.0:
            raise L.YfsError(f"HipDropout: p and slope must lie in [0, 1], got {p} and {slope}")
        self.p, self.slope = p, slope

    def forward(self, x):
        p = self.p if self.training else 0.0
        if p == 0.0 and self.slope == 1.0:
            return x
        if p == 0.0:
            seed = 0
        elif x.is_cuda and torch.cuda.is_current_stream_capturing():
            seed = torch.randint(0, 2 ** 62, (1,), device=x.device)
        else:
            seed = int(torch.randint(0, 2 ** 62, (1,)).item())
        return dropout(x, p, seed, self.slope)

    def extra_repr(self):
        return f"p={self.p}, slope={self.slope}"
