"""Dropout from a counter-based generator, without a stored mask (csrc/dropout_kernels.hip, include/yfs.h: yfs_dropout_*).

The reference's head drops with nn.Dropout(0.2) behind a LeakyReLU (yolo_toy_regressor_torch.py:260-261).  ``fc_ops`` does
both in the epilogue of one product and stores a byte per element for the backward pass; this form stands on its own behind
any layer and keeps the seed alone: the backward pass draws the same numbers again.  The rule is the epilogue's, so the
same seed and p keep the same elements.
"""
import torch
import torch.nn as nn

from . import _lib as L

_MASK64 = (1 << 64) - 1


def _run(name, src, y, p, slope, seed):
    out = torch.empty_like(src)
    if src.numel() == 0:
        return out
    dev_seed = isinstance(seed, torch.Tensor)
    with L.on_device("dropout", src, y, seed if dev_seed else None) as stream:
        lib, code = L.lib(), L.DTYPES[src.dtype]
        where = seed.data_ptr() if dev_seed else None
        value = 0 if dev_seed else seed & _MASK64
        if name == "yfs_dropout_fwd":
            rc = lib.yfs_dropout_fwd(src.data_ptr(), out.data_ptr(), src.numel(), p, slope, value, where, code, stream)
        else:
            rc = lib.yfs_dropout_bwd(src.data_ptr(), y.data_ptr() if y is not None else None, out.data_ptr(), src.numel(), p,
                                     slope, value, where, code, stream)
    L.check(rc, name)
    return out


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, slope):
        y = _run("yfs_dropout_fwd", x.detach().contiguous(), None, p, slope, seed)
        # y is kept for the sign of its elements, a seed in device memory so that a change before backward is noticed
        keep = [y] if slope != 1.0 else []
        if isinstance(seed, torch.Tensor):
            keep.append(seed)
        ctx.save_for_backward(*keep)
        ctx.args = (p, slope, seed if not isinstance(seed, torch.Tensor) else None)
        ctx.dtype = x.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, slope, seed = ctx.args
        kept = ctx.saved_tensors
        y = kept[0] if slope != 1.0 else None
        dy = (dy if dy.dtype == ctx.dtype else dy.to(ctx.dtype)).contiguous()
        return _run("yfs_dropout_bwd", dy, y, p, slope, kept[-1] if seed is None else seed), None, None, None


def dropout(x, p, seed, slope=1.0):
    """LeakyReLU(slope) (1.0: none) and dropout of ``x`` (fp32, bf16 or fp16, any shape) as one kernel; element e of the
    row-major tensor is kept iff (philox4x32_10(key=seed, counter=e // 4)[e % 4] >> 8) * 2**-24 >= p and then scaled by
    1 / (1 - p).  ``seed``: an int (64 bits are used), or an int64 tensor of one element on x's GPU that the kernels read
    when they run (a captured graph then draws a new mask when the tensor is changed between replays; it must keep its value
    from the forward to the backward pass).  Nothing but the seed, and y where there is an activation, is kept for the
    backward pass.  0 <= p <= 1, 0 <= slope <= 1."""
    if x.dtype not in L.DTYPES:
        raise L.YfsError(f"dropout: x must be fp32, bf16 or fp16, got {x.dtype}")
    if not 0.0 <= p <= 1.0:
        raise L.YfsError(f"dropout: p must lie in [0, 1], got {p}")
    if not 0.0 <= slope <= 1.0:
        raise L.YfsError(f"dropout: slope must lie in [0, 1], got {slope}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise L.YfsError(f"dropout: a seed tensor must hold one int64, got {tuple(seed.shape)} {seed.dtype}")
    elif not isinstance(seed, int):
        raise L.YfsError(f"dropout: seed must be an int or an int64 tensor, got {type(seed).__name__}")
    L.require_cuda(x, seed if isinstance(seed, torch.Tensor) else None)
    if torch.is_grad_enabled() and x.requires_grad:
        return _DropoutFn.apply(x, float(p), seed, float(slope))
    return _run("yfs_dropout_fwd", x.detach().contiguous(), None, float(p), float(slope), seed)


class HipDropout(nn.Module):
    """nn.LeakyReLU(slope) (1.0: none) and nn.Dropout(p) as one kernel without a stored mask.  In training each call draws
    its seed from torch's CPU generator, as ``HipLinear`` does (reproducible under torch.manual_seed); in eval mode the
    activation alone is applied."""

    def __init__(self, p=0.5, slope=1.0):
        super().__init__()
        if not 0.0 <= p <= 1.0 or not 0.0 <= slope <= 1.0:
            raise L.YfsError(f"HipDropout: p and slope must lie in [0, 1], got {p} and {slope}")
        self.p, self.slope = p, slope

    def forward(self, x):
        p = self.p if self.training else 0.0
        if p == 0.0 and self.slope == 1.0:
            return x
        seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if p > 0 else 0
        return dropout(x, p, seed, self.slope)

    def extra_repr(self):
        return f"p={self.p}, slope={self.slope}"
