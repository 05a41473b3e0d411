"""Layer norm over the last axis, forward and backward (csrc/norm_kernels.hip, include/yfs.h: yfs_layer_norm_*).

The reference's blocks have no normalisation (yolo_toy_regressor_torch.py:206-211, :258-266); its roadmap names it as the
next step (README.md:30).  ``HipLayerNorm`` is the form that trains: in the head it stands between ``fc.1`` and its
activation (``model.YoloRegressorModel(head_norm=True)``), over channels-last feature maps it normalises each cell.
"""
import torch
import torch.nn as nn

from . import _lib as L


def _rows(t):
    """``t`` as rows of its last axis: (a tensor that keeps the memory, rows, cols, elements from row to row)."""
    cols = t.shape[-1]
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.dim() != 2 or (cols > 1 and t.stride(1) != 1):
        t = t.contiguous().view(-1, cols)
    return t, t.shape[0], cols, t.stride(0)


def _f32_vector(t):
    if t is None:
        return None
    t = t.detach()
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _p(t):
    return t.data_ptr() if t is not None else None


def _check(x, weight, bias, eps):
    if x.dtype not in L.DTYPES:
        raise L.YfsError(f"layer_norm: x must be fp32, bf16 or fp16, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise L.YfsError(f"layer_norm: x needs a last axis of at least one element, got {tuple(x.shape)}")
    if not eps >= 0:
        raise L.YfsError(f"layer_norm: eps must not be negative, got {eps}")
    for what, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dim() != 1 or t.shape[0] != x.shape[-1] or not t.is_floating_point()):
            raise L.YfsError(f"layer_norm: {what} must be floating point [{x.shape[-1]}], got {t.dtype} {tuple(t.shape)}")


def _forward(x, weight, bias, eps, keep_stats):
    x2, rows, cols, stride = _rows(x.detach())
    w, b = _f32_vector(weight), _f32_vector(bias)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty(2, rows, device=x.device, dtype=torch.float32) if keep_stats else None
    if rows:
        mean = stats.data_ptr() if keep_stats else None
        with L.on_device("layer_norm", x2, w, b) as stream:
            L.check(L.lib().yfs_layer_norm_fwd(x2.data_ptr(), stride, _p(w), _p(b), y.data_ptr(), mean,
                                               mean + 4 * rows if keep_stats else None, rows, cols, eps, L.DTYPES[x.dtype],
                                               stream), "yfs_layer_norm_fwd")
    return y, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x2, rows, cols, xs = _rows(x.detach())
        dy2, _, _, dys = _rows(dy if dy.dtype == x.dtype else dy.to(x.dtype))
        w = _f32_vector(weight)
        dev = x.device
        dx = torch.empty(x.shape, device=dev, dtype=x.dtype) if need_x else None
        make = torch.empty if rows else torch.zeros
        dw = make(cols, device=dev, dtype=torch.float32) if need_w else None
        db = make(cols, device=dev, dtype=torch.float32) if need_b else None
        if rows:
            lib, code = L.lib(), L.DTYPES[x.dtype]
            nbytes = lib.yfs_layer_norm_bwd_workspace_bytes(rows, cols, code) if (need_w or need_b) else 0
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
            with L.on_device("layer_norm backward", x2, dy2, w) as stream:
                L.check(lib.yfs_layer_norm_bwd(dy2.data_ptr(), dys, x2.data_ptr(), xs, _p(w), stats.data_ptr(),
                                               stats.data_ptr() + 4 * rows, _p(dx), _p(dw), _p(db), rows, cols, code, _p(ws),
                                               nbytes, stream), "yfs_layer_norm_bwd")
        if need_w and weight.dtype != torch.float32:
            dw = dw.to(weight.dtype)
        if need_b and ctx.bias_dtype != torch.float32:
            db = db.to(ctx.bias_dtype)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of ``x`` [..., C] (fp32, bf16 or fp16; rows with any stride) over its last axis, ``weight`` and ``bias``
    [C] or None; the result is a dense tensor of x's dtype.  Statistics, products and sums are fp32.  Differentiable in x,
    weight and bias; the gradients of weight and bias are summed over the rows in a fixed order."""
    _check(x, weight, bias, eps)
    L.require_cuda(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


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
