"""Matrix product in 8-bit floating point with a scale for each block of 128 (csrc/fp8_kernels.hip, include/yfs.h: yfs_fp8_*).

What the head's linear layers (yolo_toy_regressor_torch.py:259, :262) multiply in 16 bits, in 8: weights are e4m3 with a
power-of-two scale for each 128 x 128 block, activations and gradients with one for each row and 128 columns.

* serving: ``quantize_fp8`` once, then ``fp8_matmul(x, w)`` per call, or ``FrozenFp8Linear`` / ``freeze_fp8(model)``;
* training: ``fp8_linear(x, weight, bias)`` / ``Fp8Linear``: 32-bit master weights, three 8-bit products
  (y = x W^T, dx = dy W, dW = dy^T x), each operand scaled along the axis that its product sums over.

A block's scale is the smallest power of two s >= 2^-127 with max|x| <= 448 s over its finite elements (1 for zeros);
x / s is rounded to nearest, ties to even.  NaN and infinities become NaN, without touching the scale.
"""
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib as L

BLOCK = 128


def _pad(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


class Fp8Tensor:
    """A weight [n, k] in 8 bits: ``data`` float8_e4m3fn [n, k rounded up to 128] (zeros behind k), ``scale`` float8_e8m0fnu
    [ceil(n / 128), ceil(k / 128)]: the values are data * scale, block by block."""
    __slots__ = ("data", "scale", "k")

    def __init__(self, data, scale, k, block=(BLOCK, BLOCK)):
        if tuple(block) != (BLOCK, BLOCK):
            raise L.YfsError(f"Fp8Tensor: blocks are {BLOCK} x {BLOCK}, got {tuple(block)}")
        if data.dim() != 2 or data.dtype != torch.float8_e4m3fn or not 0 < k <= data.shape[1] or data.shape[1] != _pad(k):
            raise L.YfsError(f"Fp8Tensor: data must be float8_e4m3fn [n, {_pad(k)}] for k = {k}, got {data.dtype} {tuple(data.shape)}")
        want = (_pad(data.shape[0]) // BLOCK, data.shape[1] // BLOCK)
        if tuple(scale.shape) != want or scale.dtype != torch.float8_e8m0fnu:
            raise L.YfsError(f"Fp8Tensor: scale must be float8_e8m0fnu {want}, got {scale.dtype} {tuple(scale.shape)}")
        if not data.is_contiguous() or not scale.is_contiguous() or data.data_ptr() % 16:
            raise L.YfsError("Fp8Tensor: data and scale must be contiguous, data 16-byte aligned")
        self.data, self.scale, self.k = data, scale, k

    @property
    def shape(self):
        return torch.Size((self.data.shape[0], self.k))

    @property
    def device(self):
        return self.data.device

    def dequantize(self):
        """The fp32 values [n, k]."""
        s = self.scale.float().repeat_interleave(BLOCK, 0)[: self.data.shape[0]].repeat_interleave(BLOCK, 1)
        return (self.data.float() * s)[:, : self.k].contiguous()

    def __repr__(self):
        return f"Fp8Tensor({tuple(self.shape)}, device={self.device})"


def _matrix(t, what):
    """[..., k] -> rows with unit stride inside a row, the count of rows and the row stride."""
    if t.dtype not in L.DTYPES:
        raise L.YfsError(f"{what}: expected fp32, bf16 or fp16, got {t.dtype}")
    k = t.shape[-1]
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.dim() != 2 or (k > 1 and t.stride(1) != 1):
        t = t.contiguous().view(-1, k)
    return t, t.shape[0], t.stride(0)


def _p(t):
    return t.data_ptr() if t is not None else None


def _check_weight(w):
    if w.dim() != 2 or w.shape[0] == 0 or w.shape[1] == 0 or w.dtype not in L.DTYPES:
        raise L.YfsError(f"quantize_fp8: expected a non-empty fp32, bf16 or fp16 matrix, got {w.dtype} {tuple(w.shape)}")


def _settled(w):
    """A parameter whose overlapped step (train.FlatSGD.overlap_tail) is still running on the side stream is waited for."""
    owner = getattr(w, "_yfs_tail_owner", None)
    if owner is not None:
        owner.join()


def _quantize_weight(w, transposed):
    """-> (data, scale) and, when asked, (data, scale) of the transpose: the same bytes, block by block."""
    w2, n, ld = _matrix(w.detach(), "quantize_fp8")
    k, dev = w2.shape[1], w2.device
    nb, kb = _pad(n) // BLOCK, _pad(k) // BLOCK
    q = torch.empty(n, kb * BLOCK, device=dev, dtype=torch.float8_e4m3fn)
    s = torch.empty(nb, kb, device=dev, dtype=torch.float8_e8m0fnu)
    qt = torch.empty(k, nb * BLOCK, device=dev, dtype=torch.float8_e4m3fn) if transposed else None
    st = torch.empty(kb, nb, device=dev, dtype=torch.float8_e8m0fnu) if transposed else None
    with L.on_device("quantize_fp8", w2) as stream:
        L.check(L.lib().yfs_fp8_quantize_weight(w2.data_ptr(), L.DTYPES[w2.dtype], ld, n, k, q.data_ptr(), s.data_ptr(), _p(qt),
                                                _p(st), stream), "yfs_fp8_quantize_weight")
    return q, s, qt, st


@torch.no_grad()
def quantize_fp8(w):
    """A weight matrix [n, k] (fp32, bf16 or fp16, rows with any stride) as ``Fp8Tensor``."""
    _check_weight(w)
    if forward_ad.unpack_dual(w).tangent is not None:
        raise L.YfsError("quantize_fp8: forward-mode derivatives are not implemented, and w carries a tangent")
    L.require_cuda(w)
    _settled(w)
    q, s, _, _ = _quantize_weight(w, False)
    return Fp8Tensor(q, s, w.shape[1])


def _bias(b, n, what):
    if b is None:
        return None
    if b.dim() != 1 or b.shape[0] != n or not b.is_floating_point():
        raise L.YfsError(f"{what}: bias must be floating point [{n}], got {b.dtype} {tuple(b.shape)}")
    b = b.detach()
    if b.dtype != torch.float32:
        b = b.float()
    return b if b.is_contiguous() else b.contiguous()


def fp8_matmul(x, w, bias=None, slope=None, out_dtype=None):
    """y [..., n] = leaky(Q(x) W^T + bias) for x [..., k] (fp32, bf16 or fp16; quantised by rows inside the call) and an
    ``Fp8Tensor`` w [n, k].  ``slope``: of a LeakyReLU behind the product (None: none).  ``out_dtype``: fp32, bf16 or fp16
    (default: x's).  Sums are fp32 when the output is; towards 16 bits the 8-bit matrix instruction keeps 16 bits behind the
    largest product of a block of 128: an output is off by 2^-9 of that product for each block at most (1.5e-5 of the outputs'
    norm), which outputs whose products cancel can see beside their own rounding.  Not differentiable: ``backward()`` through the
    result raises (``torch.autograd.grad`` for tensors in front of it leaves its part out); for gradients ``fp8_linear``."""
    if not isinstance(w, Fp8Tensor):
        raise L.YfsError(f"fp8_matmul: w must be an Fp8Tensor (quantize_fp8), got {type(w).__name__}")
    return (L._binding or L.binding()).fp8_matmul(x, w.data, w.scale, w.k, bias, slope, out_dtype)


class _SinkLinearFn(torch.autograd.Function):
    """The node of a layer whose gradients go straight into their place in an optimiser's arena (train.FlatSGD); any other
    weight's is the extension module's."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        n, k = weight.shape
        need_x, need_w, need_b = ctx.needs_input_grad
        x2, m, ldx = _matrix(x, "fp8_linear")
        w2, _, ldw = _matrix(weight, "fp8_linear")
        # db alone is a sum of dy: nothing is kept for it
        needs = (1 if need_x else 0) + (2 if need_w else 0) + (4 if need_b and (need_x or need_w) else 0)
        ctx.meta = (x.shape, x.dtype, m, n, k, needs)
        ctx.wb = (weight, bias)          # for their gradient sinks and types; their values are not read again
        y = x.new_empty(x.shape[:-1] + (n,))
        if m == 0:
            return y
        lib = L.lib()
        saved_bytes = lib.yfs_fp8_linear_saved_bytes(m, n, k, needs)
        space_bytes = lib.yfs_fp8_linear_fwd_workspace_bytes(m, n, k)
        saved = x.new_empty(saved_bytes, dtype=torch.uint8) if saved_bytes else None
        space = x.new_empty(space_bytes, dtype=torch.uint8)
        b = _bias(bias, n, "fp8_linear")
        with L.on_device("fp8_linear", x2, w2, b) as stream:
            L.check(lib.yfs_fp8_linear_fwd(x2.data_ptr(), L.DTYPES[x2.dtype], ldx, w2.data_ptr(), L.DTYPES[w2.dtype], ldw, _p(b),
                                           y.data_ptr(), L.DTYPES[y.dtype], m, n, k, needs, _p(saved), saved_bytes,
                                           space.data_ptr(), space_bytes, stream), "yfs_fp8_linear_fwd")
        if saved is not None:
            ctx.save_for_backward(saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        from .train import settle_deferred, write_grad
        shape, dtype, m, n, k, needs = ctx.meta
        weight, bias = ctx.wb
        need_x, need_w, need_b = ctx.needs_input_grad
        if need_w:
            settle_deferred(weight)      # a layer in 16 bits that shares it may have left its gradient as factors
        if m == 0:
            return (dy.new_empty(shape) if need_x else None, torch.zeros_like(weight) if need_w else None,
                    torch.zeros_like(bias) if need_b else None)
        dy2, _, ldy = _matrix(dy, "fp8_linear")
        if not needs:
            def put_alone(sink, acc):
                total = dy2.float().sum(0).to(bias.dtype)
                if sink is None:
                    return total
                sink.add_(total) if acc else sink.copy_(total)
            return None, None, write_grad(bias, put_alone) if need_b else None
        (saved,) = ctx.saved_tensors
        dx = dy.new_empty(shape) if need_x else None
        # a gradient sink (train.FlatSGD) that the kernels can write is written by them; any other gets the result afterwards
        outs, results = [], []
        for param, shape_, need in ((weight, (n, k), need_w), (bias, (n,), need_b)):
            sink = getattr(param, "_yfs_grad_sink", None) if need else None
            direct = sink is not None and sink.dtype == torch.float32 and sink.is_contiguous()
            acc = direct and not param._yfs_grad_fresh
            outs.append(((sink if direct else dy.new_empty(shape_, dtype=torch.float32)) if need else None, acc, direct))
        (dw, acc_w, _), (db, acc_b, _) = outs
        lib = L.lib()
        nbytes = lib.yfs_fp8_linear_bwd_workspace_bytes(m, n, k, needs)
        space = dy.new_empty(nbytes, dtype=torch.uint8)
        with L.on_device("fp8_linear", dy2, saved, dw, db) as stream:
            L.check(lib.yfs_fp8_linear_bwd(dy2.data_ptr(), L.DTYPES[dy2.dtype], ldy, _p(dx), L.DTYPES[dtype], _p(dw), int(acc_w), _p(db),
                                           int(acc_b), m, n, k, needs, saved.data_ptr(), saved.numel(), space.data_ptr(), nbytes,
                                           stream), "yfs_fp8_linear_bwd")
        for param, (out, acc, direct) in zip((weight, bias), outs):
            def put(sink, accumulate):
                if sink is None:
                    return out if out.dtype == param.dtype else out.to(param.dtype)
                if not direct:
                    sink.add_(out) if accumulate else sink.copy_(out)
            results.append(write_grad(param, put) if out is not None else None)
        return dx, results[0], results[1]


def fp8_linear(x, weight, bias=None):
    """y [..., n] = Q(x) Q(weight)^T + bias, differentiable, in x's dtype: x [..., k] and weight [n, k] fp32, bf16 or fp16.
    The backward pass multiplies in 8 bits too: dx = Q(dy) Q(weight), dW = Q(dy^T) Q(x^T)^T (summed in fp32, as the bias's
    gradient is); for it the transposed 8-bit weight and x are kept, not the 16-bit x."""
    ext = L._binding or L.binding()
    if getattr(weight, "_yfs_grad_sink", None) is None and getattr(bias, "_yfs_grad_sink", None) is None:
        return ext.fp8_linear(x, weight, bias)
    _settled(weight)
    if not torch.is_grad_enabled():
        return ext.fp8_linear(x, weight, bias)
    ext.fp8_linear_check(x, weight, bias)
    return _SinkLinearFn.apply(x, weight, bias)


class Fp8Linear(nn.Linear):
    """nn.Linear (same parameter names and initialisation, fp32 master weights) whose three products run in 8 bits.  Takes
    fp32, bf16 or fp16 rows and answers in bf16, as ``HipLinear`` does; its gradients go straight into FlatSGD's arena."""

    def __init__(self, in_features, out_features, bias=True):
        super().__init__(in_features, out_features, bias=bias)
        self.weight._yfs_sink_capable = True
        if bias:
            self.bias._yfs_sink_capable = True

    def forward(self, x):
        return fp8_linear(x.to(torch.bfloat16), self.weight, self.bias)


class FrozenFp8Linear(nn.Module):
    """A linear layer for serving: 8-bit weights as buffers (a quarter of the fp32 bytes), bias, and the LeakyReLU(slope)
    that follows (None: none).  Not trainable."""

    def __init__(self, linear, slope=None):
        super().__init__()
        w = quantize_fp8(linear.weight)
        self.out_features, self.in_features = w.shape
        self.slope = slope
        self.register_buffer("weight_data", w.data)
        self.register_buffer("weight_scale", w.scale)
        self.register_buffer("bias", linear.bias.detach().float().clone() if linear.bias is not None else None)

    def forward(self, x):
        w = Fp8Tensor(self.weight_data, self.weight_scale, self.in_features)
        return fp8_matmul(x, w, self.bias, self.slope, torch.bfloat16)

    def extra_repr(self):
        return f"{self.in_features}, {self.out_features}, slope={self.slope}"


def freeze_fp8(model):
    """Replaces every linear layer of ``model`` (on the GPU) by its 8-bit form for serving, a fused LeakyReLU included, and
    puts the model into eval mode.  In place, all layers or (where one cannot be converted) none; a layer that stands in several
    places is converted once.  Returns the model."""
    from .model import HipLinear
    if isinstance(model, nn.Linear):
        raise L.YfsError("freeze_fp8: replaces the linear layers inside a module; for a layer alone: FrozenFp8Linear(layer)")
    places = [(m, name, c) for m in model.modules() for name, c in m._modules.items() if isinstance(c, nn.Linear)]
    frozen = {}
    for _, _, child in places:
        if child not in frozen:
            frozen[child] = FrozenFp8Linear(child, child.fused_act if isinstance(child, HipLinear) else None)
    for module, name, child in places:
        module._modules[name] = frozen[child]
    return model.eval()
